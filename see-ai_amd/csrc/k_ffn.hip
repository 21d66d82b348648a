// k_ffn.hip -- the gated feed-forward block, forward and backward.
//
//   G = X Wg, U = X Wu, H = act(G) U, Y = H Wd
//   dH = dY Wd', dG = dH U act'(G), dU = dH act(G)
//   dX = dG Wg' + dU Wu', dWg = X' dG, dWu = X' dU, dWd = H' dY
#include "common.h"

namespace seeai {
namespace {

template <class T> __device__ __forceinline__ float Get(const T* p, size_t i);
template <> __device__ __forceinline__ float Get<float>(const float* p, size_t i) { return p[i]; }
template <> __device__ __forceinline__ float Get<uint16_t>(const uint16_t* p, size_t i) {
  return Bf16ToF32(p[i]);
}
template <class T> __device__ __forceinline__ void Put(T* p, size_t i, float v);
template <> __device__ __forceinline__ void Put<float>(float* p, size_t i, float v) { p[i] = v; }
template <> __device__ __forceinline__ void Put<uint16_t>(uint16_t* p, size_t i, float v) {
  p[i] = F32ToBf16(v);
}

// The activation's derivative.
__device__ __forceinline__ float ActGrad(int act, float x) {
  switch (act) {
    case 1: return x > 0.0f ? 1.0f : 0.0f;
    case 2: {
      const float kC = 0.7978845608028654f, kA = 0.044715f;
      const float t = tanhf(kC * (x + kA * x * x * x));
      return 0.5f * (1.0f + t) + 0.5f * x * (1.0f - t * t) * (kC * (1.0f + 3.0f * kA * x * x));
    }
    case 3: {
      const float s = SigmoidExpr(x);
      return s * (1.0f + x * (1.0f - s));
    }
    default: return 1.0f;
  }
}

// One product (or two of them) of a pass: element (i, k) of A at i am + k ak,
// (k, j) of B at k bk + j bn.
struct Product {
  const void *A, *B, *A2, *B2;
  size_t am, ak, bk, bn;
  size_t M, N, K;
  void *o1, *o2, *o3;
  const void *e1, *e2;
  int act;
};

// kKind 0: o1 = A B; 1: o1 = A B + A2 B2; 2: G = A B, U = A B2 (o1, o2 where
// given), o3 = act(G) U; 3: d = A B, with G = e1 and U = e2, o1 = d U act'(G),
// o2 = d act(G), o3 = act(G) U.
constexpr int kT = 64, kK = 16;
template <class T, int kKind>
__global__ void __launch_bounds__(256) FfnProductKernel(Product p) {
  __shared__ float sa[kK][kT + 1], sb[kK][kT + 1], sb2[kKind == 2 ? kK : 1][kT + 1];
  const size_t m0 = static_cast<size_t>(blockIdx.y) * kT, n0 = static_cast<size_t>(blockIdx.x) * kT;
  const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
  float c[4][4] = {}, c2[4][4] = {};
  for (int seg = 0; seg < (kKind == 1 ? 2 : 1); ++seg) {
    const T* A = static_cast<const T*>(seg ? p.A2 : p.A);
    const T* B = static_cast<const T*>(seg ? p.B2 : p.B);
    for (size_t k0 = 0; k0 < p.K; k0 += kK) {
      for (int i = threadIdx.x; i < kT * kK; i += 256) {
        // Neighbouring threads along the operand's own contiguous axis.
        const int ka = p.ak == 1 ? i % kK : i / kT, ma = p.ak == 1 ? i / kK : i % kT;
        const int kb = p.bk == 1 ? i % kK : i / kT, nb = p.bk == 1 ? i / kK : i % kT;
        const bool ina = m0 + ma < p.M && k0 + ka < p.K, inb = n0 + nb < p.N && k0 + kb < p.K;
        sa[ka][ma] = ina ? Get(A, (m0 + ma) * p.am + (k0 + ka) * p.ak) : 0.0f;
        sb[kb][nb] = inb ? Get(B, (k0 + kb) * p.bk + (n0 + nb) * p.bn) : 0.0f;
        if constexpr (kKind == 2)
          sb2[kb][nb] = inb ? Get(static_cast<const T*>(p.B2), (k0 + kb) * p.bk + (n0 + nb) * p.bn) : 0.0f;
      }
      __syncthreads();
      for (int k = 0; k < kK; ++k)
        for (int i = 0; i < 4; ++i)
          for (int j = 0; j < 4; ++j) {
            c[i][j] = fmaf(sa[k][ty * 4 + i], sb[k][tx * 4 + j], c[i][j]);
            if constexpr (kKind == 2) c2[i][j] = fmaf(sa[k][ty * 4 + i], sb2[k][tx * 4 + j], c2[i][j]);
          }
      __syncthreads();
    }
  }
  for (int i = 0; i < 4; ++i)
    for (int j = 0; j < 4; ++j) {
      const size_t m = m0 + ty * 4 + i, n = n0 + tx * 4 + j;
      if (m >= p.M || n >= p.N) continue;
      const size_t o = m * p.N + n;
      T *o1 = static_cast<T*>(p.o1), *o2 = static_cast<T*>(p.o2), *o3 = static_cast<T*>(p.o3);
      if constexpr (kKind < 2) Put(o1, o, c[i][j]);
      if constexpr (kKind == 2) {
        if (o1) Put(o1, o, c[i][j]), Put(o2, o, c2[i][j]);
        Put(o3, o, ActExpr(p.act, c[i][j]) * c2[i][j]);
      }
      if constexpr (kKind == 3) {
        const float g = Get(static_cast<const T*>(p.e1), o), u = Get(static_cast<const T*>(p.e2), o);
        const float a = ActExpr(p.act, g);
        Put(o1, o, c[i][j] * u * ActGrad(p.act, g));
        Put(o2, o, c[i][j] * a);
        Put(o3, o, a * u);
      }
    }
}

template <class T, int kKind>
hipError_t Go(const Product& p, hipStream_t s) {
  if (p.M == 0) return hipSuccess;
  hipLaunchKernelGGL((FfnProductKernel<T, kKind>),
                     dim3(static_cast<unsigned>((p.N + kT - 1) / kT),
                          static_cast<unsigned>((p.M + kT - 1) / kT)),
                     dim3(256), 0, s, p);
  return hipGetLastError();
}

template <class T>
hipError_t Fwd(const FfnArgs& a, hipStream_t s) {
  void* h = a.ws;
  Product p{a.x, a.wg, nullptr, a.wu, a.D, 1, a.F, 1, a.M, a.F, a.D, a.gate, a.up, h, nullptr, nullptr, a.act};
  if (hipError_t e = Go<T, 2>(p, s); e != hipSuccess) return e;
  p = Product{h, a.wd, nullptr, nullptr, a.F, 1, a.D, 1, a.M, a.D, a.F, a.y};
  return Go<T, 0>(p, s);
}

template <class T>
hipError_t Bwd(const FfnArgs& a, hipStream_t s) {
  T* dg = static_cast<T*>(a.ws);
  T *du = dg + a.M * a.F, *h = du + a.M * a.F;
  Product p{a.dy, a.wd, nullptr, nullptr, a.D, 1, 1, a.D, a.M, a.F, a.D, dg, du, h, a.gate, a.up, a.act};
  if (hipError_t e = Go<T, 3>(p, s); e != hipSuccess) return e;
  p = Product{dg, a.wg, du, a.wu, a.F, 1, 1, a.F, a.M, a.D, a.F, a.dx};
  if (hipError_t e = Go<T, 1>(p, s); e != hipSuccess) return e;
  p = Product{a.x, dg, nullptr, nullptr, 1, a.D, a.F, 1, a.D, a.F, a.M, a.dwg};
  if (hipError_t e = Go<T, 0>(p, s); e != hipSuccess) return e;
  p.B = du, p.o1 = a.dwu;
  if (hipError_t e = Go<T, 0>(p, s); e != hipSuccess) return e;
  p = Product{h, a.dy, nullptr, nullptr, 1, a.F, a.D, 1, a.F, a.D, a.M, a.dwd};
  return Go<T, 0>(p, s);
}

}  // namespace

size_t FfnWorkspaceBytes(int bf16, size_t M, size_t D, size_t F, int backward) {
  (void)D;
  return (backward ? 3 : 1) * M * F * (bf16 ? 2 : 4);
}

hipError_t LaunchFfnFwd(const FfnArgs& a, hipStream_t s) {
  return a.bf16 ? Fwd<uint16_t>(a, s) : Fwd<float>(a, s);
}
hipError_t LaunchFfnBwd(const FfnArgs& a, hipStream_t s) {
  return a.bf16 ? Bwd<uint16_t>(a, s) : Bwd<float>(a, s);
}

}  // namespace seeai
