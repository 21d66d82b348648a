// k_pref.hip -- learning from preferences: the labels' log-probabilities from
// logits [N, C] (f32 or bf16, rows ld apart), forward and backward, the paired
// loss on log ratios, and the clipped policy loss with its gradient.
//
//   m = max z, s = sum exp(z - m), logp = (z_l - m) - log s
//   dz = dlogp (1[c = l] - exp(z - m) / s)
//   paired: R_q = sum over q's judged rows of logp - ref (or their mean),
//     margin = beta (R_chosen - R_rejected) - offset,
//     loss = scale sum of (1 - eps) softplus(-margin) + eps softplus(margin),
//     dlogp = +- scale beta (sigmoid(margin) - (1 - eps))
//   policy: ratio = exp(logp - old),
//     l = -min(ratio A, clip(ratio, 1 - low, 1 + high) A) + kl (e - (ref - logp) - 1),
//     e = exp(ref - logp), loss = scale sum w l,
//     dlogp = scale w (-ratio A where the unclipped term is the smaller, + kl (1 - e))
//
// Bound by HBM: the logits read once (twice where a gradient needs a sum over
// other rows first) and the gradient written once.  A row whose label is
// negative is not judged: it is not read, and its gradient is zero.
// Everything between is f32, sums over rows and the pairs' terms are f64.
#include <type_traits>

#include "rows.h"

namespace seeai {
namespace {

constexpr float kLog2e = 1.4426950408889634f;

// exp(x) for x <= 0: the hardware's exp2.  Rounding x log2 e moves a term by
// |x| 2^-24 of itself, and terms far down hardly count.
__device__ __forceinline__ float ExpNeg(float x) { return __builtin_amdgcn_exp2f(x * kLog2e); }

// A running maximum and the sum of exp(z - max) under it.  While all z are -inf
// the maximum is, too, and the sum zero; a NaN or +inf makes the sum a NaN.
struct Lse {
  float m = -INFINITY, s = 0.0f;
  __device__ __forceinline__ float Base() const { return m == -INFINITY ? 0.0f : m; }
  template <int n>
  __device__ __forceinline__ void Take(const float (&v)[n]) {
    float top = m;
#pragma unroll
    for (int i = 0; i < n; ++i) top = fmaxf(top, v[i]);
    const float was = m;
    m = top;
    const float base = Base();
    s *= ExpNeg(was - base);
#pragma unroll
    for (int i = 0; i < n; ++i) s += ExpNeg(v[i] - base);
  }
};

// The row's, from its kTPR threads'; `label` of the row's first thread (the
// label's logit, read before any thread may write over it) comes to all of them.
template <int kTPR>
__device__ __forceinline__ Lse RowLse(Lse a, float* lds, float& label) {
  Lse r;
  r.m = WaveMaxF(a.m);
  r.s = WaveSumF(a.s * ExpNeg(a.m - r.Base()));
  label = __shfl(label, 0, kWave);
  if constexpr (kTPR > kWave) {
    constexpr int kWaves = kTPR / kWave;
    const int w = threadIdx.x / kWave, first = w / kWaves * kWaves;
    __syncthreads();  // the sums before these have been read
    if (threadIdx.x % kWave == 0) lds[2 * w] = r.m, lds[2 * w + 1] = r.s;
    if (w == first && threadIdx.x % kWave == 0) lds[32] = label;
    __syncthreads();
    label = lds[32];
    Lse all;
#pragma unroll
    for (int k = 0; k < kWaves; ++k) all.m = fmaxf(all.m, lds[2 * (first + k)]);
    const float base = all.Base();
#pragma unroll
    for (int k = 0; k < kWaves; ++k) all.s += lds[2 * (first + k) + 1] * ExpNeg(lds[2 * (first + k)] - base);
    r = all;
  }
  return r;
}

// kV neighbours from column c on, -inf past the row.
template <class T>
__device__ __forceinline__ void Columns(const T* row, size_t c, size_t C, float (&v)[Io<T>::kV]) {
  constexpr int kV = Io<T>::kV;
  if (c + kV <= C) {
    Io<T>::LoadAny(row + c, v);
  } else {
#pragma unroll
    for (int i = 0; i < kV; ++i) v[i] = c + i < C ? Io<T>::Get(row + c + i) : -INFINITY;
  }
}

template <class T, int kTPR>
__device__ __forceinline__ Lse SweepLse(const T* row, int t, size_t C) {
  constexpr int kV = Io<T>::kV;
  Lse a;
  for (size_t c = static_cast<size_t>(t) * kV; c < C; c += kTPR * kV) {
    float v[kV];
    Columns(row, c, C, v);
    a.Take(v);
  }
  return a;
}

// dz = d (1[c = l] - exp(z - m) inv): columns of a lane are read before they are
// written, so out may be row.
template <class T, int kTPR>
__device__ __forceinline__ void SweepGrad(const T* row, T* out, int t, size_t C, size_t label, float d,
                                          float m, float inv) {
  constexpr int kV = Io<T>::kV;
  for (size_t c = static_cast<size_t>(t) * kV; c < C; c += kTPR * kV) {
    float v[kV];
    Columns(row, c, C, v);
#pragma unroll
    for (int i = 0; i < kV; ++i) v[i] = -d * (ExpNeg(v[i] - m) * inv);
    if (label - c < kV) {
#pragma unroll
      for (int i = 0; i < kV; ++i)
        if (label == c + i) v[i] = d + v[i];
    }
    if (c + kV <= C) {
      Io<T>::StoreAny(out + c, v);
    } else {
#pragma unroll
      for (int i = 0; i < kV; ++i)
        if (c + i < C) Io<T>::Put(out + c + i, v[i]);
    }
  }
}
template <class T, int kTPR>
__device__ __forceinline__ void SweepZero(T* out, int t, size_t C) {
  constexpr int kV = Io<T>::kV;
  const float v[kV] = {};
  for (size_t c = static_cast<size_t>(t) * kV; c < C; c += kTPR * kV) {
    if (c + kV <= C) {
      Io<T>::StoreAny(out + c, v);
    } else {
#pragma unroll
      for (int i = 0; i < kV; ++i)
        if (c + i < C) Io<T>::Put(out + c + i, 0.0f);
    }
  }
}

// A label's logit; one past the vocabulary has none.
template <class T>
__device__ __forceinline__ float LabelLogit(const T* row, int label, size_t C) {
  return label < 0 ? 0.0f : static_cast<size_t>(label) < C ? Io<T>::Get(row + label) : NAN;
}

constexpr int GroupOf(int tpr) { return tpr > 256 ? tpr : 256; }

template <class T, int kTPR>
__global__ void __launch_bounds__(GroupOf(kTPR))
TokenLogpKernel(const T* __restrict__ z, size_t ld, const int32_t* __restrict__ labels,
                float* __restrict__ logp, float* __restrict__ stats, size_t N, size_t C) {
  constexpr int kRows = GroupOf(kTPR) / kTPR;
  __shared__ float lds[33];
  const int t = threadIdx.x % kTPR;
  for (size_t base = static_cast<size_t>(blockIdx.x) * kRows; base < N;
       base += static_cast<size_t>(gridDim.x) * kRows) {
    const size_t r = base + threadIdx.x / kTPR;
    const int label = r < N ? labels[r] : -1;
    const T* row = z + r * ld;
    float zl = t == 0 ? LabelLogit(row, label, C) : 0.0f;
    const Lse a = RowLse<kTPR>(SweepLse<T, kTPR>(row, t, label < 0 ? 0 : C), lds, zl);
    if (t == 0 && r < N) {
      logp[r] = label < 0 ? 0.0f : (zl - a.m) - logf(a.s);
      if (stats) stats[2 * r] = label < 0 ? 0.0f : a.m, stats[2 * r + 1] = label < 0 ? 0.0f : a.s;
    }
  }
}

template <class T, int kTPR>
__global__ void __launch_bounds__(GroupOf(kTPR))
TokenLogpBwdKernel(const T* z, size_t ld, const int32_t* __restrict__ labels,
                   const float* __restrict__ stats, const float* __restrict__ dlogp, T* dz, size_t N,
                   size_t C) {
  constexpr int kRows = GroupOf(kTPR) / kTPR;
  const int t = threadIdx.x % kTPR;
  for (size_t r = static_cast<size_t>(blockIdx.x) * kRows + threadIdx.x / kTPR; r < N;
       r += static_cast<size_t>(gridDim.x) * kRows) {
    const int label = labels[r];
    if (label < 0) {
      SweepZero<T, kTPR>(dz + r * ld, t, C);
    } else {
      const float d = static_cast<size_t>(label) < C ? dlogp[r] : NAN;
      SweepGrad<T, kTPR>(z + r * ld, dz + r * ld, t, C, label, d, stats[2 * r], 1.0f / stats[2 * r + 1]);
    }
  }
}

// A judged token's loss and the loss's derivative by its log-probability.
__device__ __forceinline__ float2 PolicyToken(const PolicyTerms& P, size_t r, float logp) {
  const float ratio = expf(logp - P.old_logp[r]), adv = P.adv[r];
  // (a NaN passes both bounds)
  const float held = ratio < 1.0f - P.low ? 1.0f - P.low : ratio > 1.0f + P.high ? 1.0f + P.high : ratio;
  const float whole = ratio * adv, cut = held * adv;
  float loss = cut < whole ? -cut : -whole, d = cut < whole ? 0.0f : -whole;
  if (P.ref_logp) {
    const float back = P.ref_logp[r] - logp, e = expf(back);
    loss += P.kl * ((e - back) - 1.0f);
    d += P.kl * (1.0f - e);
  }
  return make_float2(loss, d);
}

template <class T, int kTPR>
__global__ void __launch_bounds__(GroupOf(kTPR))
PolicyKernel(const T* z, size_t ld, const int32_t* __restrict__ labels, PolicyTerms P,
             float* __restrict__ logp, T* dz, double* __restrict__ part, size_t N, size_t C) {
  constexpr int kRows = GroupOf(kTPR) / kTPR;
  __shared__ float lds[33];
  __shared__ double sum[kRows];
  const int t = threadIdx.x % kTPR;
  double mine = 0.0;  // of the row's first thread
  for (size_t base = static_cast<size_t>(blockIdx.x) * kRows; base < N;
       base += static_cast<size_t>(gridDim.x) * kRows) {
    const size_t r = base + threadIdx.x / kTPR;
    const int label = r < N ? labels[r] : -1;
    const T* row = z + r * ld;
    float zl = t == 0 ? LabelLogit(row, label, C) : 0.0f;
    const Lse a = RowLse<kTPR>(SweepLse<T, kTPR>(row, t, label < 0 ? 0 : C), lds, zl);
    if (r >= N) continue;  // (no barrier is left in this turn)
    if (label < 0) {
      if (t == 0 && logp) logp[r] = 0.0f;
      if (dz) SweepZero<T, kTPR>(dz + r * ld, t, C);
      continue;
    }
    const float lp = (zl - a.m) - logf(a.s);
    const float2 term = PolicyToken(P, r, lp);
    const float w = (P.weight ? P.weight[r] : 1.0f) * P.scale;
    if (t == 0) {
      if (logp) logp[r] = lp;
      mine += static_cast<double>(w) * static_cast<double>(term.x);
    }
    if (dz) SweepGrad<T, kTPR>(row, dz + r * ld, t, C, label, w * term.y, a.m, 1.0f / a.s);
  }
  if (t == 0) sum[threadIdx.x / kTPR] = mine;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int k = 1; k < kRows; ++k) mine += sum[k];
    part[blockIdx.x] = mine;
  }
}

constexpr int kSumThreads = 1024;
__global__ void __launch_bounds__(kSumThreads)
SumTermsKernel(const double* __restrict__ part, size_t n, double scale, float* __restrict__ loss) {
  __shared__ double red[kSumThreads / kWave];
  double s = 0.0;
#pragma unroll 4
  for (size_t i = threadIdx.x; i < n; i += kSumThreads) s += part[i];
  s = BlockSumD<kSumThreads>(s, red);
  if (threadIdx.x == 0) *loss = static_cast<float>(scale * s);
}

__device__ __forceinline__ double Softplus(double x) {
  return fmax(x, 0.0) + log1p(exp(-fabs(x)));
}

// A workgroup a pair: its two sequences' log ratios, its loss, its rows' dlogp.
// Rows outside every sequence get a zero.
constexpr int kPairThreads = 512;
__global__ void __launch_bounds__(kPairThreads)
PrefPairKernel(PrefArgs P, double* __restrict__ terms) {
  __shared__ double red[kPairThreads / kWave];
  const auto at = [&](uint64_t q) {  // where sequence q begins
    const int64_t s = P.starts[q];
    return static_cast<size_t>(s < 0 ? 0 : s > static_cast<int64_t>(P.N) ? static_cast<int64_t>(P.N) : s);
  };
  const auto clear = [&](size_t from, size_t to) {
    for (size_t r = from + threadIdx.x; r < to; r += kPairThreads) P.dlogp[r] = 0.0f;
  };
  if (P.pairs == 0) {
    clear(0, P.N);
    return;
  }
  const uint64_t i = blockIdx.x;
  const size_t cut[3] = {at(2 * i), at(2 * i + 1), at(2 * i + 2)};
  double ratio[2], count[2];
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    double s = 0.0, n = 0.0;
    for (size_t r = cut[k] + threadIdx.x; r < cut[k + 1]; r += kPairThreads) {
      if (P.labels[r] < 0) continue;
      s += static_cast<double>(P.logp[r]) - (P.ref_logp ? static_cast<double>(P.ref_logp[r]) : 0.0);
      n += 1.0;
    }
    ratio[k] = BlockSumD<kPairThreads>(s, red);
    count[k] = P.average ? fmax(BlockSumD<kPairThreads>(n, red), 1.0) : 1.0;
  }
  const double beta = P.beta, eps = P.smoothing;
  const double margin = beta * (ratio[0] / count[0] - ratio[1] / count[1]) - P.offset;
  const double d = P.scale * beta * (1.0 / (1.0 + exp(-margin)) - (1.0 - eps));
  if (threadIdx.x == 0) {
    // (a smoothing of zero takes no part in an infinite margin)
    terms[i] = (eps < 1.0 ? (1.0 - eps) * Softplus(-margin) : 0.0) + (eps > 0.0 ? eps * Softplus(margin) : 0.0);
    if (P.margin) P.margin[i] = static_cast<float>(margin);
  }
  if (!P.dlogp) return;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const float dk = static_cast<float>((k ? -d : d) / count[k]);
    for (size_t r = cut[k] + threadIdx.x; r < cut[k + 1]; r += kPairThreads)
      P.dlogp[r] = P.labels[r] < 0 ? 0.0f : dk;
  }
  if (i == 0) clear(0, cut[0]);
  if (i + 1 == P.pairs) clear(cut[2], P.N);
}

// Workgroups of the row kernels: they walk what rows are left.
constexpr size_t kMaxGroups = 8192;
unsigned Groups(size_t rows, int per) {
  const size_t g = (rows + per - 1) / per;
  return static_cast<unsigned>(g < kMaxGroups ? g : kMaxGroups);
}

template <class F>
hipError_t ByRow(size_t N, size_t C, F&& go) {
  if (C <= 2048) return go(std::integral_constant<int, 64>{});
  if (N >= 2048) return go(std::integral_constant<int, 256>{});
  return go(std::integral_constant<int, 1024>{});
}

}  // namespace

size_t PolicyWorkspaceBytes(size_t N) { return (N < kMaxGroups ? N : kMaxGroups) * sizeof(double); }
size_t PrefWorkspaceBytes(size_t pairs) { return pairs * sizeof(double); }

hipError_t LaunchTokenLogpFwd(int bf16, const void* z, size_t ld, const int32_t* labels, float* logp,
                              float* stats, size_t N, size_t C, hipStream_t s) {
  if (N == 0) return hipSuccess;
  return ByRow(N, C, [&](auto tpr) {
    constexpr int kT = decltype(tpr)::value, kG = GroupOf(kT);
    if (bf16)
      hipLaunchKernelGGL((TokenLogpKernel<uint16_t, kT>), dim3(Groups(N, kG / kT)), dim3(kG), 0, s,
                         static_cast<const uint16_t*>(z), ld, labels, logp, stats, N, C);
    else
      hipLaunchKernelGGL((TokenLogpKernel<float, kT>), dim3(Groups(N, kG / kT)), dim3(kG), 0, s,
                         static_cast<const float*>(z), ld, labels, logp, stats, N, C);
    return hipGetLastError();
  });
}

hipError_t LaunchTokenLogpBwd(int bf16, const void* z, size_t ld, const int32_t* labels,
                              const float* stats, const float* dlogp, void* dz, size_t N, size_t C,
                              hipStream_t s) {
  if (N == 0) return hipSuccess;
  return ByRow(N, C, [&](auto tpr) {
    constexpr int kT = decltype(tpr)::value, kG = GroupOf(kT);
    if (bf16)
      hipLaunchKernelGGL((TokenLogpBwdKernel<uint16_t, kT>), dim3(Groups(N, kG / kT)), dim3(kG), 0, s,
                         static_cast<const uint16_t*>(z), ld, labels, stats, dlogp,
                         static_cast<uint16_t*>(dz), N, C);
    else
      hipLaunchKernelGGL((TokenLogpBwdKernel<float, kT>), dim3(Groups(N, kG / kT)), dim3(kG), 0, s,
                         static_cast<const float*>(z), ld, labels, stats, dlogp,
                         static_cast<float*>(dz), N, C);
    return hipGetLastError();
  });
}

hipError_t LaunchPrefLoss(const PrefArgs& a, float* loss, void* ws, hipStream_t s) {
  double* terms = static_cast<double*>(ws);
  if (a.pairs || (a.dlogp && a.N)) {
    hipLaunchKernelGGL(PrefPairKernel, dim3(static_cast<unsigned>(a.pairs ? a.pairs : 1)),
                       dim3(kPairThreads), 0, s, a, terms);
    if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
  }
  hipLaunchKernelGGL(SumTermsKernel, dim3(1), dim3(kSumThreads), 0, s, terms, a.pairs,
                     static_cast<double>(a.scale), loss);
  return hipGetLastError();
}

hipError_t LaunchPolicyLoss(int bf16, const void* z, size_t ld, const int32_t* labels,
                            const PolicyTerms& P, float* loss, float* logp, void* dz, size_t N, size_t C,
                            void* ws, hipStream_t s) {
  double* part = static_cast<double*>(ws);
  size_t groups = 0;
  if (N) {
    const hipError_t e = ByRow(N, C, [&](auto tpr) {
      constexpr int kT = decltype(tpr)::value, kG = GroupOf(kT);
      groups = Groups(N, kG / kT);
      if (bf16)
        hipLaunchKernelGGL((PolicyKernel<uint16_t, kT>), dim3(static_cast<unsigned>(groups)), dim3(kG), 0,
                           s, static_cast<const uint16_t*>(z), ld, labels, P, logp,
                           static_cast<uint16_t*>(dz), part, N, C);
      else
        hipLaunchKernelGGL((PolicyKernel<float, kT>), dim3(static_cast<unsigned>(groups)), dim3(kG), 0, s,
                           static_cast<const float*>(z), ld, labels, P, logp, static_cast<float*>(dz),
                           part, N, C);
      return hipGetLastError();
    });
    if (e != hipSuccess) return e;
  }
  hipLaunchKernelGGL(SumTermsKernel, dim3(1), dim3(kSumThreads), 0, s, part, groups, 1.0, loss);
  return hipGetLastError();
}

}  // namespace seeai
