// k_norm.hip -- layer and root-mean-square normalisation of rows in f32 or
// bf16, forward, and backward with the reduction of the weight's (and the
// bias's) gradient: the trained form of the norms whose frozen form
// k_elementwise.hip runs (normalization.cc computes no weight gradient).
//
//   mu = mean(x), r = 1 / sqrt(mean((x - mu)^2) + eps)   (RMS: mu = 0)
//   y  = (x - mu) r w + b
//   dx = r (w dy - mean(w dy) - xhat mean(w dy xhat)),  xhat = (x - mu) r
//   dw = sum over rows of dy xhat,  db = sum over rows of dy
//
// Bound by HBM: forward x in, y out; backward dy and x in, dx out.  A row is
// held in registers (kE elements a lane) between its statistics and its
// output, so it is read once; the variance is taken about the mean in a
// second sweep of the registers.  Statistics and sums are f32 for both types.
// 8192 x 2048 bf16 on MI355X: RMS forward 12.9 us (5.2 TB/s, a copy's rate),
// layer backward 29.8, of which the fold below 4.3 (the copy rate would be 19).
//
// The weight's gradient runs down the columns while dx needs sums along the
// rows: a workgroup walks rows strided over the grid, a lane keeps the same
// columns throughout and sums them in registers; the workgroups' partial rows
// go to the workspace and NormFoldKernel adds them in a fixed order -- no
// atomics, the same bits every run.
#include "common.h"

namespace seeai {
namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

// Sixteen bytes on a float's or a bf16's own alignment: global memory takes them.
typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4), may_alias));
typedef uint32_t u32x4u __attribute__((ext_vector_type(4), aligned(2), may_alias));

template <class T> struct Io;
template <> struct Io<float> {
  static constexpr int kV = 4;  // elements of a 16-byte access
  static __device__ __forceinline__ void Load(const float* p, float* v) {
    const float4 a = *reinterpret_cast<const float4*>(p);
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w;
  }
  static __device__ __forceinline__ void Store(float* p, const float* v) {
    *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
  }
  static __device__ __forceinline__ void LoadAny(const float* p, float* v) {
    const f32x4u a = *reinterpret_cast<const f32x4u*>(p);
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w;
  }
  static __device__ __forceinline__ void StoreAny(float* p, const float* v) {
    *reinterpret_cast<f32x4u*>(p) = f32x4u{v[0], v[1], v[2], v[3]};
  }
  static __device__ __forceinline__ float Get(const float* p) { return *p; }
  static __device__ __forceinline__ void Put(float* p, float v) { *p = v; }
};
template <> struct Io<uint16_t> {  // bf16
  static constexpr int kV = 8;
  static __device__ __forceinline__ void Load(const uint16_t* p, float* v) {
    const uint4 a = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = __uint_as_float(w[i] << 16);
      v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
    }
  }
  static __device__ __forceinline__ bf16x8 Pack(const float* v) {
    bf16x8 o;
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = static_cast<__bf16>(v[i]);
    return o;
  }
  static __device__ __forceinline__ void Store(uint16_t* p, const float* v) {
    *reinterpret_cast<bf16x8*>(p) = Pack(v);
  }
  static __device__ __forceinline__ void LoadAny(const uint16_t* p, float* v) {
    const u32x4u a = *reinterpret_cast<const u32x4u*>(p);
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = __uint_as_float(w[i] << 16);
      v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
    }
  }
  static __device__ __forceinline__ void StoreAny(uint16_t* p, const float* v) {
    *reinterpret_cast<u32x4u*>(p) = __builtin_bit_cast(u32x4u, Pack(v));
  }
  static __device__ __forceinline__ float Get(const uint16_t* p) { return Bf16ToF32(*p); }
  static __device__ __forceinline__ void Put(uint16_t* p, float v) { *p = F32ToBf16(v); }
};

// Where lane t's element e of a row lies, and whether it lies in the row.
// kVec: groups of kV neighbours, kTPR groups apart (16-byte accesses, rows a
// multiple of kV long); else single elements kTPR apart.  kAny, with kVec: the
// same groups where rows are of any length and begin anywhere, the row's last,
// short group element by element.
template <class T, int kTPR, bool kVec>
__device__ __forceinline__ int ColOf(int t, int e) {
  constexpr int kV = Io<T>::kV;
  return kVec ? ((e / kV) * kTPR + t) * kV + e % kV : e * kTPR + t;
}
template <class T, int kTPR, int kE, bool kVec, bool kAny>
__device__ __forceinline__ void LoadRow(const T* row, int t, int cols, float (&v)[kE]) {
  constexpr int kV = Io<T>::kV;
  if constexpr (kAny) {
#pragma unroll
    for (int e = 0; e < kE; e += kV) {
      const int c = ColOf<T, kTPR, true>(t, e);
      if (c + kV <= cols) {
        Io<T>::LoadAny(row + c, v + e);
      } else {
#pragma unroll
        for (int i = 0; i < kV; ++i) v[e + i] = c + i < cols ? Io<T>::Get(row + c + i) : 0.0f;
      }
    }
  } else if constexpr (kVec) {
#pragma unroll
    for (int e = 0; e < kE; e += kV) {
      const int c = ColOf<T, kTPR, true>(t, e);
      if (c < cols) {
        Io<T>::Load(row + c, v + e);
      } else {
#pragma unroll
        for (int i = 0; i < kV; ++i) v[e + i] = 0.0f;
      }
    }
  } else {
#pragma unroll
    for (int e = 0; e < kE; ++e) {
      const int c = ColOf<T, kTPR, false>(t, e);
      v[e] = c < cols ? Io<T>::Get(row + c) : 0.0f;
    }
  }
}
template <class T, int kTPR, int kE, bool kVec, bool kAny = false>
__device__ __forceinline__ void StoreRow(T* row, int t, int cols, const float (&v)[kE]) {
  constexpr int kV = Io<T>::kV;
  if constexpr (kAny) {
#pragma unroll
    for (int e = 0; e < kE; e += kV) {
      const int c = ColOf<T, kTPR, true>(t, e);
      if (c + kV <= cols) {
        Io<T>::StoreAny(row + c, v + e);
      } else {
#pragma unroll
        for (int i = 0; i < kV; ++i)
          if (c + i < cols) Io<T>::Put(row + c + i, v[e + i]);
      }
    }
  } else if constexpr (kVec) {
#pragma unroll
    for (int e = 0; e < kE; e += kV) {
      const int c = ColOf<T, kTPR, true>(t, e);
      if (c < cols) Io<T>::Store(row + c, v + e);
    }
  } else {
#pragma unroll
    for (int e = 0; e < kE; ++e) {
      const int c = ColOf<T, kTPR, false>(t, e);
      if (c < cols) Io<T>::Put(row + c, v[e]);
    }
  }
}
// The f32 vector at the same columns.
template <class T, int kTPR, int kE, bool kVec, bool kAny = false>
__device__ __forceinline__ void LoadVec(const float* w, int t, int cols, float (&v)[kE]) {
  if constexpr (kAny) {
#pragma unroll
    for (int e = 0; e < kE; e += 4) {
      const int c = ColOf<T, kTPR, true>(t, e);
      if (c + 4 <= cols) {
        Io<float>::LoadAny(w + c, v + e);
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[e + i] = c + i < cols ? w[c + i] : 0.0f;
      }
    }
  } else if constexpr (kVec) {
#pragma unroll
    for (int e = 0; e < kE; e += 4) {
      const int c = ColOf<T, kTPR, true>(t, e);
      if (c < cols) {
        Io<float>::Load(w + c, v + e);
      } else {
        v[e] = v[e + 1] = v[e + 2] = v[e + 3] = 0.0f;
      }
    }
  } else {
#pragma unroll
    for (int e = 0; e < kE; ++e) {
      const int c = ColOf<T, kTPR, false>(t, e);
      v[e] = c < cols ? w[c] : 0.0f;
    }
  }
}

// Sums over the kTPR threads of each row of a workgroup: within the wave, then
// over a row's waves through LDS (two floats a wave).
template <int kTPR, int kN>
__device__ __forceinline__ void RowSum(float (&s)[kN], float* lds) {
#pragma unroll
  for (int i = 0; i < kN; ++i) s[i] = WaveSumF(s[i]);
  if constexpr (kTPR > kWave) {
    constexpr int kWaves = kTPR / kWave;
    const int w = threadIdx.x / kWave, first = w / kWaves * kWaves;
    __syncthreads();  // the sums before these have been read
    if (threadIdx.x % kWave == 0)
#pragma unroll
      for (int i = 0; i < kN; ++i) lds[w * kN + i] = s[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      s[i] = 0.0f;
#pragma unroll
      for (int k = 0; k < kWaves; ++k) s[i] += lds[(first + k) * kN + i];
    }
  }
}

constexpr int Threads(int tpr) { return tpr > 256 ? tpr : 256; }
// The backward's workgroup: eight waves, so that few workgroups fill the chip
// and few partial rows are left.
constexpr int kBwdPerSimd = 4;
constexpr int BwdThreads(int tpr) { return tpr > 512 ? tpr : 512; }

template <class T, int kTPR, int kE, bool kVec, bool kAny>
__global__ void __launch_bounds__(Threads(kTPR))
NormFwdKernel(int rms, const T* __restrict__ x, const float* __restrict__ w,
              const float* __restrict__ b, T* __restrict__ y, float* __restrict__ mean,
              float* __restrict__ rstd, size_t rows, int cols, float eps) {
  __shared__ float lds[16];
  constexpr int kRows = Threads(kTPR) / kTPR;
  const int t = threadIdx.x % kTPR;
  // (the loop is uniform over the workgroup, its barriers too)
  for (size_t base = static_cast<size_t>(blockIdx.x) * kRows; base < rows;
       base += static_cast<size_t>(gridDim.x) * kRows) {
    const size_t r = base + threadIdx.x / kTPR;
    const bool in = r < rows;
    float v[kE];
    LoadRow<T, kTPR, kE, kVec, kAny>(x + r * cols, t, in ? cols : 0, v);
    float mu[1] = {0.0f};
    if (!rms) {
#pragma unroll
      for (int e = 0; e < kE; ++e) mu[0] += v[e];
      RowSum<kTPR>(mu, lds);
      mu[0] /= static_cast<float>(cols);
#pragma unroll
      for (int e = 0; e < kE; ++e)
        v[e] = ColOf<T, kTPR, kVec>(t, e) < cols ? v[e] - mu[0] : 0.0f;
    }
    float sq[1] = {0.0f};
#pragma unroll
    for (int e = 0; e < kE; ++e) sq[0] += v[e] * v[e];
    RowSum<kTPR>(sq, lds);
    const float rs = 1.0f / sqrtf(sq[0] / static_cast<float>(cols) + eps);
    float ww[kE];
    LoadVec<T, kTPR, kE, kVec, kAny>(w, t, cols, ww);
#pragma unroll
    for (int e = 0; e < kE; ++e) v[e] = v[e] * rs * ww[e];
    if (b) {
      LoadVec<T, kTPR, kE, kVec, kAny>(b, t, cols, ww);
#pragma unroll
      for (int e = 0; e < kE; ++e) v[e] += ww[e];
    }
    if (!in) continue;
    StoreRow<T, kTPR, kE, kVec, kAny>(y + r * cols, t, cols, v);
    if (t == 0) {
      if (mean) mean[r] = mu[0];
      if (rstd) rstd[r] = rs;
    }
  }
}

// A row as it lies in memory, for loads that run ahead of their use.
template <class T, int kTPR, int kE, bool kVec>
struct RawRow {
  static constexpr int kV = Io<T>::kV;
  uint4 q[kVec ? kE / kV : 1];
  T e[kVec ? 1 : kE];
  __device__ __forceinline__ void Load(const T* row, int t, int cols) {
    if constexpr (kVec) {
#pragma unroll
      for (int i = 0; i < kE / kV; ++i) {
        const int c = ColOf<T, kTPR, true>(t, i * kV);
        q[i] = c < cols ? *reinterpret_cast<const uint4*>(row + c) : make_uint4(0, 0, 0, 0);
      }
    } else {
#pragma unroll
      for (int i = 0; i < kE; ++i) {
        const int c = ColOf<T, kTPR, false>(t, i);
        e[i] = c < cols ? row[c] : T(0);
      }
    }
  }
  __device__ __forceinline__ void Get(float (&v)[kE]) const {
    if constexpr (kVec) {
#pragma unroll
      for (int i = 0; i < kE / kV; ++i) Io<T>::Load(reinterpret_cast<const T*>(&q[i]), v + i * kV);
    } else {
#pragma unroll
      for (int i = 0; i < kE; ++i) v[i] = Io<T>::Get(&e[i]);
    }
  }
};

// Workgroup g takes rows g kRows + i, stepping the grid; out: [gridDim][2][cols]
// partials (db behind dw), or dw and db themselves when the grid is one.  A
// row's loads go out while the row before it is reduced: with a wave a row
// there is nothing else to cover their latency (8192 x 2048 bf16 on MI355X: 30
// us with, 41 without; the copy rate would be 20).  The weight sits in LDS, a
// lane's own columns together, to leave the registers to that row.
template <class T, int kTPR, int kE, bool kVec>
__global__ void __launch_bounds__(BwdThreads(kTPR), kBwdPerSimd)
NormBwdKernel(int rms, const T* __restrict__ dy, const T* __restrict__ x,
              const float* __restrict__ w, const float* __restrict__ mean,
              const float* __restrict__ rstd, T* __restrict__ dx, float* __restrict__ dw,
              float* __restrict__ db, float* __restrict__ part, size_t rows, int cols) {
  constexpr int kRows = BwdThreads(kTPR) / kTPR;
  __shared__ float lds[32];
  __shared__ float own[kTPR * kE];  // element e of thread t at ((e / 4) kTPR + t) 4 + e % 4
  const int t = threadIdx.x % kTPR, sub = threadIdx.x / kTPR;
  auto at = [&](int e) { return (e / 4 * kTPR + t) * 4 + e % 4; };
  const float inv = 1.0f / static_cast<float>(cols);
  float sw[kE], sb[kE];
  if (sub == 0) {
    LoadVec<T, kTPR, kE, kVec>(w, t, cols, sw);
#pragma unroll
    for (int e = 0; e < kE; ++e) own[at(e)] = sw[e];
  }
  __syncthreads();
#pragma unroll
  for (int e = 0; e < kE; ++e) sw[e] = sb[e] = 0.0f;
  const size_t step = static_cast<size_t>(gridDim.x) * kRows;
  size_t base = static_cast<size_t>(blockIdx.x) * kRows;  // of the workgroup's next rows
  RawRow<T, kTPR, kE, kVec> rx, rd;
  float mu = 0.0f, rs = 0.0f;
  auto fetch = [&]() {  // past the last row: dy = 0 adds nothing
    const size_t r = base + sub;
    const int in = r < rows ? cols : 0;
    rx.Load(x + r * cols, t, in);
    rd.Load(dy + r * cols, t, in);
    mu = rms || !in ? 0.0f : mean[r], rs = in ? rstd[r] : 0.0f;
  };
  fetch();
  while (base < rows) {  // (uniform over the workgroup, its barriers too)
    float v[kE], d[kE];
    rx.Get(v);
    rd.Get(d);
    const float m = mu, q = rs;
    const bool in = base + sub < rows;
    T* out = dx + (base + sub) * cols;
    base += step;
    fetch();
    float s[2] = {0.0f, 0.0f};
#pragma unroll
    for (int e = 0; e < kE; e += 4) {  // (columns past the row: d = 0, so no term)
      const float4 w4 = *reinterpret_cast<const float4*>(own + at(e));
      const float ww[4] = {w4.x, w4.y, w4.z, w4.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v[e + i] = (v[e + i] - m) * q;
        sw[e + i] += d[e + i] * v[e + i];
        sb[e + i] += d[e + i];
        d[e + i] *= ww[i];
        s[0] += d[e + i];
        s[1] += d[e + i] * v[e + i];
      }
    }
    RowSum<kTPR>(s, lds);
    const float c1 = rms ? 0.0f : s[0] * inv, c2 = s[1] * inv;
#pragma unroll
    for (int e = 0; e < kE; ++e) d[e] = q * (d[e] - c1 - v[e] * c2);
    if (in) StoreRow<T, kTPR, kE, kVec>(out, t, cols, d);
  }
  // The workgroup's row groups add up in order; the last holds the sum.
  if constexpr (kRows > 1) {
    for (int pass = 0; pass < (db ? 2 : 1); ++pass) {
      float (&s)[kE] = pass ? sb : sw;
      for (int g = 0; g < kRows; ++g) {
        __syncthreads();
        if (sub == g) {
#pragma unroll
          for (int e = 0; e < kE; ++e) {
            if (g > 0) s[e] = own[at(e)] + s[e];
            own[at(e)] = s[e];
          }
        }
      }
    }
  }
  if (sub == kRows - 1) {
    float* ow = gridDim.x > 1 ? part + static_cast<size_t>(blockIdx.x) * 2 * cols : dw;
    float* ob = gridDim.x > 1 ? ow + cols : db;
#pragma unroll
    for (int e = 0; e < kE; ++e) {
      const int c = ColOf<T, kTPR, kVec>(t, e);
      if (c < cols) {
        ow[c] = sw[e];
        if (db) ob[c] = sb[e];
      }
    }
  }
}

// Rows past the registers: one workgroup of 1024 a row, the row read again
// (from L2 mostly) for each sweep.
constexpr int kLong = 1024;
template <class T>
__global__ void __launch_bounds__(kLong)
NormFwdLongKernel(int rms, const T* __restrict__ x, const float* __restrict__ w,
                  const float* __restrict__ b, T* __restrict__ y, float* __restrict__ mean,
                  float* __restrict__ rstd, size_t rows, size_t cols, float eps) {
  __shared__ float lds[16];
  for (size_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const T* row = x + r * cols;
    float mu[1] = {0.0f}, sq[1] = {0.0f};
    if (!rms) {
      for (size_t c = threadIdx.x; c < cols; c += kLong) mu[0] += Io<T>::Get(row + c);
      RowSum<kLong>(mu, lds);
      mu[0] /= static_cast<float>(cols);
    }
    for (size_t c = threadIdx.x; c < cols; c += kLong) {
      const float v = Io<T>::Get(row + c) - mu[0];
      sq[0] += v * v;
    }
    RowSum<kLong>(sq, lds);
    const float rs = 1.0f / sqrtf(sq[0] / static_cast<float>(cols) + eps);
    for (size_t c = threadIdx.x; c < cols; c += kLong) {
      const float v = (Io<T>::Get(row + c) - mu[0]) * rs * w[c];
      Io<T>::Put(y + r * cols + c, b ? v + b[c] : v);
    }
    if (threadIdx.x == 0) {
      if (mean) mean[r] = mu[0];
      if (rstd) rstd[r] = rs;
    }
  }
}
template <class T>
__global__ void __launch_bounds__(kLong)
NormDxLongKernel(int rms, const T* __restrict__ dy, const T* __restrict__ x,
                 const float* __restrict__ w, const float* __restrict__ mean,
                 const float* __restrict__ rstd, T* __restrict__ dx, size_t rows, size_t cols) {
  __shared__ float lds[32];
  for (size_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const float mu = rms ? 0.0f : mean[r], rs = rstd[r];
    float s[2] = {0.0f, 0.0f};
    for (size_t c = threadIdx.x; c < cols; c += kLong) {
      const float d = Io<T>::Get(dy + r * cols + c) * w[c];
      s[0] += d;
      s[1] += d * ((Io<T>::Get(x + r * cols + c) - mu) * rs);
    }
    RowSum<kLong>(s, lds);
    const float inv = 1.0f / static_cast<float>(cols);
    const float c1 = rms ? 0.0f : s[0] * inv, c2 = s[1] * inv;
    for (size_t c = threadIdx.x; c < cols; c += kLong) {
      const float d = Io<T>::Get(dy + r * cols + c) * w[c];
      const float v = (Io<T>::Get(x + r * cols + c) - mu) * rs;
      Io<T>::Put(dx + r * cols + c, rs * (d - c1 - v * c2));
    }
  }
}
// Column sums of long rows: a thread a column over the rows blockIdx.y takes.
template <class T>
__global__ void __launch_bounds__(256)
NormDwLongKernel(int rms, const T* __restrict__ dy, const T* __restrict__ x,
                 const float* __restrict__ mean, const float* __restrict__ rstd,
                 float* __restrict__ dw, float* __restrict__ db, float* __restrict__ part,
                 size_t rows, size_t cols) {
  const size_t c = static_cast<size_t>(blockIdx.x) * 256 + threadIdx.x;
  if (c >= cols) return;
  float sw = 0.0f, sb = 0.0f;
  for (size_t r = blockIdx.y; r < rows; r += gridDim.y) {
    const float d = Io<T>::Get(dy + r * cols + c);
    sw += d * ((Io<T>::Get(x + r * cols + c) - (rms ? 0.0f : mean[r])) * rstd[r]);
    sb += d;
  }
  float* ow = gridDim.y > 1 ? part + static_cast<size_t>(blockIdx.y) * 2 * cols : dw;
  ow[c] = sw;
  if (db) (gridDim.y > 1 ? ow + cols : db)[c] = sb;
}

// dw and db from `n` partial rows: 32 columns a workgroup, eight threads a
// column, each over every eighth partial, joined in order.
constexpr int kFoldCols = 32, kFoldParts = 8;
__global__ void __launch_bounds__(kFoldCols * kFoldParts)
NormFoldKernel(const float* __restrict__ part, int n, size_t cols, float* __restrict__ dw,
               float* __restrict__ db) {
  __shared__ float lds[kFoldParts][kFoldCols];
  const int i = threadIdx.x % kFoldCols, k = threadIdx.x / kFoldCols;
  const size_t c = static_cast<size_t>(blockIdx.x) * kFoldCols + i;
  const size_t width = db ? 2 * cols : cols;
  float s = 0.0f;
  if (c < width) {
#pragma unroll 8
    for (int p = k; p < n; p += kFoldParts) s += part[static_cast<size_t>(p) * 2 * cols + c];
  }
  lds[k][i] = s;
  __syncthreads();
  if (k == 0 && c < width) {
#pragma unroll
    for (int j = 1; j < kFoldParts; ++j) s += lds[j][i];
    (c < cols ? dw[c] : db[c - cols]) = s;
  }
}

// Workgroups of the backward pass: two a CU where two of them fit and each has
// rows to walk (four turns), else one; each leaves a partial row to be written
// and added.  us over 256 and 512 (layer, bf16): 8192 x 2048 30.6 and 29.0,
// 32000 x 2048 108 and 80, but 3001 x 1023 13.8 and 15.2, 600 x 2048 12.8 and
// 15.7, and with 1024 threads a workgroup 2000 x 8192 35 and 48, 16000 x 8192
// 180 and 194.
constexpr size_t kBwdGroups = 512;
size_t BwdGroups(int threads, size_t groups) {
  const size_t most = threads > 512 || groups < 4 * kBwdGroups ? kBwdGroups / 2 : kBwdGroups;
  return groups < most ? groups : most;
}
constexpr size_t kRegCols = 16384;  // the longest row held in registers

// A launch's workgroups (the kernels walk the rows past them).
dim3 Grid(size_t groups) {
  return dim3(static_cast<unsigned>(groups < (1u << 20) ? groups : 1u << 20));
}

struct NormCall {
  int rms;
  const void *dy, *x;
  const float *w, *b, *mean, *rstd;
  void* out;  // y or dx
  float *o1, *o2;  // mean and rstd, or dw and db
  float* part;
  size_t rows, cols;
  float eps;
};

template <class T, int kTPR, int kE, bool kVec, bool kAny>
hipError_t Run(const NormCall& a, bool bwd, hipStream_t s) {
  const int cols = static_cast<int>(a.cols);
  if (kAny || !bwd) {  // (kAny: Dispatch asks for the forward alone)
    constexpr int kRows = Threads(kTPR) / kTPR;
    const size_t groups = (a.rows + kRows - 1) / kRows;
    hipLaunchKernelGGL((NormFwdKernel<T, kTPR, kE, kVec, kAny>), Grid(groups), dim3(Threads(kTPR)), 0, s, a.rms,
                       static_cast<const T*>(a.x), a.w, a.b,
                       static_cast<T*>(a.out), a.o1, a.o2, a.rows, cols, a.eps);
    return hipGetLastError();
  }
  constexpr int kThreads = BwdThreads(kTPR), kRows = kThreads / kTPR;
  const size_t groups = (a.rows + kRows - 1) / kRows;
  const unsigned grid = groups ? static_cast<unsigned>(BwdGroups(kThreads, groups)) : 1;
  hipLaunchKernelGGL((NormBwdKernel<T, kTPR, kE, kVec>), dim3(grid), dim3(kThreads), 0, s,
                     a.rms, static_cast<const T*>(a.dy), static_cast<const T*>(a.x), a.w, a.mean,
                     a.rstd, static_cast<T*>(a.out), a.o1, a.o2, a.part, a.rows, cols);
  if (hipError_t e = hipGetLastError(); e != hipSuccess || grid == 1) return e;
  const size_t width = a.o2 ? 2 * a.cols : a.cols;
  hipLaunchKernelGGL(NormFoldKernel, dim3(static_cast<unsigned>((width + kFoldCols - 1) / kFoldCols)),
                     dim3(kFoldCols * kFoldParts), 0, s, a.part, static_cast<int>(grid), a.cols,
                     a.o1, a.o2);
  return hipGetLastError();
}

template <class T, bool kVec, bool kAny>
hipError_t Pick(const NormCall& a, bool bwd, hipStream_t s) {
  // Eight elements a lane: four waves a SIMD.  With sixteen the backward's sums
  // and the row in flight leave it two (8192 x 2048 bf16: 30 us either way;
  // 3001 x 1023 f32, single elements: 17 us against 16).
  if (a.cols <= 512) return Run<T, 64, 8, kVec, kAny>(a, bwd, s);
  if (a.cols <= 1024) return Run<T, 128, 8, kVec, kAny>(a, bwd, s);
  if (a.cols <= 2048) return Run<T, 256, 8, kVec, kAny>(a, bwd, s);
  if (a.cols <= 4096) return Run<T, 512, 8, kVec, kAny>(a, bwd, s);
  if (a.cols <= 8192) return Run<T, 1024, 8, kVec, kAny>(a, bwd, s);
  return Run<T, 1024, 16, kVec, kAny>(a, bwd, s);
}

template <class T>
hipError_t Long(const NormCall& a, bool bwd, hipStream_t s) {
  const T *dy = static_cast<const T*>(a.dy), *x = static_cast<const T*>(a.x);
  if (!bwd) {
    hipLaunchKernelGGL((NormFwdLongKernel<T>), Grid(a.rows), dim3(kLong), 0, s, a.rms, x, a.w,
                       a.b, static_cast<T*>(a.out), a.o1, a.o2, a.rows, a.cols, a.eps);
    return hipGetLastError();
  }
  if (a.rows) {
    hipLaunchKernelGGL((NormDxLongKernel<T>), Grid(a.rows), dim3(kLong), 0, s, a.rms, dy, x, a.w,
                       a.mean, a.rstd, static_cast<T*>(a.out), a.rows, a.cols);
    if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
  }
  // (Past 2^24 the columns fill the chip by themselves.)
  const size_t bands = a.rows < 128 || a.cols >> 24 ? 1 : a.rows / 64 < 64 ? a.rows / 64 : 64;
  hipLaunchKernelGGL((NormDwLongKernel<T>),
                     dim3(static_cast<unsigned>((a.cols + 255) / 256), static_cast<unsigned>(bands)),
                     dim3(256), 0, s, a.rms, dy, x, a.mean, a.rstd, a.o1, a.o2, a.part, a.rows,
                     a.cols);
  if (hipError_t e = hipGetLastError(); e != hipSuccess || bands == 1) return e;
  const size_t width = a.o2 ? 2 * a.cols : a.cols;
  hipLaunchKernelGGL(NormFoldKernel, dim3(static_cast<unsigned>((width + kFoldCols - 1) / kFoldCols)),
                     dim3(kFoldCols * kFoldParts), 0, s, a.part, static_cast<int>(bands), a.cols,
                     a.o1, a.o2);
  return hipGetLastError();
}

template <class T>
hipError_t Dispatch(const NormCall& a, bool bwd, hipStream_t s) {
  if (a.cols > kRegCols) return Long<T>(a, bwd, s);
  // 16-byte accesses where every row and vector begins on 16 bytes.
  const uintptr_t at = reinterpret_cast<uintptr_t>(a.dy) | reinterpret_cast<uintptr_t>(a.x) |
                       reinterpret_cast<uintptr_t>(a.w) | reinterpret_cast<uintptr_t>(a.b) |
                       reinterpret_cast<uintptr_t>(a.out);
  if (a.cols % Io<T>::kV == 0 && (at & 15) == 0) return Pick<T, true, false>(a, bwd, s);
  // Off that, the forward of wide rows still takes 16 bytes at a time, against
  // single elements, us (layer): bf16 30000 x 500 19.8 and 23.6, 4000 x 4095 26
  // and 42, but 30000 x 77 17.7 and 12.8 (most lanes have the short group); f32
  // 4000 x 4095 25 and 29, but 16384 x 1001 23.7 and 22.8.  The backward loses at
  // every width (bf16 4000 x 4095 52 and 32): its rows in flight would wait for
  // the short group's branch.
  if (!bwd && a.cols > (sizeof(T) == 2 ? 256 : 2048)) return Pick<T, true, true>(a, bwd, s);
  return Pick<T, false, false>(a, bwd, s);
}

}  // namespace

size_t NormBwdWorkspaceBytes(size_t rows, size_t cols) {
  const size_t n = rows < kBwdGroups ? rows : kBwdGroups;  // every pass's partial rows are fewer
  return n * 2 * cols * sizeof(float);
}

hipError_t LaunchNormFwd(int rms, int bf16, const void* x, const float* w, const float* b, void* y,
                         float* mean, float* rstd, size_t rows, size_t cols, float eps,
                         hipStream_t s) {
  if (rows == 0) return hipSuccess;
  const NormCall a{rms, nullptr, x, w, b, nullptr, nullptr, y, mean, rstd, nullptr, rows, cols, eps};
  return bf16 ? Dispatch<uint16_t>(a, false, s) : Dispatch<float>(a, false, s);
}

hipError_t LaunchNormBwd(int rms, int bf16, const void* dy, const void* x, const float* w,
                         const float* mean, const float* rstd, void* dx, float* dw, float* db,
                         size_t rows, size_t cols, void* ws, hipStream_t s) {
  const NormCall a{rms, dy, x, w, nullptr, mean, rstd, dx, dw, db, static_cast<float*>(ws),
                   rows, cols, 0.0f};
  return bf16 ? Dispatch<uint16_t>(a, true, s) : Dispatch<float>(a, true, s);
}

}  // namespace seeai
