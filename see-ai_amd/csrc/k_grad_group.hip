// k_grad_group.hip -- the global norm of a step's gradients over many tensors
// (f32 and bf16 beside each other), the factor that clips it, and the clip in
// place.
//
//   norm = sqrt(sum of g^2 over all tensors),  factor = min(1, max_norm / norm)
//
// The verdicts are the per-tensor clip's (k_optim.hip; optimizer.cc:40-85): a
// norm that is not finite sets the refusal word, and no step behind it writes
// anything.  Squares are f64 (an f32 square overflows from 1.8e19 on) and so
// are their sums: a workgroup adds its share of the chunks, one the shares, in an
// order that the group's sizes alone decide -- the same bits every run.  Up to a
// million elements the workgroup that is done last adds the shares (a counter in
// the group's own memory says which), past that a second launch: counting makes
// each workgroup write back and drop its L2's lines, 3.5 us for 64 of them, where
// a launch costs as much on the host, but 50 us for 2048.  Bound by HBM: every
// gradient read once (four chunks' loads at a time instead of one: 22 us against
// 17 for 34.6 M bf16; eight waves a SIMD hide them already).  The factor stays on
// the device, where the step multiplies by it (k_adamw_group.hip), so that
// clipping costs no pass of its own.
#include "rows.h"

namespace seeai {
namespace {

constexpr int kThreads = 256, kPer = 8;
static_assert(kThreads * kPer == kGradChunk, "a chunk is a workgroup's turn");
constexpr int kOneParts = 64;
constexpr uint64_t kOneChunks = 512;

__device__ __forceinline__ int TensorOf(const GradGroupTensor* tab, int count, uint64_t chunk) {
  int lo = 0, hi = count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) / 2;
    if (tab[mid].first_chunk <= chunk) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

// Eight neighbours from element `at` on, zeros past the tensor.
__device__ __forceinline__ void Load(const GradGroupTensor& T, uint64_t at, float (&v)[kPer]) {
  const bool whole = T.vec && at + kPer <= T.n;
  if (T.bf16) {
    const uint16_t* g = static_cast<const uint16_t*>(T.g) + at;
    if (whole) {
      Io<uint16_t>::Load(g, v);
    } else {
#pragma unroll
      for (int e = 0; e < kPer; ++e) v[e] = at + e < T.n ? Bf16ToF32(g[e]) : 0.0f;
    }
  } else {
    const float* g = static_cast<const float*>(T.g) + at;
    if (whole) {
      Io<float>::Load(g, v);
      Io<float>::Load(g + 4, v + 4);
    } else {
#pragma unroll
      for (int e = 0; e < kPer; ++e) v[e] = at + e < T.n ? g[e] : 0.0f;
    }
  }
}

struct NormOut {
  float max_norm;
  float *norm, *factor;
  int* flag;
  __device__ void Put(double sum) const {
    const double s = sqrt(sum);
    if (norm) *norm = static_cast<float>(s);
    if (!(max_norm > 0.0f)) return;
    const double cap = static_cast<double>(max_norm);
    if (!isfinite(s)) *flag = 1;
    *factor = isfinite(s) && s > cap ? static_cast<float>(cap / s) : 1.0f;
  }
};

template <int kN>
__device__ __forceinline__ double BlockSum(double v, double* red) {  // on thread 0
  v = WaveSumD(v);
  if (threadIdx.x % kWave == 0) red[threadIdx.x / kWave] = v;
  __syncthreads();
#pragma unroll
  for (int w = 1; w < kN / kWave; ++w) v += red[w];
  return v;
}

// A workgroup's share of the chunks.  kOne: the workgroup that is done last adds
// the shares, in order, and puts the count of those done back to zero.
template <bool kOne>
__global__ void __launch_bounds__(kThreads)
GradNormKernel(const GradGroupTensor* __restrict__ tab, int count, uint64_t chunks, double* part,
               unsigned* done, NormOut out) {
  __shared__ double red[2][kThreads / kWave];
  __shared__ bool last;
  const uint64_t first = chunks * blockIdx.x / gridDim.x, end = chunks * (blockIdx.x + 1) / gridDim.x;
  int i = TensorOf(tab, count, first);
  GradGroupTensor T = tab[i];
  double sq = 0.0;
  for (uint64_t c = first; c < end; ++c) {
    while (i + 1 < count && tab[i + 1].first_chunk <= c) T = tab[++i];
    float v[kPer];
    Load(T, (c - T.first_chunk) * kGradChunk + threadIdx.x * kPer, v);
#pragma unroll
    for (int e = 0; e < kPer; ++e) sq += static_cast<double>(v[e]) * static_cast<double>(v[e]);
  }
  sq = BlockSum<kThreads>(sq, red[0]);
  if (threadIdx.x == 0) {
    part[blockIdx.x] = sq;
    if constexpr (kOne)
      last = __hip_atomic_fetch_add(done, 1u, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT) + 1 == gridDim.x;
  }
  if constexpr (kOne) {
    static_assert(kOneParts <= kThreads, "a share a thread");
    __syncthreads();
    if (!last) return;
    sq = threadIdx.x < gridDim.x
             ? __hip_atomic_load(part + threadIdx.x, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) : 0.0;
    sq = BlockSum<kThreads>(sq, red[1]);
    if (threadIdx.x != 0) return;
    __hip_atomic_store(done, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    out.Put(sq);
  }
}

constexpr int kFoldThreads = 512, kMostParts = 2048;
__global__ void __launch_bounds__(kFoldThreads)
GradFactorKernel(const double* __restrict__ part, int n, NormOut out) {
  __shared__ double red[kFoldThreads / kWave];
  double s = 0.0;
#pragma unroll
  for (int k = 0; k < kMostParts / kFoldThreads; ++k) {  // all loads together
    const int i = threadIdx.x + k * kFoldThreads;
    s += i < n ? part[i] : 0.0;
  }
  s = BlockSum<kFoldThreads>(s, red);
  if (threadIdx.x == 0) out.Put(s);
}

__global__ void __launch_bounds__(kThreads)
GradScaleKernel(const GradGroupTensor* __restrict__ tab, int count, const float* __restrict__ factor,
                const int* __restrict__ flag) {
  const float f = *factor;
  if (*flag || f == 1.0f) return;
  const GradGroupTensor T = tab[TensorOf(tab, count, blockIdx.x)];
  const uint64_t at = (blockIdx.x - T.first_chunk) * kGradChunk + threadIdx.x * kPer;
  if (at >= T.n) return;
  float v[kPer];
  Load(T, at, v);
#pragma unroll
  for (int e = 0; e < kPer; ++e) v[e] *= f;
  const bool whole = T.vec && at + kPer <= T.n;
  if (T.bf16) {
    uint16_t* g = static_cast<uint16_t*>(T.g) + at;
    if (whole) {
      Io<uint16_t>::Store(g, v);
    } else {
#pragma unroll
      for (int e = 0; e < kPer; ++e)
        if (at + e < T.n) g[e] = F32ToBf16(v[e]);
    }
  } else {
    float* g = static_cast<float*>(T.g) + at;
    if (whole) {
      Io<float>::Store(g, v);
      Io<float>::Store(g + 4, v + 4);
    } else {
#pragma unroll
      for (int e = 0; e < kPer; ++e)
        if (at + e < T.n) g[e] = v[e];
    }
  }
}

}  // namespace

// Workgroups of the norm: up to kOneChunks chunks one launch of few workgroups,
// whose count is soon kept.
int GradNormParts(uint64_t chunks) {
  const uint64_t most = chunks <= kOneChunks ? kOneParts : kMostParts;
  return static_cast<int>(chunks < most ? chunks : most);
}

hipError_t LaunchGradNorm(const GradGroupTensor* tab, int count, uint64_t chunks, double* part,
                          unsigned* done, float max_norm, float* norm, float* factor, int* flag,
                          hipStream_t s) {
  const int n = GradNormParts(chunks);
  const NormOut out{max_norm, norm, factor, flag};
  if (n && chunks <= kOneChunks) {
    hipLaunchKernelGGL((GradNormKernel<true>), dim3(n), dim3(kThreads), 0, s, tab, count, chunks, part,
                       done, out);
    return hipGetLastError();
  }
  if (n) {
    hipLaunchKernelGGL((GradNormKernel<false>), dim3(n), dim3(kThreads), 0, s, tab, count, chunks, part,
                       done, out);
    if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
  }
  hipLaunchKernelGGL(GradFactorKernel, dim3(1), dim3(kFoldThreads), 0, s, part, n, out);
  return hipGetLastError();
}

hipError_t LaunchGradScale(const GradGroupTensor* tab, int count, uint64_t chunks,
                           const float* factor, const int* flag, hipStream_t s) {
  if (chunks == 0) return hipSuccess;
  hipLaunchKernelGGL(GradScaleKernel, dim3(static_cast<unsigned>(chunks)), dim3(kThreads), 0, s, tab,
                     count, factor, flag);
  return hipGetLastError();
}

}  // namespace seeai
