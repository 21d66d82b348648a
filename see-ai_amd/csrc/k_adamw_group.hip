// k_adamw_group.hip -- one AdamW step over a group of tensors in one launch,
// the moments in f32 or in 8 bits.
//
// The update is AdamWElement's of k_optim.hip (optimizer.cc:104-132), every
// product and sum rounded in that order, so with 32-bit moments a tensor's
// bytes are seeai_adamw_step's.
//
// 8-bit moments: 128 elements share a scale, the power of two that brings the
// block's largest finite magnitude into (224, 448]; a moment is a float of
// four significant bits (e4m3, no infinities) under it.  m is held as it is,
// v as r = sqrt(v): half the exponent range, and the root is at hand.  A code
// is 6 to 12 % from the next, while v moves by a thousandth of itself a step:
// rounded to the nearest it would never move, so both moments are rounded
// stochastically, q up with the chance of its remainder, by 16 bits each that
// Mix draws from (seed, step, the element's number in the group) -- the mean
// is right and the same call gives the same bytes.  A power of two scales
// without rounding, so the codes hold the f32 moments' own leading bits.
// r > 0 keeps at least the smallest code, 2^-9 of the scale: no element with a
// gradient behind it divides by eps alone, and below that code r is held too
// large (at 0.3 of it v is eleven times itself), so such an element's steps
// are smaller than f32 moments would make them.  v = r^2 gains r's variance: of
// what it climbs up to gap / 2r, 1/16 among the normal codes, half among the
// subnormal.  A NaN or infinite moment takes the NaN code and
// stays with its element; it does not count towards the block's scale.
//
// Bound by HBM: per element p in and out, g in, m and v in and out.  A lane
// takes eight neighbours (a block is 16 lanes), a workgroup 2048 elements;
// which tensor they lie in comes from a binary search of the device table.
// 34.6 M parameters in five tensors, bf16 gradients and copy, on MI355X: 32-bit
// moments 185 us (28 bytes each, 5.2 TB/s; a copy runs 5.1), 8-bit 113 to 131
// (16 1/8 bytes; the hashes and the coding are not hidden entirely); 96 tensors
// of 0.6 M together 6.9, a launch's length.
#include "common.h"

namespace seeai {
namespace {

constexpr int kThreads = 256, kPer = 8;
static_assert(kThreads * kPer == kAdamWChunk && kAdamWChunk % kAdamWBlock == 0, "whole blocks");

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f2 __attribute__((ext_vector_type(2)));

__device__ __forceinline__ uint32_t Mix(uint32_t h) {
  h = (h ^ (h >> 15)) * 0x6C8E9CF5u;
  h = (h ^ (h >> 13)) * 0x3A5D2B97u;
  return h ^ (h >> 16);
}

// The largest of a value over the 16 lanes of a block (their max on each).
__device__ __forceinline__ float BlockMax16(float v) {
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o, 16));
  return v;
}

// 2^e as a float's exponent field: the scale of a block whose largest finite
// magnitude is `big`, clamped to normal floats whose reciprocal is one too.
__device__ __forceinline__ float ScaleOf(float big) {
  const uint32_t b = __float_as_uint(big);
  int e = static_cast<int>(b >> 23) - 8 + ((b & 0x7FFFFFu) > 0x600000u);  // above 1.75: one more
  e = e < 1 ? 1 : e;
  return __uint_as_float(static_cast<uint32_t>(e) << 23);
}

// |v| / scale rounded to e4m3 by 16 random bits: q + 2^-6 lays the subnormals'
// grid (2^-9) on the same mantissa bits as the normals'.
__device__ __forceinline__ uint32_t Encode(float v, float inv_scale, uint32_t bits16, bool least) {
  const float q = fabsf(v) * inv_scale;
  if (!(q <= 448.0f)) return 0x7Fu | (v < 0.0f ? 0x80u : 0u);  // NaN or infinite
  const bool small = q < 0.015625f;
  const uint32_t b = __float_as_uint(small ? q + 0.015625f : q) + (bits16 << 4);
  uint32_t code = (b >> 20) - (small ? 968u : 960u);
  if (least && code == 0 && q > 0.0f) code = 1;
  return code | (v < 0.0f ? 0x80u : 0u);
}

__device__ __forceinline__ void Decode8(uint2 c, float scale, float (&v)[kPer]) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int w = static_cast<int>(i ? c.y : c.x);
    const f2 lo = __builtin_amdgcn_cvt_pk_f32_fp8(w, false);
    const f2 hi = __builtin_amdgcn_cvt_pk_f32_fp8(w, true);
    v[4 * i] = lo[0] * scale, v[4 * i + 1] = lo[1] * scale;
    v[4 * i + 2] = hi[0] * scale, v[4 * i + 3] = hi[1] * scale;
  }
}

// Eight neighbours of an f32 tensor, 16 bytes at a time where they may be.
__device__ __forceinline__ void Load8(const float* p, bool vec, int cnt, float (&v)[kPer]) {
  if (vec && cnt == kPer) {
    const float4 a = *reinterpret_cast<const float4*>(p);
    const float4 b = *reinterpret_cast<const float4*>(p + 4);
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
  } else {
#pragma unroll
    for (int e = 0; e < kPer; ++e) v[e] = e < cnt ? p[e] : 0.0f;
  }
}
// As vector types: the compiler splits a float4 struct's stores into 4 and 12 bytes
// (34.6 M parameters, bf16 gradients, 186 us against 172).  Stored past the caches the
// moments save nothing, and cost 3 to 6 % where the last cache holds them from one step
// to the next (12 M, f32 gradients, 56 against 53).
__device__ __forceinline__ void Store8(float* p, bool vec, int cnt, const float (&v)[kPer]) {
  if (vec && cnt == kPer) {
    *reinterpret_cast<v4f*>(p) = v4f{v[0], v[1], v[2], v[3]};
    *reinterpret_cast<v4f*>(p + 4) = v4f{v[4], v[5], v[6], v[7]};
  } else {
#pragma unroll
    for (int e = 0; e < kPer; ++e)
      if (e < cnt) p[e] = v[e];
  }
}
__device__ __forceinline__ void Load8(const uint16_t* p, bool vec, int cnt, float (&v)[kPer]) {
  if (vec && cnt == kPer) {
    const uint4 a = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = __uint_as_float(w[i] << 16);
      v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
    }
  } else {
#pragma unroll
    for (int e = 0; e < kPer; ++e) v[e] = e < cnt ? Bf16ToF32(p[e]) : 0.0f;
  }
}
__device__ __forceinline__ uint2 LoadCodes(const uint8_t* p, bool vec, int cnt) {
  if (vec && cnt == kPer) return *reinterpret_cast<const uint2*>(p);
  uint32_t w[2] = {0, 0};
#pragma unroll
  for (int e = 0; e < kPer; ++e)
    if (e < cnt) w[e / 4] |= static_cast<uint32_t>(p[e]) << (8 * (e % 4));
  return make_uint2(w[0], w[1]);
}
__device__ __forceinline__ void StoreCodes(uint8_t* p, bool vec, int cnt, const uint32_t (&c)[kPer]) {
  if (vec && cnt == kPer) {
    *reinterpret_cast<uint2*>(p) =
        make_uint2(c[0] | c[1] << 8 | c[2] << 16 | c[3] << 24, c[4] | c[5] << 8 | c[6] << 16 | c[7] << 24);
  } else {
#pragma unroll
    for (int e = 0; e < kPer; ++e)
      if (e < cnt) p[e] = static_cast<uint8_t>(c[e]);
  }
}

template <int kBits, class G>
__global__ void __launch_bounds__(kThreads)
AdamWGroupKernel(const AdamWGroupTensor* __restrict__ tab, int count, AdamWGroupStep args,
                 const AdamWGroupStep* __restrict__ held, const float* __restrict__ factor,
                 const int* __restrict__ flag) {
  if (*flag) return;
  const AdamWGroupStep P = held ? *held : args;
  // The tensor this chunk lies in: the last whose first chunk is not past it.
  int lo = 0, hi = count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) / 2;
    if (tab[mid].first_chunk <= blockIdx.x) lo = mid;
    else hi = mid - 1;
  }
  const AdamWGroupTensor T = tab[lo];
  const uint64_t at = static_cast<uint64_t>(blockIdx.x - T.first_chunk) * kAdamWChunk +
                      threadIdx.x * kPer;
  const int cnt = at >= T.n ? 0 : T.n - at < kPer ? static_cast<int>(T.n - at) : kPer;
  const bool vec = T.vec;
  float p[kPer], g[kPer], m[kPer], v[kPer];
  Load8(T.p + at, vec, cnt, p);
  Load8(static_cast<const G*>(T.g) + at, vec, cnt, g);
  if constexpr (kBits == 32) {
    Load8(static_cast<const float*>(T.m) + at, vec, cnt, m);
    Load8(static_cast<const float*>(T.v) + at, vec, cnt, v);
  } else {
    const uint64_t blk = at / kAdamWBlock;
    const float ms = cnt ? T.m_scale[blk] : 0.0f, vs = cnt ? T.v_scale[blk] : 0.0f;
    Decode8(LoadCodes(static_cast<const uint8_t*>(T.m) + at, vec, cnt), ms, m);
    Decode8(LoadCodes(static_cast<const uint8_t*>(T.v) + at, vec, cnt), vs, v);
#pragma unroll
    for (int e = 0; e < kPer; ++e) v[e] = v[e] * v[e];
  }
  if (factor) {  // a clipped step
    const float f = *factor;
#pragma unroll
    for (int e = 0; e < kPer; ++e) g[e] *= f;
  }
  const float om_b1 = 1.0f - P.beta1, om_b2 = 1.0f - P.beta2, wd = P.weight_decay * T.decay;
#pragma unroll
  for (int e = 0; e < kPer; ++e) {
    m[e] = P.beta1 * m[e] + om_b1 * g[e];
    v[e] = P.beta2 * v[e] + om_b2 * g[e] * g[e];
    const float m_hat = m[e] * P.inv_bc1, v_hat = v[e] * P.inv_bc2;
    p[e] = p[e] - P.lr * (m_hat / (sqrtf(v_hat) + P.eps) + wd * p[e]);
  }
  Store8(T.p + at, vec, cnt, p);
  if (T.p_bf16) {
    if (vec && cnt == kPer) {
      bf16x8 o;
#pragma unroll
      for (int e = 0; e < kPer; ++e) o[e] = static_cast<__bf16>(p[e]);
      *reinterpret_cast<bf16x8*>(T.p_bf16 + at) = o;
    } else {
#pragma unroll
      for (int e = 0; e < kPer; ++e)
        if (e < cnt) T.p_bf16[at + e] = F32ToBf16(p[e]);
    }
  }
  if constexpr (kBits == 32) {
    Store8(static_cast<float*>(T.m) + at, vec, cnt, m);
    Store8(static_cast<float*>(T.v) + at, vec, cnt, v);
  } else {
    float big_m = 0.0f, big_v = 0.0f;
#pragma unroll
    for (int e = 0; e < kPer; ++e) {  // elements past the tensor's end do not count
      v[e] = sqrtf(v[e]);
      const float am = fabsf(m[e]), av = v[e];
      big_m = fmaxf(big_m, e < cnt && am <= 3.4028234663852886e38f ? am : 0.0f);
      big_v = fmaxf(big_v, e < cnt && av <= 3.4028234663852886e38f ? av : 0.0f);
    }
    const float ms = ScaleOf(BlockMax16(big_m)), vs = ScaleOf(BlockMax16(big_v));
    const float im = 1.0f / ms, iv = 1.0f / vs;
    const uint64_t number = T.first_block * kAdamWBlock + at;  // a multiple of 8
    const uint32_t key = Mix(P.key ^ static_cast<uint32_t>(number >> 32));
    uint32_t cm[kPer], cv[kPer];
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
      const uint32_t bits = Mix((static_cast<uint32_t>(number) + e) ^ key);
      cm[e] = Encode(m[e], im, bits & 0xFFFFu, false);
      cv[e] = Encode(v[e], iv, bits >> 16, true);
    }
    StoreCodes(static_cast<uint8_t*>(T.m) + at, vec, cnt, cm);
    StoreCodes(static_cast<uint8_t*>(T.v) + at, vec, cnt, cv);
    if (at % kAdamWBlock == 0 && cnt) {
      T.m_scale[at / kAdamWBlock] = ms;
      T.v_scale[at / kAdamWBlock] = vs;
    }
  }
}

__global__ void AdamWGroupHoldKernel(AdamWGroupStep* held, AdamWGroupStep args) { *held = args; }

// What codes stand for: m, or v = r^2.
template <class T>
__global__ void __launch_bounds__(kThreads)
AdamWValuesKernel(int second, const uint8_t* __restrict__ codes, const float* __restrict__ scales,
                  uint64_t n, T* __restrict__ out, bool vec) {
  const uint64_t at = (static_cast<uint64_t>(blockIdx.x) * kThreads + threadIdx.x) * kPer;
  if (at >= n) return;
  const int cnt = n - at < kPer ? static_cast<int>(n - at) : kPer;
  float v[kPer];
  Decode8(LoadCodes(codes + at, vec, cnt), scales[at / kAdamWBlock], v);
  if (second) {
#pragma unroll
    for (int e = 0; e < kPer; ++e) v[e] = v[e] * v[e];
  }
  if constexpr (sizeof(T) == 4) {
    Store8(out + at, vec, cnt, v);
  } else if (vec && cnt == kPer) {
    bf16x8 o;
#pragma unroll
    for (int e = 0; e < kPer; ++e) o[e] = static_cast<__bf16>(v[e]);
    *reinterpret_cast<bf16x8*>(out + at) = o;
  } else {
#pragma unroll
    for (int e = 0; e < kPer; ++e)
      if (e < cnt) out[at + e] = F32ToBf16(v[e]);
  }
}

uint32_t HostMix(uint32_t h) {
  h = (h ^ (h >> 15)) * 0x6C8E9CF5u;
  h = (h ^ (h >> 13)) * 0x3A5D2B97u;
  return h ^ (h >> 16);
}

}  // namespace

uint32_t AdamWGroupKey(uint32_t seed, uint64_t step) {
  return HostMix(HostMix(seed) ^ static_cast<uint32_t>(step));
}

hipError_t LaunchAdamWGroup(const AdamWGroupTensor* tab, int count, uint64_t chunks, int bits,
                            int grads_bf16, const AdamWGroupStep& args, const AdamWGroupStep* held,
                            const float* factor, const int* flag, hipStream_t s) {
  if (chunks == 0) return hipSuccess;
  auto go = [&](auto* kernel) {
    hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(chunks)), dim3(kThreads), 0, s, tab,
                       count, args, held, factor, flag);
    return hipGetLastError();
  };
  if (bits == 32) return grads_bf16 ? go(AdamWGroupKernel<32, uint16_t>) : go(AdamWGroupKernel<32, float>);
  return grads_bf16 ? go(AdamWGroupKernel<8, uint16_t>) : go(AdamWGroupKernel<8, float>);
}

hipError_t LaunchAdamWGroupHold(AdamWGroupStep* held, const AdamWGroupStep& args, hipStream_t s) {
  hipLaunchKernelGGL(AdamWGroupHoldKernel, dim3(1), dim3(1), 0, s, held, args);
  return hipGetLastError();
}

hipError_t LaunchAdamWValues(int second, int bf16, const uint8_t* codes, const float* scales,
                             uint64_t n, void* out, hipStream_t s) {
  if (n == 0) return hipSuccess;
  const bool vec = ((reinterpret_cast<uintptr_t>(codes) & 7) | (reinterpret_cast<uintptr_t>(out) & 15)) == 0;
  const unsigned grid = static_cast<unsigned>((n + kAdamWChunk - 1) / kAdamWChunk);
  if (bf16)
    hipLaunchKernelGGL((AdamWValuesKernel<uint16_t>), dim3(grid), dim3(kThreads), 0, s, second,
                       codes, scales, n, static_cast<uint16_t*>(out), vec);
  else
    hipLaunchKernelGGL((AdamWValuesKernel<float>), dim3(grid), dim3(kThreads), 0, s, second, codes,
                       scales, n, static_cast<float*>(out), vec);
  return hipGetLastError();
}

}  // namespace seeai
