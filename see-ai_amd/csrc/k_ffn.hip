// k_ffn.hip -- the gated feed-forward block, forward and backward.
//
//   G = X Wg, U = X Wu, H = act(G) U, Y = H Wd
//   dH = dY Wd', dG = dH U act'(G), dU = dH act(G)
//   dX = dG Wg' + dU Wu', dWg = X' dG, dWu = X' dU, dWd = H' dY
//
// Every product runs on FfnMma, a bf16 MFMA tile kernel whose epilogue does the
// rest: the forward's first launch holds a gate tile and the up tile of the
// same columns side by side and stores act(G) U; the backward's first forms
// dG, dU and H from its dH accumulators, so dH is never stored.  Two launches
// forward (G and U; Y), four backward (dH; dX; dWg and dWu; dWd).
//
// bf16: the operands as they are.  f32: each operand is split into three bf16
// planes (x = hi + mid + lo, eight bits each, truncated, so exactly x), and a
// product is the six plane products down to 2^-16 of it, all into the same f32
// accumulators: f32's accuracy at a sixth of the bf16 rate, 1.6 times the f32
// MFMA's.  An infinity's remainder is a NaN, so what an infinity reaches is
// not finite but may be a NaN where f32 arithmetic has an infinity.
#include <algorithm>
#include <type_traits>

#include "common.h"

namespace seeai {
namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) void* LdsPtr;

constexpr int kStageK = 32;            // K of one stage
constexpr int kRsrcWord3 = 0x00020000;  // raw buffer, out-of-range reads give 0
constexpr int kFar = 0x7FFFFFFF;        // an offset past every range

// s_waitcnt vmcnt(n), other counters untouched (gfx9 encoding).
template <int n>
__device__ __forceinline__ void WaitVm() {
  static_assert(n >= 0 && n < 64, "vmcnt range");
  __builtin_amdgcn_s_waitcnt((n & 15) | (7 << 4) | (15 << 8) | ((n >> 4) << 14));
}

// 16 bytes a lane, lane after lane, straight into LDS.
__device__ __forceinline__ void LoadLds(__amdgpu_buffer_rsrc_t rs, uint8_t* lds, int voff, int soff) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (LdsPtr)lds, 16, voff, soff, 0, 0);
}

// The workgroup's barrier, which no access may be moved across.
__device__ __forceinline__ void Barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
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

template <class T> __device__ __forceinline__ float Get(const T* p);
template <> __device__ __forceinline__ float Get<float>(const float* p) { return *p; }
template <> __device__ __forceinline__ float Get<uint16_t>(const uint16_t* p) { return Bf16ToF32(*p); }
template <class T> __device__ __forceinline__ void Put(T* p, float v);
template <> __device__ __forceinline__ void Put<float>(float* p, float v) { *p = v; }
template <> __device__ __forceinline__ void Put<uint16_t>(uint16_t* p, float v) { *p = F32ToBf16(v); }

__device__ __forceinline__ void Get4(const float* p, bool vec, int cnt, float (&v)[4]) {
  if (vec) {
    const float4 a = *reinterpret_cast<const float4*>(p);
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w;
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = e < cnt ? p[e] : 0.0f;
  }
}
__device__ __forceinline__ void Get4(const uint16_t* p, bool vec, int cnt, float (&v)[4]) {
  if (vec) {
    const uint2 a = *reinterpret_cast<const uint2*>(p);
    v[0] = __uint_as_float(a.x << 16), v[1] = __uint_as_float(a.x & 0xFFFF0000u);
    v[2] = __uint_as_float(a.y << 16), v[3] = __uint_as_float(a.y & 0xFFFF0000u);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = e < cnt ? Bf16ToF32(p[e]) : 0.0f;
  }
}
__device__ __forceinline__ void Put4(float* p, bool vec, int cnt, const float (&v)[4]) {
  if (vec) {
    *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (e < cnt) p[e] = v[e];
  }
}
__device__ __forceinline__ void Put4(uint16_t* p, bool vec, int cnt, const float (&v)[4]) {
  if (vec) {
    StoreBf16x4(p, v);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (e < cnt) p[e] = F32ToBf16(v[e]);
  }
}

// The next bf16 plane of a value: its top eight bits, taken off it.
__device__ __forceinline__ uint32_t TakePlane(float& x) {
  const uint32_t hi = __float_as_uint(x) & 0xFFFF0000u;
  x -= __uint_as_float(hi);
  return hi >> 16;
}

// A [rows, ld] operand in bf16 planes: one for bf16, three for f32.
struct Planes {
  uint16_t* p = nullptr;
  size_t plane = 0;  // elements of one plane
  int ld = 0;        // a multiple of 8, zeros past the row's own width
};
// Four neighbours into the planes (8-byte aligned: ld and the column are
// multiples of four).
template <class T>
__device__ __forceinline__ void PutPlanes(const Planes& out, size_t at, float (&v)[4]) {
  if constexpr (sizeof(T) == 2) {
    StoreBf16x4(out.p + at, v);
  } else {
#pragma unroll
    for (int k = 0; k < 3; ++k) {
      const uint32_t a = TakePlane(v[0]), b = TakePlane(v[1]), c = TakePlane(v[2]), d = TakePlane(v[3]);
      *reinterpret_cast<uint2*>(out.p + k * out.plane + at) = make_uint2(a | b << 16, c | d << 16);
    }
  }
}

// rows x cols (packed) into padded planes: operands whose rows or base are off
// 16 bytes, and every f32 operand.
template <class T>
__global__ void __launch_bounds__(256)
FfnPackKernel(const T* __restrict__ in, size_t rows, int cols, bool vec, Planes out) {
  const int quads = out.ld / 4;
  const size_t n = rows * quads, step = static_cast<size_t>(gridDim.x) * 256;
  for (size_t i = static_cast<size_t>(blockIdx.x) * 256 + threadIdx.x; i < n; i += step) {
    const size_t r = i / quads;
    const int c = static_cast<int>(i % quads) * 4;
    float v[4];
    Get4(in + r * cols + c, vec && c + 4 <= cols, cols - c, v);
    PutPlanes<T>(out, r * out.ld + c, v);
  }
}

template <class T>
__global__ void __launch_bounds__(256) FfnZeroKernel(T* __restrict__ out, size_t n) {
  const size_t step = static_cast<size_t>(gridDim.x) * 256;
  for (size_t i = static_cast<size_t>(blockIdx.x) * 256 + threadIdx.x; i < n; i += step) out[i] = 0;
}

// The products of one launch.  Operand element (i, k) lies at i ld + k, or,
// "strided", at k ld + i.  Segments are products of the same shape added up.
constexpr int kMaxSeg = 12;
struct MmaArgs {
  const uint16_t *A[kMaxSeg], *B[kMaxSeg], *B2[kMaxSeg];
  int nseg, lda, ldb;
  int M, N, K;
  int act;
  bool vec;           // outputs (and G, U) take four neighbours at once
  void *o1, *o2;      // plain: o1 (and o2 of B2); gate: G and U or null
  const void *g, *u;  // gradient: G and U
  Planes h, dg, du;
};

enum Epilogue {
  kPlain,  // o1 = sum A B
  kTwo,    // o1 = sum A B, o2 = sum A B2
  kGate,   // G = sum A B, U = sum A B2: o1, o2 where kept, h = act(G) U
  kGrad    // d = sum A B: dg = d U act'(G), du = d act(G), h = act(G) U
};

// Tile -> workgroup order: the 8 XCDs each take a contiguous run of tiles
// (workgroup b runs on XCD b % 8) walked in bands of row tiles, so concurrent
// tiles of one XCD share operand panels in its L2.
constexpr int kBand = 4;
__device__ __forceinline__ void TileOf(int b, int tiles_m, int tiles_n, int& tm, int& tn) {
  const int n = tiles_m * tiles_n;
  int t = b;
  if (n % 8 == 0) t = (b % 8) * (n / 8) + b / 8;
  const int per = kBand * tiles_n, first = t / per * kBand;
  const int rows = min(tiles_m - first, kBand), off = t % per;
  tm = first + off % rows;
  tn = off / rows;
}

// Transposing reads of `n` fragments, each two reads four K rows apart.  The
// compiler's own read waits for every load into LDS still in flight, so the
// reads are written out; each block waits for them itself.  Fragments are at
// LDS addresses a[] plus kA (plus kB from the fourth on).
template <int kOff, int kRow>
__device__ __forceinline__ void ReadTr(const uint32_t (&a)[1], bf16x8 (&f)[1]) {
  s16x4 r[2];
  asm volatile(
      "ds_read_b64_tr_b16 %0, %2 offset:%3\n\t"
      "ds_read_b64_tr_b16 %1, %2 offset:%4\n\t"
      "s_waitcnt lgkmcnt(0)"
      : "=&v"(r[0]), "=&v"(r[1])
      : "v"(a[0]), "n"(kOff), "n"(kOff + 4 * kRow)
      : "memory");
  f[0] = __builtin_bit_cast(bf16x8, __builtin_shufflevector(r[0], r[1], 0, 1, 2, 3, 4, 5, 6, 7));
}
template <int kOff, int kRow>
__device__ __forceinline__ void ReadTr(const uint32_t (&a)[2], bf16x8 (&f)[2]) {
  s16x4 r[4];
  asm volatile(
      "ds_read_b64_tr_b16 %0, %4 offset:%6\n\t"
      "ds_read_b64_tr_b16 %1, %4 offset:%7\n\t"
      "ds_read_b64_tr_b16 %2, %5 offset:%6\n\t"
      "ds_read_b64_tr_b16 %3, %5 offset:%7\n\t"
      "s_waitcnt lgkmcnt(0)"
      : "=&v"(r[0]), "=&v"(r[1]), "=&v"(r[2]), "=&v"(r[3])
      : "v"(a[0]), "v"(a[1]), "n"(kOff), "n"(kOff + 4 * kRow)
      : "memory");
#pragma unroll
  for (int i = 0; i < 2; ++i)
    f[i] = __builtin_bit_cast(bf16x8, __builtin_shufflevector(r[2 * i], r[2 * i + 1], 0, 1, 2, 3, 4, 5, 6, 7));
}
// Two operands' fragments in one block.
template <int kOffA, int kRowA, int kOffB, int kRowB>
__device__ __forceinline__ void ReadTr2(const uint32_t (&a)[1], bf16x8 (&fa)[1], const uint32_t (&b)[1],
                                        bf16x8 (&fb)[1]) {
  s16x4 r[4];
  asm volatile(
      "ds_read_b64_tr_b16 %0, %4 offset:%6\n\t"
      "ds_read_b64_tr_b16 %1, %4 offset:%7\n\t"
      "ds_read_b64_tr_b16 %2, %5 offset:%8\n\t"
      "ds_read_b64_tr_b16 %3, %5 offset:%9\n\t"
      "s_waitcnt lgkmcnt(0)"
      : "=&v"(r[0]), "=&v"(r[1]), "=&v"(r[2]), "=&v"(r[3])
      : "v"(a[0]), "v"(b[0]), "n"(kOffA), "n"(kOffA + 4 * kRowA), "n"(kOffB), "n"(kOffB + 4 * kRowB)
      : "memory");
  fa[0] = __builtin_bit_cast(bf16x8, __builtin_shufflevector(r[0], r[1], 0, 1, 2, 3, 4, 5, 6, 7));
  fb[0] = __builtin_bit_cast(bf16x8, __builtin_shufflevector(r[2], r[3], 0, 1, 2, 3, 4, 5, 6, 7));
}
template <int kOffA, int kRowA, int kOffB, int kRowB>
__device__ __forceinline__ void ReadTr2(const uint32_t (&a)[1], bf16x8 (&fa)[1], const uint32_t (&b)[2],
                                        bf16x8 (&fb)[2]) {
  s16x4 r[6];
  asm volatile(
      "ds_read_b64_tr_b16 %0, %6 offset:%9\n\t"
      "ds_read_b64_tr_b16 %1, %6 offset:%10\n\t"
      "ds_read_b64_tr_b16 %2, %7 offset:%11\n\t"
      "ds_read_b64_tr_b16 %3, %7 offset:%12\n\t"
      "ds_read_b64_tr_b16 %4, %8 offset:%11\n\t"
      "ds_read_b64_tr_b16 %5, %8 offset:%12\n\t"
      "s_waitcnt lgkmcnt(0)"
      : "=&v"(r[0]), "=&v"(r[1]), "=&v"(r[2]), "=&v"(r[3]), "=&v"(r[4]), "=&v"(r[5])
      : "v"(a[0]), "v"(b[0]), "v"(b[1]), "n"(kOffA), "n"(kOffA + 4 * kRowA), "n"(kOffB),
        "n"(kOffB + 4 * kRowB)
      : "memory");
  fa[0] = __builtin_bit_cast(bf16x8, __builtin_shufflevector(r[0], r[1], 0, 1, 2, 3, 4, 5, 6, 7));
#pragma unroll
  for (int i = 0; i < 2; ++i)
    fb[i] = __builtin_bit_cast(bf16x8, __builtin_shufflevector(r[2 + 2 * i], r[3 + 2 * i], 0, 1, 2, 3, 4, 5, 6, 7));
}
template <int kOffA, int kRowA, int kOffB, int kRowB>
__device__ __forceinline__ void ReadTr2(const uint32_t (&a)[2], bf16x8 (&fa)[2], const uint32_t (&b)[2],
                                        bf16x8 (&fb)[2]) {
  s16x4 r[8];
  asm volatile(
      "ds_read_b64_tr_b16 %0, %8 offset:%12\n\t"
      "ds_read_b64_tr_b16 %1, %8 offset:%13\n\t"
      "ds_read_b64_tr_b16 %2, %9 offset:%12\n\t"
      "ds_read_b64_tr_b16 %3, %9 offset:%13\n\t"
      "ds_read_b64_tr_b16 %4, %10 offset:%14\n\t"
      "ds_read_b64_tr_b16 %5, %10 offset:%15\n\t"
      "ds_read_b64_tr_b16 %6, %11 offset:%14\n\t"
      "ds_read_b64_tr_b16 %7, %11 offset:%15\n\t"
      "s_waitcnt lgkmcnt(0)"
      : "=&v"(r[0]), "=&v"(r[1]), "=&v"(r[2]), "=&v"(r[3]), "=&v"(r[4]), "=&v"(r[5]), "=&v"(r[6]),
        "=&v"(r[7])
      : "v"(a[0]), "v"(a[1]), "v"(b[0]), "v"(b[1]), "n"(kOffA), "n"(kOffA + 4 * kRowA), "n"(kOffB),
        "n"(kOffB + 4 * kRowB)
      : "memory");
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    fa[i] = __builtin_bit_cast(bf16x8, __builtin_shufflevector(r[2 * i], r[2 * i + 1], 0, 1, 2, 3, 4, 5, 6, 7));
    fb[i] = __builtin_bit_cast(bf16x8, __builtin_shufflevector(r[4 + 2 * i], r[5 + 2 * i], 0, 1, 2, 3, 4, 5, 6, 7));
  }
}
template <int kOffA, int kRowA, int kOffB, int kRowB>
__device__ __forceinline__ void ReadTr2(const uint32_t (&a)[4], bf16x8 (&fa)[4], const uint32_t (&b)[2],
                                        bf16x8 (&fb)[2]) {
  s16x4 r[12];
  asm volatile(
      "ds_read_b64_tr_b16 %0, %12 offset:%18\n\t"
      "ds_read_b64_tr_b16 %1, %12 offset:%19\n\t"
      "ds_read_b64_tr_b16 %8, %16 offset:%20\n\t"
      "ds_read_b64_tr_b16 %9, %16 offset:%21\n\t"
      "ds_read_b64_tr_b16 %10, %17 offset:%20\n\t"
      "ds_read_b64_tr_b16 %11, %17 offset:%21\n\t"
      "ds_read_b64_tr_b16 %2, %13 offset:%18\n\t"
      "ds_read_b64_tr_b16 %3, %13 offset:%19\n\t"
      "ds_read_b64_tr_b16 %4, %14 offset:%18\n\t"
      "ds_read_b64_tr_b16 %5, %14 offset:%19\n\t"
      "ds_read_b64_tr_b16 %6, %15 offset:%18\n\t"
      "ds_read_b64_tr_b16 %7, %15 offset:%19\n\t"
      "s_waitcnt lgkmcnt(0)"
      : "=&v"(r[0]), "=&v"(r[1]), "=&v"(r[2]), "=&v"(r[3]), "=&v"(r[4]), "=&v"(r[5]), "=&v"(r[6]),
        "=&v"(r[7]), "=&v"(r[8]), "=&v"(r[9]), "=&v"(r[10]), "=&v"(r[11])
      : "v"(a[0]), "v"(a[1]), "v"(a[2]), "v"(a[3]), "v"(b[0]), "v"(b[1]), "n"(kOffA),
        "n"(kOffA + 4 * kRowA), "n"(kOffB), "n"(kOffB + 4 * kRowB)
      : "memory");
#pragma unroll
  for (int i = 0; i < 4; ++i)
    fa[i] = __builtin_bit_cast(bf16x8, __builtin_shufflevector(r[2 * i], r[2 * i + 1], 0, 1, 2, 3, 4, 5, 6, 7));
#pragma unroll
  for (int i = 0; i < 2; ++i)
    fb[i] = __builtin_bit_cast(bf16x8, __builtin_shufflevector(r[8 + 2 * i], r[9 + 2 * i], 0, 1, 2, 3, 4, 5, 6, 7));
}

// One operand's tile of kW rows (or strided columns): how its 64 kW bytes of a
// stage come into LDS and leave as fragments.
//
// Contiguous in K: LDS rows of 64 bytes, four 16-byte chunks, chunk c of row r
// at physical (c + r / 4) % 4: the 32 rows of a fragment read are free of bank
// conflicts.
// Strided: LDS rows are K, kW elements long; a fragment is two transposing
// reads, each of four K rows by 64 bytes a half-wave, so the 64-byte slots of
// four neighbouring rows are rotated against each other onto different banks.
template <bool kStrided, int kW, int kWaves>
struct Tile {
  static constexpr int kLoads = kW / 16 / kWaves;  // wave-loads of a stage, per wave
  static_assert(kLoads * 16 * kWaves == kW, "loads cover the tile");
  static constexpr int kBytes = kW * 64;
  static constexpr int kChunks = kStrided ? kW / 8 : 4;  // 16-byte chunks of an LDS row
  static constexpr int kRow = kW * 2;                    // bytes of a strided LDS row
  // Where 64-byte slot s of strided row k lies: rotated among the slots of
  // 256 bytes (64 columns: the rows 128 bytes apart rotate by pairs).
  static __device__ __forceinline__ int Slot(int s, int k) {
    if constexpr (kW >= 128) return (s & ~3) | ((s + k) & 3);
    else return (s + (k >> 1)) & 1;
  }
  static __device__ __forceinline__ int SlotAt(int phys, int k) {  // its inverse
    if constexpr (kW >= 128) return (phys & ~3) | ((phys - k) & 3);
    else return (phys - (k >> 1)) & 1;
  }

  int ld, extent, k8;  // rows (contiguous) or columns (strided) from the corner on; K up to 8s
  int voff[kLoads], kc[kLoads];

  __device__ __forceinline__ void Init(int ld_, int extent_, int K, int wave, int lane) {
    ld = ld_, extent = extent_, k8 = (K + 7) & ~7;
#pragma unroll
    for (int j = 0; j < kLoads; ++j) {
      const int row = (j * kWaves + wave) * (64 / kChunks) + lane / kChunks, p = lane % kChunks;
      if constexpr (kStrided) {
        voff[j] = row * ld * 2 + (SlotAt(p / 4, row) * 4 + p % 4) * 16;
        kc[j] = 0;
      } else {
        const int c = (p - row / 4) & 3;
        voff[j] = row * ld * 2 + c * 16;
        kc[j] = c * 8;
      }
    }
  }
  // Stage [k0, k0 + 32) of the operand at `at` (its tile's corner) into LDS.
  __device__ __forceinline__ void Issue(const uint16_t* at, int k0, int K, uint8_t* lds, int wave) {
    if constexpr (kStrided) {
      const int rows = min(K - k0, kStageK);
      const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(
          const_cast<uint16_t*>(at) + static_cast<size_t>(k0) * ld, 0,
          Uniform(((rows - 1) * ld + extent) * 2), kRsrcWord3);
#pragma unroll
      for (int j = 0; j < kLoads; ++j)
        LoadLds(rs, lds + Uniform((j * kWaves + wave) * 1024), voff[j], 0);
    } else {
      const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(
          const_cast<uint16_t*>(at), 0, Uniform(extent * ld * 2), kRsrcWord3);
      const bool tail = k0 + kStageK > k8;
#pragma unroll
      for (int j = 0; j < kLoads; ++j)
        LoadLds(rs, lds + Uniform((j * kWaves + wave) * 1024),
                tail && k0 + kc[j] >= k8 ? kFar : voff[j], k0 * 2);
    }
  }
  // Byte offset in the tile of lane l's part of the fragment of rows (columns)
  // [first, first + 32) at K = 0: row l % 32, K 8 (l / 32) on.
  static __device__ __forceinline__ uint32_t Frag(int first, int lane) {
    if constexpr (kStrided) {
      const int i = lane % 16, k = 8 * (lane / 32) + i / 4;
      return k * kRow + Slot(first / 32, k) * 64 + ((lane / 16) & 1) * 32 + (i % 4) * 8;
    } else {
      const int r = lane % 32;
      return (first + r) * 64 + ((lane / 32 + r / 4) & 3) * 16;
    }
  }
  // The same 16 K later (contiguous: two chunks on).
  static constexpr int kNext = kStrided ? 16 * kRow : 32;
};

template <class T, int kEpi, bool kAS, bool kBS, int BM, int BN, int WGM, int WGN, int kStages>
__global__ void __launch_bounds__(WGM * WGN * kWave) FfnMma(MmaArgs p) {
  constexpr int kWaves = WGM * WGN;
  constexpr bool kDual = kEpi == kTwo || kEpi == kGate;
  constexpr int BNs = kDual ? BN / 2 : BN;  // columns of the output
  constexpr int WM = BM / WGM, WN = BNs / WGN;
  constexpr int TM = WM / 32, TN = WN / 32, TB = kDual ? 2 * TN : TN;
  static_assert(TM * 32 * WGM == BM && TN * 32 * WGN == BNs, "waves cover the tile");
  using TA = Tile<kAS, BM, kWaves>;
  using TBt = Tile<kBS, BNs, kWaves>;
  constexpr int kStage = TA::kBytes + (kDual ? 2 : 1) * TBt::kBytes;
  constexpr int kPerStage = TA::kLoads + (kDual ? 2 : 1) * TBt::kLoads;
  __shared__ __attribute__((aligned(1024))) uint8_t smem[kStages * kStage];

  const int wave = threadIdx.x / kWave, lane = threadIdx.x % kWave;
  int tm, tn;
  TileOf(blockIdx.x, (p.M + BM - 1) / BM, (p.N + BNs - 1) / BNs, tm, tn);
  const int m0 = tm * BM, n0 = tn * BNs;
  TA ta;
  TBt tb;
  // A strided operand's last row ends where its columns do.
  ta.Init(p.lda, kAS ? p.lda - m0 : min(p.M - m0, BM), p.K, wave, lane);
  tb.Init(p.ldb, kBS ? p.ldb - n0 : min(p.N - n0, BNs), p.K, wave, lane);
  const size_t a_at = kAS ? static_cast<size_t>(m0) : static_cast<size_t>(m0) * p.lda;
  const size_t b_at = kBS ? static_cast<size_t>(n0) : static_cast<size_t>(n0) * p.ldb;

  const int per_seg = (p.K + kStageK - 1) / kStageK, last = p.nseg * per_seg - 1;
  int seg = 0, k0 = 0;  // the next stage to load
  auto issue = [&](int buf) {
    uint8_t* s = smem + buf * kStage;
    ta.Issue(p.A[seg] + a_at, k0, p.K, s, wave);
    tb.Issue(p.B[seg] + b_at, k0, p.K, s + TA::kBytes, wave);
    if constexpr (kDual) tb.Issue(p.B2[seg] + b_at, k0, p.K, s + TA::kBytes + TBt::kBytes, wave);
    // Past the last stage the loads repeat it, into a buffer nothing reads.
    if (k0 + kStageK < p.K) {
      k0 += kStageK;
    } else if (seg + 1 < p.nseg) {
      ++seg;
      k0 = 0;
    }
  };

  v16f acc[TM][TB];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TB; ++j) acc[i][j] = v16f{};
  const int wm = (wave / WGN) * WM, wn = (wave % WGN) * WN;
  // Where this lane's fragments lie in a stage.
  uint32_t oa[TM], ob[TB];
#pragma unroll
  for (int i = 0; i < TM; ++i) oa[i] = TA::Frag(wm + i * 32, lane);
#pragma unroll
  for (int j = 0; j < TB; ++j)
    ob[j] = TA::kBytes + (j / TN) * TBt::kBytes + TBt::Frag(wn + (j % TN) * 32, lane);
  const uint32_t lds0 = static_cast<uint32_t>(
      reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) uint8_t*)smem));

  bf16x8 fa[2][TM], fb[2][TB];
  // Contiguous operands' fragments come by the compiler's own reads, ahead of
  // the products of the half-stage before; strided ones behind them, while the
  // SIMD's other wave multiplies.
  auto read_ahead = [&](int buf, auto ks_tag) {
    constexpr int ks = decltype(ks_tag)::value;
    const uint8_t* s = smem + buf * kStage;
    // (chunk c + 2 ks of four, so the second half-stage is the other pair)
    if constexpr (!kAS) {
#pragma unroll
      for (int i = 0; i < TM; ++i) fa[ks][i] = *reinterpret_cast<const bf16x8*>(s + (oa[i] ^ (ks * 32)));
    }
    if constexpr (!kBS) {
#pragma unroll
      for (int j = 0; j < TB; ++j) fb[ks][j] = *reinterpret_cast<const bf16x8*>(s + (ob[j] ^ (ks * 32)));
    }
  };
  auto read_behind = [&](int buf, auto ks_tag) {
    constexpr int ks = decltype(ks_tag)::value;
    const uint32_t s = lds0 + buf * kStage;
    uint32_t a[TM], b[TB];
#pragma unroll
    for (int i = 0; i < TM; ++i) a[i] = s + oa[i];
#pragma unroll
    for (int j = 0; j < TB; ++j) b[j] = s + ob[j];
    if constexpr (kAS && kBS)
      ReadTr2<ks * TA::kNext, TA::kRow, ks * TBt::kNext, TBt::kRow>(a, fa[ks], b, fb[ks]);
    else if constexpr (kBS)
      ReadTr<ks * TBt::kNext, TBt::kRow>(b, fb[ks]);
  };
  auto mfmas = [&](auto ks_tag) {
    constexpr int ks = decltype(ks_tag)::value;
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int j = 0; j < TB; ++j)
        acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fb[ks][j], fa[ks][i], acc[i][j], 0, 0, 0);
    if constexpr (kAS || kBS) __builtin_amdgcn_sched_barrier(0);
  };
  constexpr std::integral_constant<int, 0> k0_{};
  constexpr std::integral_constant<int, 1> k1_{};

#pragma unroll
  for (int s = 0; s < kStages - 1; ++s) issue(s);
  WaitVm<(kStages - 2) * kPerStage>();
  Barrier();
  read_ahead(0, k0_);
  read_behind(0, k0_);
  for (int it = 0; it < last; ++it) {
    const int buf = it % kStages;
    read_ahead(buf, k1_);
    mfmas(k0_);
    read_behind(buf, k1_);
    WaitVm<(kStages - 3) * kPerStage>();
    Barrier();
    issue((it + kStages - 1) % kStages);
    read_ahead((it + 1) % kStages, k0_);
    mfmas(k1_);
    read_behind((it + 1) % kStages, k0_);
  }
  read_ahead(last % kStages, k1_);
  mfmas(k0_);
  read_behind(last % kStages, k1_);
  mfmas(k1_);
  WaitVm<0>();  // the repeated loads have landed

  // Accumulator element 4 q + e of block (i, j) is row lane % 32, column
  // 8 q + 4 (lane / 32) + e: four neighbours of one row at a time.
  const int h = lane / 32;
#pragma unroll
  for (int i = 0; i < TM; ++i) {
    const int m = m0 + wm + i * 32 + lane % 32;
#pragma unroll
    for (int j = 0; j < TN; ++j)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int n = n0 + wn + j * 32 + 8 * q + 4 * h;
        const int cnt = p.N - n;  // columns left
        if (m >= p.M) continue;
        const size_t o = static_cast<size_t>(m) * p.N + n;
        const bool vec = p.vec && cnt >= 4;
        float c[4], d[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          c[e] = acc[i][j][4 * q + e];
          if constexpr (kDual) d[e] = acc[i][TN + j][4 * q + e];
        }
        if constexpr (kEpi == kPlain || kEpi == kTwo) {
          Put4(static_cast<T*>(p.o1) + o, vec, cnt, c);
          if constexpr (kEpi == kTwo) Put4(static_cast<T*>(p.o2) + o, vec, cnt, d);
        }
        if constexpr (kEpi == kGate) {
          if (n >= p.h.ld) continue;
          if (p.o1) {
            Put4(static_cast<T*>(p.o1) + o, vec, cnt, c);
            Put4(static_cast<T*>(p.o2) + o, vec, cnt, d);
          }
#pragma unroll
          for (int e = 0; e < 4; ++e) c[e] = e < cnt ? ActExpr(p.act, c[e]) * d[e] : 0.0f;
          PutPlanes<T>(p.h, static_cast<size_t>(m) * p.h.ld + n, c);
        }
        if constexpr (kEpi == kGrad) {
          if (n >= p.h.ld) continue;
          float g[4], u[4];
          Get4(static_cast<const T*>(p.g) + o, vec, cnt, g);
          Get4(static_cast<const T*>(p.u) + o, vec, cnt, u);
          float x[4], y[4], z[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float a = ActExpr(p.act, g[e]);
            const bool in = e < cnt;
            x[e] = in ? c[e] * u[e] * ActGrad(p.act, g[e]) : 0.0f;
            y[e] = in ? c[e] * a : 0.0f;
            z[e] = in ? a * u[e] : 0.0f;
          }
          const size_t w = static_cast<size_t>(m) * p.h.ld + n;
          PutPlanes<T>(p.dg, w, x);
          PutPlanes<T>(p.du, w, y);
          PutPlanes<T>(p.h, w, z);
        }
      }
  }
}

// --- host ---------------------------------------------------------------------------------------

template <class T, int kEpi, bool kAS, bool kBS, int BM, int BN, int WGM, int WGN, int kStages>
hipError_t LaunchTile(const MmaArgs& a, hipStream_t s) {
  constexpr int BNs = kEpi == kTwo || kEpi == kGate ? BN / 2 : BN;
  const int64_t tiles = static_cast<int64_t>((a.M + BM - 1) / BM) * ((a.N + BNs - 1) / BNs);
  auto* kernel = &FfnMma<T, kEpi, kAS, kBS, BM, BN, WGM, WGN, kStages>;
  hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(tiles)), dim3(WGM * WGN * kWave), 0, s, a);
  return hipGetLastError();
}

template <class T, int kEpi, bool kAS, bool kBS>
hipError_t Mma(const MmaArgs& a, hipStream_t s) {
  constexpr bool dual = kEpi == kTwo || kEpi == kGate;
  auto tiles = [&](int bm, int bn) {
    return static_cast<int64_t>((a.M + bm - 1) / bm) * ((a.N + (dual ? bn / 2 : bn) - 1) / (dual ? bn / 2 : bn));
  };
  // (f32's gradient epilogue, nine planes a quad, is past the registers beside 256 x 256.)
  if constexpr (!(kEpi == kGrad && sizeof(T) == 4))
    if (tiles(256, 256) >= 192) return LaunchTile<T, kEpi, kAS, kBS, 256, 256, 2, 4, 4>(a, s);
  if (tiles(128, 128) >= 192) return LaunchTile<T, kEpi, kAS, kBS, 128, 128, 2, 2, 4>(a, s);
  if constexpr (dual) return LaunchTile<T, kEpi, kAS, kBS, 64, 128, 2, 2, 4>(a, s);
  else return LaunchTile<T, kEpi, kAS, kBS, 64, 64, 2, 2, 4>(a, s);
}

int Up8(size_t n) { return static_cast<int>((n + 7) / 8 * 8); }

// The workspace, handed out in 256-byte steps; with a null base it only counts.
class Space {
 public:
  explicit Space(void* base) : base_(static_cast<uint8_t*>(base)) {}
  Planes Take(size_t rows, size_t cols, int planes) {
    Planes p;
    p.ld = Up8(cols);
    p.plane = rows * p.ld;
    p.p = reinterpret_cast<uint16_t*>(base_ + used_);
    used_ += (p.plane * planes * 2 + 255) / 256 * 256;
    return p;
  }
  size_t used() const { return used_; }

 private:
  uint8_t* base_;
  size_t used_ = 0;
};

struct Layout {
  Planes x, wg, wu, wd, dy, h, dg, du;
  size_t bytes;
};
Layout Lay(void* ws, int planes, size_t M, size_t D, size_t F, bool backward) {
  Space s(ws);
  Layout l;
  l.x = s.Take(M, D, planes);
  l.wg = s.Take(D, F, planes);
  l.wu = s.Take(D, F, planes);
  l.wd = s.Take(F, D, planes);
  l.h = s.Take(M, F, planes);
  if (backward) {
    l.dy = s.Take(M, D, planes);
    l.dg = s.Take(M, F, planes);
    l.du = s.Take(M, F, planes);
  }
  l.bytes = s.used();
  return l;
}

// An operand as planes: itself where its rows begin on 16 bytes, else packed.
template <class T>
hipError_t Pack(const void* in, size_t rows, size_t cols, Planes& out, hipStream_t s) {
  const uintptr_t at = reinterpret_cast<uintptr_t>(in);
  if (sizeof(T) == 2 && cols % 8 == 0 && (at & 15) == 0) {
    out.p = static_cast<uint16_t*>(const_cast<void*>(in));
    return hipSuccess;
  }
  const size_t n = rows * (out.ld / 4);
  const bool vec = cols % 4 == 0 && at % (4 * sizeof(T)) == 0;
  hipLaunchKernelGGL((FfnPackKernel<T>), dim3(GridFor(n, 256, 4096)), dim3(256), 0, s,
                     static_cast<const T*>(in), rows, static_cast<int>(cols), vec, out);
  return hipGetLastError();
}

// The plane products of A B (and A B2), smallest first.
template <class T>
void AddProduct(MmaArgs& a, const Planes& A, const Planes& B, const Planes* B2 = nullptr) {
  constexpr int pairs[6][2] = {{2, 0}, {0, 2}, {1, 1}, {1, 0}, {0, 1}, {0, 0}};
  a.lda = A.ld, a.ldb = B.ld;
  for (int i = sizeof(T) == 2 ? 5 : 0; i < 6; ++i) {
    a.A[a.nseg] = A.p + pairs[i][0] * A.plane;
    a.B[a.nseg] = B.p + pairs[i][1] * B.plane;
    if (B2) a.B2[a.nseg] = B2->p + pairs[i][1] * B2->plane;
    ++a.nseg;
  }
}

template <class T>
bool Quads(size_t N, std::initializer_list<const void*> ptrs) {
  uintptr_t at = 0;
  for (const void* p : ptrs) at |= reinterpret_cast<uintptr_t>(p);
  return N % 4 == 0 && at % (4 * sizeof(T)) == 0;
}

MmaArgs Shape(size_t M, size_t N, size_t K) {
  MmaArgs a{};
  a.M = static_cast<int>(M), a.N = static_cast<int>(N), a.K = static_cast<int>(K);
  return a;
}

#define FFN_TRY(expr)                                       \
  do {                                                      \
    if (hipError_t e_ = (expr); e_ != hipSuccess) return e_; \
  } while (0)

template <class T>
hipError_t Fwd(const FfnArgs& f, hipStream_t s) {
  if (f.M == 0) return hipSuccess;
  Layout l = Lay(f.ws, sizeof(T) == 2 ? 1 : 3, f.M, f.D, f.F, false);
  FFN_TRY(Pack<T>(f.x, f.M, f.D, l.x, s));
  FFN_TRY(Pack<T>(f.wg, f.D, f.F, l.wg, s));
  FFN_TRY(Pack<T>(f.wu, f.D, f.F, l.wu, s));
  FFN_TRY(Pack<T>(f.wd, f.F, f.D, l.wd, s));
  MmaArgs a = Shape(f.M, f.F, f.D);
  AddProduct<T>(a, l.x, l.wg, &l.wu);
  a.act = f.act, a.o1 = f.gate, a.o2 = f.up, a.h = l.h, a.vec = Quads<T>(f.F, {f.gate, f.up});
  FFN_TRY((Mma<T, kGate, false, true>(a, s)));
  a = Shape(f.M, f.D, f.F);
  AddProduct<T>(a, l.h, l.wd);
  a.o1 = f.y, a.vec = Quads<T>(f.D, {f.y});
  return Mma<T, kPlain, false, true>(a, s);
}

template <class T>
hipError_t Bwd(const FfnArgs& f, hipStream_t s) {
  if (f.M == 0) {  // no tokens: no gradient
    const size_t n = f.D * f.F;
    for (void* w : {f.dwg, f.dwu, f.dwd}) {
      hipLaunchKernelGGL((FfnZeroKernel<T>), dim3(GridFor(n, 256, 4096)), dim3(256), 0, s,
                         static_cast<T*>(w), n);
      FFN_TRY(hipGetLastError());
    }
    return hipSuccess;
  }
  Layout l = Lay(f.ws, sizeof(T) == 2 ? 1 : 3, f.M, f.D, f.F, true);
  FFN_TRY(Pack<T>(f.x, f.M, f.D, l.x, s));
  FFN_TRY(Pack<T>(f.wg, f.D, f.F, l.wg, s));
  FFN_TRY(Pack<T>(f.wu, f.D, f.F, l.wu, s));
  FFN_TRY(Pack<T>(f.wd, f.F, f.D, l.wd, s));
  FFN_TRY(Pack<T>(f.dy, f.M, f.D, l.dy, s));
  MmaArgs a = Shape(f.M, f.F, f.D);
  AddProduct<T>(a, l.dy, l.wd);
  a.act = f.act, a.g = f.gate, a.u = f.up, a.h = l.h, a.dg = l.dg, a.du = l.du;
  a.vec = Quads<T>(f.F, {f.gate, f.up});
  FFN_TRY((Mma<T, kGrad, false, false>(a, s)));
  a = Shape(f.M, f.D, f.F);
  AddProduct<T>(a, l.dg, l.wg);
  AddProduct<T>(a, l.du, l.wu);
  a.o1 = f.dx, a.vec = Quads<T>(f.D, {f.dx});
  FFN_TRY((Mma<T, kPlain, false, false>(a, s)));
  a = Shape(f.D, f.F, f.M);
  AddProduct<T>(a, l.x, l.dg, &l.du);
  a.o1 = f.dwg, a.o2 = f.dwu, a.vec = Quads<T>(f.F, {f.dwg, f.dwu});
  FFN_TRY((Mma<T, kTwo, true, true>(a, s)));
  a = Shape(f.F, f.D, f.M);
  AddProduct<T>(a, l.h, l.dy);
  a.o1 = f.dwd, a.vec = Quads<T>(f.D, {f.dwd});
  return Mma<T, kPlain, true, true>(a, s);
}

}  // namespace

size_t FfnWorkspaceBytes(int bf16, size_t M, size_t D, size_t F, int backward) {
  return M ? Lay(nullptr, bf16 ? 1 : 3, M, D, F, backward != 0).bytes : 0;
}

hipError_t LaunchFfnFwd(const FfnArgs& a, hipStream_t s) {
  return a.bf16 ? Fwd<uint16_t>(a, s) : Fwd<float>(a, s);
}
hipError_t LaunchFfnBwd(const FfnArgs& a, hipStream_t s) {
  return a.bf16 ? Bwd<uint16_t>(a, s) : Bwd<float>(a, s);
}

}  // namespace seeai
