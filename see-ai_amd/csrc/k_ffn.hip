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
// forward (G and U; Y), three backward (dH; dX; the three weights' gradients),
// besides the joins of shared-out K and the packing of operands.
//
// Many tokens are bound by the matrix unit's power: 8192 x 2048 x 5632 bf16 runs
// 528 us forward and 1039 backward, 1,070 and 1,090 TFLOP/s (the same products
// of a library, without what the epilogues do, 472 and 947 us; 1,030 to 1,550
// TFLOP/s by layout and K), at 1.7 of 2.4 GHz; the down projection alone 161 us,
// the gate's launch 361 for twice its work and 277 MB stored.  Few are bound by
// the weights' bytes: one token of the same block 25 us for 69 MB.
//
// bf16: the operands as they are; what passes between launches (H, dG, dU) is
// rounded to bf16 once, as the stored G and U are, because the next product's
// operands are bf16: at most 2^-8 of each value, as the inputs' own rounding.
// f32: each operand is split into three bf16 planes (x = hi + mid + lo, eight
// bits each, truncated, so exactly x), and a product is its six largest plane
// products, all into the same f32 accumulators.  What is left out
// (mid lo, lo mid, lo lo; mid < 2^-7 and lo < 2^-15 of x's leading bit) is below
// 2^-21 of the term and has its sign: 0.7 2^-24 of it on average over random
// operands, 7.8 2^-24 for the square of 1 + 2^-7 - 2^-23.  So f32's accuracy but
// for a loss of that size towards zero, at a sixth of the bf16 rate, 1.6 times
// the f32 MFMA's (up to 128 tokens the f32 MFMA itself, below, which leaves
// nothing out).  Bits of an operand below 2^-133 are past bf16's last.  An
// infinity's remainder is a NaN, so past 128 tokens what an infinity reaches is
// not finite but may be a NaN where f32 arithmetic has an infinity.
#include <algorithm>
#include <type_traits>
#include <utility>

#include "common.h"
#include "ffn_plan.h"

namespace seeai {
namespace {

using namespace ffn;

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) uint8_t* LdsPtr;
typedef __attribute__((address_space(3))) s16x4* LdsTr;

constexpr int kRsrcWord3 = 0x00020000;  // raw buffer, out-of-range reads give 0
constexpr int kFar = 0x7FFFFFFF;        // an offset past every range

// Until at most n of this wave's loads are in flight.
template <int n>
__device__ __forceinline__ void WaitVm() {
  static_assert(n >= 0 && n < 64, "vmcnt range");
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(n) : "memory");
}

// A raw buffer over [base, base + bytes): reads past it give 0.
typedef int v4i_ __attribute__((ext_vector_type(4)));
__device__ __forceinline__ v4i_ Buffer(const uint16_t* base, int bytes) {
  const uint64_t a = reinterpret_cast<uint64_t>(base);
  return v4i_{Uniform(static_cast<int>(a)), Uniform(static_cast<int>(a >> 32)), Uniform(bytes), kRsrcWord3};
}
// kN loads of 16 bytes a lane, lane after lane, straight into LDS at `lds` and
// every kStep bytes on.  Written out because the compiler lets no transposing
// read of LDS pass a load into LDS it knows of: with its own builtin every
// step's reads would wait for every stage in flight.  They have no output
// register; WaitVm and a barrier stand between them and the reads of what they
// bring.  (The wait states are those between a scalar register's write, m0's
// included, and this use of it.)
template <int kN, int kStep>
__device__ __forceinline__ void LoadLds(v4i_ rs, uint32_t lds, const int* voff, int soff) {
  if constexpr (kN == 1) {
    asm volatile(
        "s_mov_b32 m0, %0\n\t"
        "s_nop 4\n\t"
        "buffer_load_dwordx4 %1, %2, %3 offen lds"
        :
        : "s"(Uniform(lds)), "v"(voff[0]), "s"(rs), "s"(Uniform(soff))
        : "memory", "m0");
  } else if constexpr (kN == 2) {
    asm volatile(
        "s_mov_b32 m0, %0\n\t"
        "s_nop 4\n\t"
        "buffer_load_dwordx4 %1, %3, %4 offen lds\n\t"
        "s_add_u32 m0, m0, %5\n\t"
        "s_nop 0\n\t"
        "buffer_load_dwordx4 %2, %3, %4 offen lds"
        :
        : "s"(Uniform(lds)), "v"(voff[0]), "v"(voff[1]), "s"(rs), "s"(Uniform(soff)), "n"(kStep)
        : "memory", "m0", "scc");
  } else if constexpr (kN != 4) {
    LoadLds<2, kStep>(rs, lds, voff, soff);
    LoadLds<kN - 2, kStep>(rs, lds + 2 * kStep, voff + 2, soff);
  } else {
    asm volatile(
        "s_mov_b32 m0, %0\n\t"
        "s_nop 4\n\t"
        "buffer_load_dwordx4 %1, %5, %6 offen lds\n\t"
        "s_add_u32 m0, m0, %7\n\t"
        "s_nop 0\n\t"
        "buffer_load_dwordx4 %2, %5, %6 offen lds\n\t"
        "s_add_u32 m0, m0, %7\n\t"
        "s_nop 0\n\t"
        "buffer_load_dwordx4 %3, %5, %6 offen lds\n\t"
        "s_add_u32 m0, m0, %7\n\t"
        "s_nop 0\n\t"
        "buffer_load_dwordx4 %4, %5, %6 offen lds"
        :
        : "s"(Uniform(lds)), "v"(voff[0]), "v"(voff[1]), "v"(voff[2]), "v"(voff[3]), "s"(rs),
          "s"(Uniform(soff)), "n"(kStep)
        : "memory", "m0", "scc");
  }
}

// Until this wave's LDS reads have returned.
__device__ __forceinline__ void WaitLds() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

// The workgroup's barrier, which no access may be moved across.
__device__ __forceinline__ void Barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// The activation (ActExpr's functions, but a NaN passes ReLU) and its derivative.
// GELU's 1 + tanh(t) is 2 sigmoid(2 t), so both smooth ones are x s(.) with one
// exponential.
// kFast: the hardware's exponential and reciprocal, a few f32 steps off, for
// results that leave in bf16.
template <bool kFast>
__device__ __forceinline__ float Sigmoid(float x) {
  if constexpr (kFast)
    return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-1.4426950408889634f * x));
  else
    return SigmoidExpr(x);
}
template <bool kFast>
__device__ __forceinline__ void Activate(int act, float x, float& a, float& da) {
  const float kC = 0.7978845608028654f, kA = 0.044715f;
  if (act == 3) {
    const float s = Sigmoid<kFast>(x);
    a = x * s;
    da = s * (1.0f + x * (1.0f - s));
  } else if (act == 2) {
    const float s = Sigmoid<kFast>(2.0f * (kC * (x + kA * x * x * x)));
    a = x * s;
    // Past 32 either way s is 0 or 1 and the second term 0, x^2 short of infinity or not.
    const float y = fminf(fmaxf(x, -32.0f), 32.0f);
    da = s + y * s * (1.0f - s) * (2.0f * kC * (1.0f + 3.0f * kA * y * y));
  } else {
    const bool off = act == 1 && x <= 0.0f;
    a = off ? 0.0f : x;
    da = off ? 0.0f : act == 1 && x != x ? x : 1.0f;
  }
}

// Eight of them, the activation chosen once.
template <bool kFast>
__device__ __forceinline__ void Activate8(int act, const float (&x)[8], float (&a)[8], float (&da)[8]) {
  if (act == 3) {
#pragma unroll
    for (int e = 0; e < 8; ++e) Activate<kFast>(3, x[e], a[e], da[e]);
  } else if (act == 2) {
#pragma unroll
    for (int e = 0; e < 8; ++e) Activate<kFast>(2, x[e], a[e], da[e]);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) Activate<kFast>(act, x[e], a[e], da[e]);
  }
}

// Up to eight neighbours of a row, 16 bytes at a time where they may be.
__device__ __forceinline__ void Load8(const float* p, bool vec, int cnt, float (&v)[8]) {
  if (vec && cnt >= 8) {
    const float4 a = *reinterpret_cast<const float4*>(p);
    const float4 b = *reinterpret_cast<const float4*>(p + 4);
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = e < cnt ? p[e] : 0.0f;
  }
}
__device__ __forceinline__ void Load8(const uint16_t* p, bool vec, int cnt, float (&v)[8]) {
  if (vec && cnt >= 8) {
    const uint4 a = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = __uint_as_float(w[i] << 16);
      v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = e < cnt ? Bf16ToF32(p[e]) : 0.0f;
  }
}
__device__ __forceinline__ void Store8(float* p, bool vec, int cnt, const float (&v)[8]) {
  if (vec && cnt >= 8) {
    *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
    *reinterpret_cast<float4*>(p + 4) = make_float4(v[4], v[5], v[6], v[7]);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < cnt) p[e] = v[e];
  }
}
__device__ __forceinline__ bf16x8 Bf16x8(const float (&v)[8]) {
  bf16x8 o;
#pragma unroll
  for (int e = 0; e < 8; ++e) o[e] = static_cast<__bf16>(v[e]);
  return o;
}
__device__ __forceinline__ void Store8(uint16_t* p, bool vec, int cnt, const float (&v)[8]) {
  if (vec && cnt >= 8) {
    *reinterpret_cast<bf16x8*>(p) = Bf16x8(v);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < cnt) p[e] = F32ToBf16(v[e]);
  }
}
// Eight neighbours as they lie in memory, for loads that run ahead.
template <class T>
struct Raw8 {
  uint4 q[sizeof(T) / 2];
  __device__ __forceinline__ void Load(const T* p) {
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i) q[i] = reinterpret_cast<const uint4*>(p)[i];
  }
  __device__ __forceinline__ void Get(float (&v)[8]) const {
    Load8(reinterpret_cast<const T*>(q), true, 8, v);
  }
};
__device__ __forceinline__ float One(const float* p) { return *p; }
__device__ __forceinline__ float One(const uint16_t* p) { return Bf16ToF32(*p); }
__device__ __forceinline__ void Put(float* p, float v) { *p = v; }
__device__ __forceinline__ void Put(uint16_t* p, float v) { *p = F32ToBf16(v); }

// The next bf16 plane of a value: its top eight bits, taken off it.
__device__ __forceinline__ uint32_t TakePlane(float& x) {
  const uint32_t hi = __float_as_uint(x) & 0xFFFF0000u;
  x -= __uint_as_float(hi);
  return hi >> 16;
}

// A [rows, ld] operand in bf16 planes: one for bf16, three for f32; with kWhole
// (FfnRows32's) in f32 itself.
struct Planes {
  uint16_t* p = nullptr;
  size_t plane = 0;  // elements of one plane
  int ld = 0;        // a multiple of 8, zeros past the row's own width
};
// Eight neighbours into the planes (16-byte aligned: the column is a multiple
// of eight).
template <class T, bool kWhole = false>
__device__ __forceinline__ void PutPlanes(const Planes& out, size_t at, float (&v)[8]) {
  if constexpr (kWhole) {
    Store8(reinterpret_cast<float*>(out.p) + at, true, 8, v);
  } else if constexpr (sizeof(T) == 2) {
    *reinterpret_cast<bf16x8*>(out.p + at) = Bf16x8(v);
  } else {
#pragma unroll
    for (int k = 0; k < 3; ++k) {
      uint32_t w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t lo = TakePlane(v[2 * i]);
        w[i] = lo | TakePlane(v[2 * i + 1]) << 16;
      }
      *reinterpret_cast<uint4*>(out.p + k * out.plane + at) = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
}

// rows x cols (packed) into padded planes: operands whose rows or base are off
// 16 bytes, and every f32 operand; all of a call's in one launch.
struct Piece {
  const void* in;
  size_t rows;
  int cols;
  bool vec;
  Planes out;
  unsigned first;  // its first workgroup
};
struct Pieces {
  Piece q[5];
  int count;
  unsigned blocks;
};
template <class T>
__global__ void __launch_bounds__(256) FfnPackKernel(Pieces p) {
  const unsigned block = blockIdx.y * gridDim.x + blockIdx.x;
  if (block >= p.blocks) return;
  int k = 0;
  while (k + 1 < p.count && block >= p.q[k + 1].first) ++k;
  const Piece& q = p.q[k];
  // 2048 elements of the padded rows a workgroup, eight a thread; rows off 16
  // bytes come a lane an element through LDS.
  __shared__ float st[256 * 8];
  const size_t base = static_cast<size_t>(block - q.first) * 2048, r0 = base / q.out.ld;
  const uint32_t ld = q.out.ld, c0 = static_cast<uint32_t>(base - r0 * ld);
  if (!q.vec) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const uint32_t x = e * 256 + threadIdx.x, rr = (c0 + x) / ld, cc = c0 + x - rr * ld;
      const bool in = r0 + rr < q.rows && cc < static_cast<uint32_t>(q.cols);
      st[x] = in ? One(static_cast<const T*>(q.in) + (r0 + rr) * q.cols + cc) : 0.0f;
    }
    __syncthreads();
  }
  const uint32_t at = c0 + threadIdx.x * 8, rr = at / ld, c = at - rr * ld;
  const size_t r = r0 + rr;
  if (r >= q.rows) return;
  float v[8];
  if (q.vec) Load8(static_cast<const T*>(q.in) + r * q.cols + c, true, q.cols - static_cast<int>(c), v);
  else Load8(st + threadIdx.x * 8, true, 8, v);
  PutPlanes<T>(q.out, r * ld + c, v);
}

template <class T>
__global__ void __launch_bounds__(256) FfnZeroKernel(T* __restrict__ out, size_t n) {
  const size_t step = static_cast<size_t>(gridDim.x) * 256;
  for (size_t i = static_cast<size_t>(blockIdx.x) * 256 + threadIdx.x; i < n; i += step) out[i] = 0;
}

// f(0), f(1), ... f(n - 1) with the index a constant: accumulators stay in
// registers where a loop too large to unroll would index them in memory.
template <class F, int... kI>
__device__ __forceinline__ void EachOf(F&& f, std::integer_sequence<int, kI...>) {
  (f(std::integral_constant<int, kI>{}), ...);
}
template <int kN, class F>
__device__ __forceinline__ void Each(F&& f) {
  EachOf(f, std::make_integer_sequence<int, kN>{});
}

// One product of a launch.  Operand element (i, k) lies at i ld + k, or,
// "strided", at k ld + i.  Segments are products of the same shape added up.
constexpr int kMaxSeg = 2;
struct Product {
  const uint16_t *A[kMaxSeg], *B[kMaxSeg], *B2[kMaxSeg];
  size_t a_plane, b_plane;  // elements between an operand's planes
  int lda, ldb, M, N;
  bool vec;       // outputs (and G, U) take eight neighbours at once
  bool vec_a;     // FfnOuter32: A takes four, and `vec` is of four too
  void *o1, *o2;  // plain: o1; gate: G and U or null
  int first;      // its first tile in the launch
};
// What an epilogue works on beside its sums.
struct Side {
  int act;
  const void *g, *u;  // gradient: G and U
  Planes h, dg, du;
};
// A launch's products share K, segments and kind.  Tiles [0, whole) are a
// workgroup each; the rest share K out over `splits` workgroups, `per_split`
// stages each, whose f32 sums [tile][split][rows][columns, of both operands]
// FfnJoin adds and finishes.  (FfnRows32's tiles all share K out.)
struct MmaArgs : Side {
  Product q[3];
  int count, nseg, K;
  int tiles, whole, splits, per_split;
  float* part;
};

enum Epilogue {
  kPlain,  // o1 = sum A B
  kGate,   // G = sum A B, U = sum A B2: o1, o2 where kept, h = act(G) U
  kGrad    // d = sum A B: dg = d U act'(G), du = d act(G), h = act(G) U
};

// Workgroup -> tile order: the 8 XCDs each take a contiguous run of the n tiles
// (workgroup b runs on XCD b % 8), walked in bands of row tiles, so concurrent
// tiles of one XCD share operand panels in its L2.
constexpr int kBand = 4;
__device__ __forceinline__ int XcdRun(int b, int n) {
  const int x = b % 8;
  return x * (n / 8) + min(x, n % 8) + b / 8;
}
__device__ __forceinline__ void TileOf(int t, int tiles_m, int tiles_n, int& tm, int& tn) {
  const int per = kBand * tiles_n, first = t / per * kBand;
  const int rows = min(tiles_m - first, kBand), off = t % per;
  tm = first + off % rows;
  tn = off / rows;
}
// The product tile t belongs to, and its corner.
__device__ __forceinline__ int ProductOf(const MmaArgs& p, int t, int bm, int bn, int& m0, int& n0) {
  int i = 0;
  while (i + 1 < p.count && t >= p.q[i + 1].first) ++i;
  TileOf(t - p.q[i].first, (p.q[i].M + bm - 1) / bm, (p.q[i].N + bn - 1) / bn, m0, n0);
  m0 *= bm;
  n0 *= bn;
  return i;
}

// One operand's tile of kW rows (or strided columns): how the kW kBK elements of
// a stage come into LDS and leave as fragments.
//
// Contiguous in K: LDS rows of 2 kBK bytes, kBK / 8 chunks of 16.  A fragment
// read takes one chunk of 32 rows; a row's chunks are rotated by the rows
// already in its 256 bytes, so sixteen lanes meet all the banks.
// Strided: LDS rows are K, kW elements long; a fragment is two transposing
// reads, each of four K rows by 64 bytes a half-wave, so the 64-byte slots of
// four neighbouring rows are rotated against each other onto different banks.
template <bool kStrided, int kW, int kBK, int kWaves>
struct Tile {
  static constexpr int kBytes = kW * kBK * 2;
  static constexpr int kLoads = kBytes / 1024 / kWaves;  // wave-loads of a stage, per wave
  static_assert(kLoads * 1024 * kWaves == kBytes, "loads cover the tile");
  static constexpr int kRow = kStrided ? kW * 2 : kBK * 2;  // bytes of an LDS row
  static constexpr int kChunks = kRow / 16;
  static constexpr int kPer256 = 256 / kRow;  // contiguous rows in 256 bytes
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
        const int c = (p - row / kPer256) & (kChunks - 1);
        voff[j] = row * ld * 2 + c * 16;
        kc[j] = c * 8;
      }
    }
  }
  // Wave-loads [j, j + kN) of stage [k0, k0 + kBK) of the operand at `at` (its
  // tile's corner) into LDS.
  template <int kN>
  __device__ __forceinline__ void Load(const uint16_t* at, int k0, int K, uint32_t lds, int wave, int j) {
    const uint32_t to = lds + (j * kWaves + wave) * 1024;
    if constexpr (kStrided) {
      const int rows = min(K - k0, kBK);
      LoadLds<kN, kWaves * 1024>(
          Buffer(at + static_cast<size_t>(k0) * ld, ((rows - 1) * ld + extent) * 2), to, voff + j, 0);
    } else {
      int v[kN];
#pragma unroll
      for (int l = 0; l < kN; ++l) v[l] = k0 + kc[j + l] >= k8 ? kFar : voff[j + l];
      LoadLds<kN, kWaves * 1024>(Buffer(at, extent * ld * 2), to, v, k0 * 2);
    }
  }
  // Byte offset in the tile of lane l's part of the fragment of rows (columns)
  // [first, first + 32) at K = 0: row l % 32, K 8 (l / 32) on.
  static __device__ __forceinline__ uint32_t Frag(int first, int lane) {
    if constexpr (kStrided) {
      const int i = lane % 16, k = 8 * (lane / 32) + i / 4;
      return k * kRow + Slot(first / 32, k) * 64 + ((lane / 16) & 1) * 32 + (i % 4) * 8;
    } else {
      return (first + lane % 32) * kRow + ((lane / 32 + lane % 32 / kPer256) & (kChunks - 1)) * 16;
    }
  }
  // The fragment 16 ks further in K.
  static __device__ __forceinline__ bf16x8 Read(const uint8_t* stage, uint32_t off, int ks) {
    if constexpr (kStrided) {
      const uint8_t* a = stage + off + ks * 16 * kRow;
      const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsTr)a);
      const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsTr)(a + 4 * kRow));
      return __builtin_bit_cast(bf16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
    } else {  // two chunks on, round the row's chunks
      const uint32_t row = off & ~static_cast<uint32_t>(kRow - 1);
      return *reinterpret_cast<const bf16x8*>(stage + row + ((off + ks * 32) & (kRow - 1)));
    }
  }
  static constexpr int kReads = kStrided ? 2 : 1;  // LDS reads of a fragment
};

// The gradient's eight from dH, G and U.
template <class T, bool kWhole>
__device__ __forceinline__ void FinishGrad(const Side& p, int m, int n, int cnt, const float (&c)[8],
                                           const float (&g)[8], float (&u)[8]) {
  float a[8], da[8];
  Activate8<sizeof(T) == 2>(p.act, g, a, da);
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const bool in = e < cnt;
    da[e] = in ? c[e] * u[e] * da[e] : 0.0f;
    u[e] = in ? a[e] * u[e] : 0.0f;
    a[e] = in ? c[e] * a[e] : 0.0f;
  }
  const size_t w = static_cast<size_t>(m) * p.h.ld + n;
  PutPlanes<T, kWhole>(p.dg, w, da);
  PutPlanes<T, kWhole>(p.du, w, a);
  PutPlanes<T, kWhole>(p.h, w, u);
}
// Eight neighbours of an output row from their sums: c of A B, d of A B2.  Off
// 16 bytes (!q.vec) what is stored there is Finish1's, the planes' rows are not.
template <class T, int kEpi, bool kWhole = false>
__device__ __forceinline__ void Finish(const Side& p, const Product& q, int m, int n, float (&c)[8],
                                       float (&d)[8]) {
  const int cnt = q.N - n;
  const size_t o = static_cast<size_t>(m) * q.N + n;
  if constexpr (kEpi == kPlain) Store8(static_cast<T*>(q.o1) + o, true, cnt, c);
  if constexpr (kEpi == kGate) {
    if (q.o1 && q.vec) {
      Store8(static_cast<T*>(q.o1) + o, true, cnt, c);
      Store8(static_cast<T*>(q.o2) + o, true, cnt, d);
    }
    float a[8], da[8];
    Activate8<sizeof(T) == 2>(p.act, c, a, da);
#pragma unroll
    for (int e = 0; e < 8; ++e) c[e] = e < cnt ? a[e] * d[e] : 0.0f;
    PutPlanes<T, kWhole>(p.h, static_cast<size_t>(m) * p.h.ld + n, c);
  }
  if constexpr (kEpi == kGrad) {
    float g[8], u[8];
    Load8(static_cast<const T*>(p.g) + o, q.vec, cnt, g);
    Load8(static_cast<const T*>(p.u) + o, q.vec, cnt, u);
    FinishGrad<T, kWhole>(p, m, n, cnt, c, g, u);
  }
}
// The outputs of one element, for rows off 16 bytes (a lane a column: a lane of
// eight would touch a line of its own with every access).
template <class T, int kEpi>
__device__ __forceinline__ void Finish1(const Product& q, int m, int n, float c, float d) {
  const size_t o = static_cast<size_t>(m) * q.N + n;
  if constexpr (kEpi == kPlain) Put(static_cast<T*>(q.o1) + o, c);
  if constexpr (kEpi == kGate) {
    if (!q.o1) return;
    Put(static_cast<T*>(q.o1) + o, c);
    Put(static_cast<T*>(q.o2) + o, d);
  }
}

// The sums of the tiles whose K was shared out, added in order and finished:
// workgroup (x, y) takes 2048 elements of the x-th of them, bm x bn large.
template <class T, int kEpi, bool kWhole = false>
__global__ void __launch_bounds__(256) FfnJoin(MmaArgs p, int bm, int bn) {
  constexpr int kBoth = kEpi == kGate ? 2 : 1;
  int m0, n0;
  const Product& q = p.q[ProductOf(p, p.whole + blockIdx.x, bm, bn, m0, n0)];
  const size_t row = static_cast<size_t>(kBoth) * bn, split = bm * row;
  const float* at = p.part + blockIdx.x * p.splits * split;
  __shared__ float st[kBoth][256 * 8];
  const int i = (blockIdx.y * 256 + threadIdx.x) * 8, r = i / bn, col = i % bn;
  const bool in = r < bm && m0 + r < q.M && n0 + col < q.N;
  float s[2][8] = {};
  for (int k0 = 0; in && k0 < p.splits; k0 += 4) {  // four sums' loads in flight
    float v[4][kBoth][8];
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
      for (int b = 0; b < kBoth; ++b)
        Load8(at + min(k0 + k, p.splits - 1) * split + r * row + b * bn + col, true, 8, v[k][b]);
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
      for (int b = 0; b < kBoth; ++b)
#pragma unroll
        for (int e = 0; e < 8; ++e) s[b][e] += k0 + k < p.splits ? v[k][b][e] : 0.0f;
  }
  if (kEpi != kGrad && !q.vec) {
#pragma unroll
    for (int b = 0; b < kBoth; ++b) Store8(&st[b][threadIdx.x * 8], true, 8, s[b]);
    __syncthreads();
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int x = e * 256 + threadIdx.x, j = blockIdx.y * 2048 + x;
      if (j < bm * bn && m0 + j / bn < q.M && n0 + j % bn < q.N)
        Finish1<T, kEpi>(q, m0 + j / bn, n0 + j % bn, st[0][x], st[kBoth - 1][x]);
    }
    if constexpr (kEpi == kPlain) return;
  }
  if (in) Finish<T, kEpi, kWhole>(p, q, m0 + r, n0 + col, s[0], s[1]);
}

template <class T, int kEpi, bool kAS, bool kBS, int BM, int BN, int BK, int WGM, int WGN, int kStages>
__global__ void __launch_bounds__(WGM * WGN * kWave) FfnMma(MmaArgs p) {
  constexpr int kWaves = WGM * WGN;
  constexpr bool kDual = kEpi == kGate;
  constexpr int BNs = kDual ? BN / 2 : BN;  // columns of the output
  constexpr int WM = BM / WGM, WN = BNs / WGN;
  constexpr int TM = WM / 32, TN = WN / 32, TB = kDual ? 2 * TN : TN;
  static_assert(TM * 32 * WGM == BM && TN * 32 * WGN == BNs, "waves cover the tile");
  using TA = Tile<kAS, BM, BK, kWaves>;
  using TBt = Tile<kBS, BNs, BK, kWaves>;
  constexpr int kSub = BK / 16;  // half-waves of K in a stage
  // A stage holds A's planes, B's and B2's.
  constexpr int kPl = sizeof(T) == 4 ? 3 : 1, kA = kPl * TA::kBytes, kB = kPl * TBt::kBytes;
  constexpr int kStage = kA + (kDual ? 2 : 1) * kB;
  constexpr int kPerStage = kPl * (TA::kLoads + (kDual ? 2 : 1) * TBt::kLoads);
  __shared__ __attribute__((aligned(1024))) uint8_t smem[kStages * kStage];

  const int wave = Uniform(threadIdx.x / kWave), lane = threadIdx.x % kWave;
  // This workgroup's tile, and of its K the stages from `first` on.
  const int per_seg = (p.K + BK - 1) / BK, total = p.nseg * per_seg;
  int b = blockIdx.x, tile, first = 0, stages = total, split = 0;
  const bool shared = b >= p.whole;
  if (!shared) {
    tile = XcdRun(b, p.whole);
  } else {
    b -= p.whole;
    const int rest = p.tiles - p.whole;
    split = b / rest;
    tile = p.whole + XcdRun(b - split * rest, rest);
    first = split * p.per_split;
    stages = min(total - first, p.per_split);
  }
  // (Copied: the arguments stay in their own memory only while few places use them.)
  const Side side = p;
  int m0, n0;
  const Product& q = p.q[ProductOf(p, tile, BM, BNs, m0, n0)];
  TA ta;
  TBt tb;
  // A strided operand's last row ends where its columns do.
  ta.Init(q.lda, kAS ? q.lda - m0 : min(q.M - m0, BM), p.K, wave, lane);
  tb.Init(q.ldb, kBS ? q.ldb - n0 : min(q.N - n0, BNs), p.K, wave, lane);
  const size_t a_at = kAS ? static_cast<size_t>(m0) : static_cast<size_t>(m0) * q.lda;
  const size_t b_at = kBS ? static_cast<size_t>(n0) : static_cast<size_t>(n0) * q.ldb;
  const uint32_t lds0 = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((LdsPtr)smem));

  const int last = stages - 1;
  // The next stage to load, and its segment's operands.
  int seg = first / per_seg, k0 = (first - seg * per_seg) * BK;
  const uint16_t *pa = q.A[seg] + a_at, *pb = q.B[seg] + b_at;
  const uint16_t* pb2 = kDual ? q.B2[seg] + b_at : nullptr;
  // Part `part` of kParts of the next stage's loads into buffer `buf`.  With
  // two buffers the stage is wanted at this one's end: its first half's steps.
  constexpr int kParts = kPl == 3 ? 1 : kStages == 2 ? kSub / 2 : kSub;
  auto issue = [&](int buf, auto part_tag) __attribute__((always_inline)) {
    constexpr int part = decltype(part_tag)::value;
    const uint32_t s = lds0 + buf * kStage;
    if constexpr (kPl == 3) {
#pragma unroll
      for (int k = 0; k < kPl; ++k) {
        ta.template Load<TA::kLoads>(pa + k * q.a_plane, k0, p.K, s + k * TA::kBytes, wave, 0);
        tb.template Load<TBt::kLoads>(pb + k * q.b_plane, k0, p.K, s + kA + k * TBt::kBytes, wave, 0);
        if constexpr (kDual)
          tb.template Load<TBt::kLoads>(pb2 + k * q.b_plane, k0, p.K, s + kA + kB + k * TBt::kBytes, wave, 0);
      }
      return;
    }
    // The stage's loads are A's, B's and B2's in turn; a part is a run of them
    // from one operand or a whole number of operands.
    constexpr int kLo = part * kPerStage / kParts, kHi = (part + 1) * kPerStage / kParts;
    constexpr int kToB = TA::kLoads, kToB2 = TA::kLoads + TBt::kLoads;
    constexpr int a0 = kLo, an = std::min(kHi, kToB) - a0;
    constexpr int b0 = std::max(kLo, kToB), bn = std::min(kHi, kToB2) - b0;
    constexpr int c0 = std::max(kLo, kToB2), cn = kHi - c0;
    if constexpr (kPl == 1 && an > 0) ta.template Load<an>(pa, k0, p.K, s, wave, a0);
    if constexpr (kPl == 1 && bn > 0) tb.template Load<bn>(pb, k0, p.K, s + kA, wave, b0 - kToB);
    if constexpr (kPl == 1 && cn > 0) tb.template Load<cn>(pb2, k0, p.K, s + kA + kB, wave, c0 - kToB2);
  };
  // Past this workgroup's last stage the loads go on, past the product's they
  // repeat, into buffers nothing reads.
  auto advance = [&]() __attribute__((always_inline)) {
    if (k0 + BK < p.K) {
      k0 += BK;
    } else if (seg + 1 < p.nseg) {
      ++seg;
      k0 = 0;
      pa = q.A[seg] + a_at, pb = q.B[seg] + b_at;
      if constexpr (kDual) pb2 = q.B2[seg] + b_at;
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
    ob[j] = kA + (j / TN) * kB + TBt::Frag(wn + (j % TN) * 32, lane);

  // K in steps of 16: the step's fragments are read while the one before is
  // multiplied, into the other half of fa and fb.
  bf16x8 fa[2][kPl][TM], fb[2][kPl][TB];
  auto read = [&](int buf, auto ks_tag) __attribute__((always_inline)) {
    constexpr int ks = decltype(ks_tag)::value;
    const uint8_t* s = smem + buf * kStage;
#pragma unroll
    for (int k = kPl - 1; k >= 0; --k) {
#pragma unroll
      for (int i = 0; i < TM; ++i) fa[ks % 2][k][i] = TA::Read(s + k * TA::kBytes, oa[i], ks);
#pragma unroll
      for (int j = 0; j < TB; ++j) fb[ks % 2][k][j] = TBt::Read(s + k * TBt::kBytes, ob[j], ks);
    }
  };
  // (f32: the six plane products, smallest first.)
  constexpr int kPairs = kPl == 3 ? 6 : 1;
  auto mfmas = [&](int half) __attribute__((always_inline)) {
    constexpr int pairs[6][2] = {{2, 0}, {0, 2}, {1, 1}, {1, 0}, {0, 1}, {0, 0}};
#pragma unroll
    for (int k = 6 - kPairs; k < 6; ++k)
#pragma unroll
      for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TB; ++j)
          acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fb[half][pairs[k][1]][j], fa[half][pairs[k][0]][i],
                                                              acc[i][j], 0, 0, 0);
  };
  // The next step's reads spread over the products of this one.
  constexpr int kMfmas = kPairs * TM * TB, kReads = kPl * (TM * TA::kReads + TB * TBt::kReads);
  constexpr int kPerSlot = (kReads + kMfmas - 1) / kMfmas;
  auto interleave = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int s = 0; s < kMfmas; ++s) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      if (s * kPerSlot < kReads) __builtin_amdgcn_sched_group_barrier(0x100, kPerSlot, 0);
    }
  };
  // A stage's steps but the last, each behind the next one's reads.  The loads
  // of the stage that takes the buffer freed last (`to`) go out a few a step:
  // all at once they would hold up the products behind them.
  auto steps = [&](int buf, int to, auto load) __attribute__((always_inline)) {
    Each<kSub - 1>([&](auto ks) __attribute__((always_inline)) {
      if constexpr (decltype(load)::value && decltype(ks)::value < kParts) issue(to, ks);
      read(buf, std::integral_constant<int, decltype(ks)::value + 1>{});
      mfmas(decltype(ks)::value % 2);
      interleave();
    });
    if constexpr (decltype(load)::value && kParts == kSub)
      issue(to, std::integral_constant<int, kSub - 1>{});
  };

  // kStages buffers: one multiplied, one taking loads, the others in flight or
  // landed.  Before the last step of stage `it` every wave has its fragments of
  // it and stage it + 1 has landed.
  // f32's short stages take a buffer's next loads as soon as it is free.
  constexpr bool kEarly = kPl == 3;
  constexpr int kAhead = kEarly ? kStages : kStages - 1;
  for (int s = 0; s < kAhead; ++s) {
    Each<kParts>([&](auto part) __attribute__((always_inline)) { issue(s, part); });
    advance();
  }
  WaitVm<(kAhead - 1) * kPerStage>();
  Barrier();
  read(0, std::integral_constant<int, 0>{});
  for (int it = 0; it < last; ++it) {
    steps(it % kStages, (it + kStages - 1) % kStages, std::bool_constant<!kEarly>{});
    WaitVm<(kStages - 2) * kPerStage>();
    WaitLds();
    Barrier();
    if constexpr (kEarly) issue(it % kStages, std::integral_constant<int, 0>{});
    advance();
    read((it + 1) % kStages, std::integral_constant<int, 0>{});
    mfmas((kSub - 1) % 2);
    interleave();
  }
  steps(last % kStages, 0, std::false_type{});
  mfmas((kSub - 1) % 2);
  // The repeated loads have landed and this wave's fragments are in registers:
  // past the next barrier other waves write over the stages.
  WaitVm<0>();
  WaitLds();

  // The epilogue: kW columns of 32 rows at a time through this wave's slice of
  // LDS.  Accumulator element 4 q + e of block (i, j) is row lane % 32, column
  // 8 q + 4 (lane / 32) + e; a lane takes eight neighbours of a row away.
  constexpr int kW = WN >= 64 ? 64 : 32, kPad = kW + 4, kBoth = kDual ? 2 : 1;
  static_assert(kWaves * kBoth * 32 * kPad * 4 <= kStages * kStage, "staging fits");
  constexpr int kPerRow = kW / 8, kRows = kWave / kPerRow;
  float* st = reinterpret_cast<float*>(smem) + wave * kBoth * 32 * kPad;
  const int h = lane / 32;
  // The gradient's G and U, a part ahead of their use: nothing else covers
  // their latency (8192 x 2048 x 5632 bf16: 251 us, 316 with the loads where
  // they are used; the product alone is 165).
  constexpr int kT = 32 / kRows, kEpiParts = TM * (WN / kW);
  Raw8<T> rg[2][kT], ru[2][kT];
  const bool ahead = kEpi == kGrad && q.vec && !shared;
  auto fetch = [&](auto part) __attribute__((always_inline)) {
    constexpr int i = decltype(part)::value / (WN / kW), jb = decltype(part)::value % (WN / kW);
    const int n = min(n0 + wn + jb * kW + (lane % kPerRow) * 8, q.N - 8);
    Each<kT>([&](auto t) __attribute__((always_inline)) {
      const size_t o = static_cast<size_t>(min(m0 + wm + i * 32 + lane / kPerRow + t * kRows, q.M - 1)) * q.N + n;
      rg[decltype(part)::value % 2][t].Load(static_cast<const T*>(side.g) + o);
      ru[decltype(part)::value % 2][t].Load(static_cast<const T*>(side.u) + o);
    });
  };
  if constexpr (kEpi == kGrad) {
    if (ahead) fetch(std::integral_constant<int, 0>{});
  }
  Barrier();  // every wave is done with the stages
  Each<kEpiParts>([&](auto part) __attribute__((always_inline)) {
    constexpr int i = decltype(part)::value / (WN / kW), jb = decltype(part)::value % (WN / kW);
#pragma unroll
    for (int b = 0; b < kBoth; ++b)
#pragma unroll
      for (int jj = 0; jj < kW / 32; ++jj)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const v16f& c = acc[i][b * TN + jb * (kW / 32) + jj];
          *reinterpret_cast<float4*>(st + (b * 32 + lane % 32) * kPad + jj * 32 + 8 * q + 4 * h) =
              make_float4(c[4 * q], c[4 * q + 1], c[4 * q + 2], c[4 * q + 3]);
        }
    __builtin_amdgcn_wave_barrier();
    const int mb = m0 + wm + i * 32, nb = n0 + wn + jb * kW;
    if (kEpi != kGrad && !q.vec && !shared) {
      const int n = nb + lane % kW;
      for (int r = lane / kW; r < 32; r += kWave / kW)
        if (mb + r < q.M && n < q.N)
          Finish1<T, kEpi>(q, mb + r, n, st[r * kPad + lane % kW], kDual ? st[(32 + r) * kPad + lane % kW] : 0.0f);
    }
    if (ahead) {
      if constexpr (kEpi == kGrad) {
        if constexpr (decltype(part)::value + 1 < kEpiParts)
          fetch(std::integral_constant<int, decltype(part)::value + 1>{});
        const int n = nb + (lane % kPerRow) * 8;
        Each<kT>([&](auto t) __attribute__((always_inline)) {
          const int r = lane / kPerRow + t * kRows, m = mb + r;
          if (m >= q.M || n >= q.N) return;
          float c[8], g[8], u[8];
          Load8(st + r * kPad + (lane % kPerRow) * 8, true, 8, c);
          rg[decltype(part)::value % 2][t].Get(g);
          ru[decltype(part)::value % 2][t].Get(u);
          FinishGrad<T, false>(side, m, n, 8, c, g, u);
        });
      }
    } else if (kEpi != kPlain || q.vec || shared) {
      const int n = nb + (lane % kPerRow) * 8;
#pragma unroll
      for (int t = 0; t < 32 / kRows; ++t) {
        const int r = lane / kPerRow + t * kRows, m = mb + r;
        if (m >= q.M || n >= q.N) continue;
        float c[8], d[8];
        Load8(st + r * kPad + (lane % kPerRow) * 8, true, 8, c);
        if constexpr (kDual) Load8(st + (32 + r) * kPad + (lane % kPerRow) * 8, true, 8, d);
        if (shared) {
          float* out = p.part + ((static_cast<size_t>(tile - p.whole) * p.splits + split) * BM + (m - m0)) *
                                    (kBoth * BNs) + (n - n0);
          Store8(out, true, 8, c);
          if constexpr (kDual) Store8(out + BNs, true, 8, d);
        } else {
          Finish<T, kEpi>(side, q, m, n, c, d);
        }
      }
    }
    __builtin_amdgcn_wave_barrier();
  });
}

// Few f32 tokens: splitting the weights into planes would move three times
// their bytes, so the products run on the f32 MFMA (32 x 32 x 2) straight from
// memory, and H, dG and dU stay f32.  FfnRows32 runs those with the weights: a
// workgroup takes 32 kR rows by 32 kC columns, its waves K in turns of 32; K's
// order within eight is the lanes': half-wave h of product j takes k = 4 h + j,
// so a lane's four values of a row are one load.  Weights contiguous in K have
// a lane's columns 32 apart; strided ones have kC neighbours a lane, one load.
// The waves' sums are added in LDS in wave order.  Bound by the weights' bytes up
// to 32 tokens (8 x 2048 x 5632: the gate's 92 MB in 27 us, 3.4 TB/s; through
// planes the forward took 135 us, now 48, the backward 214, now 80) and by the
// f32 MFMA's rate and its operands' loads past them (64: 53 us, floor 21).
constexpr int kRowsWaves = 8, kRowsK = 32;
template <bool kGuard>
__device__ __forceinline__ void Row4(const float* p, bool vec, int left, float (&v)[4]) {
  if (vec && (!kGuard || left >= 4)) {
    const float4 a = *reinterpret_cast<const float4*>(p);
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w;
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = !kGuard || e < left ? p[e] : 0.0f;
  }
}
// An element's epilogue, H, dG and dU in f32.
template <int kEpi>
__device__ __forceinline__ void FinishWhole(const MmaArgs& p, const Product& q, int m, int n, float c, float d) {
  const bool in = n < q.N;
  if (kEpi != kGrad && in) Finish1<float, kEpi>(q, m, n, c, d);
  if (kEpi == kPlain || n >= p.h.ld) return;
  const size_t at = static_cast<size_t>(m) * p.h.ld + n, o = static_cast<size_t>(m) * q.N + n;
  auto put = [&](const Planes& out, float v) { reinterpret_cast<float*>(out.p)[at] = in ? v : 0.0f; };
  float a, da;
  if constexpr (kEpi == kGate) {
    Activate<false>(p.act, c, a, da);
    put(p.h, a * d);
  } else if constexpr (kEpi == kGrad) {
    const float g = in ? static_cast<const float*>(p.g)[o] : 0.0f, u = in ? static_cast<const float*>(p.u)[o] : 0.0f;
    Activate<false>(p.act, g, a, da);
    put(p.dg, c * u * da);
    put(p.du, c * a);
    put(p.h, a * u);
  }
}
template <bool kGuard, bool kVec, int kC>
__device__ __forceinline__ void Cols(const float* p, const size_t (&col)[kC], bool in, float (&v)[kC]) {
#pragma unroll
  for (int c = 0; c < kC; ++c) v[c] = 0.0f;
  if (kGuard && !in) return;
  if constexpr (kVec && kC == 4) {
    const float4 a = *reinterpret_cast<const float4*>(p + col[0]);
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w;
  } else if constexpr (kVec && kC == 2) {
    const float2 a = *reinterpret_cast<const float2*>(p + col[0]);
    v[0] = a.x, v[1] = a.y;
  } else {
#pragma unroll
    for (int c = 0; c < kC; ++c) v[c] = p[col[c]];
  }
}
template <int kEpi, bool kBS, bool kVec, int kR, int kC>
__global__ void __launch_bounds__(kRowsWaves * kWave) FfnRows32(MmaArgs p) {
  constexpr int kBoth = kEpi == kGate ? 2 : 1, BM = 32 * kR, BN = 32 * kC;
  __shared__ float sums[kRowsWaves][32][32 + 4];
  const int wave = Uniform(threadIdx.x / kWave), lane = threadIdx.x % kWave;
  const int i = lane % 32, h = lane / 32;
  const int per_seg = (p.K + kRowsK - 1) / kRowsK, total = p.nseg * per_seg;
  const int split = blockIdx.x / p.tiles, tile = blockIdx.x - split * p.tiles;
  const int first = split * p.per_split, end = min(total, first + p.per_split);
  int m0, n0;
  const Product& q = p.q[ProductOf(p, tile, BM, BN, m0, n0)];
  // Rows and columns past the end repeat the last: nothing of theirs is stored.
  size_t row[kR], col[kC];
#pragma unroll
  for (int r = 0; r < kR; ++r) row[r] = static_cast<size_t>(min(m0 + 32 * r + i, q.M - 1)) * q.lda;
#pragma unroll
  for (int c = 0; c < kC; ++c)
    col[c] = kBS ? (kVec ? min(n0 + kC * i, q.N - kC) + c : min(n0 + kC * i + c, q.N - 1))
                 : min(n0 + 32 * c + i, q.N - 1) * static_cast<size_t>(q.ldb);
  v16f acc[kBoth][kR][kC];
#pragma unroll
  for (int b = 0; b < kBoth; ++b)
#pragma unroll
    for (int r = 0; r < kR; ++r)
#pragma unroll
      for (int c = 0; c < kC; ++c) acc[b][r][c] = v16f{};
  for (int s = first + wave; s < end; s += kRowsWaves) {
    const int seg = s / per_seg, k0 = (s - seg * per_seg) * kRowsK;
    auto step = [&](auto guard) __attribute__((always_inline)) {
      constexpr bool kGuard = decltype(guard)::value;
      float a[kR][kRowsK / 8][4], w[kBoth][kRowsK / 8][4][kC];
#pragma unroll
      for (int u = 0; u < kRowsK / 8; ++u) {
        const int k = k0 + 8 * u + 4 * h, left = p.K - k;
#pragma unroll
        for (int r = 0; r < kR; ++r)
          Row4<kGuard>(reinterpret_cast<const float*>(q.A[seg]) + row[r] + k, kVec, left, a[r][u]);
#pragma unroll
        for (int b = 0; b < kBoth; ++b) {
          const float* B = reinterpret_cast<const float*>(b ? q.B2[seg] : q.B[seg]);
          if constexpr (kBS) {
#pragma unroll
            for (int j = 0; j < 4; ++j) Cols<kGuard, kVec>(B + static_cast<size_t>(k + j) * q.ldb, col, j < left, w[b][u][j]);
          } else {
#pragma unroll
            for (int c = 0; c < kC; ++c) {
              float v[4];
              Row4<kGuard>(B + col[c] + k, kVec, left, v);
#pragma unroll
              for (int j = 0; j < 4; ++j) w[b][u][j][c] = v[j];
            }
          }
        }
      }
#pragma unroll
      for (int u = 0; u < kRowsK / 8; ++u)
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int b = 0; b < kBoth; ++b)
#pragma unroll
            for (int r = 0; r < kR; ++r)
#pragma unroll
              for (int c = 0; c < kC; ++c)
                acc[b][r][c] =
                    __builtin_amdgcn_mfma_f32_32x32x2f32(w[b][u][j][c], a[r][u][j], acc[b][r][c], 0, 0, 0);
    };
    if (k0 + kRowsK <= p.K) step(std::false_type{});
    else step(std::true_type{});
  }
  // The waves' sums of 32 x 32 after 32 x 32, two elements a thread.
  constexpr int kEach = 1024 / (kRowsWaves * kWave);
  Each<kR * kC>([&](auto t) __attribute__((always_inline)) {
    constexpr int r = decltype(t)::value / kC, c = decltype(t)::value % kC;
    float v[kBoth][kEach];
#pragma unroll
    for (int b = 0; b < kBoth; ++b) {
      __syncthreads();
#pragma unroll
      for (int e = 0; e < 4; ++e)
        *reinterpret_cast<float4*>(&sums[wave][i][8 * e + 4 * h]) =
            make_float4(acc[b][r][c][4 * e], acc[b][r][c][4 * e + 1], acc[b][r][c][4 * e + 2], acc[b][r][c][4 * e + 3]);
      __syncthreads();
#pragma unroll
      for (int e = 0; e < kEach; ++e) {
        const int x = e * kRowsWaves * kWave + threadIdx.x;
        v[b][e] = 0.0f;
#pragma unroll
        for (int k = 0; k < kRowsWaves; ++k) v[b][e] += sums[k][x / 32][x % 32];
      }
    }
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
      const int x = e * kRowsWaves * kWave + threadIdx.x;
      const int m = 32 * r + x / 32, n = kBS ? x % 32 * kC + c : 32 * c + x % 32;
      if (m0 + m >= q.M) continue;
      if (p.splits > 1) {
        float* out = p.part + ((static_cast<size_t>(tile) * p.splits + split) * BM + m) * (kBoth * BN) + n;
#pragma unroll
        for (int b = 0; b < kBoth; ++b) out[b * BN] = v[b][e];
      } else {
        FinishWhole<kEpi>(p, q, m0 + m, n0 + n, v[0][e], v[kBoth - 1][e]);
      }
    }
  });
}

// The weights' gradients of few f32 tokens: K is the tokens, so what there is to
// move is the stores.  A workgroup takes 128 x 128, a wave 32 rows of it and four
// neighbouring columns a lane: stores of 512 bytes.  The operands' 128 columns
// of up to 32 tokens are staged in LDS (64 tokens of 2048 x 5632: 69 us, with
// operands straight from memory 90).  8 tokens: 26 us for 138 MB stored, 5.3 TB/s.
constexpr int kOuterWaves = 4, kOuterK = 32;
// Tokens [k0, k0 + rows) of operand columns [c0, c0 + 128), zeros past K and
// past `cols`.
__device__ __forceinline__ void StageOuter(float (*to)[128], const float* p, int ld, int c0, int cols, bool vec,
                                           int k0, int K) {
  constexpr int kThreads = kOuterWaves * kWave;
#pragma unroll
  for (int j = 0; j < kOuterK * 32 / kThreads; ++j) {
    const int x = j * kThreads + threadIdx.x, k = k0 + x / 32, c = c0 + x % 32 * 4;
    const int left = k < K ? cols - c : 0;
    float v[4] = {};
    if (left > 0) Row4<true>(p + static_cast<size_t>(k) * ld + c, vec, left, v);
    *reinterpret_cast<float4*>(&to[x / 32][x % 32 * 4]) = make_float4(v[0], v[1], v[2], v[3]);
  }
}
__global__ void __launch_bounds__(kOuterWaves * kWave, 4) FfnOuter32(MmaArgs p) {
  __shared__ float A[kOuterK][128], B[kOuterK][128];
  const int wave = Uniform(threadIdx.x / kWave), lane = threadIdx.x % kWave;
  const int i = lane % 32, h = lane / 32;
  int m0, n0;
  const Product& q = p.q[ProductOf(p, XcdRun(blockIdx.x, p.tiles), 128, 128, m0, n0)];
  v16f acc[4] = {};
  for (int k0 = 0; k0 < p.K; k0 += kOuterK) {
    if (k0) __syncthreads();
    StageOuter(A, reinterpret_cast<const float*>(q.A[0]), q.lda, m0, q.M, q.vec_a, k0, p.K);
    StageOuter(B, reinterpret_cast<const float*>(q.B[0]), q.ldb, n0, q.N, q.vec, k0, p.K);
    __syncthreads();
    const int turns = (min(p.K - k0, kOuterK) + 1) / 2;
#pragma unroll 4
    for (int u = 0; u < turns; ++u) {
      const float a = A[2 * u + h][32 * wave + i];
      const float4 b = *reinterpret_cast<const float4*>(&B[2 * u + h][4 * i]);
      acc[0] = __builtin_amdgcn_mfma_f32_32x32x2f32(a, b.x, acc[0], 0, 0, 0);
      acc[1] = __builtin_amdgcn_mfma_f32_32x32x2f32(a, b.y, acc[1], 0, 0, 0);
      acc[2] = __builtin_amdgcn_mfma_f32_32x32x2f32(a, b.z, acc[2], 0, 0, 0);
      acc[3] = __builtin_amdgcn_mfma_f32_32x32x2f32(a, b.w, acc[3], 0, 0, 0);
    }
  }
  const int n = n0 + 4 * i;
#pragma unroll
  for (int e = 0; e < 16; ++e) {
    const int m = m0 + 32 * wave + 8 * (e / 4) + 4 * h + e % 4;
    if (m >= q.M) continue;
    float* out = static_cast<float*>(q.o1) + static_cast<size_t>(m) * q.N + n;
    if (q.vec) {
      if (n < q.N) *reinterpret_cast<float4*>(out) = make_float4(acc[0][e], acc[1][e], acc[2][e], acc[3][e]);
    } else {
#pragma unroll
      for (int c = 0; c < 4; ++c)
        if (n + c < q.N) out[c] = acc[c][e];
    }
  }
}

// --- host ---------------------------------------------------------------------------------------

size_t PartBytes(bool f32, const Plan& plan, bool dual) {
  const TileShape& s = ShapeOf(f32, plan.tile);
  return static_cast<size_t>(plan.tiles - plan.whole) * plan.splits * s.bm(dual) * s.bn(dual) * (dual ? 8 : 4);
}

template <class T, int kEpi, bool kAS, bool kBS, int BM, int BN, int BK, int WGM, int WGN, int kStages>
hipError_t LaunchTile(const MmaArgs& a, hipStream_t s) {
  static_assert(BK == Deep(sizeof(T) == 4), "per_split counts such stages");
  const unsigned grid = a.whole + static_cast<unsigned>(a.tiles - a.whole) * a.splits;
  auto* kernel = &FfnMma<T, kEpi, kAS, kBS, BM, BN, BK, WGM, WGN, kStages>;
  hipLaunchKernelGGL(kernel, dim3(grid), dim3(WGM * WGN * kWave), 0, s, a);
  return hipGetLastError();
}

// `part`: where the shared-out sums go (PartBytes).
template <class T, int kEpi, bool kAS, bool kBS>
hipError_t Mma(MmaArgs a, float* part, hipStream_t s) {
  constexpr bool dual = kEpi == kGate;
  const Shape shape[3] = {{static_cast<size_t>(a.q[0].M), static_cast<size_t>(a.q[0].N)},
                          {static_cast<size_t>(a.q[1].M), static_cast<size_t>(a.q[1].N)},
                          {static_cast<size_t>(a.q[2].M), static_cast<size_t>(a.q[2].N)}};
  constexpr bool f32 = sizeof(T) == 4;
  const Plan plan = a.count == 1 ? Choose(f32, dual, {shape[0]}, a.K, a.nseg)
                                 : Choose(f32, dual, {shape[0], shape[1], shape[2]}, a.K, a.nseg);
  const TileShape& t = ShapeOf(f32, plan.tile);
  const int bm = t.bm(dual), bn = t.bn(dual);
  for (int i = 0, first = 0; i < a.count; ++i) {
    a.q[i].first = first;
    first += ((a.q[i].M + bm - 1) / bm) * ((a.q[i].N + bn - 1) / bn);
  }
  a.tiles = plan.tiles, a.whole = plan.whole, a.splits = plan.splits, a.per_split = plan.per_split;
  a.part = part;
  hipError_t e;
  if constexpr (f32) {
    if (plan.tile == 0) e = LaunchTile<T, kEpi, kAS, kBS, dual ? 128 : 256, dual ? 256 : 128, 32, dual ? 2 : 4, dual ? 4 : 2, 2>(a, s);
    else e = LaunchTile<T, kEpi, kAS, kBS, 64, 128, 32, 2, 2, 2>(a, s);
  } else {
    if (plan.tile == 0) e = LaunchTile<T, kEpi, kAS, kBS, 256, 256, 64, 2, 4, 2>(a, s);
    else if (plan.tile == 1) e = LaunchTile<T, kEpi, kAS, kBS, 128, 128, 64, 2, 2, 2>(a, s);
    else e = LaunchTile<T, kEpi, kAS, kBS, 64, dual ? 128 : 64, 64, 2, 2, dual ? 3 : 4>(a, s);
  }
  if (e != hipSuccess || plan.whole == plan.tiles) return e;
  auto* kernel = &FfnJoin<T, kEpi>;
  hipLaunchKernelGGL(kernel, dim3(plan.tiles - plan.whole, bm * bn / 2048), dim3(256), 0, s, a, bm, bn);
  return hipGetLastError();
}

// f32 tokens up to which FfnRows32 and FfnOuter32 run the products.  Forward and
// backward at 2048 x 5632, us, against the planes: 16 tokens 48, 83 (138, 214);
// 64 tokens 82, 152 (155, 241); 128 tokens 133, 247 (170, 282); 192 tokens 250,
// 443 (206, 345).  Smaller weights turn at 192 or later.
constexpr size_t kRowsMost = 128;
bool FewRows(int planes, size_t M) { return planes == 3 && M <= kRowsMost; }
// FfnRows32's tile, and how it shares K out: over workgroups enough for the
// chip, with a turn for every wave.  Measured on 4 and 64 tokens of 2048 x 5632
// (forward, whole): gate tiles 32 wide over 768 workgroups 53 and 106 us, over
// 256 56 and 108, 64 wide 56 and 161; plain ones 64 wide over 256 53 and 100,
// 32 wide over 512 59 and 116.  Where that leaves the chip short of workgroups
// the 32 x 32 tile is better: 64 tokens of 333 x 1111 26 us against 43.
struct RowsPlan {
  int rows, cols, tiles, splits, per_split;
};
RowsPlan ChooseRows(Epilogue epi, const Shape& q, size_t K, int nseg) {
  const int steps = static_cast<int>((K + kRowsK - 1) / kRowsK) * nseg;
  const int groups = epi == kPlain ? 256 : 768;
  RowsPlan plan;
  const int most = std::max(1, steps / kRowsWaves);
  const bool small = (q.M + 31) / 32 * ((q.N + 31) / 32) * most < 512;
  plan.rows = q.M > 32 && !small ? 64 : 32;
  plan.cols = epi == kPlain && !small ? 64 : 32;
  plan.tiles = static_cast<int>(((q.M + plan.rows - 1) / plan.rows) * ((q.N + plan.cols - 1) / plan.cols));
  const int splits = std::min(most, std::max(1, (groups + plan.tiles / 2) / plan.tiles));
  plan.per_split = (steps + splits - 1) / splits;
  plan.splits = (steps + plan.per_split - 1) / plan.per_split;
  return plan;
}
size_t RowsPartBytes(const RowsPlan& plan, bool dual) {
  return plan.splits == 1 ? 0 : static_cast<size_t>(plan.tiles) * plan.splits * plan.rows * plan.cols * (dual ? 8 : 4);
}
template <int kEpi, bool kBS>
hipError_t Rows32(MmaArgs a, bool vec, float* part, hipStream_t s) {
  const Shape shape{static_cast<size_t>(a.q[0].M), static_cast<size_t>(a.q[0].N)};
  const RowsPlan plan = ChooseRows(static_cast<Epilogue>(kEpi), shape, a.K, a.nseg);
  a.tiles = plan.tiles, a.splits = plan.splits, a.per_split = plan.per_split;
  a.part = part;
  constexpr int kC = kEpi == kPlain ? 2 : 1;
  using Kernel = void (*)(MmaArgs);
  Kernel kernel = vec ? &FfnRows32<kEpi, kBS, true, 1, 1> : &FfnRows32<kEpi, kBS, false, 1, 1>;
  if (plan.rows == 32 && plan.cols == 32 * kC)
    kernel = vec ? &FfnRows32<kEpi, kBS, true, 1, kC> : &FfnRows32<kEpi, kBS, false, 1, kC>;
  if (plan.rows == 64)
    kernel = vec ? &FfnRows32<kEpi, kBS, true, 2, kC> : &FfnRows32<kEpi, kBS, false, 2, kC>;
  hipLaunchKernelGGL(kernel, dim3(plan.tiles * plan.splits), dim3(kRowsWaves * kWave), 0, s, a);
  if (hipError_t e = hipGetLastError(); e != hipSuccess || plan.splits == 1) return e;
  auto* join = &FfnJoin<float, kEpi, true>;
  const unsigned parts = (plan.rows * plan.cols + 2047) / 2048;
  hipLaunchKernelGGL(join, dim3(plan.tiles, parts), dim3(256), 0, s, a, plan.rows, plan.cols);
  return hipGetLastError();
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
  float* Floats(size_t bytes) {
    float* p = reinterpret_cast<float*>(base_ + used_);
    used_ += (bytes + 255) / 256 * 256;
    return p;
  }
  size_t used() const { return used_; }

 private:
  uint8_t* base_;
  size_t used_ = 0;
};

struct Layout {
  Planes x, wg, wu, wd, dy, h, dg, du;
  float* part;
  size_t bytes;
};
Layout Lay(void* ws, int planes, size_t M, size_t D, size_t F, bool backward) {
  Space s(ws);
  Layout l;
  if (FewRows(planes, M)) {
    l.h = s.Take(M, F, 2);  // (two planes' bytes are f32's)
    if (backward) {
      l.dg = s.Take(M, F, 2);
      l.du = s.Take(M, F, 2);
    }
    auto rows = [&](Epilogue epi, size_t n, size_t k, int segs) {
      return RowsPartBytes(ChooseRows(epi, {M, n}, k, segs), epi == kGate);
    };
    l.part = s.Floats(backward ? std::max(rows(kGrad, F, D, 1), rows(kPlain, D, F, 2))
                               : std::max(rows(kGate, F, D, 1), rows(kPlain, D, F, 1)));
    l.bytes = s.used();
    return l;
  }
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
  auto part = [&](bool dual, std::initializer_list<Shape> q, size_t k, int segs) {
    return PartBytes(planes == 3, Choose(planes == 3, dual, q, k, segs), dual);
  };
  l.part = s.Floats(backward ? std::max({part(false, {{M, F}}, D, 1), part(false, {{M, D}}, F, 2),
                                         part(false, {{D, F}, {D, F}, {F, D}}, M, 1)})
                             : std::max(part(true, {{M, F}}, D, 1), part(false, {{M, D}}, F, 1)));
  l.bytes = s.used();
  return l;
}

// An operand as planes: itself where its rows begin on 16 bytes, else to be
// packed.
template <class T>
void Take(const void* in, size_t rows, size_t cols, Planes& out, Pieces& pieces) {
  const uintptr_t at = reinterpret_cast<uintptr_t>(in);
  if (sizeof(T) == 2 && cols % 8 == 0 && (at & 15) == 0) {
    out.p = static_cast<uint16_t*>(const_cast<void*>(in));
    return;
  }
  pieces.q[pieces.count++] = {in, rows, static_cast<int>(cols),
                              cols % (16 / sizeof(T)) == 0 && (at & 15) == 0, out, pieces.blocks};
  pieces.blocks += static_cast<unsigned>((rows * (out.ld / 8) + 255) / 256);
}
template <class T>
hipError_t Pack(const Pieces& pieces, hipStream_t s) {
  if (pieces.count == 0) return hipSuccess;
  auto* kernel = &FfnPackKernel<T>;
  // In rows of workgroups: past 2^35 elements one row would be over 2^32 threads.
  const unsigned row = std::min(pieces.blocks, 1u << 16);
  hipLaunchKernelGGL(kernel, dim3(row, (pieces.blocks + row - 1) / row), dim3(256), 0, s, pieces);
  return hipGetLastError();
}

// Rows that begin on 16 bytes.
template <class T>
bool Octs(size_t N, std::initializer_list<const void*> ptrs) {
  uintptr_t at = 0;
  for (const void* p : ptrs) at |= reinterpret_cast<uintptr_t>(p);
  return N % 8 == 0 && (at & 15) == 0;
}

// A launch's next product, its first segment A B (and A B2).
Product& AddProduct(MmaArgs& a, size_t M, size_t N, const Planes& A, const Planes& B,
                    const Planes* B2 = nullptr) {
  Product& q = a.q[a.count++];
  q.M = static_cast<int>(M), q.N = static_cast<int>(N);
  q.lda = A.ld, q.ldb = B.ld;
  q.A[0] = A.p, q.B[0] = B.p, q.B2[0] = B2 ? B2->p : nullptr;
  q.a_plane = A.plane, q.b_plane = B.plane;
  a.nseg = 1;
  return q;
}

MmaArgs Launch(size_t K) {
  MmaArgs a{};
  a.K = static_cast<int>(K);
  return a;
}

#define FFN_TRY(expr)                                       \
  do {                                                      \
    if (hipError_t e_ = (expr); e_ != hipSuccess) return e_; \
  } while (0)

// A product of f32 operands as they are, rows of A by B (and B2).
Product& AddRaw(MmaArgs& a, size_t M, size_t N, const void* A, size_t lda, const void* B, size_t ldb,
                const void* B2 = nullptr) {
  Product& q = a.q[a.count++];
  q.M = static_cast<int>(M), q.N = static_cast<int>(N);
  q.lda = static_cast<int>(lda), q.ldb = static_cast<int>(ldb);
  q.A[0] = static_cast<const uint16_t*>(A);
  q.B[0] = static_cast<const uint16_t*>(B);
  q.B2[0] = static_cast<const uint16_t*>(B2);
  a.nseg = 1;
  return q;
}
bool Fours(size_t n, std::initializer_list<const void*> ptrs) {
  uintptr_t at = 0;
  for (const void* p : ptrs) at |= reinterpret_cast<uintptr_t>(p);
  return n % 4 == 0 && (at & 15) == 0;
}

hipError_t FwdRows(const FfnArgs& f, const Layout& l, hipStream_t s) {
  MmaArgs a = Launch(f.D);
  Product& gate = AddRaw(a, f.M, f.F, f.x, f.D, f.wg, f.F, f.wu);
  gate.o1 = f.gate, gate.o2 = f.up, gate.vec = Octs<float>(f.F, {f.gate, f.up});
  a.act = f.act, a.h = l.h;
  FFN_TRY((Rows32<kGate, true>(a, Fours(f.D, {f.x}) && Fours(f.F, {f.wg, f.wu}), l.part, s)));
  a = Launch(f.F);
  Product& down = AddRaw(a, f.M, f.D, l.h.p, l.h.ld, f.wd, f.D);
  down.o1 = f.y, down.vec = Octs<float>(f.D, {f.y});
  return Rows32<kPlain, true>(a, Fours(f.D, {f.wd}), l.part, s);
}
hipError_t BwdRows(const FfnArgs& f, const Layout& l, hipStream_t s) {
  MmaArgs a = Launch(f.D);
  AddRaw(a, f.M, f.F, f.dy, f.D, f.wd, f.D).vec = Octs<float>(f.F, {f.gate, f.up});
  a.act = f.act, a.g = f.gate, a.u = f.up, a.h = l.h, a.dg = l.dg, a.du = l.du;
  FFN_TRY((Rows32<kGrad, false>(a, Fours(f.D, {f.dy, f.wd}), l.part, s)));
  a = Launch(f.F);
  Product& dx = AddRaw(a, f.M, f.D, l.dg.p, l.dg.ld, f.wg, f.F);
  dx.A[1] = l.du.p, dx.B[1] = static_cast<const uint16_t*>(f.wu), a.nseg = 2;
  dx.o1 = f.dx, dx.vec = Octs<float>(f.D, {f.dx});
  FFN_TRY((Rows32<kPlain, false>(a, Fours(f.F, {f.wg, f.wu}), l.part, s)));
  a = Launch(f.M);
  const void* left[3] = {f.x, f.x, l.h.p};
  const void* right[3] = {l.dg.p, l.du.p, f.dy};
  void* out[3] = {f.dwg, f.dwu, f.dwd};
  for (int i = 0; i < 3; ++i) {
    const size_t M = i == 2 ? f.F : f.D, N = i == 2 ? f.D : f.F;
    Product& q = AddRaw(a, M, N, left[i], i == 2 ? l.h.ld : f.D, right[i], i == 2 ? f.D : l.dg.ld);
    q.o1 = out[i], q.vec = Fours(N, {out[i], right[i]}), q.vec_a = Fours(M, {left[i]}), q.first = a.tiles;
    a.tiles += static_cast<int>((M + 127) / 128 * ((N + 127) / 128));
  }
  hipLaunchKernelGGL(FfnOuter32, dim3(a.tiles), dim3(kOuterWaves * kWave), 0, s, a);
  return hipGetLastError();
}

template <class T>
hipError_t Fwd(const FfnArgs& f, hipStream_t s) {
  if (f.M == 0) return hipSuccess;
  Layout l = Lay(f.ws, sizeof(T) == 2 ? 1 : 3, f.M, f.D, f.F, false);
  if (sizeof(T) == 4 && FewRows(3, f.M)) return FwdRows(f, l, s);
  Pieces pieces{};
  Take<T>(f.x, f.M, f.D, l.x, pieces);
  Take<T>(f.wg, f.D, f.F, l.wg, pieces);
  Take<T>(f.wu, f.D, f.F, l.wu, pieces);
  Take<T>(f.wd, f.F, f.D, l.wd, pieces);
  FFN_TRY(Pack<T>(pieces, s));
  MmaArgs a = Launch(f.D);
  Product& gate = AddProduct(a, f.M, f.F, l.x, l.wg, &l.wu);
  gate.o1 = f.gate, gate.o2 = f.up, gate.vec = Octs<T>(f.F, {f.gate, f.up});
  a.act = f.act, a.h = l.h;
  FFN_TRY((Mma<T, kGate, false, true>(a, l.part, s)));
  a = Launch(f.F);
  Product& down = AddProduct(a, f.M, f.D, l.h, l.wd);
  down.o1 = f.y, down.vec = Octs<T>(f.D, {f.y});
  return Mma<T, kPlain, false, true>(a, l.part, s);
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
  if (sizeof(T) == 4 && FewRows(3, f.M)) return BwdRows(f, l, s);
  Pieces pieces{};
  Take<T>(f.x, f.M, f.D, l.x, pieces);
  Take<T>(f.wg, f.D, f.F, l.wg, pieces);
  Take<T>(f.wu, f.D, f.F, l.wu, pieces);
  Take<T>(f.wd, f.F, f.D, l.wd, pieces);
  Take<T>(f.dy, f.M, f.D, l.dy, pieces);
  FFN_TRY(Pack<T>(pieces, s));
  MmaArgs a = Launch(f.D);
  AddProduct(a, f.M, f.F, l.dy, l.wd).vec = Octs<T>(f.F, {f.gate, f.up});
  a.act = f.act, a.g = f.gate, a.u = f.up, a.h = l.h, a.dg = l.dg, a.du = l.du;
  FFN_TRY((Mma<T, kGrad, false, false>(a, l.part, s)));
  a = Launch(f.F);
  Product& dx = AddProduct(a, f.M, f.D, l.dg, l.wg);
  dx.A[1] = l.du.p, dx.B[1] = l.wu.p, a.nseg = 2;
  dx.o1 = f.dx, dx.vec = Octs<T>(f.D, {f.dx});
  FFN_TRY((Mma<T, kPlain, false, false>(a, l.part, s)));
  a = Launch(f.M);
  const Planes* left[3] = {&l.x, &l.x, &l.h};
  const Planes* right[3] = {&l.dg, &l.du, &l.dy};
  void* out[3] = {f.dwg, f.dwu, f.dwd};
  for (int i = 0; i < 3; ++i) {
    const size_t M = i == 2 ? f.F : f.D, N = i == 2 ? f.D : f.F;
    Product& q = AddProduct(a, M, N, *left[i], *right[i]);
    q.o1 = out[i], q.vec = Octs<T>(N, {out[i]});
  }
  return Mma<T, kPlain, true, true>(a, l.part, s);
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
