// k_join.hip -- what stands between two blocks, forward and backward, in f32 or
// bf16: the norm after a block, its gate, the scaled residual, and the norm
// before the next block, each part but the residual optional.
//
//   n = norm(o) w + b,  y = res x + gate n,  h = norm(y) w' + b'
//   backward, from dh and dy (the gradient that reaches y past h), with
//   ohat, yhat the normalised o and y, and norm'(d, vhat, r) = r (d - mean(d)
//   - vhat mean(d vhat)) (root mean square: without mean(d)):
//   t  = dy + norm'(dh w', yhat),  dx = res t,  do = norm'(t gate w, ohat)
//   dw' = sum of dh yhat, db' = sum of dh;  with S1 = sum of t ohat and
//   S0 = sum of t over the rows of one gate: dgate = w S1 + b S0,
//   dw = sum over gates of gate S1, db = of gate S0
//
// Bound by HBM: forward o and x in, y and h out, backward dh, dy, y and o in,
// dx and do out; apart, a norm, a product, an addition and another norm move
// twice that.  A row is held in registers throughout, kE elements a lane.  The
// forward's second norm takes y before its rounding to bf16.  Sums and
// statistics are f32.
//
// The vectors' gradients run down the columns: a workgroup takes a band of
// neighbouring rows, a lane keeps its columns, and S1 and S0 serve the gate and
// the norm's weight both.  Where a gate's rows are more than a band's, a band
// lies within one gate's rows and leaves its S1 and S0; where they are fewer, a
// band holds whole gates' rows and writes their dgate itself.  JoinFoldKernel
// adds the bands in order -- no atomics, the same bits every run.
// 8192 x 2048 bf16, root mean square, one gate, on MI355X: forward 25.7 us (5.2
// TB/s; a copy runs 5.1), backward 34 and the fold 4.7.
#include "rows.h"

namespace seeai {
namespace {

constexpr int kRsrcWord3 = 0x00020000;  // raw buffer, out-of-range reads give 0
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ u32x4 ReadBuffer(__amdgpu_buffer_rsrc_t rs, int byte) {
  return __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(rs, byte, 0, 0));
}
__device__ __forceinline__ __amdgpu_buffer_rsrc_t Buffer(const void* p, int bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, bytes, kRsrcWord3);
}

__device__ __forceinline__ float UniformF(float v) {
  return __int_as_float(__builtin_amdgcn_readfirstlane(__float_as_int(v)));
}

// A row of T over kTPR threads, 16 bytes an access: lane t's group i holds the
// kV columns from (i kTPR + t) kV on.  Rows on dwords (f32; bf16 of an even
// width) go through buffer ranges.  With a wave or more a row the range is
// exactly the row, its address a scalar: a dword past it reads as zero and is
// not stored, each dword by itself, so no access asks where the row ends.  With
// several rows a wave (kTPR 16 or 32) the range is the wave's rows, neighbours in
// memory, lanes past their row's columns point past it, and a row's last, short
// group is cut by hand.  Other bf16 rows (kOff) are read 16 bytes at a time from
// wherever they lie; the row's last, short group reads the row's last 16 bytes
// and is shifted into place, so its load, too, can run ahead of its use.
template <class T, int kTPR, int kE, bool kOff>
struct Row {
  static constexpr int kV = Io<T>::kV, kN = kE / kV, kSize = sizeof(T);
  static constexpr bool kNarrow = kTPR < kWave;
  u32x4 q[kN];
  static __device__ __forceinline__ int Col(int t, int i) { return (i * kTPR + t) * kV; }
  static constexpr int kPast = 0x40000000;  // past every range
  // The wave's rows from its first on, and where this lane's group i lies.
  static __device__ __forceinline__ size_t First(size_t r) {
    const size_t lane_row = (threadIdx.x % kWave) / kTPR;
    const size_t f = r - lane_row;
    return (static_cast<size_t>(Uniform(static_cast<int>(f >> 32))) << 32) |
           static_cast<uint32_t>(Uniform(static_cast<int>(f)));
  }
  static __device__ __forceinline__ int Byte(int t, int i, int cols) {
    const int c = Col(t, i), lane_row = (threadIdx.x % kWave) / kTPR;
    return c < cols ? (lane_row * cols + c) * kSize : kPast;
  }
  static __device__ __forceinline__ __amdgpu_buffer_rsrc_t Rows(const T* x, size_t r, size_t end, int cols) {
    const size_t f = First(r), left = f < end ? end - f : 0;
    const int n = left < kWave / kTPR ? static_cast<int>(left) : kWave / kTPR;
    return Buffer(x + f * cols, n * cols * kSize);
  }
  // Row r of x, zeros where it is not before `end`.
  __device__ __forceinline__ void Load(const T* x, size_t r, size_t end, int t, int cols) {
    const T* row = x + r * cols;
    const int here = r < end ? cols : 0;
    if constexpr (!kOff && kNarrow) {
      const auto rs = Rows(x, r, end, cols);
#pragma unroll
      for (int i = 0; i < kN; ++i) q[i] = ReadBuffer(rs, Byte(t, i, cols));
    } else if constexpr (!kOff) {
      const auto rs = Buffer(row, here * kSize);
#pragma unroll
      for (int i = 0; i < kN; ++i) q[i] = ReadBuffer(rs, Col(t, i) * kSize);
    } else if (here >= kV) {
#pragma unroll
      for (int i = 0; i < kN; ++i) {
        const int c = Col(t, i), last = here - kV;
        q[i] = *reinterpret_cast<const u32x4u*>(row + (c < last ? c : last));
      }
    } else {  // fewer columns than a group, the first lane's
#pragma unroll
      for (int i = 0; i < kN; ++i) q[i] = u32x4{0, 0, 0, 0};
      if (t == 0) {
#pragma unroll
        for (int c = 0; c < kV - 1; ++c)
          if (c < here) q[0][c / 2] |= static_cast<uint32_t>(row[c]) << (16 * (c % 2));
      }
    }
  }
  __device__ __forceinline__ void Get(int t, int cols, float (&v)[kE]) const {
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      u32x4 w = q[i];
      if constexpr (kOff) {
        const int by = cols >= kV ? Col(t, i) - (cols - kV) : 0;  // elements to shift out
        if (by & 4) w = u32x4{w[2], w[3], 0, 0};
        if (by & 2) w = u32x4{w[1], w[2], w[3], 0};
        if (by & 1)
          w = u32x4{__builtin_amdgcn_alignbit(w[1], w[0], 16), __builtin_amdgcn_alignbit(w[2], w[1], 16),
                    __builtin_amdgcn_alignbit(w[3], w[2], 16), w[3] >> 16};
        if (by >= kV) w = u32x4{0, 0, 0, 0};
        if (by <= 0) w = q[i];  // a group before the last
      }
      if constexpr (kSize == 4) {
#pragma unroll
        for (int k = 0; k < 4; ++k) v[i * kV + k] = __uint_as_float(w[k]);
      } else {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          v[i * kV + 2 * k] = __uint_as_float(w[k] << 16);
          v[i * kV + 2 * k + 1] = __uint_as_float(w[k] & 0xFFFF0000u);
        }
      }
      if constexpr (!kOff && kNarrow) {
#pragma unroll
        for (int k = 1; k < kV; ++k)
          if (Col(t, i) + k >= cols) v[i * kV + k] = 0.0f;
      }
    }
  }
  static __device__ __forceinline__ u32x4 Bits(const float* v) {
    if constexpr (kSize == 4)
      return u32x4{__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])};
    else
      return __builtin_bit_cast(u32x4, Io<uint16_t>::Pack(v));
  }
  static __device__ __forceinline__ void Store(T* x, size_t r, size_t end, int t, int cols, const float (&v)[kE]) {
    if constexpr (!kOff && kNarrow) {
      const auto rs = Rows(x, r, end, cols);
#pragma unroll
      for (int i = 0; i < kN; ++i) {
        const u32x4 w = Bits(v + i * kV);
        const int c = Col(t, i), byte = Byte(t, i, cols);
        if (c + kV <= cols) {
          __builtin_amdgcn_raw_buffer_store_b128(w, rs, byte, 0, 0);
        } else {
#pragma unroll
          for (int k = 0; k < 4; ++k)
            if (c + k * 4 / kSize < cols) __builtin_amdgcn_raw_buffer_store_b32(w[k], rs, byte + 4 * k, 0, 0);
        }
      }
      return;
    }
    if (r >= end) return;
    T* row = x + r * cols;
    if constexpr (!kOff) {
      const auto rs = Buffer(row, cols * kSize);
#pragma unroll
      for (int i = 0; i < kN; ++i)
        __builtin_amdgcn_raw_buffer_store_b128(Bits(v + i * kV), rs, Col(t, i) * kSize, 0, 0);
    } else {
#pragma unroll
      for (int i = 0; i < kN; ++i) {
        const int c = Col(t, i);
        const float* at = v + i * kV;
        if (c + kV <= cols) {
          Io<T>::StoreAny(row + c, at);
        } else {
#pragma unroll
          for (int k = 0; k < kV; ++k)
            if (c + k < cols) Io<T>::Put(row + c + k, at[k]);
        }
      }
    }
  }
};

// The row group of a thread: a scalar where a row has whole waves.
template <int kTPR>
__device__ __forceinline__ int RowGroup() {
  if constexpr (kTPR >= kWave) return Uniform(threadIdx.x / kTPR);
  else return threadIdx.x / kTPR;
}
template <int kTPR>
__device__ __forceinline__ float RowFloat(float v) {  // a value of a row
  if constexpr (kTPR >= kWave) return UniformF(v);
  else return v;
}

// The f32 vector at the same columns, zeros past it.
template <class T, int kTPR, int kE>
__device__ __forceinline__ void Vector(const float* w, int t, int cols, float (&v)[kE]) {
  const auto rs = Buffer(w, cols * 4);
#pragma unroll
  for (int e = 0; e < kE; e += 4) {
    const u32x4 x = ReadBuffer(rs, ColOf<T, kTPR, true>(t, e) * 4);
#pragma unroll
    for (int k = 0; k < 4; ++k) v[e + k] = __uint_as_float(x[k]);
  }
}

constexpr int FwdThreads(int tpr) { return tpr > 256 ? tpr : 256; }
// The backward's workgroup, and its bands: two workgroups a CU, whose turns of
// load, sum and store interleave.  us, against one of 1024 threads a CU (half the
// bands): 20000 x 200 bf16 with gates of 300 rows 25 and 35, 4000 x 4095 bf16 51
// and 54, 8192 x 2048 bf16 39 both, 3001 x 1023 f32 27 and 25.
constexpr int BwdThreads(int tpr) { return tpr > 512 ? tpr : 512; }

template <int kTPR>
__device__ __forceinline__ float LaneSum(float v) {
  if constexpr (kTPR >= kWave) {
    return LanesSum(v);
  } else {  // over 16 or 32 lanes, each of them gets it
    v = MoveAdd<0xB1>(v);   // the neighbour's
    v = MoveAdd<0x4E>(v);   // the neighbouring pair's
    v = MoveAdd<0x141>(v);  // the other four of eight
    v = MoveAdd<0x140>(v);  // the other eight of sixteen
    if constexpr (kTPR == 32) v += __shfl_xor(v, 16, kWave);
    return v;
  }
}
template <int kTPR>
__device__ __forceinline__ float RowSum1(float a, float* lds, int& turn) {
  a = LaneSum<kTPR>(a);
  if constexpr (kTPR > kWave) {
    constexpr int kWaves = kTPR / kWave;
    const int w = threadIdx.x / kWave, first = w / kWaves * kWaves;
    float* at = lds + 32 * turn;
    turn ^= 1;
    if (threadIdx.x % kWave == 0) at[w] = a;
    __syncthreads();
    a = 0.0f;
#pragma unroll
    for (int k = 0; k < kWaves; ++k) a += at[first + k];
  }
  return a;
}
// Two sums over the kTPR threads of each row; `lds` [2][2 x 16], used in turn,
// so that one barrier keeps a sum's reads from the next one's writes.
template <int kTPR>
__device__ __forceinline__ float2 RowSum2(float a, float b, float* lds, int& turn) {
  a = LaneSum<kTPR>(a), b = LaneSum<kTPR>(b);
  if constexpr (kTPR > kWave) {
    constexpr int kWaves = kTPR / kWave;
    const int w = threadIdx.x / kWave, first = w / kWaves * kWaves;
    float* at = lds + 32 * turn;
    turn ^= 1;
    if (threadIdx.x % kWave == 0) at[2 * w] = a, at[2 * w + 1] = b;
    __syncthreads();
    a = b = 0.0f;
#pragma unroll
    for (int k = 0; k < kWaves; ++k) a += at[2 * (first + k)], b += at[2 * (first + k) + 1];
  }
  return make_float2(a, b);
}

// v normalised in place; its mean and 1 / deviation.
template <class T, int kTPR, int kE>
__device__ __forceinline__ float2 Normalise(float (&v)[kE], int rms, int t, int cols, float inv, float eps,
                                            float* lds, int& turn) {
  float mu = 0.0f, sq = 0.0f;
  if (!rms) {
#pragma unroll
    for (int e = 0; e < kE; ++e) mu += v[e];
    mu = RowSum1<kTPR>(mu, lds, turn) * inv;
#pragma unroll
    for (int e = 0; e < kE; ++e) v[e] = ColOf<T, kTPR, true>(t, e) < cols ? v[e] - mu : 0.0f;
  }
#pragma unroll
  for (int e = 0; e < kE; ++e) sq += v[e] * v[e];
  const float rs = rsqrtf(RowSum1<kTPR>(sq, lds, turn) * inv + eps);
#pragma unroll
  for (int e = 0; e < kE; ++e) v[e] *= rs;
  return make_float2(mu, rs);
}

// v = v w + b (b null: without).
template <class T, int kTPR, int kE>
__device__ __forceinline__ void Scale(float (&v)[kE], const float* w, const float* b, int t, int cols) {
  float u[kE];
  Vector<T, kTPR, kE>(w, t, cols, u);
#pragma unroll
  for (int e = 0; e < kE; ++e) v[e] *= u[e];
  if (!b) return;
  Vector<T, kTPR, kE>(b, t, cols, u);
#pragma unroll
  for (int e = 0; e < kE; ++e) v[e] += u[e];
}

template <class T, int kTPR, int kE, bool kOff>
__global__ void __launch_bounds__(FwdThreads(kTPR))
JoinFwdKernel(JoinArgs a) {
  using R = Row<T, kTPR, kE, kOff>;
  __shared__ float lds[64];
  constexpr int kRows = FwdThreads(kTPR) / kTPR;
  const int t = threadIdx.x % kTPR, sub = RowGroup<kTPR>(), cols = static_cast<int>(a.cols);
  const float inv = 1.0f / static_cast<float>(cols);
  int turn = 0;
  // (the loop is uniform over the workgroup, its barriers too)
  for (size_t base = static_cast<size_t>(blockIdx.x) * kRows; base < a.rows;
       base += static_cast<size_t>(gridDim.x) * kRows) {
    const size_t r = base + sub;
    const bool in = r < a.rows;
    R ro, rx;
    ro.Load(static_cast<const T*>(a.o), r, a.rows, t, cols);
    rx.Load(static_cast<const T*>(a.x), r, a.rows, t, cols);
    float v[kE], x[kE];
    ro.Get(t, cols, v);
    float2 so = make_float2(0.0f, 0.0f), sy = so;
    if (a.post_w) {
      so = Normalise<T, kTPR, kE>(v, a.rms, t, cols, inv, a.eps, lds, turn);
      Scale<T, kTPR, kE>(v, a.post_w, a.post_b, t, cols);
    }
    if (a.gate) {
      const size_t g = (in ? r : 0) / a.gate_rows;
      if constexpr (kTPR >= kWave) {
        Scale<T, kTPR, kE>(v, a.gate + g * cols, nullptr, t, cols);
      } else {  // rows of one wave may differ in their gates
#pragma unroll
        for (int e = 0; e < kE; ++e) {
          const int c = ColOf<T, kTPR, true>(t, e);
          v[e] *= c < cols ? a.gate[g * cols + c] : 0.0f;
        }
      }
    }
    rx.Get(t, cols, x);
#pragma unroll
    for (int e = 0; e < kE; ++e) v[e] = a.res * x[e] + v[e];
    R::Store(static_cast<T*>(a.y), r, a.rows, t, cols, v);
    if (a.pre_w) {
      sy = Normalise<T, kTPR, kE>(v, a.rms, t, cols, inv, a.eps, lds, turn);
      Scale<T, kTPR, kE>(v, a.pre_w, a.pre_b, t, cols);
      R::Store(static_cast<T*>(a.h), r, a.rows, t, cols, v);
    }
    if (in && t == 0 && a.stats) {
      float* s = a.stats + 4 * r;
      s[0] = so.x, s[1] = so.y, s[2] = sy.x, s[3] = sy.y;
    }
  }
}

// How the rows are shared out: `bands` of `len` rows, `per` to a gate, or of
// `gates` whole gates' rows.
struct Plan {
  unsigned bands, per;
  size_t len, gates;
};
// A row's threads, for rows of `cols`.
int RowThreads(size_t cols) {
  return cols <= 128 ? 16 : cols <= 256 ? 32 : cols <= 512 ? 64 : cols <= 1024 ? 128 : cols <= 2048 ? 256 : cols <= 4096 ? 512 : 1024;
}
constexpr size_t kBands = 512;
Plan PlanOf(size_t rows, size_t cols, size_t gate_rows) {
  if (rows == 0) return {1, 1, 0, 0};  // sums of zero
  const int tpr = RowThreads(cols), threads = BwdThreads(tpr);
  const size_t slots = static_cast<size_t>(threads / tpr), most = threads > 512 ? kBands / 2 : kBands;
  const auto whole = [&](size_t n) { return (n + slots - 1) / slots * slots; };
  size_t len = whole((rows + most - 1) / most);
  const size_t gr = gate_rows == 0 || gate_rows > rows ? rows : gate_rows, groups = (rows + gr - 1) / gr;
  if (gr <= len) {
    const size_t k = len / gr;
    return {static_cast<unsigned>((groups + k - 1) / k), 1, k * gr, k};
  }
  const size_t per = (gr + len - 1) / len;
  len = whole((gr + per - 1) / per);
  return {static_cast<unsigned>(groups * per), static_cast<unsigned>(per), len, 0};
}

// bands' sums: [bands][4][cols]: dw', db', S1 and S0 (or dw and db where a
// band's gates are whole), or the gradients themselves where there is one band.
// A row's loads go out while the row before it is reduced (kAhead; not with 16
// elements a lane).  128 registers a lane, four waves a SIMD, are enough for bf16 rows
// on dwords of up to 8192 columns (one instance spills 12 bytes).  Root mean squares in f32 up to
// 256 columns and f32 layer norms spill 20 to 144 bytes a lane, some layer norms of bf16
// rows off dwords 28 to 60, and 16 elements a lane up to 324: such reloads wait behind
// the next row's loads.
template <class T, int kTPR, int kE, bool kOff, bool kRms>
__global__ void __launch_bounds__(BwdThreads(kTPR), 4)
JoinBwdKernel(JoinArgs a, Plan plan) {
  using R = Row<T, kTPR, kE, kOff>;
  constexpr int kThreads = BwdThreads(kTPR), kRows = kThreads / kTPR;
  constexpr bool kAhead = kE == 8;
  __shared__ float lds[64];
  // Element e of thread t at ((e / 4) kTPR + t) 4 + e % 4: w', and gate w.
  __shared__ float wpre[kTPR * kE], wpost[kTPR * kE];
  // Sums of the row groups' columns; over wpost, which is read no more by then,
  // where there is one group.
  __shared__ float groups[kRows > 1 ? kRows * kTPR * kE : 4];
  float* stage = kRows > 1 ? groups : wpost;
  const int t = threadIdx.x % kTPR, sub = RowGroup<kTPR>(), cols = static_cast<int>(a.cols);
  const auto slot = [&](int e) { return (e / 4 * kTPR + t) * 4 + e % 4; };
  const float inv = 1.0f / static_cast<float>(cols);
  const bool pre = a.pre_w != nullptr, post = a.post_w != nullptr, tail = post || a.gate;
  const size_t all = a.rows ? a.rows : 1, gr = !a.gate || a.gate_rows > all ? all : a.gate_rows;
  const bool whole = plan.gates > 0;  // whole gates in a band
  int turn = 0;
  // This band's rows.
  size_t first, last;
  if (whole) {
    first = blockIdx.x * plan.len, last = first + plan.len;
  } else {
    const unsigned g = blockIdx.x / plan.per, k = blockIdx.x % plan.per;
    first = g * gr + k * plan.len;
    last = first + plan.len < (g + 1) * gr ? first + plan.len : (g + 1) * gr;
  }
  if (last > a.rows) last = a.rows;
  // Column sums over the row groups, in order, a thread a column: `use(c, sum)`.
  auto join = [&](const auto& s, auto&& use) {
    __syncthreads();  // what the memory held has been read
#pragma unroll
    for (int e = 0; e < kE; e += 4)
      *reinterpret_cast<float4*>(stage + sub * (kTPR * kE) + ColOf<T, kTPR, true>(t, e)) =
          make_float4(s[e], s[e + 1], s[e + 2], s[e + 3]);
    __syncthreads();
    for (int c = threadIdx.x; c < cols; c += kThreads) {
      float sum = stage[c];
#pragma unroll
      for (int g = 1; g < kRows; ++g) sum += stage[g * (kTPR * kE) + c];
      use(c, sum);
    }
  };
  auto four = [&](const float* own, int e, float (&w)[4]) {  // from column e on
    const float4 q = *reinterpret_cast<const float4*>(own + slot(e));
    w[0] = q.x, w[1] = q.y, w[2] = q.z, w[3] = q.w;
  };
  float* part = a.part + static_cast<size_t>(blockIdx.x) * 4 * cols;
  const bool one = gridDim.x == 1;
  float pw[kE], pb[kRms ? 1 : kE];
#pragma unroll
  for (int e = 0; e < kE; ++e) pw[e] = 0.0f;
  if constexpr (!kRms) {
#pragma unroll
    for (int e = 0; e < kE; ++e) pb[e] = 0.0f;
  }
  R rh, ry, ro, rd;
  float4 st;
  size_t base = first;
  auto fetch = [&](size_t end) {  // (past the gate's last row: zeros, which add nothing)
    const size_t r = base + sub;
    rh.Load(static_cast<const T*>(a.dh), r, pre ? end : 0, t, cols);
    ry.Load(static_cast<const T*>(a.y), r, pre ? end : 0, t, cols);
    rd.Load(static_cast<const T*>(a.dy), r, a.dy ? end : 0, t, cols);
    ro.Load(static_cast<const T*>(a.o), r, tail ? end : 0, t, cols);
    st = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (r < end) {
      const float* s = a.stats + 4 * r;
      st = make_float4(s[0], s[1], s[2], s[3]);
    }
  };
  if (pre && sub == 0) {
    float v[kE];
    Vector<T, kTPR, kE>(a.pre_w, t, cols, v);
#pragma unroll
    for (int e = 0; e < kE; ++e) wpre[slot(e)] = v[e];
  }
  for (size_t at = first;;) {  // a gate's rows in this band (at least one turn: no rows, sums of zero)
    const size_t g = at / gr, end = whole && (g + 1) * gr < last ? (g + 1) * gr : last;
    const float* gate = a.gate && at < a.rows ? a.gate + g * cols : nullptr;
    base = at;
    if constexpr (kAhead) fetch(end);
    __syncthreads();  // (the gate before has been read)
    if (sub == 0) {
      float v[kE], u[kE];
#pragma unroll
      for (int e = 0; e < kE; ++e) v[e] = u[e] = 1.0f;
      if (post) Vector<T, kTPR, kE>(a.post_w, t, cols, v);
      if (gate) Vector<T, kTPR, kE>(gate, t, cols, u);
#pragma unroll
      for (int e = 0; e < kE; ++e) wpost[slot(e)] = v[e] * u[e];
    }
    __syncthreads();
    float s1[kE], s0[kRms ? 1 : kE];
#pragma unroll
    for (int e = 0; e < kE; ++e) s1[e] = 0.0f;
    if constexpr (!kRms) {
#pragma unroll
      for (int e = 0; e < kE; ++e) s0[e] = 0.0f;
    }
    while (base < end) {  // (uniform over the workgroup, its barriers too)
      const size_t r = base + sub;
      if constexpr (!kAhead) fetch(end);
      const float4 q = make_float4(RowFloat<kTPR>(st.x), RowFloat<kTPR>(st.y), RowFloat<kTPR>(st.z),
                                   RowFloat<kTPR>(st.w));
      float d[kE], v[kE];
      const R md = rd, mo = ro;
      rh.Get(t, cols, d);
      ry.Get(t, cols, v);
      base += kRows;
      if constexpr (kAhead) fetch(end);
      if (pre) {
        float c1 = 0.0f, c2 = 0.0f;
        const float mu = kRms ? 0.0f : q.z;
#pragma unroll
        for (int e = 0; e < kE; e += 4) {  // (columns past the row: d = 0, so no term)
          float ww[4];
          four(wpre, e, ww);
#pragma unroll
          for (int i = e; i < e + 4; ++i) {
            v[i] = (v[i] - mu) * q.w;
            pw[i] += d[i] * v[i];
            if constexpr (!kRms) pb[i] += d[i];
            d[i] *= ww[i - e];
            c1 += d[i];
            c2 += d[i] * v[i];
          }
        }
        const float2 c = RowSum2<kTPR>(c1, c2, lds, turn);
        c1 = kRms ? 0.0f : c.x * inv, c2 = c.y * inv;
#pragma unroll
        for (int e = 0; e < kE; ++e) {
          d[e] = q.w * (d[e] - c1 - v[e] * c2);
          // (a layer norm's columns past the row would hold its mean's part)
          if (!kRms && ColOf<T, kTPR, true>(t, e) >= cols) d[e] = 0.0f;
        }
      }
      md.Get(t, cols, v);
#pragma unroll
      for (int e = 0; e < kE; ++e) d[e] += v[e];
#pragma unroll
      for (int e = 0; e < kE; ++e) v[e] = a.res * d[e];
      R::Store(static_cast<T*>(a.dx), r, end, t, cols, v);
      if (tail) {
        mo.Get(t, cols, v);
        if (post) {
          const float mu = kRms ? 0.0f : q.x;
#pragma unroll
          for (int e = 0; e < kE; ++e) v[e] = (v[e] - mu) * q.y;
        }
        float c1 = 0.0f, c2 = 0.0f;
#pragma unroll
        for (int e = 0; e < kE; e += 4) {
          float ww[4];
          four(wpost, e, ww);
#pragma unroll
          for (int i = e; i < e + 4; ++i) {
            s1[i] += d[i] * v[i];
            if constexpr (!kRms) s0[i] += d[i];
            d[i] *= ww[i - e];
            c1 += d[i];
            c2 += d[i] * v[i];
          }
        }
        if (post) {
          const float2 c = RowSum2<kTPR>(c1, c2, lds, turn);
          c1 = kRms ? 0.0f : c.x * inv, c2 = c.y * inv;
#pragma unroll
          for (int e = 0; e < kE; ++e) d[e] = q.y * (d[e] - c1 - v[e] * c2);
        }
      }
      R::Store(static_cast<T*>(a.d_o), r, end, t, cols, d);
    }
    if (tail) {
      const bool mine = a.dgate && (whole || plan.per == 1) && at < a.rows;  // all of the gate's rows are here
      const bool weighted = whole || one;
      float* o1 = one ? a.dpost_w : part + 2 * cols;
      float* o0 = one ? a.dpost_b : part + 3 * cols;
      join(s1, [&](int c, float sum) {
        if (mine) a.dgate[g * cols + c] = post ? a.post_w[c] * sum : sum;
        if (!weighted) o1[c] = sum;
        else if (post) o1[c] = (gate ? gate[c] : 1.0f) * sum + (at == first ? 0.0f : o1[c]);
      });
      if constexpr (!kRms) {
        if (a.post_b) {
          join(s0, [&](int c, float sum) {
            if (mine) a.dgate[g * cols + c] += a.post_b[c] * sum;
            if (!weighted) o0[c] = sum;
            else if (a.dpost_b) o0[c] = (gate ? gate[c] : 1.0f) * sum + (at == first ? 0.0f : o0[c]);
          });
        }
      }
    }
    at = end;
    if (!whole || at >= last) break;
  }
  if (pre) {
    float* o1 = one ? a.dpre_w : part;
    join(pw, [&](int c, float sum) { o1[c] = sum; });
    if constexpr (!kRms) {
      if (a.dpre_b) {
        float* o0 = one ? a.dpre_b : part + cols;
        join(pb, [&](int c, float sum) { o0[c] = sum; });
      }
    }
  }
}

// The bands' sums, 32 columns a workgroup, 32 threads a column, each over every
// 32nd band, joined in order.  blockIdx.y, of what there is: the norm before the
// next block's gradients; the norm after the block's, and the gate's where there
// is one for all rows; every other gate's.
constexpr int kFoldCols = 32, kFoldParts = 32;
__global__ void __launch_bounds__(kFoldCols * kFoldParts)
JoinFoldKernel(JoinArgs a, Plan plan, unsigned gates) {
  __shared__ float lds[2][kFoldParts][kFoldCols + 1];
  const int i = threadIdx.x % kFoldCols, k = threadIdx.x / kFoldCols;
  const size_t cols = a.cols, c = static_cast<size_t>(blockIdx.x) * kFoldCols + i;
  unsigned job = blockIdx.y + (a.pre_w ? 0 : 1);
  if (job > 0 && !a.post_w && !(a.dgate && gates == 1)) ++job;
  const unsigned g = job - 2;  // from job 2 on
  const unsigned b0 = job < 2 ? 0 : g * plan.per, b1 = job < 2 ? plan.bands : b0 + plan.per;
  // A band's sums count as its gate times them where its gate is one of several.
  const bool weigh = job == 1 && a.gate && plan.gates == 0 && gates > 1;
  const float* row = a.part + (job == 0 ? 0 : 2) * cols + c;
  const bool both = !a.rms && (job == 0 ? a.dpre_b != nullptr : a.post_b != nullptr);
  float s = 0.0f, z = 0.0f;
  if (c < cols) {
#pragma unroll 8
    for (unsigned b = b0 + k; b < b1; b += kFoldParts) {
      const size_t off = static_cast<size_t>(b) * 4 * cols;
      float v = row[off], u = both ? row[off + cols] : 0.0f;
      if (weigh) {
        const float by = a.gate[b / plan.per * cols + c];
        v *= by, u *= by;
      }
      s += v, z += u;
    }
  }
  lds[0][k][i] = s, lds[1][k][i] = z;
  __syncthreads();
  // Eight threads a column join four parts each, then one the eight.
  if (k < 8) {
#pragma unroll
    for (int j = 8; j < kFoldParts; j += 8) s += lds[0][k + j][i], z += lds[1][k + j][i];
    lds[0][k][i] = s, lds[1][k][i] = z;
  }
  __syncthreads();
  if (k != 0 || c >= cols) return;
#pragma unroll
  for (int j = 1; j < 8; ++j) s += lds[0][j][i], z += lds[1][j][i];
  if (job == 0) {
    a.dpre_w[c] = s;
    if (a.dpre_b) a.dpre_b[c] = z;
    return;
  }
  const float gate = a.gate && gates == 1 && plan.gates == 0 ? a.gate[c] : 1.0f;
  if (job == 1 && a.post_w) {
    a.dpost_w[c] = gate * s;
    if (a.dpost_b) a.dpost_b[c] = gate * z;
  }
  if (a.dgate && (job > 1 || (gates == 1 && plan.gates == 0)))
    a.dgate[(job > 1 ? g : 0) * cols + c] = a.post_w ? a.post_w[c] * s + (a.post_b ? a.post_b[c] * z : 0.0f) : s;
}

dim3 Grid(size_t groups) {  // a launch's workgroups (the kernels walk the rows past them)
  return dim3(static_cast<unsigned>(groups < (1u << 20) ? groups : 1u << 20));
}

template <class T, int kTPR, int kE, bool kOff>
hipError_t RunFwd(const JoinArgs& a, hipStream_t s) {
  constexpr int kThreads = FwdThreads(kTPR), kRows = kThreads / kTPR;
  hipLaunchKernelGGL((JoinFwdKernel<T, kTPR, kE, kOff>), Grid((a.rows + kRows - 1) / kRows), dim3(kThreads), 0, s, a);
  return hipGetLastError();
}

template <class T, int kTPR, int kE, bool kOff>
hipError_t RunBwd(const JoinArgs& a, hipStream_t s) {
  const Plan plan = PlanOf(a.rows, a.cols, a.gate ? a.gate_rows : 0);
  if (a.rms)
    hipLaunchKernelGGL((JoinBwdKernel<T, kTPR, kE, kOff, true>), dim3(plan.bands), dim3(BwdThreads(kTPR)), 0, s, a, plan);
  else
    hipLaunchKernelGGL((JoinBwdKernel<T, kTPR, kE, kOff, false>), dim3(plan.bands), dim3(BwdThreads(kTPR)), 0, s, a, plan);
  if (hipError_t e = hipGetLastError(); e != hipSuccess || plan.bands == 1) return e;
  // Gates whose rows lie in several bands.
  const unsigned gates = a.gate && plan.gates == 0 ? plan.bands / plan.per : 0;
  const unsigned shared = a.dgate && plan.per > 1 ? gates : 0;
  const unsigned jobs = (a.pre_w ? 1 : 0) + (a.post_w || shared == 1 ? 1 : 0) + (shared > 1 ? shared : 0);
  if (jobs == 0) return hipSuccess;
  hipLaunchKernelGGL(JoinFoldKernel,
                     dim3(static_cast<unsigned>((a.cols + kFoldCols - 1) / kFoldCols), jobs),
                     dim3(kFoldCols * kFoldParts), 0, s, a, plan, gates);
  return hipGetLastError();
}

// Past 512 columns the forward holds 16 elements a lane: fewer waves meet in a
// row's sums and share its vectors' loads (8 a lane and 16, bf16, us: layer norms
// 2000 x 8192 35 and 28, 4000 x 4095 34 and 33, 8000 x 2048 26 both; 32768 x 128,
// half the lanes without columns, 7.8 and 9.9).  From 257 to 512 columns a wave has a
// row of 8 a lane: as two rows of 16 a lane each gathers its own gate (root mean
// square, one gate, 16000 x 512: bf16 14 and 25, f32 22 and 25; without a gate 32000 x
// 512 bf16 23 both, f32 41 and 45, f32 layer norms 52 and 51).
template <class T, bool kOff>
hipError_t Forward(const JoinArgs& a, hipStream_t s) {
  if (a.cols <= 128) return RunFwd<T, 16, 8, kOff>(a, s);
  if (a.cols <= 256) return RunFwd<T, 32, 8, kOff>(a, s);
  if (a.cols <= 512) return RunFwd<T, 64, 8, kOff>(a, s);
  if (a.cols <= 1024) return RunFwd<T, 64, 16, kOff>(a, s);
  if (a.cols <= 2048) return RunFwd<T, 128, 16, kOff>(a, s);
  if (a.cols <= 4096) return RunFwd<T, 256, 16, kOff>(a, s);
  if (a.cols <= 8192) return RunFwd<T, 512, 16, kOff>(a, s);
  return RunFwd<T, 1024, 16, kOff>(a, s);
}

template <class T, bool kOff>
hipError_t Backward(const JoinArgs& a, hipStream_t s) {
  switch (RowThreads(a.cols)) {
    case 16: return RunBwd<T, 16, 8, kOff>(a, s);
    case 32: return RunBwd<T, 32, 8, kOff>(a, s);
    case 64: return RunBwd<T, 64, 8, kOff>(a, s);
    case 128: return RunBwd<T, 128, 8, kOff>(a, s);
    case 256: return RunBwd<T, 256, 8, kOff>(a, s);
    case 512: return RunBwd<T, 512, 8, kOff>(a, s);
    default: return a.cols <= 8192 ? RunBwd<T, 1024, 8, kOff>(a, s) : RunBwd<T, 1024, 16, kOff>(a, s);
  }
}

template <class T, bool kOff>
hipError_t Pick(const JoinArgs& a, bool bwd, hipStream_t s) {
  return bwd ? Backward<T, kOff>(a, s) : Forward<T, kOff>(a, s);
}

hipError_t Dispatch(int bf16, const JoinArgs& a, bool bwd, hipStream_t s) {
  if (!bf16) return Pick<float, false>(a, bwd, s);
  uintptr_t at = 2 * a.cols;  // every row on a dword
  for (const void* p : {a.o, a.x, static_cast<const void*>(a.y), static_cast<const void*>(a.h), a.dh, a.dy,
                        static_cast<const void*>(a.dx), static_cast<const void*>(a.d_o)})
    at |= reinterpret_cast<uintptr_t>(p);
  return at & 3 ? Pick<uint16_t, true>(a, bwd, s) : Pick<uint16_t, false>(a, bwd, s);
}

}  // namespace

size_t JoinWorkspaceBytes(size_t rows, size_t cols, size_t gate_rows) {
  const Plan p = PlanOf(rows, cols, gate_rows);
  return p.bands > 1 ? p.bands * 4 * cols * sizeof(float) : 0;
}

hipError_t LaunchJoinFwd(int bf16, const JoinArgs& a, hipStream_t s) {
  if (a.rows == 0) return hipSuccess;
  return Dispatch(bf16, a, false, s);
}

hipError_t LaunchJoinBwd(int bf16, const JoinArgs& a, hipStream_t s) {
  return Dispatch(bf16, a, true, s);
}

}  // namespace seeai
