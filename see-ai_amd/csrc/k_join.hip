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
#include "rows.h"

namespace seeai {
namespace {

constexpr int FwdThreads(int tpr) { return tpr > 256 ? tpr : 256; }
constexpr int BwdThreads(int tpr) { return tpr > 512 ? tpr : 512; }

// v normalised in place; its mean and 1 / deviation.
template <class T, int kTPR, int kE, bool kVec>
__device__ __forceinline__ float2 Normalise(float (&v)[kE], int rms, int t, int cols, float eps,
                                            float* lds) {
  float mu[1] = {0.0f}, sq[1] = {0.0f};
  if (!rms) {
#pragma unroll
    for (int e = 0; e < kE; ++e) mu[0] += v[e];
    RowSum<kTPR>(mu, lds);
    mu[0] /= static_cast<float>(cols);
#pragma unroll
    for (int e = 0; e < kE; ++e) v[e] = ColOf<T, kTPR, kVec>(t, e) < cols ? v[e] - mu[0] : 0.0f;
  }
#pragma unroll
  for (int e = 0; e < kE; ++e) sq[0] += v[e] * v[e];
  RowSum<kTPR>(sq, lds);
  const float rs = 1.0f / sqrtf(sq[0] / static_cast<float>(cols) + eps);
#pragma unroll
  for (int e = 0; e < kE; ++e) v[e] *= rs;
  return make_float2(mu[0], rs);
}

// v = v w + b (b null: without).
template <class T, int kTPR, int kE, bool kVec, bool kAny>
__device__ __forceinline__ void Scale(float (&v)[kE], const float* w, const float* b, int t, int cols) {
  float u[kE];
  LoadVec<T, kTPR, kE, kVec, kAny>(w, t, cols, u);
#pragma unroll
  for (int e = 0; e < kE; ++e) v[e] *= u[e];
  if (!b) return;
  LoadVec<T, kTPR, kE, kVec, kAny>(b, t, cols, u);
#pragma unroll
  for (int e = 0; e < kE; ++e) v[e] += u[e];
}

template <class T, int kTPR, int kE, bool kVec, bool kAny>
__global__ void __launch_bounds__(FwdThreads(kTPR))
JoinFwdKernel(JoinArgs a) {
  __shared__ float lds[16];
  constexpr int kRows = FwdThreads(kTPR) / kTPR;
  const int t = threadIdx.x % kTPR, cols = static_cast<int>(a.cols);
  // (the loop is uniform over the workgroup, its barriers too)
  for (size_t base = static_cast<size_t>(blockIdx.x) * kRows; base < a.rows;
       base += static_cast<size_t>(gridDim.x) * kRows) {
    const size_t r = base + threadIdx.x / kTPR;
    const bool in = r < a.rows;
    const int here = in ? cols : 0;
    float v[kE], x[kE];
    LoadRow<T, kTPR, kE, kVec, kAny>(static_cast<const T*>(a.o) + r * cols, t, here, v);
    LoadRow<T, kTPR, kE, kVec, kAny>(static_cast<const T*>(a.x) + r * cols, t, here, x);
    float2 so = make_float2(0.0f, 0.0f), sy = so;
    if (a.post_w) {
      so = Normalise<T, kTPR, kE, kVec>(v, a.rms, t, cols, a.eps, lds);
      Scale<T, kTPR, kE, kVec, kAny>(v, a.post_w, a.post_b, t, cols);
    }
    if (a.gate) Scale<T, kTPR, kE, kVec, kAny>(v, a.gate + (in ? r : 0) / a.gate_rows * cols, nullptr, t, cols);
#pragma unroll
    for (int e = 0; e < kE; ++e) v[e] = a.res * x[e] + v[e];
    if (in) StoreRow<T, kTPR, kE, kVec, kAny>(static_cast<T*>(a.y) + r * cols, t, cols, v);
    if (a.pre_w) {
      sy = Normalise<T, kTPR, kE, kVec>(v, a.rms, t, cols, a.eps, lds);
      Scale<T, kTPR, kE, kVec, kAny>(v, a.pre_w, a.pre_b, t, cols);
      if (in) StoreRow<T, kTPR, kE, kVec, kAny>(static_cast<T*>(a.h) + r * cols, t, cols, v);
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
  size_t bands, len, per, gates;
};
// A row's threads, for rows of `cols`.
int RowThreads(size_t cols) {
  return cols <= 512 ? 64 : cols <= 1024 ? 128 : cols <= 2048 ? 256 : cols <= 4096 ? 512 : 1024;
}
constexpr size_t kBands = 512;
Plan PlanOf(size_t rows, size_t cols, size_t gate_rows) {
  if (rows == 0) return {1, 0, 1, 0};  // sums of zero
  const int tpr = RowThreads(cols), threads = BwdThreads(tpr);
  const size_t slots = static_cast<size_t>(threads / tpr), turns = (rows + slots - 1) / slots;
  const size_t most = threads > 512 || turns < 4 * kBands ? kBands / 2 : kBands;
  const auto whole = [&](size_t n) { return (n + slots - 1) / slots * slots; };
  size_t len = whole((rows + most - 1) / most);
  const size_t gr = gate_rows == 0 || gate_rows > rows ? rows : gate_rows, groups = (rows + gr - 1) / gr;
  if (gr < len) {
    const size_t k = len / gr;
    return {(groups + k - 1) / k, k * gr, 1, k};
  }
  const size_t per = (gr + len - 1) / len;
  len = whole((gr + per - 1) / per);
  return {groups * per, len, per, 0};
}

// bands' sums: [bands][4][cols]: dw', db', S1 and S0 (or dw and db where a
// band's gates are whole), or the gradients themselves where there is one band.
template <class T, int kTPR, int kE, bool kVec>
__global__ void __launch_bounds__(BwdThreads(kTPR), BwdThreads(kTPR) / 256)
JoinBwdKernel(JoinArgs a, Plan plan) {
  constexpr int kRows = BwdThreads(kTPR) / kTPR;
  __shared__ float lds[32];
  __shared__ float own[kRows > 1 ? kTPR * kE : 4];  // element e of thread t at ((e / 4) kTPR + t) 4 + e % 4
  const int t = threadIdx.x % kTPR, sub = threadIdx.x / kTPR, cols = static_cast<int>(a.cols);
  const float inv = 1.0f / static_cast<float>(cols);
  const bool pre = a.pre_w != nullptr, post = a.post_w != nullptr;
  const size_t all = a.rows ? a.rows : 1, gr = !a.gate || a.gate_rows > all ? all : a.gate_rows;
  const bool whole = plan.gates > 0;  // whole gates in a band
  // This band's rows.
  size_t first, last;
  if (whole) {
    first = blockIdx.x * plan.len, last = first + plan.len;
  } else {
    const size_t g = blockIdx.x / plan.per, k = blockIdx.x % plan.per;
    first = g * gr + k * plan.len;
    last = first + plan.len < (g + 1) * gr ? first + plan.len : (g + 1) * gr;
  }
  if (last > a.rows) last = a.rows;
  // The row groups' sums add up in order; the last group holds them.
  auto join = [&](float (&s)[kE]) {
    if constexpr (kRows > 1) {
      for (int g = 0; g < kRows; ++g) {
        __syncthreads();
        if (sub == g) {
#pragma unroll
          for (int e = 0; e < kE; ++e) {
            float* at = own + (e / 4 * kTPR + t) * 4 + e % 4;
            if (g > 0) s[e] = *at + s[e];
            *at = s[e];
          }
        }
      }
    }
  };
  float* part = a.part + static_cast<size_t>(blockIdx.x) * 4 * cols;
  const bool one = gridDim.x == 1;
  float pw[kE], pb[kE];
#pragma unroll
  for (int e = 0; e < kE; ++e) pw[e] = pb[e] = 0.0f;
  for (size_t at = first;;) {  // a gate's rows in this band (at least one turn: no rows, sums of zero)
    const size_t g = at / gr, end = whole && (g + 1) * gr < last ? (g + 1) * gr : last;
    const float* gate = a.gate && at < a.rows ? a.gate + g * cols : nullptr;
    float s1[kE], s0[kE];
#pragma unroll
    for (int e = 0; e < kE; ++e) s1[e] = s0[e] = 0.0f;
    for (size_t base = at; base < end; base += kRows) {  // (uniform over the workgroup, its barriers too)
      const size_t r = base + sub;
      const bool in = r < end;
      const int here = in ? cols : 0;
      const size_t off = r * cols;
      float d[kE], v[kE], w[kE];
      float4 st = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      if (in) {
        const float* s = a.stats + 4 * r;
        st = make_float4(s[0], s[1], s[2], s[3]);
      }
#pragma unroll
      for (int e = 0; e < kE; ++e) d[e] = 0.0f;
      if (pre) {
        float s[2] = {0.0f, 0.0f};
        LoadRow<T, kTPR, kE, kVec>(static_cast<const T*>(a.dh) + off, t, here, d);
        LoadRow<T, kTPR, kE, kVec>(static_cast<const T*>(a.y) + off, t, here, v);
        LoadVec<T, kTPR, kE, kVec>(a.pre_w, t, cols, w);
        const float mu = a.rms ? 0.0f : st.z;
#pragma unroll
        for (int e = 0; e < kE; ++e) {  // (columns past the row: d = 0, so no term)
          v[e] = (v[e] - mu) * st.w;
          pw[e] += d[e] * v[e];
          pb[e] += d[e];
          d[e] *= w[e];
          s[0] += d[e];
          s[1] += d[e] * v[e];
        }
        RowSum<kTPR>(s, lds);
        const float c1 = a.rms ? 0.0f : s[0] * inv, c2 = s[1] * inv;
#pragma unroll
        for (int e = 0; e < kE; ++e) d[e] = ColOf<T, kTPR, kVec>(t, e) < here ? st.w * (d[e] - c1 - v[e] * c2) : 0.0f;
      }
      if (a.dy) {
        LoadRow<T, kTPR, kE, kVec>(static_cast<const T*>(a.dy) + off, t, here, v);
#pragma unroll
        for (int e = 0; e < kE; ++e) d[e] += v[e];
      }
#pragma unroll
      for (int e = 0; e < kE; ++e) v[e] = a.res * d[e];
      if (in) StoreRow<T, kTPR, kE, kVec>(static_cast<T*>(a.dx) + off, t, cols, v);
      if (post || gate) {
        LoadRow<T, kTPR, kE, kVec>(static_cast<const T*>(a.o) + off, t, here, v);
        if (post) {
          const float mu = a.rms ? 0.0f : st.x;
#pragma unroll
          for (int e = 0; e < kE; ++e) v[e] = (v[e] - mu) * st.y;
        }
#pragma unroll
        for (int e = 0; e < kE; ++e) s1[e] += d[e] * v[e], s0[e] += d[e];
      }
      if (gate) {
        LoadVec<T, kTPR, kE, kVec>(gate, t, cols, w);
#pragma unroll
        for (int e = 0; e < kE; ++e) d[e] *= w[e];
      }
      if (post) {
        float s[2] = {0.0f, 0.0f};
        LoadVec<T, kTPR, kE, kVec>(a.post_w, t, cols, w);
#pragma unroll
        for (int e = 0; e < kE; ++e) {
          d[e] *= w[e];
          s[0] += d[e];
          s[1] += d[e] * v[e];
        }
        RowSum<kTPR>(s, lds);
        const float c1 = a.rms ? 0.0f : s[0] * inv, c2 = s[1] * inv;
#pragma unroll
        for (int e = 0; e < kE; ++e) d[e] = st.y * (d[e] - c1 - v[e] * c2);
      }
      if (in) StoreRow<T, kTPR, kE, kVec>(static_cast<T*>(a.d_o) + off, t, cols, d);
    }
    if (post || gate) {
      join(s1);
      join(s0);
      if (sub == kRows - 1) {
        const bool mine = whole || plan.per == 1;  // all of the gate's rows
#pragma unroll
        for (int e = 0; e < kE; ++e) {
          const int c = ColOf<T, kTPR, kVec>(t, e);
          if (c >= cols) continue;
          if (a.dgate && mine && at < a.rows)
            a.dgate[g * cols + c] = post ? a.post_w[c] * s1[e] + (a.post_b ? a.post_b[c] * s0[e] : 0.0f) : s1[e];
          if (whole || one) {
            const float by = gate ? gate[c] : 1.0f;
            float* ow = one ? a.dpost_w : part + 2 * cols;
            float* ob = one ? a.dpost_b : part + 3 * cols;
            if (post) ow[c] = by * s1[e] + (at == first ? 0.0f : ow[c]);
            if (post && a.dpost_b) ob[c] = by * s0[e] + (at == first ? 0.0f : ob[c]);
          } else {
            part[2 * cols + c] = s1[e];
            part[3 * cols + c] = s0[e];
          }
        }
      }
    }
    at = end;
    if (!whole || at >= last) break;
  }
  if (pre) {
    join(pw);
    join(pb);
    if (sub == kRows - 1) {
#pragma unroll
      for (int e = 0; e < kE; ++e) {
        const int c = ColOf<T, kTPR, kVec>(t, e);
        if (c >= cols) continue;
        (one ? a.dpre_w : part)[c] = pw[e];
        if (a.dpre_b) (one ? a.dpre_b : part + cols)[c] = pb[e];
      }
    }
  }
}

// The bands' sums, 32 columns a workgroup, eight threads a column, each over
// every eighth band, joined in order.  blockIdx.y: 0 dw', 1 db', 2 dw, 3 db,
// 4 + g gate g.
constexpr int kFoldCols = 32, kFoldParts = 8;
__global__ void __launch_bounds__(kFoldCols * kFoldParts)
JoinFoldKernel(JoinArgs a, Plan plan) {
  __shared__ float lds[2][kFoldParts][kFoldCols];
  const int i = threadIdx.x % kFoldCols, k = threadIdx.x / kFoldCols;
  const size_t cols = a.cols, c = static_cast<size_t>(blockIdx.x) * kFoldCols + i;
  const unsigned job = blockIdx.y;
  float* out = job == 0 ? a.dpre_w : job == 1 ? a.dpre_b : job == 2 ? a.dpost_w : job == 3 ? a.dpost_b
                                                                              : a.dgate;
  if (!out) return;  // (uniform)
  const bool by_gate = (job == 2 || job == 3) && a.gate && plan.gates == 0;
  const size_t b0 = job >= 4 ? (job - 4) * plan.per : 0, b1 = job >= 4 ? b0 + plan.per : plan.bands;
  const float* row = a.part + (job >= 4 ? 2 : job) * cols + c;
  float s = 0.0f, s0 = 0.0f;
  if (c < cols) {
#pragma unroll 8
    for (size_t b = b0 + k; b < b1; b += kFoldParts) {
      const float v = row[b * 4 * cols];
      s += by_gate ? a.gate[b / plan.per * cols + c] * v : v;
      if (job >= 4 && a.post_b) s0 += row[(b * 4 + 1) * cols];
    }
  }
  lds[0][k][i] = s, lds[1][k][i] = s0;
  __syncthreads();
  if (k != 0 || c >= cols) return;
#pragma unroll
  for (int j = 1; j < kFoldParts; ++j) s += lds[0][j][i], s0 += lds[1][j][i];
  if (job < 4) {
    out[c] = s;
  } else {
    out[(job - 4) * cols + c] = a.post_w ? a.post_w[c] * s + (a.post_b ? a.post_b[c] * s0 : 0.0f) : s;
  }
}

dim3 Grid(size_t groups) {  // a launch's workgroups (the kernels walk the rows past them)
  return dim3(static_cast<unsigned>(groups < (1u << 20) ? groups : 1u << 20));
}

template <class T, int kTPR, int kE, bool kVec, bool kAny>
hipError_t Run(const JoinArgs& a, bool bwd, hipStream_t s) {
  if (kAny || !bwd) {  // (kAny: Dispatch asks for the forward alone)
    constexpr int kThreads = FwdThreads(kTPR), kRows = kThreads / kTPR;
    hipLaunchKernelGGL((JoinFwdKernel<T, kTPR, kE, kVec, kAny>), Grid((a.rows + kRows - 1) / kRows),
                       dim3(kThreads), 0, s, a);
    return hipGetLastError();
  }
  const Plan plan = PlanOf(a.rows, a.cols, a.gate ? a.gate_rows : 0);
  hipLaunchKernelGGL((JoinBwdKernel<T, kTPR, kE, kVec>), dim3(static_cast<unsigned>(plan.bands)),
                     dim3(BwdThreads(kTPR)), 0, s, a, plan);
  if (hipError_t e = hipGetLastError(); e != hipSuccess || plan.bands == 1) return e;
  if (!a.pre_w && !a.post_w && !(a.dgate && plan.per > 1)) return hipSuccess;
  const size_t gates = a.dgate && plan.per > 1 ? plan.bands / plan.per : 0;
  hipLaunchKernelGGL(JoinFoldKernel,
                     dim3(static_cast<unsigned>((a.cols + kFoldCols - 1) / kFoldCols),
                          static_cast<unsigned>(4 + gates)),
                     dim3(kFoldCols * kFoldParts), 0, s, a, plan);
  return hipGetLastError();
}

template <class T, bool kVec, bool kAny>
hipError_t Pick(const JoinArgs& a, bool bwd, hipStream_t s) {
  switch (RowThreads(a.cols)) {
    case 64: return Run<T, 64, 8, kVec, kAny>(a, bwd, s);
    case 128: return Run<T, 128, 8, kVec, kAny>(a, bwd, s);
    case 256: return Run<T, 256, 8, kVec, kAny>(a, bwd, s);
    case 512: return Run<T, 512, 8, kVec, kAny>(a, bwd, s);
    default:
      return a.cols <= 8192 ? Run<T, 1024, 8, kVec, kAny>(a, bwd, s) : Run<T, 1024, 16, kVec, kAny>(a, bwd, s);
  }
}

template <class T>
hipError_t Dispatch(const JoinArgs& a, bool bwd, hipStream_t s) {
  // 16-byte accesses where every row and vector begins on 16 bytes.
  uintptr_t at = 0;
  for (const void* p : {a.o, a.x, static_cast<const void*>(a.post_w), static_cast<const void*>(a.post_b),
                        static_cast<const void*>(a.gate), static_cast<const void*>(a.pre_w),
                        static_cast<const void*>(a.pre_b), static_cast<const void*>(a.y),
                        static_cast<const void*>(a.h), a.dh, a.dy, static_cast<const void*>(a.dx),
                        static_cast<const void*>(a.d_o)})
    at |= reinterpret_cast<uintptr_t>(p);
  if (a.cols % Io<T>::kV == 0 && (at & 15) == 0) return Pick<T, true, false>(a, bwd, s);
  if (!bwd && a.cols > (sizeof(T) == 2 ? 256 : 2048)) return Pick<T, true, true>(a, bwd, s);
  return Pick<T, false, false>(a, bwd, s);
}

}  // namespace

size_t JoinWorkspaceBytes(size_t rows, size_t cols, size_t gate_rows) {
  const Plan p = PlanOf(rows, cols, gate_rows);
  return p.bands > 1 ? p.bands * 4 * cols * sizeof(float) : 0;
}

hipError_t LaunchJoinFwd(int bf16, const JoinArgs& a, hipStream_t s) {
  if (a.rows == 0) return hipSuccess;
  return bf16 ? Dispatch<uint16_t>(a, false, s) : Dispatch<float>(a, false, s);
}

hipError_t LaunchJoinBwd(int bf16, const JoinArgs& a, hipStream_t s) {
  return bf16 ? Dispatch<uint16_t>(a, true, s) : Dispatch<float>(a, true, s);
}

}  // namespace seeai
