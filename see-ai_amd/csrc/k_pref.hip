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
// A row's label stands apart from its other logits: where it is nearly sure, its
// log-probability and its gradient are as small as the others' share of the sum and
// come from that share, not from differences of numbers near 1.  Setting it apart
// costs rows of one wave 3 to 5 % (16384 x 1000 bf16 log-probabilities 11.6 and 12.2
// us), large ones nothing or 1 %.
// Everything between is f32; sums along a row past its groups of 16 bytes, a
// log-probability before its one rounding, sums over rows and the pairs' terms are f64.
// 8192 x 32000 bf16 with 70 % of the rows judged, on MI355X: log-probabilities 66
// us (5.6 TB/s; a copy runs 5.1), their backward 146 (6.1, part of the logits from
// the last cache), the policy loss with its gradient 163 (5.5, VALU issue 70 %
// busy).
#include <type_traits>

#include "rows.h"

namespace seeai {
namespace {

constexpr float kLog2e = 1.4426950408889634f;

// exp(x) for x <= 0: the hardware's exp2.  Rounding x log2 e moves a term by
// |x| 2^-24 of itself, and terms far down hardly count.
__device__ __forceinline__ float ExpNeg(float x) { return __builtin_amdgcn_exp2f(x * kLog2e); }

// A running maximum and the sum of exp(z - max) under it, of a row's logits but the
// label's.  While all z are -inf the maximum is, too, and the sum zero; a NaN or
// +inf makes the sum a NaN.  A group's terms add up in pairs, groups in f64.
struct Lse {
  float m = -INFINITY;
  double s = 0.0;
  __device__ __forceinline__ float Base() const { return m == -INFINITY ? 0.0f : m; }
};

// The whole row, from the sum of the others under the row's maximum and the label's
// logit: the sum, and the label's log-probability.  Where the label is nearly sure
// the sum is 1 and a little, and the log-probability as small: the logarithm of the
// sum's leading bits, and what they leave of that little, which has its own digits as
// the label stands apart from it.
struct Soft {
  float m, s, logp, rest;  // rest: s without the label's term
  __device__ __forceinline__ Soft(const Lse& others, float zl) : m(others.m), rest(static_cast<float>(others.s)) {
    const float own = ExpNeg(zl - others.Base());
    s = static_cast<float>(others.s + static_cast<double>(own));
    // log s from 2^k f, f within 1 / sqrt 2 and sqrt 2, so that f32's logarithm is of
    // a number near 1; the sum is rounded once.
    int k = __builtin_amdgcn_frexp_expf(s);
    float f = __builtin_amdgcn_frexp_mantf(s);
    if (f < 0.70710678f) f += f, --k;
    const float left = static_cast<float>(others.s - static_cast<double>(s - own)) * __builtin_amdgcn_rcpf(s);
    const double log_s = fma(static_cast<double>(k), 0.6931471805599453, static_cast<double>(logf(f) + left));
    logp = static_cast<float>((static_cast<double>(zl) - static_cast<double>(m)) - log_s);
  }
};

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// A row on 16-byte groups of kV elements: wherever the row begins, the groups
// begin on 16 bytes, the first with `skip` elements before the row, the last
// with what lies behind it.  A softmax asks nothing of which lane holds which
// column, so rows of any alignment cost no more than aligned ones; a group's
// elements outside the row, which share 16 aligned bytes with one of the row's,
// are read and become -inf, and are never written.
template <class T>
struct Line {
  static constexpr int kV = 16 / sizeof(T);
  const u32x4* base;
  size_t groups, end;  // end: skip + C
  int skip;
  __device__ __forceinline__ Line(const T* row, size_t C) {
    const uintptr_t at = reinterpret_cast<uintptr_t>(row);
    skip = static_cast<int>(at % 16 / sizeof(T));
    base = reinterpret_cast<const u32x4*>(at & ~uintptr_t{15});
    end = C + skip;
    groups = (end + kV - 1) / kV;
  }
  __device__ __forceinline__ bool Whole(size_t g) const { return (g > 0 || skip == 0) && (g + 1) * kV <= end; }
  // Group g's elements outside the row become -inf, all of them past the row.
  __device__ __forceinline__ u32x4 Mask(u32x4 w, size_t g) const {
    const size_t c = g * kV;
    const int first = g == 0 ? skip : 0, last = c >= end ? 0 : end - c < kV ? static_cast<int>(end - c) : kV;
#pragma unroll
    for (int k = 0; k < kV; ++k) {
      const bool out = k < first || k >= last;
      if constexpr (sizeof(T) == 4) {
        w[k] = out ? 0xFF800000u : w[k];
      } else if (k % 2) {
        w[k / 2] = out ? (w[k / 2] & 0xFFFFu) | 0xFF800000u : w[k / 2];
      } else {
        w[k / 2] = out ? (w[k / 2] & 0xFFFF0000u) | 0xFF80u : w[k / 2];
      }
    }
    return w;
  }
  // Element `at` (a scalar) of a group becomes -inf.
  static __device__ __forceinline__ u32x4 Without(u32x4 w, int at) {
    const uint32_t keep = sizeof(T) == 4 ? 0u : at % 2 ? 0xFFFFu : 0xFFFF0000u;
    const uint32_t low = sizeof(T) == 4 || at % 2 ? 0xFF800000u : 0xFF80u;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const bool here = at * static_cast<int>(sizeof(T)) / 4 == k;
      w[k] = (w[k] & (here ? keep : ~0u)) | (here ? low : 0u);
    }
    return w;
  }
  static __device__ __forceinline__ void Floats(u32x4 w, float (&v)[kV]) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if constexpr (sizeof(T) == 4) {
        v[k] = __uint_as_float(w[k]);
      } else {
        v[2 * k] = __uint_as_float(w[k] << 16);
        v[2 * k + 1] = __uint_as_float(w[k] & 0xFFFF0000u);
      }
    }
  }
  static __device__ __forceinline__ u32x4 Bits(const float (&v)[kV]) {
    if constexpr (sizeof(T) == 4)
      return u32x4{__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])};
    else
      return __builtin_bit_cast(u32x4, Io<uint16_t>::Pack(v));
  }
  // Group from + g (from a scalar, g a lane's): an address of a scalar and 32 bits.
  __device__ __forceinline__ u32x4 Read(size_t from, unsigned g) const {
    return *reinterpret_cast<const u32x4*>(reinterpret_cast<const char*>(base + from) + g * 16u);
  }
  // A whole group to the row `out`: how 0 on out's own groups (out lies on 16
  // bytes as the row does), 1 the same past the caches, 2 wherever out lies.
  __device__ __forceinline__ void Store(T* out, int how, size_t from, unsigned g, const float (&v)[kV]) const {
    char* at = reinterpret_cast<char*>(out - skip + from * kV) + g * 16u;
    if (how == 1) __builtin_nontemporal_store(Bits(v), reinterpret_cast<u32x4*>(at));
    else if (how == 0) *reinterpret_cast<u32x4*>(at) = Bits(v);
    else Io<T>::StoreAny(reinterpret_cast<T*>(at), v);
  }
  // The column that thread t sees to of the first and the last group where they
  // are not whole (kV threads each), or C for none.
  __device__ __forceinline__ size_t Edge(int t, size_t C) const {
    if (t >= 2 * kV || (t >= kV && groups == 1)) return C;
    const size_t g = t < kV ? 0 : groups - 1, c = g * kV + t % kV;
    return Whole(g) || c < static_cast<size_t>(skip) || c >= end ? C : c - skip;
  }
};

// Keeps what is formed from w before from being kept for what is formed of it
// behind: unpacked twice it takes a quarter of the registers.
__device__ __forceinline__ void Forget(u32x4& w) { asm volatile("" : "+v"(w)); }

// Of n groups, kStep apart from this thread's on, the one that is group `own` of
// them all (a scalar) loses its element `at`.  Branches, a scalar's and then a lane's:
// as selects they would be formed for every group.
template <class T, int kStep, int n>
__device__ __forceinline__ void DropLabel(u32x4 (&w)[n], unsigned own, int at, int t) {
#pragma unroll
  for (int i = 0; i < n; ++i) {
    if (own / kStep != static_cast<unsigned>(i)) continue;
    if (t == static_cast<int>(own % kStep)) {
      Forget(w[i]);
      w[i] = Line<T>::Without(w[i], at);
    }
  }
}

// The first `used` (a scalar) of several groups at once: one new maximum for all.
template <class T, int n>
__device__ __forceinline__ void Take(Lse& a, u32x4 (&w)[n], int used) {
  constexpr int kV = Line<T>::kV;
  float top = a.m;
#pragma unroll
  for (int i = 0; i < n; ++i) {
    if (i >= used) break;
    float v[kV];
    Line<T>::Floats(w[i], v);
#pragma unroll
    for (int k = 0; k < kV; ++k) top = fmaxf(top, v[k]);
    Forget(w[i]);
    __builtin_amdgcn_sched_barrier(0);
  }
  const float was = a.m;
  a.m = top;
  const float base = a.Base();
  a.s *= static_cast<double>(ExpNeg(was - base));
#pragma unroll
  for (int i = 0; i < n; ++i) {
    if (i >= used) break;
    float v[kV];
    Line<T>::Floats(w[i], v);
#pragma unroll
    for (int k = 0; k < kV; ++k) v[k] = ExpNeg(v[k] - base);
#pragma unroll
    for (int n2 = kV / 2; n2 > 0; n2 /= 2)
#pragma unroll
      for (int k = 0; k < n2; ++k) v[k] += v[k + n2];
    a.s += static_cast<double>(v[0]);
    Forget(w[i]);
    __builtin_amdgcn_sched_barrier(0);
  }
}

// The row's maximum and the sum of all but its label under it, from its kTPR threads';
// `label` of the row's first thread (the label's logit, read before any thread may
// write over it) comes to all of them.
struct RowLds {
  double s[16];
  float m[16], label[16];
};
template <int kTPR>
__device__ __forceinline__ Lse RowLse(Lse a, RowLds& lds, float& label) {
  Lse r;
  label = __int_as_float(Uniform(__float_as_int(label)));
  r.m = LanesMax(a.m);
  if constexpr (kTPR == kWave) r.m = fmaxf(r.m, label);
  r.s = LanesSumD(a.s * static_cast<double>(ExpNeg(a.m - r.Base())));
  if constexpr (kTPR > kWave) {
    constexpr int kWaves = kTPR / kWave;
    const int w = threadIdx.x / kWave, first = w / kWaves * kWaves;
    __syncthreads();  // the sums before these have been read
    if (threadIdx.x % kWave == 0) lds.m[w] = r.m, lds.s[w] = r.s, lds.label[w] = label;
    __syncthreads();
    label = lds.label[first];
    Lse all;
    all.m = fmaxf(all.m, label);
#pragma unroll
    for (int k = 0; k < kWaves; ++k) all.m = fmaxf(all.m, lds.m[first + k]);
    const float base = all.Base();
#pragma unroll
    for (int k = 0; k < kWaves; ++k) all.s += lds.s[first + k] * static_cast<double>(ExpNeg(lds.m[first + k] - base));
    r = all;
  }
  return r;
}

// Groups a lane reads before it uses them: more where few rows share a CU.
constexpr int Ahead(int tpr) { return tpr > 256 ? 8 : 4; }

// This thread's share of a row but its label (`label` from the line's first group
// on): kAhead loads go out at a time; what may lie outside the row (the first
// turn's first group, the last turn) is masked.
template <class T, int kTPR>
__device__ __forceinline__ Lse SweepLse(const Line<T>& line, size_t label, int t) {
  constexpr int kAhead = Ahead(kTPR), kV = Line<T>::kV;
  Lse a;
  for (size_t at = 0; at < line.groups; at += kAhead * kTPR) {
    u32x4 w[kAhead];
    const bool last = at + kAhead * kTPR >= line.groups;
    const unsigned left = last ? static_cast<unsigned>(line.groups - at) : kAhead * kTPR;
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const unsigned g = u * kTPR + t;
      w[u] = line.Read(at, g < left ? g : left - 1);
    }
    const int used = last ? static_cast<int>((left + kTPR - 1) / kTPR) : kAhead;
    if (at == 0 && t == 0) w[0] = line.Mask(w[0], 0);
    if (last) {
#pragma unroll
      for (int u = 0; u < kAhead; ++u)
        if (u < used && u * kTPR + t + 1u >= left) w[u] = line.Mask(w[u], at + u * kTPR + t);
    }
    if (label / kV - at < kAhead * kTPR)  // (far past this turn's where it lies before)
      DropLabel<T, kTPR>(w, static_cast<unsigned>(label / kV - at), static_cast<int>(label % kV), t);
    Take<T>(a, w, used);
  }
  return a;
}

// dz = -d exp(z - m) / s for a group, by = -d / s; whether the label lies in it, at `at`.
template <class T>
__device__ __forceinline__ bool GroupGrad(u32x4 w, unsigned g, size_t label, float by, float m,
                                          float (&v)[Line<T>::kV], int& at) {
  constexpr int kV = Line<T>::kV;
  Line<T>::Floats(w, v);
#pragma unroll
  for (int k = 0; k < kV; ++k) v[k] = by * ExpNeg(v[k] - m);
  at = static_cast<int>(label % kV);
  return label / kV <= 0xFFFFFFFFu && g == static_cast<unsigned>(label / kV);
}
template <int kV>
__device__ __forceinline__ void PutAt(float (&v)[kV], int at, float x) {
#pragma unroll
  for (int k = 0; k < kV; ++k)
    if (k == at) v[k] = x;
}

// The label's own gradient is d (1 - p), where a nearly sure label's 1 - p has to
// come from the others' terms: `own`, d rest / s, where that rest is known.
// Where it is not (kSum), d - d p, and the row's other gradients add up (a thread's
// in `sum`): they are less than half of d where p is more than a half, and then the
// label's gradient is minus their sum.  `mine`: this thread has stored the label's.
struct RowGrad {
  float d, own, by, m;
  double sum = 0.0;
  bool mine = false;
};

// One column's gradient, by itself: what groups that are not whole hold.
template <class T, bool kSum>
__device__ __forceinline__ void EdgeGrad(const Line<T>& line, const T* row, T* out, int t, size_t C, size_t label,
                                         RowGrad& G) {
  const size_t c = line.Edge(t, C);
  if (c >= C) return;
  const float v = G.by * ExpNeg(Io<T>::Get(row + c) - G.m);
  Io<T>::Put(out + c, c != label ? v : kSum ? v + G.d : G.own);
  if constexpr (kSum) {
    if (c == label) G.mine = true;
    else G.sum += static_cast<double>(v);
  }
}

// A lane's groups are read before they are written, so out may be the row.
template <class T, int kTPR, bool kSum>
__device__ __forceinline__ void SweepGrad(const Line<T>& line, const T* row, T* out, int how, int t, size_t C,
                                          size_t label, RowGrad& G) {
  constexpr int kV = Line<T>::kV, kAhead = Ahead(kTPR);
  constexpr size_t kTurn = kAhead * kTPR;
  for (size_t i = (line.groups + kTurn - 1) / kTurn; i-- > 0;) {  // the end, read last, first
    const size_t at = i * kTurn;
    u32x4 w[kAhead];
    const size_t rest = line.groups - at;
    const unsigned left = rest < kAhead * kTPR ? static_cast<unsigned>(rest) : kAhead * kTPR;
    // This turn's groups that are whole, and the label's among them.
    const unsigned from = at == 0 && line.skip ? 1 : 0, to = left - (at + left == line.groups && line.end % kV ? 1 : 0);
    const size_t lab = label + line.skip - at * kV;  // (far past this turn's where it lies before)
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const unsigned g = u * kTPR + t;
      w[u] = line.Read(at, g < left ? g : left - 1);
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const unsigned g = u * kTPR + t;
      float v[kV], own = G.own;
      int k;
      const bool here = GroupGrad<T>(w[u], g, lab, G.by, G.m, v, k);
      if constexpr (kSum) {
        if (here) {
#pragma unroll
          for (int e = 0; e < kV; ++e)
            if (e == k) own = v[e] + G.d, v[e] = 0.0f;
        }
        float part[kV];
#pragma unroll
        for (int e = 0; e < kV; ++e) part[e] = v[e];
#pragma unroll
        for (int n = kV / 2; n > 0; n /= 2)
#pragma unroll
          for (int e = 0; e < n; ++e) part[e] += part[e + n];
        if (g >= from && g < to) G.sum += static_cast<double>(part[0]), G.mine |= here;
      }
      if (here) PutAt(v, k, own);
      if (g >= from && g < to) line.Store(out, how, at, g, v);
    }
  }
  EdgeGrad<T, kSum>(line, row, out, t, C, label, G);
}
template <class T, int kTPR>
__device__ __forceinline__ void SweepZero(T* out, bool past, int t, size_t C) {
  const Line<T> line(out, C);
  const float v[Line<T>::kV] = {};
  for (size_t at = 0; at < line.groups; at += kTPR)
    if (line.Whole(at + t)) line.Store(out, past, at, t, v);
  const size_t c = line.Edge(t, C);
  if (c < C) Io<T>::Put(out + c, 0.0f);
}

// A label's logit; one past the vocabulary has none.
template <class T>
__device__ __forceinline__ float LabelLogit(const T* row, int label, size_t C) {
  return label < 0 ? 0.0f : static_cast<size_t>(label) < C ? Io<T>::Get(row + label) : NAN;
}

constexpr int GroupOf(int tpr) { return tpr > 256 ? tpr : 256; }
// The row group of a thread, a scalar: a row has whole waves.
template <int kTPR>
__device__ __forceinline__ int RowGroup() { return Uniform(threadIdx.x / kTPR); }
// How a row's gradient is stored (Line::Store).
template <class T>
__device__ __forceinline__ int StoreHow(const T* row, const T* out, bool past) {
  return ((reinterpret_cast<uintptr_t>(row) ^ reinterpret_cast<uintptr_t>(out)) & 15) == 0 ? past : 2;
}

template <class T, int kTPR>
__global__ void __launch_bounds__(GroupOf(kTPR))
TokenLogpKernel(const T* __restrict__ z, size_t ld, const int32_t* __restrict__ labels,
                float* __restrict__ logp, float* __restrict__ stats, size_t N, size_t C) {
  constexpr int kRows = GroupOf(kTPR) / kTPR;
  __shared__ RowLds lds;
  const int t = threadIdx.x % kTPR;
  for (size_t base = static_cast<size_t>(blockIdx.x) * kRows; base < N;
       base += static_cast<size_t>(gridDim.x) * kRows) {
    const size_t r = base + RowGroup<kTPR>();
    const int label = r < N ? Uniform(labels[r]) : -1;
    const T* row = z + r * ld;
    float zl = t == 0 ? LabelLogit(row, label, C) : 0.0f;
    Lse a;
    if (label >= 0) {
      const Line<T> line(row, C);
      a = SweepLse<T, kTPR>(line, static_cast<size_t>(label) + line.skip, t);
    }
    a = RowLse<kTPR>(a, lds, zl);
    if (t == 0 && r < N) {
      const Soft all(a, zl);
      logp[r] = label < 0 ? 0.0f : all.logp;
      if (stats) stats[2 * r] = label < 0 ? 0.0f : all.m, stats[2 * r + 1] = label < 0 ? 0.0f : all.s;
    }
  }
}

// The last rows first: of logits that the forward pass has just read, they are
// what the chip's last cache still holds.
template <class T, int kTPR>
__global__ void __launch_bounds__(GroupOf(kTPR))
TokenLogpBwdKernel(const T* z, size_t ld, const int32_t* __restrict__ labels,
                   const float* __restrict__ stats, const float* __restrict__ dlogp, T* dz, bool past,
                   size_t N, size_t C) {
  constexpr int kRows = GroupOf(kTPR) / kTPR, kWaves = kTPR / kWave;
  static_assert(kWaves == 1 || kRows == 1, "a row's barriers are its workgroup's");
  __shared__ double lds[2][kWaves];  // used in turn: one barrier a row
  const int t = threadIdx.x % kTPR;
  int turn = 0;
  for (size_t i = static_cast<size_t>(blockIdx.x) * kRows + RowGroup<kTPR>(); i < N;
       i += static_cast<size_t>(gridDim.x) * kRows) {
    const size_t r = N - 1 - i;
    const int label = Uniform(labels[r]);
    T* out = dz + r * ld;
    if (label < 0) {
      SweepZero<T, kTPR>(out, past, t, C);
    } else {
      const T* row = z + r * ld;
      RowGrad G{static_cast<size_t>(label) < C ? dlogp[r] : NAN, 0.0f, 0.0f, stats[2 * r]};
      G.by = -G.d / stats[2 * r + 1];
      SweepGrad<T, kTPR, true>(Line<T>(row, C), row, out, StoreHow(row, out, past), t, C, label, G);
      double sum = LanesSumD(G.sum);
      if constexpr (kWaves > 1) {
        if (threadIdx.x % kWave == 0) lds[turn][threadIdx.x / kWave] = sum;
        __syncthreads();
        sum = 0.0;
#pragma unroll
        for (int k = 0; k < kWaves; ++k) sum += lds[turn][k];
        turn ^= 1;
      }
      if (G.mine && fabs(sum) < 0.5 * fabs(static_cast<double>(G.d))) Io<T>::Put(out + label, static_cast<float>(-sum));
    }
  }
}

// A judged token's numbers, read ahead of its log-probability, and its loss with
// the derivative by it.
struct PolicyToken {
  float old, ref, adv, weight;
  __device__ PolicyToken() {}
  __device__ __forceinline__ PolicyToken(const PolicyTerms& P, size_t r)
      : old(P.old_logp[r]), ref(P.ref_logp ? P.ref_logp[r] : 0.0f), adv(P.adv[r]),
        weight((P.weight ? P.weight[r] : 1.0f) * P.scale) {}
  __device__ __forceinline__ float2 At(const PolicyTerms& P, float logp) const {
    if (weight == 0.0f) return make_float2(0.0f, 0.0f);  // whatever the rest is
    const float ratio = expf(logp - old);
    // (a NaN passes both bounds)
    const float held = ratio < 1.0f - P.low ? 1.0f - P.low : ratio > 1.0f + P.high ? 1.0f + P.high : ratio;
    // (a ratio past f32 beside an advantage of zero: no term)
    const float whole = adv == 0.0f && ratio == INFINITY ? 0.0f : ratio * adv, cut = held * adv;
    float loss = cut < whole ? -cut : -whole, d = cut < whole ? 0.0f : -whole;
    if (P.ref_logp) {
      // Near the reference e - back - 1 is about back^2 / 2, which differences of
      // numbers near 1 lose (up to 30 % of it at back = 1e-3): there its series,
      // whose first missing term is 2 back^6 / 8! of it, 2^-26 at 1/4.
      const float back = ref - logp, e = expf(back);
      const bool near = fabsf(back) < 0.25f;
      const float row = 1.0f + back * (1.0f / 3) * (1.0f + back * 0.25f * (1.0f + back * 0.2f *
                        (1.0f + back * (1.0f / 6) * (1.0f + back * (1.0f / 7)))));
      // (infinite where back is, on either side)
      const float curve = near ? 0.5f * back * back * row : e == INFINITY ? e : (e - back) - 1.0f;
      loss += P.kl * curve;
      d -= P.kl * (near ? back + curve : e - 1.0f);
    }
    return make_float2(loss, d);
  }
};

// A row of at most kT kN groups in registers: the logits are read once and their
// gradient written once.  kN = 0: rows of any length, read a second time (from
// the caches, mostly) for the gradient.
template <class T, int kT, int kN>
__global__ void __launch_bounds__(GroupOf(kT))
PolicyKernel(const T* z, size_t ld, const int32_t* __restrict__ labels, PolicyTerms P,
             float* __restrict__ logp, T* dz, bool past, double* __restrict__ part, size_t N, size_t C) {
  constexpr int kRows = GroupOf(kT) / kT, kV = Line<T>::kV;
  __shared__ RowLds lds;
  __shared__ double sum[kRows];
  double mine = 0.0;  // of the row's first thread
  for (size_t base = static_cast<size_t>(blockIdx.x) * kRows; base < N;
       base += static_cast<size_t>(gridDim.x) * kRows) {
    int t = threadIdx.x % kT;
    asm volatile("" : "+v"(t));  // (its groups' offsets are formed where they are used, not kept)
    const size_t r = base + RowGroup<kT>();
    const int label = r < N ? Uniform(labels[r]) : -1;
    const T* row = z + r * ld;
    const Line<T> line(row, C);
    Lse a;
    u32x4 q[kN ? kN : 1];
    float zl = 0.0f;
    PolicyToken tok;
    const size_t at = static_cast<size_t>(label) + line.skip;  // (a judged row's)
    if (label >= 0) {
      if (t == 0) zl = LabelLogit(row, label, C);
      tok = PolicyToken(P, r);
      if constexpr (kN > 0) {
        const unsigned groups = static_cast<unsigned>(line.groups);
        const int used = static_cast<int>((groups + kT - 1) / kT);
#pragma unroll
        for (int i = 0; i < kN; ++i) {
          if (i >= used) break;
          const unsigned g = i * kT + t;
          q[i] = line.Read(0, g < groups ? g : groups - 1);
        }
        // (outside the row: -inf; groups past it all of it)
        if (t == 0) q[0] = line.Mask(q[0], 0);
#pragma unroll
        for (int i = 0; i < kN; ++i) {
          if (i >= used) break;
          if (i * kT + t + 1u >= groups) q[i] = line.Mask(q[i], i * kT + t);
          __builtin_amdgcn_sched_barrier(0);
        }
        DropLabel<T, kT>(q, static_cast<unsigned>(at / kV), static_cast<int>(at % kV), t);
        Take<T>(a, q, used);
      } else {
        a = SweepLse<T, kT>(line, at, t);
      }
    }
    a = RowLse<kT>(a, lds, zl);
    if (r >= N) continue;  // (no barrier is left in this turn)
    T* out = dz + r * ld;
    if (label < 0) {
      if (t == 0 && logp) logp[r] = 0.0f;
      if (dz) SweepZero<T, kT>(out, past, t, C);
      continue;
    }
    const Soft all(a, zl);
    const float2 term = tok.At(P, all.logp);
    if (t == 0) {
      if (logp) logp[r] = all.logp;
      mine += static_cast<double>(tok.weight) * static_cast<double>(term.x);
    }
    if (!dz) continue;
    const int how = StoreHow(row, out, past);
    const float d = tok.weight * term.y;
    RowGrad G{d, 0.0f, -d / all.s, all.m};
    G.own = -G.by * all.rest;
    if constexpr (kN > 0) {
      const unsigned from = line.skip ? 1 : 0, to = static_cast<unsigned>(line.end / kV);
#pragma unroll
      for (int i = 0; i < kN; ++i) {
        if (static_cast<size_t>(i) * kT >= line.groups) break;
        const unsigned g = i * kT + t;
        float v[kV];
        int k;
        if (GroupGrad<T>(q[i], g, at, G.by, G.m, v, k)) PutAt(v, k, G.own);
        if (g >= from && g < to) line.Store(out, how, 0, g, v);
        __builtin_amdgcn_sched_barrier(0);  // one group's numbers at a time
      }
      EdgeGrad<T, false>(line, row, out, t, C, label, G);
    } else {
      SweepGrad<T, kT, false>(line, row, out, how, t, C, label, G);
    }
  }
  if (threadIdx.x % kT == 0) sum[threadIdx.x / kT] = mine;
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
  for (size_t i = threadIdx.x; i < n; i += 8 * kSumThreads) {  // eight loads at a time
    double v[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const size_t at = i + k * kSumThreads;
      v[k] = part[at < n ? at : 0];
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) s += i + k * kSumThreads < n ? v[k] : 0.0;
  }
  s = WaveSumD(s);
  if (threadIdx.x % kWave == 0) red[threadIdx.x / kWave] = s;
  __syncthreads();
  if (threadIdx.x != 0) return;
#pragma unroll
  for (int k = 1; k < kSumThreads / kWave; ++k) s += red[k];
  *loss = static_cast<float>(scale * s);
}

// Where sequence q begins, kept within the rows.
__device__ __forceinline__ size_t StartOf(const PrefArgs& P, uint64_t q) {
  const int64_t s = P.starts[q], N = static_cast<int64_t>(P.N);
  return static_cast<size_t>(s < 0 ? 0 : s > N ? N : s);
}
__device__ __forceinline__ void ClearRows(const PrefArgs& P, size_t from, size_t to, int threads) {
  for (size_t r = from + threadIdx.x; r < to; r += threads) P.dlogp[r] = 0.0f;
}
// A pair's margin, its loss, and the loss's derivative by its log ratios' difference.
struct Pair {
  double margin, term, d;
  __device__ __forceinline__ Pair(const PrefArgs& P, double chosen, double rejected) {
    const double beta = P.beta, eps = P.smoothing;
    margin = beta * (chosen - rejected) - P.offset;
    // softplus(x) = max(x, 0) + log(1 + exp(-|x|)), sigmoid by the same exponential.
    const double e = exp(-fabs(margin)), tail = log1p(e), up = margin > 0.0 ? margin : 0.0;
    const double down = margin < 0.0 ? -margin : 0.0;
    const double won = (margin < 0.0 ? e : 1.0) / (1.0 + e), lost = (margin > 0.0 ? e : 1.0) / (1.0 + e);
    // (a smoothing of zero takes no part in an infinite margin)
    term = (eps < 1.0 ? (1.0 - eps) * (down + tail) : 0.0) + (eps > 0.0 ? eps * (up + tail) : 0.0);
    // won - (1 - eps), without the difference from 1 where the chosen answer is far ahead.
    d = P.scale * beta * (eps * won - (1.0 - eps) * lost);
  }
};

// Eight rows a lane of a sequence from `r` on, `step` apart: their log ratios
// and how many are judged.
__device__ __forceinline__ double2 EightRows(const PrefArgs& P, size_t r, size_t end, size_t step) {
  int32_t lab[8];
  float lp[8], ref[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const size_t at = r + k * step < end ? r + k * step : r;
    lab[k] = P.labels[at], lp[k] = P.logp[at], ref[k] = P.ref_logp ? P.ref_logp[at] : 0.0f;
  }
  double s = 0.0, n = 0.0;
#pragma unroll
  for (int k = 0; k < 8; ++k)
    if (r + k * step < end && lab[k] >= 0) s += static_cast<double>(lp[k]) - static_cast<double>(ref[k]), n += 1.0;
  return make_double2(s, n);
}
// A sequence's, by `threads` threads of which this is t; every lane gets its wave's.
__device__ __forceinline__ double2 Sequence(const PrefArgs& P, size_t from, size_t to, int t, int threads) {
  double s = 0.0, n = 0.0;
  for (size_t r = from + t; r < to; r += 8 * static_cast<size_t>(threads)) {
    const double2 v = EightRows(P, r, to, threads);
    s += v.x, n += v.y;
  }
  return make_double2(WaveSumD(s), P.average ? WaveSumD(n) : 1.0);
}

// A workgroup a pair: its two sequences' log ratios, its loss, its rows' dlogp.
// Rows outside every sequence get a zero.
constexpr int kPairThreads = 512;
__global__ void __launch_bounds__(kPairThreads)
PrefPairKernel(PrefArgs P, double* __restrict__ terms) {
  constexpr int kWaves = kPairThreads / kWave;
  __shared__ double2 red[2][kWaves];
  if (P.pairs == 0) {
    ClearRows(P, 0, P.N, kPairThreads);
    return;
  }
  const uint64_t i = blockIdx.x;
  const size_t cut[3] = {StartOf(P, 2 * i), StartOf(P, 2 * i + 1), StartOf(P, 2 * i + 2)};
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const double2 v = Sequence(P, cut[k], cut[k + 1], threadIdx.x, kPairThreads);
    if (threadIdx.x % kWave == 0) red[k][threadIdx.x / kWave] = v;
  }
  __syncthreads();
  double ratio[2], count[2];
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    ratio[k] = count[k] = 0.0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) ratio[k] += red[k][w].x, count[k] += red[k][w].y;
    count[k] = P.average ? fmax(count[k], 1.0) : 1.0;
  }
  const Pair pair(P, ratio[0] / count[0], ratio[1] / count[1]);
  if (threadIdx.x == 0) {
    terms[i] = pair.term;
    if (P.margin) P.margin[i] = static_cast<float>(pair.margin);
  }
  if (!P.dlogp) return;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const float dk = static_cast<float>((k ? -pair.d : pair.d) / count[k]);
    for (size_t r = cut[k] + threadIdx.x; r < cut[k + 1]; r += kPairThreads)
      P.dlogp[r] = P.labels[r] < 0 ? 0.0f : dk;
  }
  if (i == 0) ClearRows(P, 0, cut[0], kPairThreads);
  if (i + 1 == P.pairs) ClearRows(P, cut[2], P.N, kPairThreads);
}

// All pairs in one workgroup, and their loss: a launch less.  A wave takes a sequence,
// or several a share of one each where there are fewer.
constexpr int kOneThreads = 1024, kOneWaves = kOneThreads / kWave;
constexpr size_t kOnePairs = kOneWaves / 2, kOneRows = 2048;
__global__ void __launch_bounds__(kOneThreads)
PrefOneKernel(PrefArgs P, float* __restrict__ loss) {
  __shared__ double2 red[kOneWaves];  // a wave's sum and count
  __shared__ float slope[2 * kOnePairs];
  const int wave = Uniform(threadIdx.x / kWave), lane = threadIdx.x % kWave;
  const int seqs = static_cast<int>(2 * P.pairs);
  // Sequences' shares: 8, 4, 2 or 1 waves to each.
  int shares = 1;
  while (2 * shares * seqs <= kOneWaves) shares *= 2;
  const int q = wave / shares, first = wave % shares * kWave + lane, threads = shares * kWave;
  const size_t from = q < seqs ? StartOf(P, q) : 0, to = q < seqs ? StartOf(P, q + 1) : 0;
  const double2 sum = Sequence(P, from, to, first, threads);
  if (lane == 0) red[wave] = sum;
  __syncthreads();
  if (wave == 0) {
    double term = 0.0;
    if (lane < static_cast<int>(P.pairs)) {
      double2 v[2];
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        v[k] = make_double2(0.0, 0.0);
        for (int h = 0; h < shares; ++h) {
          v[k].x += red[(2 * lane + k) * shares + h].x;
          v[k].y += red[(2 * lane + k) * shares + h].y;
        }
        v[k].y = P.average ? fmax(v[k].y, 1.0) : 1.0;
      }
      const Pair pair(P, v[0].x / v[0].y, v[1].x / v[1].y);
      term = pair.term;
      if (P.margin) P.margin[lane] = static_cast<float>(pair.margin);
      slope[2 * lane] = static_cast<float>(pair.d / v[0].y);
      slope[2 * lane + 1] = static_cast<float>(-pair.d / v[1].y);
    }
    term = WaveSumD(term);
    if (lane == 0) *loss = static_cast<float>(P.scale * term);
  }
  if (!P.dlogp) return;
  __syncthreads();
  const float d = q < seqs ? slope[q] : 0.0f;
#pragma unroll 8
  for (size_t r = from + first; r < to; r += threads) P.dlogp[r] = P.labels[r] < 0 ? 0.0f : d;
  ClearRows(P, 0, StartOf(P, 0), kOneThreads);
  ClearRows(P, StartOf(P, seqs), P.N, kOneThreads);
}

// Workgroups of the row kernels: they walk what rows are left.
constexpr size_t kMaxGroups = 8192;
unsigned Groups(size_t rows, int per) {
  const size_t g = (rows + per - 1) / per;
  return static_cast<unsigned>(g < kMaxGroups ? g : kMaxGroups);
}

// Gradients that the last cache (256 MB) cannot hold beside the logits for the
// product that reads them are stored past it: 8192 x 32000 bf16 paired loss 242 us
// against 261, policy loss 165 against 169, 2000 x 128000 paired 289 against 321; 2000 x
// 16000 (64 MB) 43 against 42.
bool GoesPast(size_t N, size_t ld, size_t size) { return N * ld * size > size_t{128} << 20; }

// The 16-byte groups that a row of C may lie on.
size_t RowGroups(int bf16, const void* z, size_t ld, size_t C) {
  const size_t kV = bf16 ? 8 : 4, size = bf16 ? 2 : 4;
  return (C + kV - 1) / kV + ((reinterpret_cast<uintptr_t>(z) | (ld * size)) % 16 ? 1 : 0);
}

// A row's threads in the kernels that walk along it: four groups each, then as
// many as fill the chip (1879 x 27328 bf16: 256 threads 21 us, 1024 34).
template <class F>
hipError_t ByRow(size_t N, size_t groups, F&& go) {
  if (groups <= 256) return go(std::integral_constant<int, 64>{});
  if (groups <= 1024 || N >= 512) return go(std::integral_constant<int, 256>{});
  return go(std::integral_constant<int, 1024>{});
}

// A row's threads and groups a thread in registers.
template <class F>
hipError_t ByRegisters(size_t N, size_t groups, F&& go) {
#define SEEAI_ROW(t, n) go(std::integral_constant<int, t>{}, std::integral_constant<int, n>{})
  if (groups <= 64 * 4) return SEEAI_ROW(64, 4);
  if (groups <= 128 * 4) return SEEAI_ROW(128, 4);
  if (groups <= 256 * 4) return SEEAI_ROW(256, 4);
  if (N >= 512) {
    if (groups <= 256 * 8) return SEEAI_ROW(256, 8);
    if (groups <= 512 * 8) return SEEAI_ROW(512, 8);
  }
  if (groups <= 1024 * 4) return SEEAI_ROW(1024, 4);
  // One such workgroup fills a CU: with rows enough it pays where its lanes are
  // (4096 x 32000 f32, 8000 groups: 205 us against 212 in two sweeps; 4824 x 49394
  // bf16, 6175 groups: 199 against 181).
  if (groups <= 1024 * 8 && (N < 512 || groups > 1024 * 7)) return SEEAI_ROW(1024, 8);
  return SEEAI_ROW(512, 0);
#undef SEEAI_ROW
}

}  // namespace

size_t PolicyWorkspaceBytes(size_t N) { return (N < kMaxGroups ? N : kMaxGroups) * sizeof(double); }
size_t PrefWorkspaceBytes(size_t pairs) { return pairs * sizeof(double); }

hipError_t LaunchTokenLogpFwd(int bf16, const void* z, size_t ld, const int32_t* labels, float* logp,
                              float* stats, size_t N, size_t C, hipStream_t s) {
  if (N == 0) return hipSuccess;
  return ByRow(N, RowGroups(bf16, z, ld, C), [&](auto tpr) {
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
  return ByRow(N, RowGroups(bf16, z, ld, C), [&](auto tpr) {
    constexpr int kT = decltype(tpr)::value, kG = GroupOf(kT);
    if (bf16)
      hipLaunchKernelGGL((TokenLogpBwdKernel<uint16_t, kT>), dim3(Groups(N, kG / kT)), dim3(kG), 0, s,
                         static_cast<const uint16_t*>(z), ld, labels, stats, dlogp,
                         static_cast<uint16_t*>(dz), GoesPast(N, ld, 2), N, C);
    else
      hipLaunchKernelGGL((TokenLogpBwdKernel<float, kT>), dim3(Groups(N, kG / kT)), dim3(kG), 0, s,
                         static_cast<const float*>(z), ld, labels, stats, dlogp,
                         static_cast<float*>(dz), GoesPast(N, ld, 4), N, C);
    return hipGetLastError();
  });
}

hipError_t LaunchPrefLoss(const PrefArgs& a, float* loss, void* ws, hipStream_t s) {
  double* terms = static_cast<double*>(ws);
  // One launch where a wave has one sequence at most, and few rows (us, one launch
  // against two: 4 pairs of 701 rows 5.4 and 7.2, 8 of 2048 5.6 and 7.5, 8 of 8192 6.8 and
  // 7.8; with 32 pairs, sequences in turn, 12 and 7.2, with 256 80 and 7.5).  How long each
  // answer is the device knows: one of 8 pairs with nearly all rows takes 12 against 7.4 of
  // 2048, 21 against 8.1 of 4096.
  if (a.pairs && a.pairs <= kOnePairs && a.N <= kOneRows) {
    hipLaunchKernelGGL(PrefOneKernel, dim3(1), dim3(kOneThreads), 0, s, a, loss);
    return hipGetLastError();
  }
  if (a.pairs || (a.dlogp && a.N)) {
    hipLaunchKernelGGL(PrefPairKernel, dim3(static_cast<unsigned>(a.pairs ? a.pairs : 1)),
                       dim3(kPairThreads), 0, s, a, terms);
    if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
  }
  hipLaunchKernelGGL(SumTermsKernel, dim3(1), dim3(kSumThreads), 0, s, terms, a.pairs,
                     static_cast<double>(a.scale), loss);
  return hipGetLastError();
}

template <class T>
hipError_t RunPolicy(const void* z, size_t ld, const int32_t* labels, const PolicyTerms& P, float* logp,
                     void* dz, size_t N, size_t C, double* part, size_t* parts, hipStream_t s) {
  return ByRegisters(N, RowGroups(sizeof(T) == 2, z, ld, C), [&](auto tpr, auto held) {
    constexpr int kT = decltype(tpr)::value, kN = decltype(held)::value, kG = GroupOf(kT);
    const unsigned groups = Groups(N, kG / kT);
    hipLaunchKernelGGL((PolicyKernel<T, kT, kN>), dim3(groups), dim3(kG), 0, s, static_cast<const T*>(z), ld,
                       labels, P, logp, static_cast<T*>(dz), GoesPast(N, ld, sizeof(T)), part, N, C);
    *parts = groups;
    return hipGetLastError();
  });
}

hipError_t LaunchPolicyLoss(int bf16, const void* z, size_t ld, const int32_t* labels,
                            const PolicyTerms& P, float* loss, float* logp, void* dz, size_t N, size_t C,
                            void* ws, hipStream_t s) {
  double* part = static_cast<double*>(ws);
  size_t parts = 0;
  if (N) {
    const hipError_t e = bf16 ? RunPolicy<uint16_t>(z, ld, labels, P, logp, dz, N, C, part, &parts, s)
                              : RunPolicy<float>(z, ld, labels, P, logp, dz, N, C, part, &parts, s);
    if (e != hipSuccess) return e;
  }
  hipLaunchKernelGGL(SumTermsKernel, dim3(1), dim3(kSumThreads), 0, s, part, parts, 1.0, loss);
  return hipGetLastError();
}

}  // namespace seeai
