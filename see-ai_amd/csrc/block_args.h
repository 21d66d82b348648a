// block_args.h -- the argument checks of the trained-block entry points
// (seeai_norm_*, seeai_ffn_*, seeai_adamw_group_*): what the kernels assume of
// their operands, decided on the host before anything is launched.  Plain C++
// without HIP, so the checks run where there is no GPU.  A check returns null,
// or why the call is refused.
#pragma once

#include <algorithm>
#include <cstddef>
#include <cstdint>
#include <initializer_list>
#include <vector>

#include "../../include/seeai_hip.h"

namespace seeai {

// The widest row (D, F) of a feed-forward block: a tile's 256 rows stay inside
// one buffer descriptor's 32-bit range.
constexpr uint64_t kFfnMaxWidth = uint64_t{1} << 20;
// Rows and columns of a norm: the kernels' column indices are 32-bit.
constexpr uint64_t kBlockMaxRows = (uint64_t{1} << 31) - 1;
// Tokens: a row tile past the last stays a 32-bit index, and 64-row tiles of a
// narrow block one launch.
constexpr uint64_t kFfnMaxTokens = uint64_t{1} << 29;

// An operand: its elements, their size, and whether the call writes it.
struct Operand {
  const void* p;
  uint64_t n, size;
  bool out;
};

// Every operand present, on its element's alignment, its bytes countable, and
// no output sharing a byte with another operand.
inline const char* CheckOperands(std::initializer_list<Operand> all) {
  for (const Operand& a : all) {
    if (a.n == 0) continue;
    uint64_t bytes;
    if (!a.p) return "null operand";
    if (reinterpret_cast<uintptr_t>(a.p) % a.size) return "operand off its element's alignment";
    if (__builtin_mul_overflow(a.n, a.size, &bytes) || bytes >> 62) return "operand too large";
  }
  for (const Operand& a : all) {
    if (!a.out || a.n == 0) continue;
    for (const Operand& b : all) {
      if (&a == &b || b.n == 0) continue;
      const uintptr_t a0 = reinterpret_cast<uintptr_t>(a.p), b0 = reinterpret_cast<uintptr_t>(b.p);
      if (a0 < b0 + b.n * b.size && b0 < a0 + a.n * a.size) return "an output overlaps an operand";
    }
  }
  return nullptr;
}

inline uint64_t TypeSize(int dtype) { return dtype ? 2 : 4; }

inline const char* CheckNormShape(int kind, int dtype, uint64_t rows, uint64_t cols) {
  if (kind < 0 || kind > 1) return "kind is 0 (layer) or 1 (root mean square)";
  if (dtype < 0 || dtype > 1) return "dtype is 0 (f32) or 1 (bf16)";
  if (cols == 0 || cols > kBlockMaxRows || rows > kBlockMaxRows) return "bad shape";
  return nullptr;
}

inline const char* CheckNormFwd(int kind, int dtype, const void* x, const float* w, const float* b,
                                const void* y, const float* mean, const float* rstd, uint64_t rows,
                                uint64_t cols, float eps) {
  if (const char* e = CheckNormShape(kind, dtype, rows, cols)) return e;
  if (!(eps >= 0.0f) || eps > 3.4028234663852886e38f) return "eps is a finite number from zero";
  if (kind == 1 && (b || mean)) return "a root-mean-square norm has no bias and no mean";
  const uint64_t n = rows * cols, size = TypeSize(dtype);
  return CheckOperands({{x, n, size, false}, {w, cols, 4, false}, {b, b ? cols : 0, 4, false},
                        {y, n, size, true}, {mean, mean ? rows : 0, 4, true},
                        {rstd, rstd ? rows : 0, 4, true}});
}

inline const char* CheckNormBwd(int kind, int dtype, const void* dy, const void* x, const float* w,
                                const float* mean, const float* rstd, const void* dx,
                                const float* dw, const float* db, uint64_t rows, uint64_t cols,
                                const void* ws, uint64_t ws_bytes, uint64_t need) {
  if (const char* e = CheckNormShape(kind, dtype, rows, cols)) return e;
  if (kind == 1 && (db || mean)) return "a root-mean-square norm has no bias and no mean";
  if (ws_bytes < need) return "workspace too small (seeai_norm_bwd_workspace)";
  const uint64_t n = rows * cols, size = TypeSize(dtype);
  return CheckOperands({{dy, n, size, false}, {x, n, size, false}, {w, cols, 4, false},
                        {mean, kind == 0 ? rows : 0, 4, false}, {rstd, rows, 4, false},
                        {dx, n, size, true}, {dw, cols, 4, true}, {db, db ? cols : 0, 4, true},
                        {ws, (need + 15) / 16, 16, true}});
}

inline const char* CheckFfnShape(int dtype, int act, uint64_t M, uint64_t D, uint64_t F) {
  if (dtype < 0 || dtype > 1) return "dtype is 0 (f32) or 1 (bf16)";
  if (act < 0 || act > 3) return "act is 0 (none), 1 (relu), 2 (gelu) or 3 (silu)";
  if (D == 0 || F == 0 || D > kFfnMaxWidth || F > kFfnMaxWidth || M > kFfnMaxTokens)
    return "bad shape (widths from 1 to 1048576, tokens to 536870912)";
  return nullptr;
}

inline const char* CheckFfnFwd(int dtype, int act, const void* x, const void* wg, const void* wu,
                               const void* wd, const void* gate, const void* up, const void* y,
                               uint64_t M, uint64_t D, uint64_t F, const void* ws,
                               uint64_t ws_bytes, uint64_t need) {
  if (const char* e = CheckFfnShape(dtype, act, M, D, F)) return e;
  if (!gate != !up) return "the projections are saved both or neither";
  if (ws_bytes < need) return "workspace too small (seeai_ffn_workspace)";
  const uint64_t size = TypeSize(dtype), kept = gate ? M * F : 0;
  return CheckOperands({{x, M * D, size, false}, {wg, D * F, size, false}, {wu, D * F, size, false},
                        {wd, D * F, size, false}, {gate, kept, size, true}, {up, kept, size, true},
                        {y, M * D, size, true}, {ws, (need + 15) / 16, 16, true}});
}

inline const char* CheckFfnBwd(int dtype, int act, const void* x, const void* wg, const void* wu,
                               const void* wd, const void* gate, const void* up, const void* dy,
                               const void* dx, const void* dwg, const void* dwu, const void* dwd,
                               uint64_t M, uint64_t D, uint64_t F, const void* ws,
                               uint64_t ws_bytes, uint64_t need) {
  if (const char* e = CheckFfnShape(dtype, act, M, D, F)) return e;
  if (ws_bytes < need) return "workspace too small (seeai_ffn_workspace)";
  const uint64_t size = TypeSize(dtype), w = D * F;
  return CheckOperands({{x, M * D, size, false}, {wg, w, size, false}, {wu, w, size, false},
                        {wd, w, size, false}, {gate, M * F, size, false}, {up, M * F, size, false},
                        {dy, M * D, size, false}, {dx, M * D, size, true}, {dwg, w, size, true},
                        {dwu, w, size, true}, {dwd, w, size, true},
                        {ws, (need + 15) / 16, 16, true}});
}

// A group of tensors: each complete and aligned, no two writing the same byte,
// none reading as gradient what another writes.
inline const char* CheckAdamWGroup(const seeai_adamw_tensor* t, uint64_t count, int state_bits,
                                   int grad_dtype) {
  if (state_bits != 8 && state_bits != 32) return "state_bits is 8 or 32";
  if (grad_dtype < 0 || grad_dtype > 1) return "grad_dtype is 0 (f32) or 1 (bf16)";
  if (count > 1 << 24) return "too many tensors";
  if (count && !t) return "null operand";
  struct Run {
    uintptr_t b, e;
    bool out;
  };
  std::vector<Run> runs;
  uint64_t chunks = 0;
  for (uint64_t i = 0; i < count; ++i) {
    const seeai_adamw_tensor& x = t[i];
    if (x.n == 0) continue;
    if (x.n >> 36) return "operand too large";
    if (!(x.decay >= 0.0f) || x.decay > 3.4028234663852886e38f)
      return "decay is a finite number from zero";
    const uint64_t blocks = (x.n + 127) / 128, state = state_bits / 8;
    const Operand all[] = {{x.p, x.n, 4, true},
                           {x.g, x.n, grad_dtype ? 2u : 4u, false},
                           {x.m, x.n, state, true},
                           {x.v, x.n, state, true},
                           {x.m_scale, state_bits == 8 ? blocks : 0, 4, true},
                           {x.v_scale, state_bits == 8 ? blocks : 0, 4, true},
                           {x.p_bf16, x.p_bf16 ? x.n : 0, 2, true}};
    for (const Operand& o : all) {
      if (o.n == 0) continue;
      if (!o.p) return "null operand";
      const uintptr_t b = reinterpret_cast<uintptr_t>(o.p);
      if (b % o.size) return "operand off its element's alignment";
      runs.push_back({b, b + o.n * o.size, o.out});
    }
    if ((chunks += (x.n + 2047) / 2048) >> 24) return "group too large";
  }
  std::sort(runs.begin(), runs.end(), [](const Run& a, const Run& b) { return a.b < b.b; });
  uintptr_t written = 0, any = 0;  // the furthest end of an output, of an operand, so far
  for (const Run& r : runs) {
    if (r.b < written || (r.out && r.b < any)) return "an output overlaps an operand";
    any = std::max(any, r.e);
    if (r.out) written = std::max(written, r.e);
  }
  return nullptr;
}

// The values of 8-bit moments: as many as a group can hold (one launch of
// 2048 elements a workgroup, below 2^32 threads).
inline const char* CheckAdamWValues(int which, int dtype, const void* codes, const float* scales,
                                    uint64_t n, const void* out) {
  if (which < 0 || which > 1) return "which is 0 (m) or 1 (v)";
  if (dtype < 0 || dtype > 1) return "dtype is 0 (f32) or 1 (bf16)";
  if (n >> 36 || (n + 2047) / 2048 >> 24) return "operand too large";
  return CheckOperands({{codes, n, 1, false}, {scales, (n + 127) / 128, 4, false},
                        {out, n, TypeSize(dtype), true}});
}

}  // namespace seeai
