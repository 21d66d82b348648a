// pref_args.h -- the argument checks of seeai_token_logp_*, seeai_pref_loss and
// seeai_policy_loss: what the kernels assume of their operands, decided on the
// host before anything is launched.  Plain C++ without HIP, so the checks run
// where there is no GPU.  A check returns null, or why the call is refused.
#pragma once

#include "block_args.h"

namespace seeai {

// Pairs: one launch of a workgroup each.
constexpr uint64_t kPrefMaxPairs = uint64_t{1} << 20;

inline bool Finite(float v) { return v - v == 0.0f; }

// The elements of N rows of C, ld apart, from the first to the last.
inline const char* CheckLogitsShape(int dtype, uint64_t ld, uint64_t N, uint64_t C) {
  if (dtype < 0 || dtype > 1) return "dtype is 0 (f32) or 1 (bf16)";
  if (C == 0 || C > kBlockMaxRows || N > kBlockMaxRows) return "bad shape";
  if (ld < C) return "rows are at least C apart";
  uint64_t span;
  if (__builtin_mul_overflow(ld, N, &span) || span >> 60) return "operand too large";
  return nullptr;
}
inline uint64_t LogitsSpan(uint64_t ld, uint64_t N, uint64_t C) { return N ? (N - 1) * ld + C : 0; }

inline const char* CheckTokenLogpFwd(int dtype, const void* z, uint64_t ld, const int32_t* labels,
                                     const float* logp, const float* stats, uint64_t N, uint64_t C) {
  if (const char* e = CheckLogitsShape(dtype, ld, N, C)) return e;
  return CheckOperands({{z, LogitsSpan(ld, N, C), TypeSize(dtype), false}, {labels, N, 4, false},
                        {logp, N, 4, true}, {stats, stats ? 2 * N : 0, 4, true}});
}

inline const char* CheckTokenLogpBwd(int dtype, const void* z, uint64_t ld, const int32_t* labels,
                                     const float* stats, const float* dlogp, const void* dz, uint64_t N,
                                     uint64_t C) {
  if (const char* e = CheckLogitsShape(dtype, ld, N, C)) return e;
  const uint64_t span = LogitsSpan(ld, N, C), size = TypeSize(dtype);
  return CheckOperands({{z, z == dz ? 0 : span, size, false}, {labels, N, 4, false},
                        {stats, 2 * N, 4, false}, {dlogp, N, 4, false}, {dz, span, size, true}});
}

inline const char* CheckPrefLoss(const float* logp, const float* ref, const int32_t* labels,
                                 const int32_t* starts, uint64_t N, uint64_t pairs, float beta,
                                 float offset, float smoothing, int average, float scale,
                                 const float* loss, const float* margin, const float* dlogp,
                                 const void* ws, uint64_t ws_bytes, uint64_t need) {
  if (N > kBlockMaxRows || pairs > kPrefMaxPairs) return "bad shape";
  if (average < 0 || average > 1) return "average is 0 or 1";
  if (!(smoothing >= 0.0f && smoothing <= 1.0f)) return "smoothing is from 0 to 1";
  if (!Finite(beta) || !Finite(offset) || !Finite(scale)) return "beta, offset and scale are finite";
  if (ws_bytes < need) return "workspace too small (seeai_pref_workspace)";
  return CheckOperands({{logp, pairs ? N : 0, 4, false}, {ref, ref && pairs ? N : 0, 4, false},
                        {labels, pairs ? N : 0, 4, false}, {starts, pairs ? 2 * pairs + 1 : 0, 4, false},
                        {loss, 1, 4, true}, {margin, margin ? pairs : 0, 4, true},
                        {dlogp, dlogp ? N : 0, 4, true}, {ws, (need + 15) / 16, 16, true}});
}

inline const char* CheckPolicyLoss(int dtype, const void* z, uint64_t ld, const int32_t* labels,
                                   const float* old_logp, const float* ref, const float* adv,
                                   const float* weight, uint64_t N, uint64_t C, float low, float high,
                                   float kl, float scale, const float* loss, const float* logp,
                                   const void* dz, const void* ws, uint64_t ws_bytes, uint64_t need) {
  if (const char* e = CheckLogitsShape(dtype, ld, N, C)) return e;
  if (!(low >= 0.0f && low <= 1.0f) || !(high >= 0.0f) || !Finite(high))
    return "clip_low is from 0 to 1, clip_high a finite number from zero";
  if (!Finite(kl) || !Finite(scale)) return "kl_coef and scale are finite";
  if (N && !ref && kl != 0.0f) return "a KL term needs ref_logp";
  if (ws_bytes < need) return "workspace too small (seeai_policy_workspace)";
  const uint64_t span = LogitsSpan(ld, N, C), size = TypeSize(dtype);
  return CheckOperands({{z, dz && z == dz ? 0 : span, size, false}, {labels, N, 4, false},
                        {old_logp, N, 4, false}, {ref, ref ? N : 0, 4, false}, {adv, N, 4, false},
                        {weight, weight ? N : 0, 4, false}, {loss, 1, 4, true},
                        {logp, logp ? N : 0, 4, true}, {dz, dz ? span : 0, size, true},
                        {ws, (need + 15) / 16, 16, true}});
}

}  // namespace seeai
