// Scores capped by a tanh and biased by distance, as the attention kernels that take them form them.
#pragma once

#include "common.h"

namespace tasft {

// cap tanh(s scale / cap) and the head's slope. All results are in units of log2 (the exponentials'
// argument).
struct ScoreParams {
  const float* slopes;  // [Hq] or null
  float scale_log2;     // scale log2(e)
  float cap_in;         // 2 log2(e) scale / cap
  float cap_out;        // cap log2(e)
  float cap_lin;        // scale / cap
  int cap_wide;         // a cap so large that tanh is taken by its series near 0
};

// tanh(x) = 1 - 2 / (1 + exp(2x)): two of the slow instructions and three others. Near x = 0 it is off by
// 2^-23 of 1, so the score by 2^-23 caps.
__device__ __forceinline__ float cap_gate(float s, const ScoreParams& p) {  // 1 / (1 + exp(2x))
  return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(s * p.cap_in));
}

__device__ __forceinline__ float cap_score(float s, float r, const ScoreParams& p) {
  return fmaf(r, -2.f * p.cap_out, p.cap_out);
}

// From a cap of kWideCap on (the error above would be 2^-23 kWideCap = 1.5e-5 and more) arguments under
// 1/4 go by the series x - x^3/3 + 2x^5/15 - 17x^7/315 + 62x^9/2835 (the next term: 2^-27 of x).
constexpr float kWideCap = 128.f;
__device__ __forceinline__ float cap_score_wide(float s, float r, const ScoreParams& p) {
  const float x = s * p.cap_lin, y = x * x;
  float t = fmaf(y, 62.f / 2835.f, -17.f / 315.f);
  t = fmaf(y, t, 2.f / 15.f);
  t = fmaf(y, t, -1.f / 3.f);
  t = fmaf(y, t, 1.f);
  return fabsf(x) < 0.25f ? x * t * p.cap_out : cap_score(s, r, p);
}

inline ScoreParams score_params(float scale, float softcap, const float* slopes) {
  ScoreParams s = {};
  s.slopes = slopes;
  s.scale_log2 = scale * kLog2e;
  if (softcap > 0.f) {
    s.cap_in = (float)(2.0 * 1.4426950408889634 * (double)scale / (double)softcap);
    s.cap_out = (float)((double)softcap * 1.4426950408889634);
    s.cap_lin = (float)((double)scale / (double)softcap);
    s.cap_wide = softcap > kWideCap;
  }
  return s;
}

}  // namespace tasft
