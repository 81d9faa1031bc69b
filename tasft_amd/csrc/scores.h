// Scores capped by a tanh and biased by distance, as the attention kernels that take them form them.
#pragma once

#include "common.h"

namespace tasft {

// A product s = q . k becomes a value x that rises with the score, and the score, in units of log2 (the
// exponentials' argument), is x mul + add:
//   without a cap x = s (biased: less slope / scale distance), mul = scale log2(e);
//   with one x = -1 / (1 + exp(2 s scale / cap)), tanh being 1 + 2x: mul = 2 cap log2(e), add = half of it;
//   a wide cap, or a cap and a bias: x is the score itself.
// The map costs nothing: the exponential's argument is a multiply-add in any case.
struct ScoreParams {
  const float* slopes;  // [Hq] or null
  float mul, add;
  float slope_mul;      // a slope in units of x
  float cap_in;         // 2 log2(e) scale / cap, 0: no cap
  float cap_out;        // cap log2(e)
  float cap_lin;        // scale / cap
  int cap_score;        // with a cap: x is the score itself
  int cap_wide;         // a cap so large that tanh is taken by its series near 0
};

// -1 / (1 + exp(2 s scale / cap)): two of the slow instructions and two others. Around s = 0 tanh so formed is
// off by some 2^-23, the score by that of the cap.
__device__ __forceinline__ float cap_gate(float s, const ScoreParams& p) {
  return __builtin_amdgcn_rcpf(-1.f - __builtin_amdgcn_exp2f(s * p.cap_in));
}

// The score from its gate. From a cap of kWideCap on (the error above would be 2^-23 kWideCap = 1.5e-5 and more)
// arguments under 1/4 go by the series x - x^3/3 + 2x^5/15 - 17x^7/315 + 62x^9/2835 (the next term: 2^-27 of x).
constexpr float kWideCap = 128.f;
__device__ __forceinline__ float cap_score(float s, float gate, const ScoreParams& p) {
  const float far = fmaf(gate, 2.f * p.cap_out, p.cap_out);
  if (!p.cap_wide) return far;
  const float x = s * p.cap_lin, y = x * x;
  float t = fmaf(y, 62.f / 2835.f, -17.f / 315.f);
  t = fmaf(y, t, 2.f / 15.f);
  t = fmaf(y, t, -1.f / 3.f);
  t = fmaf(y, t, 1.f);
  return fabsf(x) < 0.25f ? x * t * p.cap_out : far;
}

inline ScoreParams score_params(float scale, float softcap, const float* slopes) {
  ScoreParams s = {};
  s.slopes = slopes;
  s.mul = scale * kLog2e;
  s.slope_mul = (float)(1.0 / (double)scale);
  if (softcap > 0.f) {
    const double log2e = 1.4426950408889634;
    s.cap_in = (float)(2.0 * log2e * (double)scale / (double)softcap);
    s.cap_out = (float)((double)softcap * log2e);
    s.cap_lin = (float)((double)scale / (double)softcap);
    s.cap_wide = softcap > kWideCap;
    s.cap_score = s.cap_wide || slopes;
    s.mul = s.cap_score ? 1.f : 2.f * s.cap_out;
    s.add = s.cap_score ? 0.f : s.cap_out;
    s.slope_mul = kLog2e;
  }
  return s;
}

// Whether fp32 holds a scale, its cap and what is made of them (scale / cap too with all of its bits: rounded to 0
// it would make every score 0, and no cap of one).
inline bool score_range(float scale, float softcap) {
  const double most = 3e38, least = 1.2e-38, s = scale, c = softcap;
  if (!(scale > 0.f) || !(softcap >= 0.f) || !(s * 1.5 < most) || !(1.0 / s < most)) return false;
  return softcap == 0.f || (c * 3.0 < most && s / c * 3.0 < most && s / c > least);
}

}  // namespace tasft
