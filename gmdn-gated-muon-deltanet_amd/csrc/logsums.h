// Running sums of a softmax over a row of logits x: with the largest logit m,
// s = sum e^(x - m) and w = sum e^(x - m) (x - m), for the log probabilities and
// the entropy; rescaled where m grows, joined over lanes, and what they say.
#pragma once
#include <float.h>
#include "rows8.h"

namespace gmdn {
namespace {

constexpr float LOG2E = 1.44269504088896340736f;
// Differences of logits are clamped here where they multiply a sum: e^-200
// is 0 in float32, and 0 times the clamped value is 0, not NaN.
constexpr float FAR = -200.f;

GMDN_DEV float exp_of(float x) { return __builtin_amdgcn_exp2f(x * LOG2E); }

struct Sums {
  float m, s, w;
};
GMDN_DEV Sums no_sums() { return {-FLT_MAX, 0.f, 0.f}; }

// Rescale to the maximum m >= a.m.  NaN stays in s; an infinite m makes its
// own terms NaN.
GMDN_DEV void rescale(Sums& a, float m) {
  const float u = fmaxf(a.m - m, FAR), k = exp_of(u);
  a.w = k * (a.w + u * a.s);
  a.s *= k;
  a.m = m;
}

// The sums of N lanes' Sums, in each of them.
template <int N>
GMDN_DEV Sums join_lanes(Sums a) {
  rescale(a, lanes_max<N>(a.m));
  a.s = lanes_sum<N>(a.s);
  a.w = lanes_sum<N>(a.w);
  return a;
}

// What a row's sums say.  No logit above -inf: s = 0, and the row's
// distribution is empty (stats -inf, 0).
struct Row {
  float m, logs, entropy;
  bool empty;
  GMDN_DEV float logprob(float x) const { return empty ? -INFINITY : x - m - logs; }
};
GMDN_DEV Row row_of(const Sums& a) {
  if (a.s == 0.f) return {-INFINITY, 0.f, 0.f, true};
  const float logs = logf(a.s), h = logs - a.w / a.s;
  return {a.m, logs, h < 0.f ? 0.f : h, false};
}

}  // namespace
}  // namespace gmdn
