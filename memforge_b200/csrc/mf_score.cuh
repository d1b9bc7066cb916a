// Modified attention scores: capped, biased by distance, windowed, with a prefix.
#pragma once

#include "mf_internal.h"

namespace mf {

// Score modifiers, in this order: s = scale q.k; softcap > 0: s = softcap *
// tanh(s / softcap); slopes: s -= slopes[query head] * (query position - key
// position); then the mask.  Key k is visible to the row at position p iff
// k < kv_len and (k < prefix or ((not causal or k <= p) and (window == 0 or
// p - k < window))).
struct ScoreMods {
  float softcap;
  const float* slopes;    // [num_q_heads] or null
  int32_t window;         // 0: none
  const int32_t* prefix;  // [num_seqs] or null
  __host__ __device__ bool any() const {
    return softcap > 0.f || slopes != nullptr || window > 0 || prefix != nullptr;
  }
};

// Kernels take maxima of unscaled scores and mask those with -inf, which a negative or
// vanishing scale would turn into the largest.  (A NaN fails.)
inline bool scale_ok(float scale) { return scale >= 1e-9f && scale <= 1e9f; }

// (a smaller cap's reciprocal is not finite in fp32; a NaN fails both)
inline bool softcap_ok(float cap) { return cap == 0.f || (cap >= 1e-30f && cap <= 1e30f); }

// A window that reaches back behind every row's position (rows start at max_q_len - 1 before the
// first key at the earliest) hides nothing; bounded so that p - window + 1 stays in 32 bits.
inline int32_t bounded_window(int32_t window, int32_t max_q_len) {
  return window < INT32_MAX - max_q_len ? window : INT32_MAX - max_q_len;
}

constexpr float kLog2e = 1.4426950408889634f;

MF_DEVINL float rcp_approx(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// cap * tanh(s / cap) with score and result in log2 units: cap2 = cap * log2(e),
// two_over = 2 / cap (s2 = s * log2 e, so exp(2 s / cap) = 2^(s2 * 2 / cap)).
// From tanh(y) = 1 - 2 / (1 + exp(2y)): absolute error about cap2 * 2^-23, where the
// hardware's own tanh (relative 2^-11) would move a weight by cap * 2^-11.  An
// overflowing exponential gives rcp(inf) = 0, the cap itself.
MF_DEVINL float softcap_large_log2(float s2, float cap2, float two_over) {
  return fmaf(-2.f * cap2, rcp_approx(1.f + fast_exp2(s2 * two_over)), cap2);
}

// The same, and below a quarter of the cap its series (relative error 4e-7), so that the
// error stays within |s2| * 2^-21 however large the cap is.
MF_DEVINL float softcap_log2(float s2, float cap2, float two_over) {
  constexpr float H2 = 0.34657359f * 0.34657359f;  // (ln 2 / 2)^2: y = z ln 2 / 2
  const float z = s2 * two_over, u = z * z;
  const float t = fmaf(u, fmaf(u, fmaf(u, -17.f / 315.f * H2 * H2 * H2, 2.f / 15.f * H2 * H2),
                               -1.f / 3.f * H2), 1.f);
  return fabsf(z) < 0.72f ? s2 * t : softcap_large_log2(s2, cap2, two_over);
}

}  // namespace mf
