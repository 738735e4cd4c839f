// score_mod.h -- modified attention scores: the cap, the bias by distance and the key ranges that
// the kernels instantiated with MOD put between Q.K^T and the softmax (decode_kernels.h,
// prefill_kernels.h) and weights.hip recomputes.

#pragma once

#include "common.h"

namespace pkv {

// ---------------------------------------------------------------------------------
// Modified scores (kernels instantiated with MOD): what happens to a score between Q.K^T and
// the softmax, and which keys a query sees. Scores are in log2 units, d = scale log2(e) q.k:
//   cap:     d -> c2 tanh(d / c2), c2 = softcap log2(e), written c2 - 2 c2 / (1 + 2^(c1 d)) with
//            c1 = 2 / softcap (2^(c1 d) = e^(2 x) at x = s / softcap): one exp2 and one
//            reciprocal, saturating at +-c2 through exp2's infinity and zero;
//   slopes:  d -= slope[head] log2(e) |position of the query - position of the key|;
//   ranges:  the query in row r of q sees the keys ranges[r] = [first, last) of its context
//            (instead of the causal limit); a row whose range is empty gives 0.
// ---------------------------------------------------------------------------------
struct ScoreMod {
  float c1, c2;           // c2 = 0: no cap
  const float* slopes;    // [heads] or null
  const int32_t* ranges;  // [rows of q, 2] or null
  int64_t range_stride;
};

// d capped. EXACT (fp32 results): below |s / softcap| = 0.35 the difference above loses up to
// 2^-24 c2, which a weight turns into a relative error; there the odd series of tanh up to x^13
// (next term below 2^-25 x at 0.35) keeps fp32 relative to d.
template <bool EXACT>
__device__ __forceinline__ float capped(const ScoreMod& m, float d) {
  const float e = __builtin_amdgcn_exp2f(d * m.c1);
  const float t = __builtin_fmaf(-2.f * m.c2, __builtin_amdgcn_rcpf(1.f + e), m.c2);
  if constexpr (!EXACT) {
    return t;
  } else {
    const float x = d * m.c1 * 0.34657359f;  // (ln 2) / 2: s / softcap
    const float x2 = x * x;
    float p = __builtin_fmaf(x2, 21844.f / 6081075.f, -1382.f / 155925.f);
    p = __builtin_fmaf(x2, p, 62.f / 2835.f);
    p = __builtin_fmaf(x2, p, -17.f / 315.f);
    p = __builtin_fmaf(x2, p, 2.f / 15.f);
    p = __builtin_fmaf(x2, p, -1.f / 3.f);
    return fabsf(x) < 0.35f ? __builtin_fmaf(d * x2, p, d) : t;
  }
}
// d biased for a key `far` positions away (slope2 = slope log2(e)).
__device__ __forceinline__ float biased(float d, float slope2, int far) {
  return __builtin_fmaf(-slope2, fabsf((float)far), d);
}
constexpr float kLog2e = 1.4426950408889634f;

// The entry points' score arguments, checked. softcap 0: no cap. c1 and c2 stay finite and away
// from zero for every cap of fp32's normal range but its ends.
inline int score_mod(ScoreMod* m, float softcap, const float* slopes, const int32_t* ranges,
                     int64_t range_stride) {
  if (!(softcap == 0.f || (softcap >= 1e-30f && softcap <= 1e30f))) return PKV_E_SHAPE;
  if (ranges && range_stride < 0) return PKV_E_SHAPE;
  *m = {softcap > 0.f ? 2.f / softcap : 0.f, softcap * kLog2e, slopes, ranges, range_stride};
  return 0;
}

// A tile's raw scores s = q . k (RT row tiles of NB 16-key blocks, lane values [t][beta][r] =
// key 16 beta + r of row t) to modified ones in log2 units; far[t]: the distance from row t's query
// back to the lane's key beta = r = 0.
template <int RT, int NB>
__device__ __forceinline__ void modify_scores(f32x4 (&sc)[RT][NB], const ScoreMod& m, float scale_log2,
                                              const float (&slope2)[RT], const int (&far)[RT]) {
#pragma unroll
  for (int t = 0; t < RT; ++t)
#pragma unroll
    for (int beta = 0; beta < NB; ++beta) sc[t][beta] *= scale_log2;
  if (m.c2 != 0.f) {  // uniform
#pragma unroll
    for (int t = 0; t < RT; ++t)
#pragma unroll
      for (int beta = 0; beta < NB; ++beta)
#pragma unroll
        for (int r = 0; r < 4; ++r) sc[t][beta][r] = capped<false>(m, sc[t][beta][r]);
  }
  if (m.slopes) {
#pragma unroll
    for (int t = 0; t < RT; ++t)
#pragma unroll
      for (int beta = 0; beta < NB; ++beta)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          sc[t][beta][r] = biased(sc[t][beta][r], slope2[t], far[t] - 16 * beta - r);
  }
}

}  // namespace pkv
