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
  float series[2], series_max;  // cap_series; read by the matrix-core prefill
};

// Which of them a kernel is made for (prefill_kernels.h).
constexpr int kModRanges = 1, kModCap = 2, kModBias = 3, kModAny = 4;

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

// The entry points' score arguments, checked. softcap 0: no cap. Its upper bound keeps the error of
// the 16-bit kernels' cap, some 2^-21 of it, below that of their weights.
inline int score_mod(ScoreMod* m, float softcap, const float* slopes, const int32_t* ranges,
                     int64_t range_stride) {
  if (!(softcap == 0.f || (softcap >= 1e-30f && softcap <= 1000.f))) return PKV_E_SHAPE;
  if (ranges && range_stride < 0) return PKV_E_SHAPE;
  *m = {softcap > 0.f ? 2.f / softcap : 0.f, softcap * kLog2e, slopes, ranges, range_stride, {}, -1.f};
  return 0;
}

// The cap of a raw score s as an odd polynomial, for |s| <= series_max (0.3 of the cap): with
// x = scale_log2 s / c2, c2 tanh(x) = s (scale_log2 + s^2 (series[0] + s^2 series[1])). The coefficients
// are the minimax ones of tanh(x) - x over [0, 0.3] (a linear program over 4,001 points): off by at most
// 3.0e-07, relative 2.0e-06. series_max = -1 (no score) without a cap and where the coefficients could
// over- or underflow.
inline void cap_series(ScoreMod* m, float scale_log2) {
  const double f = (double)scale_log2 / m->c2, co[2] = {-0.33312109, 0.12640677};
  m->series_max = -1.f;
  if (m->c2 == 0.f || !(f <= 1e4)) return;
  double g = scale_log2;
  for (int i = 0; i < 2; ++i) m->series[i] = (float)(co[i] * (g *= f * f));
  if (m->series[1] >= 1e-37f) m->series_max = (float)(0.3 / f);  // 0 would take -inf to NaN
}

// A tile's raw scores s = q . k (RT row tiles of NB 16-key blocks, lane values [t][beta][r] =
// key 16 beta + r of row t) to capped and biased ones in log2 units; far[t]: the distance from row
// t's query back to the lane's key beta = r = 0. SERIES: the polynomial of cap_series where all of the
// wave's scores allow it.
template <bool SERIES, int RT, int NB>
__device__ __forceinline__ void modify_scores(f32x4 (&sc)[RT][NB], const ScoreMod& m, float scale_log2,
                                              const float (&slope2)[RT], const int (&far)[RT]) {
  if (m.c2 != 0.f) {  // uniform
    [[maybe_unused]] float top = 0.f;
    if constexpr (SERIES) {
#pragma unroll
      for (int t = 0; t < RT; ++t)
#pragma unroll
        for (int beta = 0; beta < NB; ++beta)
#pragma unroll
          for (int r = 0; r < 4; ++r) top = fmaxf(top, fabsf(sc[t][beta][r]));
    }
    auto each = [&](auto cap) __attribute__((always_inline)) {
#pragma unroll
      for (int t = 0; t < RT; ++t)
#pragma unroll
        for (int beta = 0; beta < NB; ++beta)
#pragma unroll
          for (int r = 0; r < 4; ++r) sc[t][beta][r] = cap(sc[t][beta][r]);
    };
    if (!SERIES || __builtin_amdgcn_ballot_w64(top > m.series_max))
      each([&](float x) { return capped<false>(m, x * scale_log2); });
    else
      each([&](float x) {
        const float y = x * x;
        return x * __builtin_fmaf(y, __builtin_fmaf(y, m.series[1], m.series[0]), scale_log2);
      });
    scale_log2 = 1.f;
  }
#pragma unroll
  for (int t = 0; t < RT; ++t) {
    const float f0 = (float)far[t];
#pragma unroll
    for (int beta = 0; beta < NB; ++beta)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        sc[t][beta][r] = __builtin_fmaf(sc[t][beta][r], scale_log2, -slope2[t] * fabsf(f0 - (float)(16 * beta + r)));
  }
}

}  // namespace pkv
