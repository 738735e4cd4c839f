// prefill_mod.hip -- chunked-prefill attention with modified scores (include/paged_kv.h:
// pkv_paged_prefill_mod) on the matrix cores: the MOD instantiations of prefill_kernels.h's
// kernel. The checks and the fp32 kernel are prefill.hip's.

#include "prefill_kernels.h"

namespace {

using namespace pkv;

template <int DT, int HD, bool V16> hipError_t launch_hd(PrefillArgs a, int64_t rows, hipStream_t st) {
  constexpr int BM = PrefillShape<HD>::BM;
  a.row_blocks = (int)((rows + BM - 1) / BM);
  const int64_t items = (int64_t)a.row_blocks * a.nkv * a.n_chunks;
  if (items > 0x7FFFFFFF) return hipErrorInvalidValue;
  const dim3 grid((unsigned)items), block(512);
  // Block sizes that are no power of two have the general kernel only; a bias in units of tiny scales
  // could overflow.
  const bool bias_only = a.mod.c2 == 0.f && a.scale_log2 >= 1e-12f;
  const int mod = a.bs_shift < 0 ? 0 : a.mod.slopes ? (bias_only ? kModBias : kModAny)
                                                    : (a.mod.c2 != 0.f ? kModCap : kModRanges);
  auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, block, 0, st, a); };
  switch (mod) {
    case kModRanges: go(paged_prefill_kernel<DT, HD, true, V16, true, kModRanges>); break;
    case kModCap: go(paged_prefill_kernel<DT, HD, true, V16, true, kModCap>); break;
    case kModBias: go(paged_prefill_kernel<DT, HD, true, V16, true, kModBias>); break;
    case kModAny: go(paged_prefill_kernel<DT, HD, true, V16, true, kModAny>); break;
    default: go(paged_prefill_kernel<DT, HD, false, V16, true, kModAny>);
  }
  return hipGetLastError();
}

template <int DT, bool V16>
hipError_t launch(const PrefillArgs& a, int hd, int64_t rows, hipStream_t st) {
  switch (hd) {
    case 32: return launch_hd<DT, 32, V16>(a, rows, st);
    case 64: return launch_hd<DT, 64, V16>(a, rows, st);
    case 128: return launch_hd<DT, 128, V16>(a, rows, st);
    default: return launch_hd<DT, 256, V16>(a, rows, st);
  }
}

}  // namespace

namespace pkv {

hipError_t launch_prefill_mod(PrefillArgs a, int kv_dtype, int head_dim, int64_t rows, hipStream_t st) {
  cap_series(&a.mod, a.scale_log2);
  if (kv_dtype == PKV_F16) return launch<PKV_F16, false>(a, head_dim, rows, st);
  return a.v16 ? launch<PKV_BF16, true>(a, head_dim, rows, st)
               : launch<PKV_BF16, false>(a, head_dim, rows, st);
}

}  // namespace pkv
