// decode_mod.hip -- paged decode attention with modified scores (include/paged_kv.h:
// pkv_paged_decode_mod): the MOD instantiations of the decode kernels and their launches. The
// checks, the split and the workspace are decode.hip's.

#include "decode_dispatch.h"

namespace {

template <int DT, int HD, int GPW> struct ModKernels {
  static constexpr int G = stream_gpw<HD, GPW>();
  using Fn = void (*)(DecodeArgs);
  // The stream pass: blocks of a multiple of 16 tokens (fast), the batch's lengths in LDS (staged).
  static Fn stream(bool fast, bool staged) {
    if constexpr (use_mfma<DT, HD>()) {
      if (fast)
        return staged ? &paged_decode_mfma_kernel<DT, G, true, HD, false, true, true, true>
                      : &paged_decode_mfma_kernel<DT, G, true, HD, false, false, true, true>;
      return staged ? &paged_decode_mfma_kernel<DT, G, false, HD, false, true, true, true>
                    : &paged_decode_mfma_kernel<DT, G, false, HD, false, false, true, true>;
    } else {
      return &paged_decode_stream_kernel<DT, HD, GPW, true, true>;
    }
  }
};

struct LaunchMod {
  const DecodeArgs* a;
  int wpg, ygrid;
  hipStream_t st;
  template <int DT, int HD, int GPW> hipError_t run() const {
    const dim3 grid((unsigned)a->num_wg, (unsigned)ygrid), block(kWave * wpg);
    const bool staged = a->batch > kWave && a->batch <= kLdsBatch;
    hipLaunchKernelGGL((ModKernels<DT, HD, GPW>::stream(a->bs % 16 == 0, staged)), grid, block,
                       (stream_lds<DT, HD, GPW>(wpg)), st, *a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || a->num_wg <= 1) return e;
    launch_combine<DT, HD, false, true, true>(*a, st);
    return hipGetLastError();
  }
};

struct LaunchModSplit {
  const DecodeArgs* a;
  int ytasks;
  hipStream_t st;
  template <int DT, int HD, int GPW> hipError_t run() const {
    if constexpr (use_mfma<DT, HD>()) {
      const dim3 grid((unsigned)a->batch, (unsigned)ytasks), block(kWave * kSplitWaves);
      const unsigned lds = pv_mfma<HD, GPW, true>() ? kSplitWaves * kVSlotBytes : 0;
      if (a->bs % 16 == 0)
        hipLaunchKernelGGL((paged_decode_mfma_kernel<DT, GPW, true, HD, true, false, false, true>),
                           grid, block, lds, st, *a);
      else
        hipLaunchKernelGGL((paged_decode_mfma_kernel<DT, GPW, false, HD, true, false, false, true>),
                           grid, block, lds, st, *a);
      return hipGetLastError();
    } else {
      return hipErrorInvalidValue;  // never chosen for these shapes
    }
  }
};

struct QueryMod {
  int wpg;
  int* per_cu;
  template <int DT, int HD, int GPW> hipError_t run() const {
    return hipOccupancyMaxActiveBlocksPerMultiprocessor(
        per_cu, reinterpret_cast<const void*>(ModKernels<DT, HD, GPW>::stream(true, false)),
        kWave * wpg, stream_lds<DT, HD, GPW>(wpg));
  }
};

}  // namespace

namespace pkv {

hipError_t launch_decode_mod(const DecodeArgs& a, int kv_dtype, int head_dim, int wpg, int ygrid,
                             bool split, hipStream_t st) {
  if (split) return by_dtype(kv_dtype, head_dim, a.gpw, LaunchModSplit{&a, ygrid, st});
  return by_dtype(kv_dtype, head_dim, a.gpw, LaunchMod{&a, wpg, ygrid, st});
}

hipError_t decode_mod_per_cu(int kv_dtype, int head_dim, int gpw, int wpg, int* per_cu) {
  return by_dtype(kv_dtype, head_dim, gpw, QueryMod{wpg, per_cu});
}

}  // namespace pkv
