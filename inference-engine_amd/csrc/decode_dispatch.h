// decode_dispatch.h -- from runtime (dtype, head_dim, heads per wave) to the decode kernels'
// instantiations, and the launch of the combine: shared by decode.hip (plain scores) and
// decode_mod.hip (modified scores).

#pragma once

#include "decode_kernels.h"

namespace {

using namespace pkv;

// The MFMA kernel serves 16-bit K/V at head_dim 64 and 128; every other shape uses the
// generic stream kernel.
template <int DT, int HD> constexpr bool use_mfma() {
  return DT != PKV_F32 && (HD == 128 || HD == 64) && PKV_DECODE_USE_MFMA;
}

// Run f.run<DT, HD, GPW>() for the runtime (dtype, head_dim, heads per wave).
template <int DT, int HD, class F> hipError_t by_gpw(int gpw, const F& f) {
  switch (gpw) {
    case 1: return f.template run<DT, HD, 1>();
    case 2: return f.template run<DT, HD, 2>();
    case 3: return f.template run<DT, HD, 3>();
    case 4: return f.template run<DT, HD, 4>();
    default:  // only planned where the MFMA kernel serves the shape (plan_decode)
      if constexpr (use_mfma<DT, HD>()) return f.template run<DT, HD, kWideHeads>();
      else return hipErrorInvalidValue;
  }
}
template <int DT, class F> hipError_t by_hd(int hd, int gpw, const F& f) {
  switch (hd) {
    case 16: return by_gpw<DT, 16>(gpw, f);
    case 32: return by_gpw<DT, 32>(gpw, f);
    case 64: return by_gpw<DT, 64>(gpw, f);
    case 128: return by_gpw<DT, 128>(gpw, f);
    default: return by_gpw<DT, 256>(gpw, f);
  }
}
template <class F> hipError_t by_dtype(int dt, int hd, int gpw, const F& f) {
  switch (dt) {
    case PKV_F32: return by_hd<PKV_F32>(hd, gpw, f);
    case PKV_F16: return by_hd<PKV_F16>(hd, gpw, f);
    default: return by_hd<PKV_BF16>(hd, gpw, f);
  }
}

// Dynamic LDS of the stream pass's workgroups of wpg waves.
template <int DT, int HD, int GPW> constexpr unsigned stream_lds(int wpg) {
  return use_mfma<DT, HD>() && pv_mfma<HD, GPW>() ? (unsigned)(wpg * kVSlotBytes) : 0u;
}

// Waves the combine gives each (sequence, head) pair: there are as many ranges for any
// batch, so with few pairs each has many records, and one wave folds them in dependent
// trips of a few rows each. Whole decode calls with 1 / 2 / 4 / 8 / 16 waves per pair (us):
//   32 pairs (1 sequence of 20,011 tokens, hd 128)  45.2 / 34.8 / 28.7 / 26.2 / 25.7
//   64 pairs (2 sequences of 3,000-9,000)           33.7 / 26.8 / 21.9 / 20.6 / 20.5
//   128 pairs (4 such)                              32.8 / 29.3 / 27.1 / 26.2 / 26.8
//   256 pairs (8 such)                              42.6 / 41.1 / 39.6 / 39.8 / 40.3
//   512 pairs (16 of 1,000-4,000)                   35.0 / 34.2 / 34.1 / 34.4 / 38.0
//   1,024 pairs (64 of 200-3,000, 16 heads)         71.3 / 71.4 / 72.1 / 74.6 / 77.9
//   1,024 pairs (32 of 128-32,768, log)            106.9 / 105.7 / 105.0 / 106.5 / 110.1
//   1,536 pairs (64 of 1,024-4,096, 24 heads)      109.8 / 110.0 / 111.6 / 115.0 / 119.8
//   768 pairs (24 of 3,000-9,000, 24 heads)        103.4 / 101.8 / 104.2 / 105.3 / 112.0
//   1,024 pairs (32 of 2,060-2,200)                 56.9 / 54.5 / 56.1 / 57.2 / 64.4
//   32 pairs, hd 256 (1 of 20,011)                  65.6 / 54.0 / 47.0 / 44.4 / 44.4
//   8 pairs, hd 256 (1 of 9,000, 8 heads)          122.2 / 74.6 / 43.8 / 34.0 / 30.3
// (Two libraries in turn on the same buffers, hd 128: four waves up to 1,024 pairs gain 0.4-0.9%
// where a few long sequences have most of the ranges, 32 or 24 of 128-32,768, and lose 1-2% where
// lengths are even: 45.3 against 45.9 us for 64 of 200-3,000, 55.9 against 56.6 for 32 of
// 2,060-2,200.)
int combine_waves(const DecodeArgs& a) {
  const int pairs = a.batch * a.nh;
  if (pairs <= 64) return 16;
  if (pairs <= 256) return 8;
  if (pairs <= 512) return 4;
  return pairs <= PKV_DECODE_COMBINE_SPLIT_PAIRS ? 2 : 1;
}
template <int DT, int HD, int SP, bool WT, bool ROWS, bool MOD = false>
void launch_combine_sp(const DecodeArgs& a, hipStream_t st) {
  constexpr int WG = SP > 4 ? SP : 4;  // waves per workgroup
  const int pairs = a.batch * a.nh;
  hipLaunchKernelGGL((paged_decode_combine_kernel<DT, HD, SP, WT, ROWS, MOD>),
                     dim3((unsigned)((pairs + WG / SP - 1) / (WG / SP))), dim3(kWave * WG), 0, st, a);
}
template <int DT, int HD, bool WT, bool ROWS, bool MOD = false>
void launch_combine(const DecodeArgs& a, hipStream_t st) {
  switch (combine_waves(a)) {
    case 16: return launch_combine_sp<DT, HD, 16, WT, ROWS, MOD>(a, st);
    case 8: return launch_combine_sp<DT, HD, 8, WT, ROWS, MOD>(a, st);
    case 4: return launch_combine_sp<DT, HD, 4, WT, ROWS, MOD>(a, st);
    case 2: return launch_combine_sp<DT, HD, 2, WT, ROWS, MOD>(a, st);
    default: return launch_combine_sp<DT, HD, 1, WT, ROWS, MOD>(a, st);
  }
}

}  // namespace

namespace pkv {

// decode_mod.hip: the stream pass and its combine (or, with split, the per-sequence split pass of
// `ygrid` tasks) with modified scores.
hipError_t launch_decode_mod(const DecodeArgs& a, int kv_dtype, int head_dim, int wpg, int ygrid,
                             bool split, hipStream_t st);
// decode_mod.hip: how many of the stream pass's workgroups of wpg waves one CU holds at once.
hipError_t decode_mod_per_cu(int kv_dtype, int head_dim, int gpw, int wpg, int* per_cu);

}  // namespace pkv
