// weights.hip -- accumulated attention weights (include/paged_kv.h: pkv_attention_weights): for
// every cached token, the softmax weights that a step's queries give it, summed over queries and
// heads, from the normalisers that the attention call left.

#include "score_mod.h"

namespace {

using namespace pkv;

struct WeightsArgs {
  float* w;  // row r, token p: w[r * w_stride + p]
  int64_t w_stride, w_num;
  const int64_t* w_rows;  // [n_chunks] or null (row c)
  float decay;
  const void* q;
  int64_t q_st, q_sh;
  const void* k;
  int64_t kv_ss, kv_sh, num_slots;
  const int32_t* tables;
  int64_t table_stride;
  int32_t max_blocks;
  const int32_t* ctx;
  const int32_t* cu_q;  // [n_chunks + 1] or null (one query per chunk)
  const float* lse;     // [tokens, nh]
  int32_t n_chunks, nh, nkv, groups, bs, bs_shift;
  int32_t max_queries;  // query tokens of a chunk that count
  int32_t tw;           // few rows: waves that take different KV heads; the others share the keys
  int32_t span;         // keys per workgroup
  int32_t kblocks;      // spans per chunk
  float* ws;            // many rows: [n_chunks, nkv, max_blocks * bs], the KV heads' sums
  float scale_log2;
  ScoreMod mod;
};

// ---------------------------------------------------------------------------------
// w[p] = decay w[p] + sum over queries t and heads h of 2^(s(t, h, p) - lse(t, h)).
//
// Scores on the matrix cores, 16 query rows (token, head of a KV head's group; A) by 16 keys (B): lane
// (col, grp) holds dims 4 VEC m + VEC grp .. of row / key col and gets the scores of rows 4 grp + r for
// key col. Every score becomes its weight; a lane adds over the rows it sees, the four rows of lanes
// are added by two swaps, and the waves (and KV heads) that share a key in a fixed order, without
// atomics.
// ---------------------------------------------------------------------------------

template <int DT, int HD> struct WShape {
  static constexpr int VEC = vec16<DT>();
  static constexpr int NF = HD >= 4 * VEC ? HD / (4 * VEC) : 1;  // 16-byte pieces of a row per lane
};

template <int DT, int HD>
__device__ __forceinline__ f32x4 score_tile(const u32x4* qf, const u32x4* kf) {
  f32x4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int m = 0; m < WShape<DT, HD>::NF; ++m) {
    if constexpr (DT == PKV_F32) {
      const f32x4 a = __builtin_bit_cast(f32x4, qf[m]), b = __builtin_bit_cast(f32x4, kf[m]);
#pragma unroll
      for (int j = 0; j < 4; ++j) s = __builtin_amdgcn_mfma_f32_16x16x4f32(a[j], b[j], s, 0, 0, 0);
    } else if constexpr (DT == PKV_BF16) {
      typedef __bf16 v8 __attribute__((ext_vector_type(8)));
      s = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8, qf[m]),
                                                  __builtin_bit_cast(v8, kf[m]), s, 0, 0, 0);
    } else {
      typedef _Float16 v8 __attribute__((ext_vector_type(8)));
      s = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8, qf[m]),
                                                 __builtin_bit_cast(v8, kf[m]), s, 0, 0, 0);
    }
  }
  return s;
}

__device__ __forceinline__ int wave_min(int x) {
#pragma unroll
  for (int off = 1; off < kWave; off <<= 1) x = min(x, __shfl_xor(x, off));
  return __builtin_amdgcn_readfirstlane(x);
}

// The workgroup's chunk.
struct WChunk {
  int c, n, q0, qlen, nrows, base_pos;
  int64_t wrow;
};
__device__ __forceinline__ WChunk w_chunk(const WeightsArgs& a, int c) {
  WChunk k;
  k.c = c;
  k.n = min(max(a.ctx[c], 0), a.max_blocks * a.bs);
  k.wrow = a.w_rows ? a.w_rows[c] : c;
  k.q0 = a.cu_q ? a.cu_q[c] : c;
  const int len = a.cu_q ? max(a.cu_q[c + 1] - k.q0, 0) : 1;
  k.base_pos = k.n - len;
  k.qlen = min(len, a.max_queries);
  k.nrows = k.qlen * a.groups;
  return k;
}

// What a wave keeps in LDS of its 16 RT query rows: visible keys [lo, hi), position, slope (as bits),
// and the normalisers, +inf (weight 0) for rows past the last and rows that saw no key.
template <int RT> struct RowLds {
  int4 meta[16 * RT];
  float lse[16 * RT];
};

// RT tiles of 16 query rows of one KV head, from row row0 on (rows past the last repeat row0).
// first .. last: the keys that any row sees; every row sees [lo_max, hi_min). Wave-uniform.
template <int DT, int HD, int RT> struct WRows {
  u32x4 q[RT][WShape<DT, HD>::NF];
  float lse[RT][4];  // of rows 16 t + 4 grp + r
  int first, last, lo_max, hi_min;

  // The bounds, and lane i's row i to LDS.
  __device__ __forceinline__ void rows(const WeightsArgs& a, const WChunk& k, int kvh, int row0, RowLds<RT>& l) {
    const int i = (threadIdx.x & (kWave - 1)) & (16 * RT - 1), rho = row0 + i, G = a.groups;
    const bool ok = rho < k.nrows;
    const int tok = (ok ? rho : row0) / G, head = kvh * G + (ok ? rho : row0) - tok * G;
    const float x = a.lse[(int64_t)(k.q0 + tok) * a.nh + head];
    const float slope = a.mod.slopes ? a.mod.slopes[head] * kLog2e : 0.f;
    int lo = 0, hi = k.base_pos + tok + 1;
    if (a.mod.ranges) {
      const int32_t* r = a.mod.ranges + (int64_t)(k.q0 + tok) * a.mod.range_stride;
      lo = max(r[0], 0);
      hi = min(r[1], k.n);
      first = wave_min(lo < hi ? lo : 0x7FFFFFFF);
      last = -wave_min(lo < hi ? -hi : 0);
      lo_max = -wave_min(-lo);
      hi_min = wave_min(hi);
    } else {  // causal: rows are in the order of their tokens
      first = lo_max = 0;
      last = k.base_pos + (min(row0 + 16 * RT, k.nrows) - 1) / G + 1;
      hi_min = k.base_pos + row0 / G + 1;
    }
    const bool empty = x == -INFINITY;
    if (__ballot(ok & empty)) hi_min = -1;  // the masked form leaves such rows out, whatever their keys hold
    l.meta[i] = make_int4(lo, hi, k.base_pos + tok, __float_as_int(slope));
    l.lse[i] = !ok | empty ? INFINITY : x;
  }
  __device__ __forceinline__ void load_q(const WeightsArgs& a, const WChunk& k, int kvh, int row0) {
    using S = typename Elt<DT>::S;
    constexpr int VEC = WShape<DT, HD>::VEC, NF = WShape<DT, HD>::NF;
    const int lane = threadIdx.x & (kWave - 1), col = lane & 15, grp = lane >> 4, G = a.groups;
    const bool dims = HD >= 4 * VEC || grp * VEC < HD;  // head_dim 16 of a 16-bit type: half the lanes
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      const int rho = row0 + 16 * t + col, rr = rho < k.nrows ? rho : row0, tok = rr / G;
      const S* qp = reinterpret_cast<const S*>(a.q) + (int64_t)(k.q0 + tok) * a.q_st +
                    (int64_t)(kvh * G + rr - tok * G) * a.q_sh + (dims ? VEC * grp : 0);
#pragma unroll
      for (int m = 0; m < NF; ++m) q[t][m] = *reinterpret_cast<const u32x4*>(qp + (dims ? 4 * VEC * m : 0));
      if (!dims) q[t][0] = u32x4{0, 0, 0, 0};
    }
  }
  __device__ __forceinline__ void load_lse(const RowLds<RT>& l) {
    const int grp = (threadIdx.x & (kWave - 1)) >> 4;
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      const float4 x = *reinterpret_cast<const float4*>(&l.lse[16 * t + 4 * grp]);
      lse[t][0] = x.x, lse[t][1] = x.y, lse[t][2] = x.z, lse[t][3] = x.w;
    }
  }
  // The same where every row sees every key of the tile and scores are as they are.
  __device__ __forceinline__ float plain_weight(const WeightsArgs& a, const f32x4 (&s)[RT]) const {
    float acc[2] = {0.f, 0.f};
#pragma unroll
    for (int t = 0; t < RT; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        acc[r & 1] += __builtin_amdgcn_exp2f(__builtin_fmaf(s[t][r], a.scale_log2, -lse[t][r]));
    return acc[0] + acc[1];
  }
  // The weights of key kt + col over this lane's rows, from the tile's scores. here: the key exists.
  __device__ __forceinline__ float weight(const WeightsArgs& a, const RowLds<RT>& l, const f32x4 (&s)[RT],
                                          int kt, bool here, bool plain) const {
    if (plain && lo_max <= kt && kt + 16 <= hi_min && __ballot(here) == ~0ull)  // uniform
      return plain_weight(a, s);
    float acc[2] = {0.f, 0.f};
    const int lane = threadIdx.x & (kWave - 1), key = kt + (lane & 15), grp = lane >> 4;
#pragma unroll
    for (int t = 0; t < RT; ++t) {
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int4 m = l.meta[16 * t + 4 * grp + r];
        float d = s[t][r] * a.scale_log2;
        if (a.mod.c2 != 0.f) d = capped<DT == PKV_F32>(a.mod, d);
        if (a.mod.slopes) d = biased(d, __int_as_float(m.w), m.z - key);
        const bool sees = (key >= m.x) & (key < m.y) & here & (lse[t][r] != INFINITY);
        acc[r & 1] += sees ? __builtin_amdgcn_exp2f(d - lse[t][r]) : 0.f;
      }
    }
    return acc[0] + acc[1];
  }
};
// x[l] + x[l ^ 32] in the lower 32 lanes, y's in the upper ones; likewise for rows of 16 lanes (x's
// in the even rows, y's in the odd ones).
__device__ __forceinline__ float swap_add32(float x, float y) {
  const auto p = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(y), false, false);
  return __uint_as_float(p[0]) + __uint_as_float(p[1]);
}
__device__ __forceinline__ float swap_add16(float x, float y) {
  const auto p = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(y), false, false);
  return __uint_as_float(p[0]) + __uint_as_float(p[1]);
}
// LDS that one wave wrote for itself may be read.
__device__ __forceinline__ void wave_lds_fence() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// Few rows (at most 16 per KV head: decode): a workgroup takes `span` keys of one chunk. Its waves
// take KV heads (or, where these are fewer than the waves, shares of the keys) and stream their K rows
// past the queries, which stay in registers, the next TP tiles in flight under the current ones.
// Bound by reading K once; the span's block ids arrive in one trip, as slots in LDS.
constexpr int kFewRows = 16, kFewWaves = 8, kFewSpan = 512;
template <int DT, int HD> constexpr int few_tiles() {  // 4 KB a wave and stage
  return WShape<DT, HD>::NF >= 4 ? 1 : 4 / WShape<DT, HD>::NF;
}
// Waves per SIMD asked for: two workgroups per CU where that spills nothing.
template <int DT, int HD> constexpr int few_occupancy() { return WShape<DT, HD>::NF <= 4 ? 4 : 2; }

template <int DT, int HD>
__global__ void __launch_bounds__(kFewWaves * kWave, (few_occupancy<DT, HD>()))
attention_weights_few_kernel(const WeightsArgs a) {
  using SH = WShape<DT, HD>;
  using S = typename Elt<DT>::S;
  constexpr int VEC = SH::VEC, NF = SH::NF, TP = few_tiles<DT, HD>(), STEP = 16 * TP;
  static_assert(kFewSpan == kFewWaves * kWave, "a thread per key");
  __shared__ __align__(16) float sums[kFewWaves][kFewSpan];
  __shared__ int slots[kFewSpan];
  __shared__ __align__(16) RowLds<1> row_lds[kFewWaves];

  const int tid = threadIdx.x, lane = tid & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  const int col = lane & 15, grp = lane >> 4;
  const unsigned item = blockIdx.y * gridDim.x + blockIdx.x;
  const int c = (int)(item / (unsigned)a.kblocks);
  if (c >= a.n_chunks) return;
  const int kg = (int)(item % (unsigned)a.kblocks) * a.span;  // the workgroup's first key
  const int pk = kg + tid;                                    // this thread's
  const int blk = a.bs_shift >= 0 ? pk >> a.bs_shift : pk / a.bs;
  const int id = tid < a.span && pk < a.max_blocks * a.bs ? a.tables[(int64_t)c * a.table_stride + blk] : -1;
  const WChunk k = w_chunk(a, c);
  if (kg >= k.n || k.wrow < 0 || k.wrow >= a.w_num) return;  // uniform
  float* const w = a.w + k.wrow * a.w_stride + pk;
  const bool mine = tid < a.span && pk < k.n;
  const float old = mine && a.decay != 0.f ? *w : 0.f;
  if (tid < a.span) {
    const int64_t sl = (int64_t)id * a.bs + (pk - blk * a.bs);
    slots[tid] = mine && id >= 0 && sl < a.num_slots ? (int)sl : -1;  // num_slots < 2^31 (launch)
#pragma unroll
    for (int v = 0; v < kFewWaves; ++v) sums[v][tid] = 0.f;
  }
  __syncthreads();

  const int sub = wave / a.tw, share = a.span / (kFewWaves / a.tw);  // this wave's keys of the span
  const int kw = kg + sub * share, kw_end = min(k.n, kw + share);
  const bool dims = HD >= 4 * VEC || grp * VEC < HD;
  const bool plain = a.mod.c2 == 0.f && !a.mod.slopes;  // scores as they are
  WRows<DT, HD, 1> rows;
  for (int kvh = wave & (a.tw - 1); k.nrows > 0 && kvh < a.nkv; kvh += a.tw) {
    rows.rows(a, k, kvh, 0, row_lds[wave]);
    // Tiles of this wave's keys that some row sees.
    const int k_beg = max(kw, kw + (max(rows.first, kw) - kw) / 16 * 16), k_end = min(kw_end, rows.last);
    const S* const kb = reinterpret_cast<const S*>(a.k) + (int64_t)kvh * a.kv_sh + (dims ? VEC * grp : 0);
    auto load_stage = [&](int k0, u32x4 (&kf)[TP][NF], int (&sl)[TP]) __attribute__((always_inline)) {
#pragma unroll
      for (int t = 0; t < TP; ++t) {
        const int p = k0 + 16 * t + col;  // past the wave's keys: no key
        sl[t] = p < kw_end ? slots[min(p - kg, a.span - 1)] : -1;
      }
#pragma unroll
      for (int t = 0; t < TP; ++t) {
        const S* row = kb + (int64_t)max(sl[t], 0) * a.kv_ss;  // no key: row 0, masked
#pragma unroll
        for (int m = 0; m < NF; ++m)
          kf[t][m] = *reinterpret_cast<const u32x4*>(row + (dims ? 4 * VEC * m : 0));
      }
    };
    u32x4 ka[TP][NF], kn[TP][NF];
    int sa[TP], sn[TP];
    if (k_beg >= k_end) continue;
    load_stage(k_beg, ka, sa);
    rows.load_q(a, k, kvh, 0);
    wave_lds_fence();
    rows.load_lse(row_lds[wave]);
    auto use_stage = [&](int k0, const u32x4 (&kf)[TP][NF], const int (&sl)[TP]) __attribute__((always_inline)) {
#pragma unroll
      for (int t = 0; t < TP; ++t) {
        const int kt = k0 + 16 * t;
        if (kt >= k_end) break;  // uniform
        const f32x4 s[1] = {score_tile<DT, HD>(rows.q[0], kf[t])};
        const float v = rows_sum(rows.weight(a, row_lds[wave], s, kt, sl[t] >= 0, plain));
        if (grp == 0) sums[wave][kt - kg + col] += v;
      }
    };
    for (int k0 = k_beg; k0 < k_end; k0 += 2 * STEP) {
      if (k0 + STEP < k_end) load_stage(k0 + STEP, kn, sn);
      use_stage(k0, ka, sa);
      if (k0 + STEP >= k_end) break;
      if (k0 + 2 * STEP < k_end) load_stage(k0 + 2 * STEP, ka, sa);
      use_stage(k0 + STEP, kn, sn);
    }
  }
  __syncthreads();
  if (mine) {
    float v = 0.f;
#pragma unroll
    for (int i = 0; i < kFewWaves; ++i) v += sums[i][tid];
    *w = a.decay != 0.f ? __builtin_fmaf(old, a.decay, v) : v;
  }
}

// Many rows (a prompt's queries): one workgroup per (chunk, KV head, `span` keys). Its 8 waves keep 16
// RT query rows each in registers and all walk over the span's keys, TK at a time through LDS (rows
// padded by 16 bytes: the operand reads of 16 keys then cover all banks), the next tile's K on its
// way under this one's scores. Each KV head's sums go to the workspace, and a second launch adds them
// up in the order of the heads, with the decay. Bound by vector instructions: an exp2, a
// multiply-add and an add per score. 8 prompts of 64 queries over 2,000-8,000 tokens, 32 / 8 heads, hd
// 128, bf16: 41 us and 4 for the second launch; 46 before tiles that every row sees whole had a path
// without a branch per 16 keys. (With all KV heads in one workgroup, no second launch, every workgroup
// read all queries, 512 KB for 64 keys, and waited for them head by head: 76 us. With runs of tiles of
// equal length over chunks and heads, one per workgroup that the card holds: as fast, and spilled.)
constexpr int kManyWaves = 8, kManySpan = 2048;
template <int DT, int HD> struct MShape {
  static constexpr int NF = WShape<DT, HD>::NF;
  static constexpr int RT = NF >= 16 ? 1 : 2;
  static constexpr int TK = NF >= 16 ? 32 : 64;         // keys per tile
  static constexpr int CPR = HD / WShape<DT, HD>::VEC;  // 16-byte granules per K row
  static constexpr int LDW = CPR + 1;                   // .. per staged row
  static constexpr int NL = (TK * CPR + 511) / 512;     // .. per thread
};

template <int DT, int HD>
__global__ void __launch_bounds__(kManyWaves * kWave, (WShape<DT, HD>::NF <= (DT == PKV_F32 ? 2 : 4) ? 4 : 2))
attention_weights_many_kernel(const WeightsArgs a) {
  using SH = WShape<DT, HD>;
  using MS = MShape<DT, HD>;
  using S = typename Elt<DT>::S;
  constexpr int VEC = SH::VEC, NF = SH::NF, RT = MS::RT, TK = MS::TK, LDW = MS::LDW, CPR = MS::CPR;
  constexpr int NL = MS::NL, NT = TK / 16, ROWS = kManyWaves * 16 * RT, THREADS = kManyWaves * kWave;
  __shared__ __align__(16) u32x4 kv[2][TK * LDW];
  __shared__ float part[2][kManyWaves][TK];
  __shared__ __align__(16) RowLds<RT> row_lds[kManyWaves];
  __shared__ int slots[kManySpan];
  __shared__ int ends[kManyWaves][2];

  const int tid = threadIdx.x, lane = tid & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  const int col = lane & 15, grp = lane >> 4;
  // Items: chunks, spans, KV heads innermost.
  const unsigned item = blockIdx.y * gridDim.x + blockIdx.x;
  const int kvh = (int)(item % (unsigned)a.nkv), rest = (int)(item / (unsigned)a.nkv);
  const int c = rest / a.kblocks, cap = a.max_blocks * a.bs;
  if (c >= a.n_chunks) return;
  const int kg = (rest - c * a.kblocks) * a.span;
  const WChunk k = w_chunk(a, c);
  if (kg >= k.n || k.wrow < 0 || k.wrow >= a.w_num) return;  // uniform
  const int k_end = min(k.n, kg + a.span);
  // The span's slots, -1 past the context or outside the pool.
  bool bad = false;  // a key of the span without a slot
  for (int i = tid; i < a.span; i += THREADS) {
    const int p = kg + i, blk = a.bs_shift >= 0 ? p >> a.bs_shift : p / a.bs;
    const int id = p < k_end ? a.tables[(int64_t)c * a.table_stride + blk] : -1;
    const int64_t sl = (int64_t)id * a.bs + (p - blk * a.bs);
    slots[i] = id >= 0 && sl < a.num_slots ? (int)sl : -1;  // num_slots < 2^31 (launch)
    bad = bad || (p < k_end && slots[i] < 0);
  }
  float* const out = a.ws + ((int64_t)c * a.nkv + kvh) * cap;
  const bool dims = HD >= 4 * VEC || grp * VEC < HD;
  const bool plain = a.mod.c2 == 0.f && !a.mod.slopes;  // scores as they are
  const S* const kp = reinterpret_cast<const S*>(a.k) + (int64_t)kvh * a.kv_sh;

  // Granule i of this thread in a tile: key e / CPR, 16-byte chunk e % CPR, e = tid + THREADS i.
  auto load_k = [&](int k0, u32x4 (&st)[NL]) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      const int e = tid + THREADS * i;
      const int sl = max(slots[min(k0 - kg + e / CPR, a.span - 1)], 0);  // no key: row 0, masked
      st[i] = *reinterpret_cast<const u32x4*>(kp + (int64_t)sl * a.kv_ss + (e % CPR) * VEC);
    }
  };
  auto store_k = [&](int buf, const u32x4 (&st)[NL]) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      const int e = tid + THREADS * i;
      if (TK * CPR % THREADS == 0 || e < TK * CPR) kv[buf][e / CPR * LDW + e % CPR] = st[i];
    }
  };
  // The waves' sums of the tile at k0 (a key is always the same thread's).
  auto put = [&](int k0, int buf, bool add) __attribute__((always_inline)) {
    if (tid >= TK || k0 + tid >= k_end) return;
    float v = 0.f;
#pragma unroll
    for (int u = 0; u < kManyWaves; ++u) v += part[buf][u][tid];
    out[k0 + tid] = add ? out[k0 + tid] + v : v;
  };

  for (int rb = 0; rb == 0 || rb < k.nrows; rb += ROWS) {
    const int row0 = rb + wave * 16 * RT;
    const bool has = row0 < k.nrows;  // uniform per wave
    WRows<DT, HD, RT> rows;
    rows.first = 0x7FFFFFFF, rows.last = 0;
    const bool holes = __syncthreads_or(bad);  // the slots; the row block before is done with its LDS
    if (has) {
      rows.rows(a, k, kvh, row0, row_lds[wave]);
      rows.load_q(a, k, kvh, row0);
    }
    if (lane == 0) ends[wave][0] = rows.first, ends[wave][1] = rows.last;
    __syncthreads();
    if (has) rows.load_lse(row_lds[wave]);
    // The tiles that some row of the workgroup sees.
    int first = ends[0][0], last = ends[0][1];
#pragma unroll
    for (int u = 1; u < kManyWaves; ++u) first = min(first, ends[u][0]), last = max(last, ends[u][1]);
    const int t_beg = kg + max(0, (min(first, k_end) - kg) / TK) * TK, t_end = min(k_end, last);
    if (rb == 0 && tid < TK)  // keys of the span that no tile below covers
      for (int p = kg + tid; p < k_end; p += TK)
        if (p < t_beg || p >= t_beg + (max(t_end - t_beg, 0) + TK - 1) / TK * TK) out[p] = 0.f;

    u32x4 st[NL];
    if (t_beg < t_end) {
      load_k(t_beg, st);
      store_k(0, st);
    }
    // The queries have arrived before the loop: a wait for them inside it would also be one for the
    // next tile's K.
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
      for (int m = 0; m < NF; ++m) __asm__ volatile("" : "+v"(rows.q[i][m]));
    int buf = 0;
    for (int k0 = t_beg; k0 < t_end; k0 += TK, buf ^= 1) {
      __syncthreads();  // tile k0 is staged, the previous tile's buffer free, its sums in `part`
      const bool more = k0 + TK < t_end;
      if (more) load_k(k0 + TK, st);
      if (k0 > t_beg) put(k0 - TK, buf ^ 1, rb > 0);
      float v[NT];
      if (has && plain && !holes && rows.lo_max <= k0 && k0 + TK <= min(rows.hi_min, k_end)) {  // uniform
#pragma unroll
        for (int t = 0; t < NT; t += 2) {  // two blocks' chains of products at a time
          f32x4 s[2][RT];
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            u32x4 kf[NF];
#pragma unroll
            for (int m = 0; m < NF; ++m) kf[m] = kv[buf][(16 * (t + u) + col) * LDW + (dims ? 4 * m + grp : 0)];
#pragma unroll
            for (int i = 0; i < RT; ++i) s[u][i] = score_tile<DT, HD>(rows.q[i], kf);
          }
#pragma unroll
          for (int u = 0; u < 2; ++u) v[t + u] = rows.plain_weight(a, s[u]);
        }
      } else {
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          v[t] = 0.f;
          const int kt = k0 + 16 * t;
          if (!has || kt >= rows.last || kt + 16 <= rows.first) continue;  // uniform
          const bool here = slots[min(kt - kg + col, a.span - 1)] >= 0;
          u32x4 kf[NF];
#pragma unroll
          for (int m = 0; m < NF; ++m) kf[m] = kv[buf][(16 * t + col) * LDW + (dims ? 4 * m + grp : 0)];
          f32x4 s[RT];
#pragma unroll
          for (int i = 0; i < RT; ++i) s[i] = score_tile<DT, HD>(rows.q[i], kf);
          v[t] = rows.weight(a, row_lds[wave], s, kt, here, plain);
        }
      }
      // Lane (col, grp) gets the sum over the rows of lanes for key 16 grp + col (two blocks: 16
      // (grp / 2) + col): each swap brings two blocks' halves side by side.
      float x = swap_add32(v[0], v[NT / 2]);
      if constexpr (NT == 4) x = swap_add16(x, swap_add32(v[1], v[3]));
      else x = swap_add16(x, x);
      if (NT == 4 || grp % 2 == 0) part[buf][wave][16 * (NT == 4 ? grp : grp / 2) + col] = x;
      if (more) store_k(buf ^ 1, st);
    }
    __syncthreads();
    if (t_beg < t_end) put(t_beg + (t_end - t_beg - 1) / TK * TK, buf ^ 1, rb > 0);
  }
}

// w = decay w + the KV heads' sums, in their order.
__global__ void __launch_bounds__(256)
attention_weights_sum_kernel(const WeightsArgs a) {
  const int cap = a.max_blocks * a.bs, c = blockIdx.y;
  for (int ch = c; ch < a.n_chunks; ch += gridDim.y) {
    const int n = min(max(a.ctx[ch], 0), cap);
    const int64_t wrow = a.w_rows ? a.w_rows[ch] : ch;
    const int p = blockIdx.x * 256 + threadIdx.x;
    if (p >= n || wrow < 0 || wrow >= a.w_num) continue;
    const float* src = a.ws + (int64_t)ch * a.nkv * cap + p;
    float v = 0.f;
    for (int h = 0; h < a.nkv; ++h) v += src[(int64_t)h * cap];
    float* w = a.w + wrow * a.w_stride + p;
    *w = a.decay != 0.f ? __builtin_fmaf(*w, a.decay, v) : v;
  }
}

template <int DT, int HD> hipError_t launch_weights_hd(WeightsArgs a, int64_t rows, hipStream_t st) {
  const int64_t cap = (int64_t)a.max_blocks * a.bs;
  const bool few = rows <= kFewRows;
  if (few) {
    a.tw = 1;
    while (a.tw < kFewWaves && 2 * a.tw <= a.nkv) a.tw *= 2;
    // Keys per workgroup: every wave's share is a multiple of 16.
    a.span = kFewSpan;
    const int least = 16 * (kFewWaves / a.tw) > 64 ? 16 * (kFewWaves / a.tw) : 64;
    while (a.span > least && a.n_chunks * ((cap + a.span - 1) / a.span) < 512) a.span /= 2;
  } else {
    // Keys per workgroup: a multiple of the tiles', about two workgroups per CU and half as many again
    // (the prompts above: 46 us with 512 keys or 1,024, 49 with 256).
    a.span = kManySpan;
    while (a.span > 128 && a.n_chunks * a.nkv * ((cap + a.span - 1) / a.span) < 768) a.span /= 2;
  }
  const int64_t kblocks = (cap + a.span - 1) / a.span, items = kblocks * a.n_chunks * (few ? 1 : a.nkv);
  if (items > 0x7FFFFFFF) return hipErrorInvalidValue;
  a.kblocks = (int32_t)kblocks;
  const int64_t gx = items < (1 << 20) ? items : (1 << 20);
  const dim3 grid((unsigned)gx, (unsigned)((items + gx - 1) / gx));
  if (few) {
    hipLaunchKernelGGL((attention_weights_few_kernel<DT, HD>), grid, dim3(kFewWaves * kWave), 0, st, a);
    return hipGetLastError();
  }
  hipLaunchKernelGGL((attention_weights_many_kernel<DT, HD>), grid, dim3(kManyWaves * kWave), 0, st, a);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(attention_weights_sum_kernel,
                     dim3((unsigned)((cap + 255) / 256), (unsigned)(a.n_chunks < 65535 ? a.n_chunks : 65535)),
                     dim3(256), 0, st, a);
  return hipGetLastError();
}

template <int DT> hipError_t launch_weights(const WeightsArgs& a, int hd, int64_t rows, hipStream_t st) {
  switch (hd) {
    case 16: return launch_weights_hd<DT, 16>(a, rows, st);
    case 32: return launch_weights_hd<DT, 32>(a, rows, st);
    case 64: return launch_weights_hd<DT, 64>(a, rows, st);
    case 128: return launch_weights_hd<DT, 128>(a, rows, st);
    default: return launch_weights_hd<DT, 256>(a, rows, st);
  }
}

}  // namespace

extern "C" {

int64_t pkv_attention_weights_workspace_bytes(int32_t num_heads, int32_t num_kv_heads,
                                              int32_t n_chunks, int32_t max_query_len,
                                              int32_t max_blocks, int32_t block_size) {
  if (num_heads <= 0 || num_kv_heads <= 0 || num_heads % num_kv_heads || n_chunks < 0 ||
      n_chunks > (1 << 24) || max_query_len < 0 || max_blocks < 0 || block_size <= 0 ||
      (int64_t)max_blocks * block_size > (int64_t)1 << 30)
    return PKV_E_SHAPE;
  if ((int64_t)max_query_len * (num_heads / num_kv_heads) <= kFewRows) return 0;
  return (int64_t)n_chunks * num_kv_heads * max_blocks * block_size * 4;
}

int pkv_attention_weights(float* weights, int64_t weight_stride, int64_t num_weight_rows,
                          const int64_t* weight_rows, float decay, const void* q,
                          int64_t q_stride_tok, int64_t q_stride_h, const void* k_cache,
                          int kv_dtype, int64_t kv_stride_slot, int64_t kv_stride_head,
                          int64_t num_slots, const int32_t* block_tables, int64_t table_stride,
                          int32_t max_blocks, const int32_t* context_lens,
                          const int32_t* cu_seqlens_q, int32_t n_chunks, int32_t max_query_len,
                          const float* lse,
                          int32_t num_heads, int32_t num_kv_heads, int32_t head_dim,
                          int32_t block_size, float scale, float softcap,
                          const float* alibi_slopes, const int32_t* key_ranges,
                          int64_t range_stride, void* workspace, int64_t workspace_bytes,
                          void* stream) {
  if (!valid_dtype(kv_dtype)) return PKV_E_DTYPE;
  if (num_heads <= 0 || num_kv_heads <= 0 || num_heads % num_kv_heads || block_size <= 0 ||
      max_blocks < 0 || n_chunks < 0 || n_chunks > (1 << 24) || num_weight_rows < 0 ||
      weight_stride < 0 || max_query_len < 0 || num_slots < 0 || num_slots > 0x7FFFFFFF)
    return PKV_E_SHAPE;
  // query rows of the longest chunk for one KV head
  const int64_t rows = (int64_t)(cu_seqlens_q ? max_query_len : 1) * (num_heads / num_kv_heads);
  if (rows > (int64_t)1 << 30) return PKV_E_SHAPE;
  if (!(head_dim == 16 || head_dim == 32 || head_dim == 64 || head_dim == 128 || head_dim == 256))
    return PKV_E_SHAPE;
  if ((int64_t)max_blocks * block_size > (int64_t)1 << 30) return PKV_E_SHAPE;
  if (!(scale > 0.f && scale < INFINITY) || !(decay >= 0.f && decay < INFINITY)) return PKV_E_SHAPE;
  if (!weight_rows && num_weight_rows < n_chunks) return PKV_E_SHAPE;
  ScoreMod mod;
  const int bad = score_mod(&mod, softcap, alibi_slopes, key_ranges, range_stride);
  if (bad) return bad;
  const int64_t need = pkv_attention_weights_workspace_bytes(
      num_heads, num_kv_heads, n_chunks, cu_seqlens_q ? max_query_len : 1, max_blocks, block_size);
  if (workspace_bytes < need || (need > 0 && !workspace)) return PKV_E_WORKSPACE;
  if (workspace && ((uintptr_t)workspace & 3u)) return PKV_E_ALIGN;
  if (n_chunks == 0 || max_blocks == 0) return 0;
  if (!weights || !q || !k_cache || !block_tables || !context_lens || !lse) return PKV_E_NULL;
  const int vec = kv_dtype == PKV_F32 ? 4 : 8;
  if (!aligned16(q) || !aligned16(k_cache) || q_stride_tok % vec || q_stride_h % vec ||
      kv_stride_slot % vec || kv_stride_head % vec)
    return PKV_E_ALIGN;
  WeightsArgs a;
  a.w = weights;
  a.w_stride = weight_stride;
  a.w_num = num_weight_rows;
  a.w_rows = weight_rows;
  a.decay = decay;
  a.q = q;
  a.q_st = q_stride_tok;
  a.q_sh = q_stride_h;
  a.k = k_cache;
  a.kv_ss = kv_stride_slot;
  a.kv_sh = kv_stride_head;
  a.num_slots = num_slots;
  a.tables = block_tables;
  a.table_stride = table_stride;
  a.max_blocks = max_blocks;
  a.ctx = context_lens;
  a.cu_q = cu_seqlens_q;
  a.lse = lse;
  a.n_chunks = n_chunks;
  a.nh = num_heads;
  a.nkv = num_kv_heads;
  a.groups = num_heads / num_kv_heads;
  a.bs = block_size;
  a.bs_shift = (block_size & (block_size - 1)) == 0 ? __builtin_ctz(block_size) : -1;
  a.max_queries = cu_seqlens_q ? max_query_len : 1;
  a.tw = a.span = a.kblocks = 0;  // set at launch
  a.ws = static_cast<float*>(workspace);
  a.scale_log2 = scale * kLog2e;
  a.mod = mod;
  hipStream_t st = (hipStream_t)stream;
  switch (kv_dtype) {
    case PKV_F32: return (int)launch_weights<PKV_F32>(a, head_dim, rows, st);
    case PKV_F16: return (int)launch_weights<PKV_F16>(a, head_dim, rows, st);
    default: return (int)launch_weights<PKV_BF16>(a, head_dim, rows, st);
  }
}

}  // extern "C"
