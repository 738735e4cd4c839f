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
  int32_t hw;       // waves that take different KV heads (a power of two, at most 8)
  int32_t kblocks;  // workgroups per chunk
  int32_t steps;    // key groups that a workgroup takes one after the other
  float scale_log2;
  ScoreMod mod;
};

// ---------------------------------------------------------------------------------
// w[p] = decay w[p] + sum over queries t and heads h of 2^(s(t, h, p) - lse(t, h)).
//
// A workgroup of 8 waves takes a group of keys of one chunk: hw waves share the KV heads, 8 / hw
// the keys, so that a key's whole sum is formed in one workgroup -- in a fixed order, without
// atomics -- and w is read and written once. A wave holds NT tiles of 16 keys of one KV head as
// MFMA A operands (lane (col, grp): key col, dims 4 VEC m + VEC grp ..) and walks over the query
// rows (token, head of the group) in tiles of 16, the B operand: S^T = K Q^T, lane (row col, grp)
// gets keys 4 grp + r, exactly the decode pass's score tile. Every score becomes its weight, lanes
// add over row tiles and KV heads, and the 16 columns are added once at the end.
// One query per chunk (decode) is bound by reading K once; there NT tiles are one batch of loads,
// and the CU's other waves stream while one waits. Many queries are bound by an exp2 per score;
// the next row tile's queries and normalisers are on their way under this one's.
// ---------------------------------------------------------------------------------

template <int DT, int HD> struct WShape {
  static constexpr int VEC = vec16<DT>();
  static constexpr int NF = HD >= 4 * VEC ? HD / (4 * VEC) : 1;  // 16-byte pieces of a row per lane
  static constexpr int NT = NF <= 2 ? 4 : NF <= 4 ? 4 : NF <= 8 ? 2 : 1;  // 16-key tiles per wave
  static constexpr int KEYS = 16 * NT;
};

template <int DT, int HD>
__device__ __forceinline__ f32x4 score_tile(const u32x4* kf, const u32x4* qf) {
  f32x4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int m = 0; m < WShape<DT, HD>::NF; ++m) {
    if constexpr (DT == PKV_F32) {
      const f32x4 a = __builtin_bit_cast(f32x4, kf[m]), b = __builtin_bit_cast(f32x4, qf[m]);
#pragma unroll
      for (int j = 0; j < 4; ++j) s = __builtin_amdgcn_mfma_f32_16x16x4f32(a[j], b[j], s, 0, 0, 0);
    } else if constexpr (DT == PKV_BF16) {
      typedef __bf16 v8 __attribute__((ext_vector_type(8)));
      s = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8, kf[m]),
                                                  __builtin_bit_cast(v8, qf[m]), s, 0, 0, 0);
    } else {
      typedef _Float16 v8 __attribute__((ext_vector_type(8)));
      s = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8, kf[m]),
                                                 __builtin_bit_cast(v8, qf[m]), s, 0, 0, 0);
    }
  }
  return s;
}

template <int DT, int HD>
__global__ void __launch_bounds__(512)
attention_weights_kernel(const WeightsArgs a) {
  using SH = WShape<DT, HD>;
  using S = typename Elt<DT>::S;
  constexpr int VEC = SH::VEC, NF = SH::NF, NT = SH::NT, KEYS = SH::KEYS;
  __shared__ float sums[8][KEYS];

  const int lane = threadIdx.x & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int col = lane & 15, grp = lane >> 4;
  const unsigned item = blockIdx.y * gridDim.x + blockIdx.x;
  const int c = (int)(item / (unsigned)a.kblocks);
  if (c >= a.n_chunks) return;
  const int kblk = (int)(item % (unsigned)a.kblocks);
  const int hw = a.hw, hid = wave & (hw - 1), sub = wave / hw;
  const int wg_keys = KEYS * (8 / hw);  // per step
  const int cap = a.max_blocks * a.bs;
  const int n = min(max(a.ctx[c], 0), cap);
  const int64_t wrow = a.w_rows ? a.w_rows[c] : c;
  const int q0 = a.cu_q ? a.cu_q[c] : c;
  const int qlen = a.cu_q ? max(a.cu_q[c + 1] - q0, 0) : 1;
  if (wrow < 0 || wrow >= a.w_num) return;  // uniform, as n
  const int G = a.groups, nrows = qlen * G, base_pos = n - qlen;
  const int32_t* trow = a.tables + (int64_t)c * a.table_stride;
  const bool lane_dims = HD >= 4 * VEC || grp * VEC < HD;  // head_dim 16 of a 16-bit type: half the lanes

  for (int step = 0; step < a.steps; ++step) {
    const int kg = (kblk * a.steps + step) * wg_keys;  // the workgroup's keys of this step
    if (kg >= n) return;                               // uniform
    const int k0 = kg + sub * KEYS;                    // this wave's
    // Slots of this lane's key (col) of every tile, -1 past the context or outside the pool.
    int64_t off[NT];
    unsigned live_col = 0;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const int p = k0 + 16 * t + col;
      off[t] = 0;
      if (p < n) {
        const int blk = a.bs_shift >= 0 ? p >> a.bs_shift : p / a.bs;
        const int id = trow[blk];
        const int64_t sl = (int64_t)id * a.bs + (p - blk * a.bs);
        if (id >= 0 && sl < a.num_slots) {
          off[t] = sl * a.kv_ss;
          live_col |= 1u << t;
        }
      }
    }
    // Keys 4 grp + r of tile t that exist: bit 4 t + r.
    unsigned live = 0;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const uint64_t b = __ballot((live_col >> t) & 1u);
      live |= (unsigned)((b >> (4 * grp)) & 15u) << (4 * t);
    }
    // Whether any query sees any of this wave's keys.
    bool any = false;
    if (a.mod.ranges) {
      for (int t = lane; t < qlen; t += kWave) {
        const int32_t* r = a.mod.ranges + (int64_t)(q0 + t) * a.mod.range_stride;
        any = any || (max(r[0], k0) < min(min(r[1], n), k0 + KEYS));
      }
      any = __ballot(any) != 0;
    } else {
      any = k0 < n && nrows > 0;
    }

    f32x4 acc[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) acc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int kvh = any ? hid : a.nkv; kvh < a.nkv; kvh += hw) {
      const u32x4 z = {0, 0, 0, 0};
      u32x4 kf[NT][NF];
      const S* kb = reinterpret_cast<const S*>(a.k) + (int64_t)kvh * a.kv_sh + VEC * grp;
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int m = 0; m < NF; ++m)
          kf[t][m] = ((live_col >> t) & 1u) && lane_dims
                         ? __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(kb + off[t] + 4 * VEC * m))
                         : z;
      // A row tile's operands: its queries, normaliser and visible keys [lo, hi) of row col.
      struct Rows {
        u32x4 q[NF];
        float lse;
        int lo, hi;
      };
      auto load_rows = [&](int rt, Rows& x) __attribute__((always_inline)) {
        const int rho = rt * 16 + col;
        const bool ok = rho < nrows;
        const int tok = ok ? rho / G : 0, head = kvh * G + (ok ? rho % G : 0);
        const S* qp = reinterpret_cast<const S*>(a.q) + (int64_t)(q0 + tok) * a.q_st +
                      (int64_t)head * a.q_sh + VEC * grp;
#pragma unroll
        for (int m = 0; m < NF; ++m)
          x.q[m] = ok && lane_dims ? *reinterpret_cast<const u32x4*>(qp + 4 * VEC * m) : z;
        x.lse = ok ? a.lse[(int64_t)(q0 + tok) * a.nh + head] : -INFINITY;
        x.lo = 0;
        x.hi = base_pos + tok + 1;
        if (a.mod.ranges) {
          const int32_t* r = a.mod.ranges + (int64_t)(q0 + tok) * a.mod.range_stride;
          x.lo = r[0];
          x.hi = r[1];
        }
        if (x.lse == -INFINITY) x.hi = -1;  // no row, or one without keys: nothing
      };
      const int rtiles = (nrows + 15) / 16;
      Rows cur;
      load_rows(0, cur);
      for (int rt = 0; rt < rtiles; ++rt) {
        Rows next = cur;
        if (rt + 1 < rtiles) load_rows(rt + 1, next);
        float slope = 0.f;
        int qpos = 0;
        if (a.mod.slopes) {
          const int rho = min(rt * 16 + col, nrows - 1);
          slope = a.mod.slopes[kvh * G + rho % G] * kLog2e;
          qpos = base_pos + rho / G;
        }
        // Keys key0 + r of tile t that row col sees: r in [lo - key0, hi - key0).
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          const f32x4 s = score_tile<DT, HD>(kf[t], cur.q);
          const int key0 = k0 + 16 * t + 4 * grp;
          const int lo = cur.lo - key0, hi = cur.hi - key0;
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            float d = s[r] * a.scale_log2;
            if (a.mod.c2 != 0.f) d = capped<DT == PKV_F32>(a.mod, d);
            if (a.mod.slopes) d = biased(d, slope, qpos - key0 - r);
            const bool sees = r >= lo && r < hi && ((live >> (4 * t + r)) & 1u);
            acc[t][r] += sees ? __builtin_amdgcn_exp2f(d - cur.lse) : 0.f;
          }
        }
        cur = next;
      }
    }
    // Over the 16 columns (query rows), then over the waves that share the keys.
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float v = group_sum<16>(acc[t][r]);
        if (col == 0) sums[wave][16 * t + 4 * grp + r] = v;
      }
    __syncthreads();
    for (int i = threadIdx.x; i < wg_keys; i += 512) {
      const int p = kg + i;
      if (p < n) {
        const int s = i / KEYS, key = i % KEYS;
        float v = 0.f;
        for (int h = 0; h < hw; ++h) v += sums[s * hw + h][key];
        float* w = a.w + wrow * a.w_stride + p;
        *w = a.decay != 0.f ? __builtin_fmaf(*w, a.decay, v) : v;
      }
    }
    __syncthreads();  // the next step's sums
  }
}

template <int DT, int HD> hipError_t launch_weights_hd(WeightsArgs a, hipStream_t st) {
  constexpr int KEYS = WShape<DT, HD>::KEYS;
  a.hw = 1;
  while (a.hw < 8 && 2 * a.hw <= a.nkv) a.hw *= 2;
  const int64_t groups = ((int64_t)a.max_blocks * a.bs + KEYS * (8 / a.hw) - 1) / (KEYS * (8 / a.hw));
  if (groups == 0) return hipSuccess;
  a.steps = 1;
  while (a.steps < 16 && a.n_chunks * ((groups + 2 * a.steps - 1) / (2 * a.steps)) >= 4096) a.steps *= 2;
  const int64_t kblocks = (groups + a.steps - 1) / a.steps, items = kblocks * a.n_chunks;
  if (items > 0x7FFFFFFF) return hipErrorInvalidValue;
  a.kblocks = (int32_t)kblocks;
  const int64_t gx = items < (1 << 20) ? items : (1 << 20);
  hipLaunchKernelGGL((attention_weights_kernel<DT, HD>),
                     dim3((unsigned)gx, (unsigned)((items + gx - 1) / gx)), dim3(512), 0, st, a);
  return hipGetLastError();
}

template <int DT> hipError_t launch_weights(const WeightsArgs& a, int hd, hipStream_t st) {
  switch (hd) {
    case 16: return launch_weights_hd<DT, 16>(a, st);
    case 32: return launch_weights_hd<DT, 32>(a, st);
    case 64: return launch_weights_hd<DT, 64>(a, st);
    case 128: return launch_weights_hd<DT, 128>(a, st);
    default: return launch_weights_hd<DT, 256>(a, st);
  }
}

}  // namespace

extern "C" {

int pkv_attention_weights(float* weights, int64_t weight_stride, int64_t num_weight_rows,
                          const int64_t* weight_rows, float decay, const void* q,
                          int64_t q_stride_tok, int64_t q_stride_h, const void* k_cache,
                          int kv_dtype, int64_t kv_stride_slot, int64_t kv_stride_head,
                          int64_t num_slots, const int32_t* block_tables, int64_t table_stride,
                          int32_t max_blocks, const int32_t* context_lens,
                          const int32_t* cu_seqlens_q, int32_t n_chunks, const float* lse,
                          int32_t num_heads, int32_t num_kv_heads, int32_t head_dim,
                          int32_t block_size, float scale, float softcap,
                          const float* alibi_slopes, const int32_t* key_ranges,
                          int64_t range_stride, void* stream) {
  if (!valid_dtype(kv_dtype)) return PKV_E_DTYPE;
  if (num_heads <= 0 || num_kv_heads <= 0 || num_heads % num_kv_heads || block_size <= 0 ||
      max_blocks < 0 || n_chunks < 0 || n_chunks > (1 << 24) || num_weight_rows < 0 ||
      weight_stride < 0)
    return PKV_E_SHAPE;
  if (!(head_dim == 16 || head_dim == 32 || head_dim == 64 || head_dim == 128 || head_dim == 256))
    return PKV_E_SHAPE;
  if ((int64_t)max_blocks * block_size > (int64_t)1 << 30) return PKV_E_SHAPE;
  if (!(scale > 0.f && scale < INFINITY) || !(decay >= 0.f && decay < INFINITY)) return PKV_E_SHAPE;
  if (!weight_rows && num_weight_rows < n_chunks) return PKV_E_SHAPE;
  ScoreMod mod;
  const int bad = score_mod(&mod, softcap, alibi_slopes, key_ranges, range_stride);
  if (bad) return bad;
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
  a.hw = a.kblocks = a.steps = 0;  // set at launch
  a.scale_log2 = scale * kLog2e;
  a.mod = mod;
  hipStream_t st = (hipStream_t)stream;
  switch (kv_dtype) {
    case PKV_F32: return (int)launch_weights<PKV_F32>(a, head_dim, st);
    case PKV_F16: return (int)launch_weights<PKV_F16>(a, head_dim, st);
    default: return (int)launch_weights<PKV_BF16>(a, head_dim, st);
  }
}

}  // extern "C"
