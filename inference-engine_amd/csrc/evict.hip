// evict.hip -- eviction from the paged pool by accumulated attention weight (include/paged_kv.h:
// pkv_evict): every layer of a sequence keeps its last tokens and the heaviest of the others,
// moved up in their order over the evicted ones' slots.

#include "common.h"

namespace {

using namespace pkv;

struct EvictArgs {
  char* k;
  char* v;
  int64_t layer_bytes, row_bytes, num_slots;
  float* w;  // layer l, row r, token p: w[l * w_layer + r * w_stride + p]
  int64_t w_layer, w_stride, w_num;
  const int64_t* w_rows;  // [batch] or null
  const int32_t* tables;
  int64_t table_stride;
  int32_t max_blocks, bs, layers, batch, keep, recent;
  const int32_t* ctx;
  int32_t* new_ctx;
  int2* head;     // [layers, batch]: first and one past the last token that moves
  int32_t* from;  // [layers, batch, keep]: slot that kept token i comes from, -1 outside the pool
  int32_t keep_stride, bs_shift;
};

// ---------------------------------------------------------------------------------
// Selection: one workgroup of 1,024 threads per (layer, sequence).
//
// Of the first n - recent tokens the k = keep - recent heaviest stay, ties by the lowest index.
// Weights become unsigned keys in their order (NaN below all); the k-th largest key is found eight
// bits at a time from the top: a histogram in LDS of the digit of the keys that share the digits found
// so far, and a suffix sum over its 256 bins by one wave. (Two bits at a time by counting compares, in
// registers, took 16 rounds of all 16 waves: 20 us for 2,112 tokens, now 8.) A wave's keys with its first
// one's digit count as one: where most weights are 0 (tokens outside a window) or alike they would all
// meet in one bin (4 layers, 32,768 zeros: 147 us a call, with this 82; 254 against 249 for random
// ones). Then rounds of 1,024
// tokens in index order give every kept token its place by prefix counts, move its weight there and
// leave its slot for the move pass. R: keys per thread in registers (R = 0: more tokens than that,
// read from L2 in every pass).
// ---------------------------------------------------------------------------------

__device__ __forceinline__ uint32_t weight_key(float x) {
  if (x != x) return 0u;
  const uint32_t u = __float_as_uint(x + 0.f);  // -0 is 0
  return u ^ ((u >> 31) ? 0xFFFFFFFFu : 0x80000000u);
}

// Sum over the 16 lanes of a row of lanes, in every one of them.
__device__ __forceinline__ int row_sum(int x) {
  x += __builtin_amdgcn_update_dpp(0, x, kQuadXor1, 0xF, 0xF, false);
  x += __builtin_amdgcn_update_dpp(0, x, kQuadXor2, 0xF, 0xF, false);
  x += __builtin_amdgcn_update_dpp(0, x, kRowHalfMirror, 0xF, 0xF, false);
  x += __builtin_amdgcn_update_dpp(0, x, kRowMirror, 0xF, 0xF, false);
  return x;
}

constexpr int kSelThreads = 1024, kSelWaves = kSelThreads / kWave;

// Inclusive prefix sum over the wave's lanes.
__device__ __forceinline__ int wave_scan(int x) {
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xF, 0xF, false);  // row_shr 1, 2, 4, 8
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xF, 0xF, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xF, 0xF, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xF, 0xF, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xA, 0xF, false);  // row_bcast 15 to rows 1 and 3
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xC, 0xF, false);  // row_bcast 31 to rows 2 and 3
  return x;
}

template <int R>
__global__ void __launch_bounds__(kSelThreads, (R <= 4 ? 8 : 4))
evict_select_kernel(const EvictArgs a) {
  static_assert(kSelWaves == 16, "a row of lanes holds the waves' counts");
  __shared__ __align__(16) int hist[2][256];
  __shared__ __align__(16) int2 counts[2][kSelWaves];
  __shared__ int2 found;  // the digit, and the keys above it
  __shared__ int first_gap;
  const int tid = threadIdx.x, lane = tid & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  const int b = blockIdx.x % a.batch, layer = blockIdx.x / a.batch;
  const int cap = a.max_blocks * a.bs;
  const int n = min(max(a.ctx[b], 0), cap);
  const int64_t wrow = a.w_rows ? a.w_rows[b] : b;
  const bool skip = wrow < 0 || wrow >= a.w_num;
  int2* head = a.head + (int64_t)layer * a.batch + b;
  if (layer == 0 && tid == 0) a.new_ctx[b] = skip ? a.ctx[b] : min(n, a.keep);
  if (skip || n <= a.keep) {  // uniform: nothing to evict
    if (tid == 0) *head = make_int2(0, 0);
    return;
  }
  float* w = a.w + layer * a.w_layer + wrow * a.w_stride;
  const int old = n - a.recent, k = a.keep - a.recent;  // 0 <= k < old
  const int rounds = (n + kSelThreads - 1) / kSelThreads;

  constexpr int RR = R > 0 ? R : 1;
  float x[RR];
  uint32_t key[RR];
  if constexpr (R > 0) {
#pragma unroll
    for (int j = 0; j < R; ++j) {
      const int i = j * kSelThreads + tid;
      x[j] = i < n ? w[i] : 0.f;
    }
#pragma unroll
    for (int j = 0; j < R; ++j) key[j] = weight_key(x[j]);
  }
  if (tid == 0) first_gap = n;
  if (tid < 256) hist[0][tid] = 0;

  // The k-th largest key t of the old tokens (k > 0), and how many of them are above it.
  uint32_t t = 0;
  int above = 0;
  for (int pass = 0; k > 0 && pass < 4; ++pass) {
    const int shift = 24 - 8 * pass;
    int* const h = hist[pass & 1];
    __syncthreads();  // the histogram is clear; the last pass's digit has been read
    auto count = [&](int i, uint32_t kk) __attribute__((always_inline)) {
      const bool on = i < old && (pass == 0 || (kk >> (shift + 8)) == t);
      const int d = (int)((kk >> shift) & 255u);
      const uint64_t live = __ballot(on);
      if (!live) return;  // uniform
      const int lead = __builtin_ctzll(live), first = __builtin_amdgcn_readlane(d, lead);
      const uint64_t same = __ballot(on && d == first);
      if (lane == lead) atomicAdd(&h[first], __popcll(same));
      else if (on && d != first) atomicAdd(&h[d], 1);
    };
    if constexpr (R > 0) {
#pragma unroll
      for (int j = 0; j < R; ++j) count(j * kSelThreads + tid, key[j]);
    } else {
      for (int j = 0; j < rounds; ++j) {
        const int i = j * kSelThreads + tid;
        count(i, i < old ? weight_key(w[i]) : 0u);
      }
    }
    __syncthreads();
    if (wave == 0) {
      // Lane l: bins 255 - 4 l down to 252 - 4 l; keys in them and in all higher bins.
      const int4 c = *reinterpret_cast<const int4*>(&h[252 - 4 * lane]);
      const int mine = c.x + c.y + c.z + c.w;
      const int upto = wave_scan(mine) + above;
      const uint64_t hit = __ballot(upto >= k);  // not empty: all of the prefix's keys and those above
      if (lane == __builtin_ctzll(hit)) {
        int over = upto - mine, d = 255 - 4 * lane;
        const int bins[4] = {c.w, c.z, c.y, c.x};
#pragma unroll
        for (int u = 0; u < 3; ++u)
          if (over + bins[u] < k && d == 255 - 4 * lane - u) over += bins[u], --d;
        found = make_int2(d, over);
      }
    } else if (wave < 5) {
      hist[(pass & 1) ^ 1][tid - kWave] = 0;
    }
    __syncthreads();
    const int2 f = found;
    t = t << 8 | (uint32_t)f.x;
    above = f.y;
  }
  const int ties = k - above;  // tokens equal to t that stay, the first ones

  __syncthreads();
  const int32_t* trow = a.tables + (int64_t)b * a.table_stride;
  auto slot_of = [&](int p) {
    const int blk = a.bs_shift >= 0 ? p >> a.bs_shift : p / a.bs, id = trow[blk];
    const int64_t sl = (int64_t)id * a.bs + (p - blk * a.bs);
    return id >= 0 && sl < a.num_slots ? (int)sl : -1;  // num_slots < 2^31 (launch)
  };
  int32_t* from = a.from + ((int64_t)layer * a.batch + b) * a.keep_stride;
  int before = 0, eq_before = 0;  // tokens kept for sure, and tokens equal to t, in earlier rounds
  auto emit = [&](int j, float xv, uint32_t kk) __attribute__((always_inline)) {
    const int i = j * kSelThreads + tid;
    const int slot = i < n ? slot_of(i) : -1;
    const bool sure = (i < old && k > 0 && kk > t) || (i >= old && i < n);
    const bool eq = i < old && k > 0 && kk == t;
    const uint64_t bs = __ballot(sure), be = __ballot(eq);
    int2* const cnt = counts[j & 1];
    if (lane == 0) cnt[wave] = make_int2(__popcll(bs), __popcll(be));
    __syncthreads();  // the round's weights are in registers; the earlier rounds' moves may be overtaken
    const int2 c = cnt[lane & 15];
    const bool prior = (lane & 15) < wave;
    int sb = before + __builtin_amdgcn_readfirstlane(row_sum(prior ? c.x : 0));
    int eb = eq_before + __builtin_amdgcn_readfirstlane(row_sum(prior ? c.y : 0));
    const int st = __builtin_amdgcn_readfirstlane(row_sum(c.x));
    const int et = __builtin_amdgcn_readfirstlane(row_sum(c.y));
    const uint64_t below = (1ull << lane) - 1;
    sb += __popcll(bs & below);
    eb += __popcll(be & below);
    const int pos = sb + min(eb, ties);
    const bool kept = sure || (eq && eb < ties);
    if (kept) {
      w[pos] = xv;
      from[pos] = slot;
    }
    const uint64_t gone = __ballot(!kept && i < n);
    if (gone && lane == 0) atomicMin(&first_gap, j * kSelThreads + wave * kWave + __builtin_ctzll(gone));
    before += st;
    eq_before += et;
  };
  if constexpr (R > 0 && R <= 4) {
#pragma unroll
    for (int j = 0; j < R; ++j)
      if (j < rounds) emit(j, x[j], key[j]);
  } else {  // read again: no round before wrote past its own tokens
    for (int j = 0; j < rounds; ++j) {
      const int i = j * kSelThreads + tid;
      const float xv = i < n ? w[i] : 0.f;
      emit(j, xv, weight_key(xv));
    }
  }
  __syncthreads();
  for (int i = a.keep + tid; i < n; i += kSelThreads) w[i] = 0.f;
  if (tid == 0) *head = make_int2(first_gap, a.keep);
}

// ---------------------------------------------------------------------------------
// Move: kept token i goes from its slot to token i's, for every i from the first gap on.
//
// A token moves down (from >= to), and moves go up in i, so where a batch of tokens is read before any
// of it is written, and the batches follow each other in order, nothing is overwritten unread: a
// later batch's sources lie at or past every earlier batch's destinations. The bytes of a row are
// independent, so a workgroup takes a slice of SLICE bytes of every row of one (layer, sequence, K
// or V) and needs no other workgroup; its W waves take shares of a batch, with one barrier between
// its reads and its writes (W = 1: a workgroup of four waves with a slice each). The next batch's rows
// are on their way while this one's are written. Bound by HBM, every row read and written once.
// Figures at the launch.
// ---------------------------------------------------------------------------------

template <int SLICE, int W>
__global__ void __launch_bounds__(W > 1 ? W * kWave : 4 * kWave)
evict_move_kernel(const EvictArgs a, int slices) {
  constexpr int LPR = SLICE / 16;      // lanes per row
  constexpr int RPL = kWave / LPR;     // rows per load
  constexpr int U = 8;                 // loads per batch
  constexpr int BATCH = RPL * U * W;
  const int lane = threadIdx.x & (kWave - 1);
  const int wave = threadIdx.x / kWave;
  const int64_t job = W > 1 ? blockIdx.x : (int64_t)blockIdx.x * 4 + wave;  // slices innermost
  const int64_t per = 2 * (int64_t)slices;
  const int64_t seq = job / per;
  if (seq >= (int64_t)a.layers * a.batch) return;
  const int2 h = a.head[seq];
  if (h.x >= h.y) return;
  const int part = (int)(job % per);
  const int slice = part % slices;
  int64_t at = (int64_t)slice * SLICE + (lane % LPR) * 16;
  const bool on = at < a.row_bytes;  // the last slice may be narrower
  if (!on) at = 0;
  char* pool = (part / slices ? a.v : a.k) + (seq / a.batch) * a.layer_bytes + at;
  const int32_t* from = a.from + seq * a.keep_stride;
  const int32_t* trow = a.tables + (seq % a.batch) * a.table_stride;
  const int r = lane / LPR + (W > 1 ? wave * (RPL * U) : 0);  // this lane's first row of a batch

  // Loads go out without conditions (a token past the end reads the last one's, a slot outside the
  // pool and a lane past the row slot 0), so that the wait for one batch does not wait for the next;
  // where a token goes is worked out only when its row is written.
  struct Moves {
    int from[U], id[U];
  };
  auto blk_of = [&](int i) { return a.bs_shift >= 0 ? i >> a.bs_shift : i / a.bs; };
  auto load_moves = [&](int i0, Moves& m) __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = min(i0 + u * RPL + r, h.y - 1);
      m.from[u] = from[i];
      m.id[u] = trow[blk_of(i)];
    }
  };
  auto load_rows = [&](const Moves& m, u32x4* d) __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < U; ++u)
      d[u] = *reinterpret_cast<const u32x4*>(pool + (int64_t)max(m.from[u], 0) * a.row_bytes);
  };
  Moves cur, next, after;
  u32x4 x[U], nx[U];
  load_moves(h.x, cur);
  load_moves(h.x + BATCH, next);
  load_rows(cur, x);
  for (int i = h.x; i < h.y; i += BATCH) {
    load_moves(i + 2 * BATCH, after);
    load_rows(next, nx);
    // Every row of this batch is in registers before any of it is overwritten: one statement that
    // takes a wave's all, and a barrier without a fence (which would wait for the next batch's rows).
    static_assert(U == 8, "the rows of a batch below");
    __asm__ volatile("" : "+v"(x[0]), "+v"(x[1]), "+v"(x[2]), "+v"(x[3]), "+v"(x[4]), "+v"(x[5]),
                          "+v"(x[6]), "+v"(x[7]) : : "memory");
    if constexpr (W > 1) __builtin_amdgcn_s_barrier();
    __asm__ volatile("" : : : "memory");
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int p = i + u * RPL + r;
      const int64_t to = (int64_t)cur.id[u] * a.bs + (p - blk_of(p) * a.bs);
      if (on && p < h.y && cur.from[u] >= 0 && cur.id[u] >= 0 && to < a.num_slots)
        *reinterpret_cast<u32x4*>(pool + to * a.row_bytes) = x[u];
    }
    cur = next;
    next = after;
#pragma unroll
    for (int u = 0; u < U; ++u) x[u] = nx[u];
  }
}

template <int SLICE, int W> int launch_move(const EvictArgs& a, int64_t seqs, hipStream_t st) {
  const int64_t slices = (a.row_bytes + SLICE - 1) / SLICE, jobs = seqs * 2 * slices;
  const int64_t wgs = W > 1 ? jobs : (jobs + 3) / 4;
  if (slices > (1 << 20) || wgs >= ((int64_t)1 << 24)) return PKV_E_SHAPE;
  hipLaunchKernelGGL((evict_move_kernel<SLICE, W>), dim3((unsigned)wgs), dim3(W > 1 ? W * kWave : 4 * kWave), 0,
                     st, a, (int)slices);
  return (int)hipGetLastError();
}

struct EvictWs {
  int64_t moves, total;
};
EvictWs evict_ws(int32_t layers, int32_t batch, int32_t keep) {
  const int64_t pairs = (int64_t)layers * batch;
  const int64_t moves = (pairs * 8 + 255) / 256 * 256;
  return {moves, moves + pairs * keep * 4};
}

}  // namespace

extern "C" {

int64_t pkv_evict_workspace_bytes(int32_t layers, int32_t batch, int32_t max_blocks,
                                  int32_t block_size, int32_t keep) {
  if (layers < 0 || batch < 0 || max_blocks < 0 || block_size <= 0 || keep < 0 ||
      (int64_t)max_blocks * block_size > (int64_t)1 << 30)
    return PKV_E_SHAPE;
  const int64_t cap = (int64_t)max_blocks * block_size;
  return evict_ws(layers, batch, (int32_t)(keep < cap ? keep : cap)).total;
}

int pkv_evict(void* k_pool, void* v_pool, int64_t layer_stride_bytes, int32_t layers,
              int64_t row_bytes, int64_t num_slots, float* weights, int64_t weight_stride_layer,
              int64_t weight_stride_row, int64_t num_weight_rows, const int64_t* weight_rows,
              const int32_t* block_tables, int64_t table_stride, int32_t max_blocks,
              int32_t block_size, const int32_t* context_lens, int32_t batch, int32_t keep,
              int32_t recent, int32_t* new_lens, void* workspace, int64_t workspace_bytes,
              void* stream) {
  if (layers < 0 || layers > 65535 || batch < 0 || batch > (1 << 20) || block_size <= 0 ||
      max_blocks < 0 || keep < 0 || recent < 0 || recent > keep || row_bytes <= 0 ||
      num_slots < 0 || num_slots > 0x7FFFFFFF || num_weight_rows < 0)
    return PKV_E_SHAPE;
  if ((int64_t)max_blocks * block_size > (int64_t)1 << 30) return PKV_E_SHAPE;
  if (!weight_rows && num_weight_rows < batch) return PKV_E_SHAPE;
  if (layers == 0 || batch == 0) return 0;
  if (!k_pool || !v_pool || !weights || !context_lens || !new_lens || !workspace ||
      (max_blocks > 0 && !block_tables))
    return PKV_E_NULL;
  if (!aligned16(k_pool) || !aligned16(v_pool) || row_bytes % 16 || layer_stride_bytes % 16 ||
      ((uintptr_t)workspace & 7u))
    return PKV_E_ALIGN;
  const int64_t cap = (int64_t)max_blocks * block_size;
  const int32_t kept = (int32_t)(keep < cap ? keep : cap);  // the moves of one sequence
  const EvictWs ws = evict_ws(layers, batch, kept);
  if (workspace_bytes < ws.total) return PKV_E_WORKSPACE;
  EvictArgs a;
  a.k = (char*)k_pool;
  a.v = (char*)v_pool;
  a.layer_bytes = layer_stride_bytes;
  a.row_bytes = row_bytes;
  a.num_slots = num_slots;
  a.w = weights;
  a.w_layer = weight_stride_layer;
  a.w_stride = weight_stride_row;
  a.w_num = num_weight_rows;
  a.w_rows = weight_rows;
  a.tables = block_tables;
  a.table_stride = table_stride;
  a.max_blocks = max_blocks;
  a.bs = block_size;
  a.layers = layers;
  a.batch = batch;
  a.keep = keep;
  a.recent = recent;
  a.ctx = context_lens;
  a.new_ctx = new_lens;
  a.head = (int2*)workspace;
  a.from = (int32_t*)((char*)workspace + ws.moves);
  a.bs_shift = (block_size & (block_size - 1)) == 0 ? __builtin_ctz(block_size) : -1;
  a.keep_stride = kept;
  hipStream_t st = (hipStream_t)stream;
  const int64_t seqs = (int64_t)layers * batch;
  if (seqs > (1 << 22)) return PKV_E_SHAPE;  // 2^32 threads
  const dim3 grid((unsigned)seqs), block(kSelThreads);
  if (cap <= 4 * kSelThreads) hipLaunchKernelGGL(evict_select_kernel<4>, grid, block, 0, st, a);
  else if (cap <= 16 * kSelThreads) hipLaunchKernelGGL(evict_select_kernel<16>, grid, block, 0, st, a);
  else hipLaunchKernelGGL(evict_select_kernel<0>, grid, block, 0, st, a);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || cap <= keep) return (int)e;
  // Slices of 256 bytes keep a row's bytes together in memory, of 128 make twice the workgroups; the
  // wide ones where they are more than one per CU. Whole calls, rows of 1 KB, wide and narrow: 16
  // layers, 4 sequences of 8,192 tokens down to 8,000 448 and 479 us; one sequence of 2,112 down to 2,048
  // 34 and 31, of 32,768 down to 30,000 532 and 508 (single waves with narrower slices, down to 32
  // bytes: 615, 37, 743). A wave per slice where that makes 16 per CU: 32 sequences of 700-4,096 down
  // to 1,000 412 us, with 8 waves 427.
  const int64_t wide = seqs * 2 * ((row_bytes + 255) / 256);
  if (wide >= 4096) return launch_move<256, 1>(a, seqs, st);
  if (wide > 256) return launch_move<256, 8>(a, seqs, st);
  return launch_move<128, 8>(a, seqs, st);
}

}  // extern "C"
