// Page tables and slot maps of the quantized KV cache, made on the GPU from request lengths; and the accepted path of a tree of drafted tokens kept.
//
// All of it is a few hundred kilobytes at most (the largest tables some megabytes) and bound by latency: launches, dependent loads, barriers. So each call is
// one launch, with nothing read back by the host.
#include <algorithm>

#include "xnq_kv_attend.cuh"

namespace xnq {
namespace {

__device__ unsigned int g_kv_plan_status;

// ---- page tables ----
//
//   needed(b, i) = i ps < length_b  and  ((i + 1) ps > first_b  or  i ps < sinks)
//   kept(b, i)   = needed, and the entry is a page                        used = the pages of kept entries
// The k-th entry (row by row) that is needed and not kept gets the k-th page, in ascending order, that is not used. What pages are free is not state of its
// own: it follows from the table, so pages that two rows name (a shared beginning) are free when the last of them lets go.
//
// One thread-block cluster. Every CTA marks the pages of its run of entries in a bitmap of its own (shared memory); the CTAs add the bitmaps up, a slice each
// (distributed shared memory), write the list of the first free pages, as many as are missing, and go over their entries again.
constexpr int RESERVE_THREADS = 1024, RESERVE_WARPS = RESERVE_THREADS / 32, RESERVE_MOST_CTAS = 16;

struct ReserveArgs {
  const int *from;
  int *to;
  long long from_stride, to_stride, num_pages, max_seq, sinks;
  const long long *length, *first; // first: null, or [batch]
  long long *room, *free;
  int *list; // [num_pages]
  long long cells;
  int batch, per, page_size; // per: entries of a row
};

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() { // every thread of every CTA; what was written before, shared or global, is seen behind it
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t in_cta(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
__device__ __forceinline__ uint32_t load_remote(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ void store_remote(uint32_t addr, uint32_t v) { asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(addr), "r"(v) : "memory"); }

// exclusive sums over a block; total: of all
template <int WARPS>
__device__ __forceinline__ unsigned block_before(unsigned v, unsigned *s_warp, unsigned &total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  unsigned inc = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const unsigned up = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += up;
  }
  if (lane == 31) s_warp[warp] = inc;
  __syncthreads();
  unsigned before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < WARPS; w++) {
    const unsigned x = s_warp[w];
    if (w < warp) before += x;
    total += x;
  }
  __syncthreads();
  return before + inc - v;
}

__global__ void __launch_bounds__(RESERVE_THREADS, 1) kv_reserve_kernel(const ReserveArgs a, int ctas) {
  extern __shared__ uint32_t bitmap[];
  __shared__ unsigned s_warp[RESERVE_WARPS], s_missing[RESERVE_WARPS];
  __shared__ uint32_t s_cta[2][RESERVE_MOST_CTAS]; // free pages and missing entries of every CTA
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t rank = cluster_rank();
  const int words = (int)((a.num_pages + 31) / 32);
  for (int i = threadIdx.x; i < words; i += RESERVE_THREADS) bitmap[i] = 0u;
  __syncthreads();
  pdl_launch_dependents();
  pdl_wait();
  for (int b = rank * RESERVE_THREADS + threadIdx.x; b < a.batch; b += ctas * RESERVE_THREADS) a.room[b] = min(max(a.length[b], 0ll), a.max_seq);

  // A warp's run of entries, in the order of the table; f(entry, needed, row, place) for each.
  const long long run = (a.cells + (long long)ctas * RESERVE_WARPS * 32 - 1) / ((long long)ctas * RESERVE_WARPS * 32) * 32;
  const long long begin = (rank * (long long)RESERVE_WARPS + warp) * run, end = min(begin + run, a.cells);
  const unsigned ps = (unsigned)a.page_size;
  auto walk = [&](auto f) {
    int row = 0, i = 0, known = -1;
    unsigned last = 0, from = 0, heads = 0; // entries [0, heads) and [from, last) are needed
    for (long long at = begin; at < end; at += 32) {
      const long long cell = at + lane;
      const bool in = cell < end;
      if (at == begin || a.per < 32) row = in ? (int)(cell / a.per) : 0, i = in ? (int)(cell - (long long)row * a.per) : 0;
      else {
        i += 32;
        if (i >= a.per) i -= a.per, row++;
      }
      if (in && row != known) {
        known = row;
        const unsigned n = (unsigned)min(max(a.length[row], 0ll), a.max_seq);
        last = (n + ps - 1) / ps;
        from = a.first ? min((unsigned)min(max(a.first[row], 0ll), a.max_seq) / ps, last) : 0u;
        heads = a.first ? min((unsigned)min(a.sinks, a.max_seq + ps) / ps + ((unsigned)min(a.sinks, a.max_seq + ps) % ps != 0), last) : 0u;
      }
      const bool needed = in && (unsigned)i < last && ((unsigned)i >= from || (unsigned)i < heads);
      f(in, needed, row, i);
    }
  };
  auto entry = [&](bool needed, int row, int i) { // -1: no page
    const int v = needed ? a.from[row * a.from_stride + i] : -1;
    return v >= 0 && v < a.num_pages ? v : -1;
  };
  unsigned missing = 0;
  walk([&](bool, bool needed, int row, int i) {
    const int v = entry(needed, row, i);
    missing += __popc(__ballot_sync(0xffffffffu, needed && v < 0));
    // Pages of neighbouring entries often share a word: one atomic for the warp.
    const unsigned have = __ballot_sync(0xffffffffu, v >= 0);
    if (have) {
      const int w = __shfl_sync(0xffffffffu, v >> 5, __ffs(have) - 1);
      if (__all_sync(0xffffffffu, v < 0 || (v >> 5) == w)) {
        const unsigned bits = __reduce_or_sync(0xffffffffu, v >= 0 ? 1u << (v & 31) : 0u);
        if (lane == 0) atomicOr(&bitmap[w], bits);
      } else if (v >= 0) atomicOr(&bitmap[v >> 5], 1u << (v & 31));
    }
  });
  if (lane == 0) s_missing[warp] = missing;
  if (ctas > 1) cluster_sync();
  else __syncthreads();

  // ---- this CTA's slice of the pages: all bitmaps together, and how many are free ----
  const int slice = (words + ctas - 1) / ctas, w0 = min((int)rank * slice, words), w1 = min(w0 + slice, words);
  const int each = (slice + RESERVE_THREADS - 1) / RESERVE_THREADS, mine0 = min(w0 + (int)threadIdx.x * each, w1), mine1 = min(mine0 + each, w1);
  const uint32_t map = (uint32_t)__cvta_generic_to_shared(bitmap);
  if (ctas > 1) {
    for (int w = w0 + threadIdx.x; w < w1; w += RESERVE_THREADS) { // (in this CTA's own bitmap nobody else looks at this slice)
      uint32_t x[RESERVE_MOST_CTAS];
#pragma unroll
      for (int c = 0; c < RESERVE_MOST_CTAS; c++) x[c] = c < ctas ? load_remote(in_cta(map + w * 4, c)) : 0u;
      uint32_t all = 0;
#pragma unroll
      for (int c = 0; c < RESERVE_MOST_CTAS; c++) all |= x[c];
      bitmap[w] = all;
    }
    __syncthreads();
  }
  auto free_in = [&](int w) {
    const long long left = a.num_pages - (long long)w * 32; // pages of the word
    return ~bitmap[w] & (left >= 32 ? 0xffffffffu : (1u << left) - 1u);
  };
  unsigned n_free = 0, free_here, missing_here = 0, missing_before = 0;
  for (int w = mine0; w < mine1; w++) n_free += __popc(free_in(w));
  unsigned free_before = block_before<RESERVE_WARPS>(n_free, s_warp, free_here);
#pragma unroll
  for (int w = 0; w < RESERVE_WARPS; w++) {
    if (w < warp) missing_before += s_missing[w];
    missing_here += s_missing[w];
  }
  unsigned free_all = free_here, missing_all = missing_here;
  if (ctas > 1) {
    if ((int)threadIdx.x < ctas) {
      store_remote(in_cta((uint32_t)__cvta_generic_to_shared(&s_cta[0][rank]), threadIdx.x), free_here);
      store_remote(in_cta((uint32_t)__cvta_generic_to_shared(&s_cta[1][rank]), threadIdx.x), missing_here);
    }
    cluster_sync();
    free_all = missing_all = 0;
    for (int c = 0; c < ctas; c++) {
      const unsigned f = s_cta[0][c], m = s_cta[1][c];
      if (c < (int)rank) free_before += f, missing_before += m;
      free_all += f, missing_all += m;
    }
  }
  if (missing_all) {
    for (int w = mine0; w < mine1 && free_before < missing_all; w++)
      for (uint32_t bits = free_in(w); bits && free_before < missing_all; bits &= bits - 1) a.list[free_before++] = w * 32 + __ffs(bits) - 1;
    if (ctas > 1) cluster_sync();
    else __syncthreads();
  }

  unsigned at = missing_before; // which of the missing entries the warp is at
  walk([&](bool in, bool needed, int row, int i) {
    int v = entry(needed, row, i);
    const unsigned none = __ballot_sync(0xffffffffu, needed && v < 0);
    if (needed && v < 0) {
      const unsigned k = at + __popc(none & ((1u << lane) - 1u));
      if (k < free_all) v = __ldcg(a.list + k);
      else atomicMin(a.room + row, (long long)i * a.page_size);
    }
    at += __popc(none);
    if (in) a.to[row * a.to_stride + i] = v;
  });
  if (rank == 0 && threadIdx.x == 0) *a.free = (long long)free_all - min(free_all, missing_all);
}

// ---- where packed tokens go ----
struct PlanArgs {
  KvView c;
  xnq_kv_plan p;
  const long long *pos, *count;
  const int *parents;
  int pos_stride, page_size;
};
__device__ __forceinline__ long long tokens_of(const PlanArgs &a, int b) { return min(max(a.count[b], 0ll), (long long)a.p.longest); }
// a place in a sequence -> a row of the cache's memory, or -1
__device__ __forceinline__ long long slot_of(const PlanArgs &a, int b, long long place) {
  if (!a.c.table) return (long long)b * a.page_size + place;
  const unsigned pi = (unsigned)place / (unsigned)a.page_size;
  const int page = __ldg(a.c.table + b * a.c.table_stride + pi);
  if (page < 0 || page >= a.c.num_pages) {
    atomicOr(&g_kv_plan_status, KV_NO_PAGE);
    return -1;
  }
  return (long long)page * a.page_size + (place - (long long)pi * a.page_size);
}

// Rows in the order of their sequences: every CTA adds up the counts (offsets in shared memory) and takes a run of tokens, each found by bisection.
constexpr int PLAN_THREADS = 256, PLAN_TOKENS = 512, PLAN_MOST_BATCH = 32768;
__global__ void __launch_bounds__(PLAN_THREADS) kv_plan_kernel(const PlanArgs a) {
  extern __shared__ int s_off[]; // [batch + 1]
  __shared__ long long s_sum[PLAN_THREADS / 32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, batch = (int)a.p.batch;
  pdl_launch_dependents();
  pdl_wait();
  const int each = (batch + PLAN_THREADS - 1) / PLAN_THREADS, b0 = min((int)threadIdx.x * each, batch), b1 = min(b0 + each, batch);
  long long sum = 0;
  bool cut = false;
  for (int b = b0; b < b1; b++) {
    const long long n = tokens_of(a, b);
    sum += n, cut |= n != a.count[b];
  }
  long long inc = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long up = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += up;
  }
  if (lane == 31) s_sum[warp] = inc;
  __syncthreads();
  long long off = inc - sum;
#pragma unroll
  for (int w = 0; w < PLAN_THREADS / 32; w++)
    if (w < warp) off += s_sum[w];
  for (int b = b0; b < b1; b++) {
    const int o = (int)min(off, (long long)a.p.tokens);
    s_off[b] = o;
    if (blockIdx.x == 0) a.p.offsets[b] = o, a.p.start[b] = a.pos[(long long)b * a.pos_stride];
    off += tokens_of(a, b);
  }
  if (b1 == batch && b0 < b1) { // (one thread)
    s_off[batch] = (int)min(off, (long long)a.p.tokens);
    if (blockIdx.x == 0) a.p.offsets[batch] = s_off[batch];
    cut |= off > a.p.tokens;
  }
  if (cut && blockIdx.x == 0) atomicOr(&g_kv_plan_status, KV_PLAN_CUT);
  __syncthreads();
  const int all = s_off[batch];
#pragma unroll
  for (int k = 0; k < PLAN_TOKENS / PLAN_THREADS; k++) {
    const long long t = (long long)blockIdx.x * PLAN_TOKENS + k * PLAN_THREADS + threadIdx.x;
    if (t >= a.p.tokens) break;
    int seq = -1;
    long long place = -1, slot = -1;
    if (t < all) {
      int lo = 0, hi = batch; // the last sequence that starts at or before t: s_off[lo] <= t < s_off[hi]
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (s_off[mid] <= t) lo = mid;
        else hi = mid;
      }
      seq = lo;
      place = a.pos[(long long)seq * a.pos_stride] + (t - s_off[seq]);
      if (place >= a.c.max_seq) {
        atomicOr(&g_kv_plan_status, KV_PAST_STORE);
        place = -1;
      }
      place = max(place, -1ll);
      if (place >= 0) slot = slot_of(a, seq, place);
    }
    a.p.sequence[t] = seq, a.p.position[t] = place, a.p.slot[t] = slot;
  }
}

// Trees: a CTA a sequence, a thread a token, which holds the bits of the tokens that it sees. In each round a token takes over what the token sees that it has
// reached, and goes on to where that one stands: the depth's logarithm of rounds.
__global__ void __launch_bounds__(XNQ_KV_TREE_MOST) kv_plan_trees_kernel(const PlanArgs a) {
  constexpr int T = XNQ_KV_TREE_MOST, W = T / 32;
  __shared__ uint32_t s_sees[T][W + 1];
  __shared__ int s_up[T];
  __shared__ uint32_t s_ok[W];
  __shared__ long long s_sum[2][W];
  const int i = threadIdx.x, lane = i & 31, warp = i >> 5, batch = (int)a.p.batch, b = blockIdx.x, words = ((int)a.p.longest + 31) / 32;
  pdl_launch_dependents();
  pdl_wait();
  long long before = 0, all = 0;
  bool cut = false;
  for (int x = i; x < batch; x += T) {
    const long long n = tokens_of(a, x);
    all += n, cut |= n != a.count[x];
    if (x < b) before += n;
  }
#pragma unroll
  for (int o = 16; o >= 1; o >>= 1) before += __shfl_xor_sync(0xffffffffu, before, o), all += __shfl_xor_sync(0xffffffffu, all, o);
  if (lane == 0) s_sum[0][warp] = before, s_sum[1][warp] = all;
  __syncthreads();
  before = all = 0;
#pragma unroll
  for (int w = 0; w < W; w++) before += s_sum[0][w], all += s_sum[1][w];
  const long long tokens = a.p.tokens, off = min(before, tokens), here = min(before + tokens_of(a, b), tokens) - off; // of this sequence
  const long long pos = a.pos[(long long)b * a.pos_stride];
  if (i == 0) {
    a.p.offsets[b] = off, a.p.start[b] = pos;
    if (b == batch - 1) a.p.offsets[batch] = off + here;
  }
  if (b == 0 && (cut || all > tokens)) atomicOr(&g_kv_plan_status, KV_PLAN_CUT);

  uint32_t sees[W];
  int up = i < here ? a.parents[off + i] : -2;
  bool ok = up >= -1 && up < i && pos >= 0;
  if (i < here && up != -2 && !(up >= -1 && up < i)) atomicOr(&g_kv_plan_status, KV_PLAN_CUT); // a parent that is none
  if (ok && pos + i >= a.c.max_seq) {
    atomicOr(&g_kv_plan_status, KV_PAST_STORE);
    ok = false;
  }
#pragma unroll
  for (int w = 0; w < W; w++) sees[w] = w == warp ? 1u << lane : 0u;
  if (!ok) up = -1;
  while (__syncthreads_or(up >= 0)) {
#pragma unroll
    for (int w = 0; w < W; w++)
      if (w < words) s_sees[i][w] = sees[w];
    s_up[i] = ok ? up : -2; // -2: none, and so is who descends from it
    __syncthreads();
    if (up >= 0) {
#pragma unroll
      for (int w = 0; w < W; w++)
        if (w < words) sees[w] |= s_sees[up][w];
      const int next = s_up[up];
      ok = next > -2, up = max(next, -1);
    }
  }
  const unsigned there = __ballot_sync(0xffffffffu, ok);
  if (lane == 0) s_ok[warp] = there;
  __syncthreads();
  if (i < words) a.p.nodes[(long long)b * words + i] = s_ok[i];
  if (i < here) {
    int depth = -1;
#pragma unroll
    for (int w = 0; w < W; w++) {
      depth += __popc(sees[w]);
      if (w < words) a.p.sees[(off + i) * words + w] = ok ? sees[w] : 0u;
    }
    a.p.sequence[off + i] = b, a.p.position[off + i] = ok ? pos + depth : -1, a.p.slot[off + i] = ok ? slot_of(a, b, pos + i) : -1;
  }
  for (long long t = min(all, tokens) + (long long)b * T + i; t < tokens; t += (long long)batch * T) { // behind the last sequence
    a.p.sequence[t] = -1, a.p.position[t] = a.p.slot[t] = -1;
    for (int w = 0; w < words; w++) a.p.sees[t * words + w] = 0u;
  }
}

// ---- the accepted path kept ----
// The tokens that `node` sees, r = 0, 1, .. in their order, move from place pos + index to pos + r; index >= r, and both ascend. A warp takes the keys or the
// values of a head, KEEP_ROWS tokens at a time: all of them are read before one is written, and what a later batch reads lies behind what this one writes.
constexpr int KEEP_WARPS = 4, KEEP_ROWS = 8;
template <int BITS, int HD>
__global__ void __launch_bounds__(KEEP_WARPS * 32) kv_keep_kernel(KvView c, xnq_kv_plan p, const long long *node, long long *pos_out) {
  using L = KvTile<BITS, HD>;
  constexpr int W = L::W, NB = L::NB;
  constexpr int K_ITEMS = 4 * W + NB / 2, V_ITEMS = 16 * W + NB, EACH = (V_ITEMS + 31) / 32; // 32-bit words of a key, 16-bit halves of a value; with scales
  __shared__ uint16_t s_path[KEEP_WARPS][XNQ_KV_TREE_MOST];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, words = ((int)p.longest + 31) / 32;
  const long long unit = (long long)blockIdx.x * KEEP_WARPS + warp; // (sequence, head, keys or values)
  pdl_launch_dependents();
  pdl_wait();
  if (unit >= p.batch * 2 * c.kv_heads) return;
  const int b = (int)(unit / (2 * c.kv_heads)), kh = (int)(unit - (long long)b * (2 * c.kv_heads)), head = kh >> 1;
  const bool is_v = kh & 1;
  const long long off = p.offsets[b], here = p.offsets[b + 1] - off, start = p.start[b], at = node[b];
  uint32_t bits = at >= 0 && at < here && lane < words ? p.sees[(off + at) * words + lane] : 0u;
  int inc = __popc(bits);
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int up = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += up;
  }
  const int n = __shfl_sync(0xffffffffu, inc, 31);
  for (int r = inc - __popc(bits); bits; bits &= bits - 1) s_path[warp][r++] = (uint16_t)(lane * 32 + __ffs(bits) - 1);
  if (kh == 0 && lane == 0) pos_out[b] = start + n;
  __syncwarp();
  auto item = [&](uint8_t *tile, int row, int x) -> uint8_t * { // item x of a row of a tile
    if (!is_v) return x < 4 * W ? tile + L::k_word(row, x / W, x % W) : tile + L::k_scale(row, 2 * (x - 4 * W));
    if (x < 8 * W) return tile + L::v_word(row / 2, x / W, x % W) + (row & 1) * 2;
    return tile + L::v_scale(row / 2, x - 8 * W) + (row & 1) * 2;
  };
  const int items = is_v ? 8 * W + NB : K_ITEMS;
  for (int r0 = 0; r0 < n; r0 += KEEP_ROWS) {
    // lanes 0 .. 7 look up where the batch's tokens are, lanes 8 .. 15 where they go
    const int r = r0 + (lane & (KEEP_ROWS - 1));
    const bool used = lane < 2 * KEEP_ROWS && r < n && s_path[warp][r] != r;
    const long long place = used ? start + (lane < KEEP_ROWS ? (int)s_path[warp][r] : r) : 0;
    uint8_t *const tile_at = used ? kv_tile_at(c, b, head, (int)(place / KV_TILE), L::BYTES) : nullptr;
    const int row_at = (int)(place % KV_TILE);
    uint32_t v[KEEP_ROWS][EACH];
    uint8_t *to[KEEP_ROWS];
    int to_row[KEEP_ROWS];
#pragma unroll
    for (int k = 0; k < KEEP_ROWS; k++) {
      uint8_t *const tile = reinterpret_cast<uint8_t *>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(tile_at), k));
      to[k] = reinterpret_cast<uint8_t *>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(tile_at), KEEP_ROWS + k));
      const int row = __shfl_sync(0xffffffffu, row_at, k);
      to_row[k] = __shfl_sync(0xffffffffu, row_at, KEEP_ROWS + k);
      if (!tile) to[k] = nullptr; // (no page: not moved)
#pragma unroll
      for (int e = 0; e < EACH; e++) {
        const int x = e * 32 + lane;
        v[k][e] = 0u;
        if (to[k] && x < items) v[k][e] = is_v ? *reinterpret_cast<const uint16_t *>(item(tile, row, x)) : *reinterpret_cast<const uint32_t *>(item(tile, row, x));
      }
    }
    __syncwarp();
#pragma unroll
    for (int k = 0; k < KEEP_ROWS; k++)
#pragma unroll
      for (int e = 0; e < EACH; e++) {
        const int x = e * 32 + lane;
        if (!to[k] || x >= items) continue;
        if (is_v) *reinterpret_cast<uint16_t *>(item(to[k], to_row[k], x)) = (uint16_t)v[k][e];
        else *reinterpret_cast<uint32_t *>(item(to[k], to_row[k], x)) = v[k][e];
      }
    __syncwarp();
  }
}

constexpr long long RESERVE_MOST_PAGES = 1ll << 20; // a bitmap of 128 KB
int reserve_ctas(int64_t cells) { return cells <= 8192 ? 1 : 8; }

} // namespace

int kv_plan_status(unsigned int *bits) {
  XNQ_CUDA(cudaMemcpyFromSymbol(bits, g_kv_plan_status, sizeof(*bits)));
  return XNQ_OK;
}
int kv_plan_init() {
  unsigned int zero = 0;
  XNQ_CUDA(cudaMemcpyToSymbol(g_kv_plan_status, &zero, sizeof(zero)));
  XNQ_CUDA(cudaFuncSetAttribute(kv_reserve_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)(RESERVE_MOST_PAGES / 8)));
  XNQ_CUDA(cudaFuncSetAttribute(kv_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (PLAN_MOST_BATCH + 1) * 4));
  return XNQ_OK;
}

int kv_plan_check(const char *who, const xnq_kv_plan *p) {
  if (!p || !p->start || !p->offsets || !p->sequence || !p->position || !p->slot) return fail(XNQ_ERR_NULL, "%s: the plan is NULL, or one of its arrays", who);
  if ((p->sees == nullptr) != (p->nodes == nullptr)) return fail(XNQ_ERR_NULL, "%s: a plan of trees has both sees and nodes", who);
  if (p->tokens < 0 || p->tokens > INT32_MAX - 1024 || p->batch < 1 || p->batch > PLAN_MOST_BATCH || p->longest < 1 || p->longest > INT32_MAX)
    return fail(XNQ_ERR_SHAPE, "%s: a plan of %lld tokens of %lld sequences (1 to %d), of up to %lld each", who, (long long)p->tokens, (long long)p->batch, PLAN_MOST_BATCH,
                (long long)p->longest);
  if (p->sees && p->longest > XNQ_KV_TREE_MOST) return fail(XNQ_ERR_UNSUPPORTED, "%s: trees of %lld tokens (up to %d are served)", who, (long long)p->longest, XNQ_KV_TREE_MOST);
  return XNQ_OK;
}

} // namespace xnq

using namespace xnq;

extern "C" {

size_t xnq_kv_reserve_workspace_bytes(int64_t num_pages) { return num_pages < 1 || num_pages > RESERVE_MOST_PAGES ? 0 : (size_t)(num_pages + 3) / 4 * 16; }

int xnq_kv_reserve(int32_t *table, int64_t table_stride, const int32_t *from, int64_t from_stride, int64_t batch, int64_t page_size, int64_t num_pages, int64_t max_seq,
                   const long long *length, const long long *first, int64_t sinks, long long *room, long long *free_pages, void *workspace, size_t ws_bytes, void *stream) {
  clear_error();
  if (batch < 0 || batch > INT32_MAX || page_size < KV_TILE || page_size % KV_TILE || page_size > INT32_MAX || num_pages < 1 || max_seq < 1 || max_seq > INT32_MAX - KV_TILE || sinks < 0)
    return fail(XNQ_ERR_SHAPE, "kv_reserve: batch %lld, page_size %lld (a multiple of %d), num_pages %lld, max_seq %lld, sinks %lld", (long long)batch, (long long)page_size, KV_TILE,
                (long long)num_pages, (long long)max_seq, (long long)sinks);
  if (num_pages > RESERVE_MOST_PAGES) return fail(XNQ_ERR_UNSUPPORTED, "kv_reserve: %lld pages (up to %lld are served)", (long long)num_pages, RESERVE_MOST_PAGES);
  if (!free_pages || (batch && (!table || !from || !length || !room))) return fail(XNQ_ERR_NULL, "kv_reserve: NULL argument");
  const int64_t per = (max_seq + page_size - 1) / page_size;
  if (table_stride < per || from_stride < per) return fail(XNQ_ERR_SIZE, "kv_reserve: rows of %lld and %lld entries; %lld positions take %lld", (long long)table_stride, (long long)from_stride, (long long)max_seq, (long long)per);
  if (batch * per > INT32_MAX - 1024) return fail(XNQ_ERR_SIZE, "kv_reserve: tables of %lld x %lld entries", (long long)batch, (long long)per);
  if (!workspace || ws_bytes < xnq_kv_reserve_workspace_bytes(num_pages)) return fail(XNQ_ERR_SIZE, "kv_reserve: workspace has %zu bytes, needs %zu", ws_bytes, xnq_kv_reserve_workspace_bytes(num_pages));
  if (reinterpret_cast<uintptr_t>(workspace) & 15) return fail(XNQ_ERR_ALIGN, "kv_reserve: the workspace must be 16-byte aligned");
  ReserveArgs a{from, table, from_stride, table_stride, num_pages, max_seq, std::min<int64_t>(sinks, INT32_MAX), length, first, room, free_pages, static_cast<int *>(workspace), batch * per, (int)batch, (int)per, (int)page_size};
  const int ctas = reserve_ctas(a.cells);
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)ctas), cfg.blockDim = dim3(RESERVE_THREADS), cfg.dynamicSmemBytes = (size_t)(num_pages + 31) / 32 * 4, cfg.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)ctas, attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr, cfg.numAttrs = 2;
  XNQ_CUDA(cudaLaunchKernelEx(&cfg, kv_reserve_kernel, a, ctas));
  count_launch();
  return XNQ_OK;
}

int xnq_kv_plan_make(const xnq_kv_cache *cache, const long long *pos, int pos_stride, const long long *count, const int32_t *parents, const xnq_kv_plan *plan, void *stream) {
  clear_error();
  PlanArgs a{};
  int rc = kv_plan_check("kv_plan", plan);
  if (rc != XNQ_OK || (rc = kv_view("kv_plan", cache, plan->batch, &a.c)) != XNQ_OK) return rc;
  if (!pos || !count) return fail(XNQ_ERR_NULL, "kv_plan: NULL argument");
  if (pos_stride < 0 || pos_stride > 1) return fail(XNQ_ERR_SHAPE, "kv_plan: pos_stride %d (0 or 1)", pos_stride);
  if ((parents == nullptr) != (plan->sees == nullptr)) return fail(XNQ_ERR_NULL, "kv_plan: parents and the plan's sees go together");
  a.p = *plan, a.pos = pos, a.count = count, a.parents = parents, a.pos_stride = pos_stride, a.page_size = (int)cache->page_size;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (parents) XNQ_CUDA(launch_pdl(kv_plan_trees_kernel, dim3((unsigned)plan->batch), dim3(XNQ_KV_TREE_MOST), 0, s, a));
  else
    XNQ_CUDA(launch_pdl(kv_plan_kernel, dim3((unsigned)std::max<int64_t>(1, (plan->tokens + PLAN_TOKENS - 1) / PLAN_TOKENS)), dim3(PLAN_THREADS), (size_t)(plan->batch + 1) * 4, s, a));
  count_launch();
  return XNQ_OK;
}

int xnq_kv_keep(const xnq_kv_cache *cache, const xnq_kv_plan *plan, const long long *node, long long *pos_out, void *stream) {
  clear_error();
  KvView c;
  int rc = kv_plan_check("kv_keep", plan);
  if (rc != XNQ_OK || (rc = kv_view("kv_keep", cache, plan->batch, &c)) != XNQ_OK) return rc;
  if (!plan->sees) return fail(XNQ_ERR_NULL, "kv_keep: the plan is not one of trees");
  if (!node || !pos_out) return fail(XNQ_ERR_NULL, "kv_keep: NULL argument");
  const int64_t warps = plan->batch * 2 * c.kv_heads;
  const dim3 grid((unsigned)((warps + KEEP_WARPS - 1) / KEEP_WARPS)), block(KEEP_WARPS * 32);
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int bits = kv_bits(cache->ggml_dtype);
  if (bits == 4) {
    if (cache->head_dim == 64) XNQ_CUDA(launch_pdl(kv_keep_kernel<4, 64>, grid, block, 0, s, c, *plan, node, pos_out));
    else XNQ_CUDA(launch_pdl(kv_keep_kernel<4, 128>, grid, block, 0, s, c, *plan, node, pos_out));
  } else if (cache->head_dim == 64) XNQ_CUDA(launch_pdl(kv_keep_kernel<8, 64>, grid, block, 0, s, c, *plan, node, pos_out));
  else XNQ_CUDA(launch_pdl(kv_keep_kernel<8, 128>, grid, block, 0, s, c, *plan, node, pos_out));
  count_launch();
  return XNQ_OK;
}

} // extern "C"
