// Page tables and slot maps of the quantized KV cache, made on the GPU from request lengths; and the accepted path of a tree of drafted tokens kept.
//
// All of it is a few hundred kilobytes at most (the largest tables some megabytes) and bound by latency: launches, dependent loads, barriers. So each call is
// one launch (page tables of more than 4096 entries three), with nothing read back by the host.
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
// Entries lie in the order of the table, 32 CELLS neighbouring ones to a warp; a lane's are asked for together. Up to RESERVE_SMALL entries: one block, a bitmap of
// the pages and the list of the free ones in shared memory (up to 1024 entries and 131072 pages a block of 128 threads: 256 entries 5.2 us, with 1024
// threads 8.2; 4096 entries, 512 threads, 6.2). More: three kernels over all SMs (clear the bitmap; mark pages and count what is missing; give pages out, every block adding up what is missing
// before it and, if it misses any itself, reading the bitmap for the free pages of its ranks): 16384 entries 8.9 us, 1024000 22 us, of which the bytes take 1.3.
// (One cluster of 8 or 16 CTAs with their bitmaps added up in distributed shared memory: 8.6 and 73 us.)
constexpr int CELLS = 8, RESERVE_THREADS = 256, RESERVE_SMALL_THREADS = 512, RESERVE_SMALL = RESERVE_SMALL_THREADS * CELLS;

struct Divisor { // n / d for n < 2^31: n m >> (31 + s), s = ceil(log2 d), m = floor(2^(31 + s) / d) + 1, whose error n (m d - 2^(31 + s)) < 2^(31 + s) never carries
  unsigned m, s;
  static Divisor of(unsigned d) {
    unsigned s = 0;
    while ((1ull << s) < d) s++;
    return Divisor{(unsigned)((1ull << (31 + s)) / d + 1), 31 + s};
  }
  __device__ __forceinline__ unsigned operator()(unsigned n) const { return (unsigned)(((unsigned long long)n * m) >> s); }
};
struct ReserveArgs {
  const int *from;
  int *to;
  long long from_stride, to_stride, max_seq, end; // end: of a row's last page, max_seq or behind it
  const long long *length, *first; // first: null, or [batch]
  long long *room, *free;
  uint32_t *bitmap; // many entries: pages that are in use
  unsigned *missing; // many entries: of a block
  unsigned num_pages, sinks, cells, per, page_size; // per: entries of a row
  int batch;
  Divisor by_per, by_page;
};

struct Cells { // a lane's entries, 32 apart
  int v[CELLS];                  // their pages; -1: none
  unsigned row[CELLS], at[CELLS];
  unsigned in, needed;           // bits: is there such an entry, is it needed
};
__device__ __forceinline__ void load_cells(const ReserveArgs &a, unsigned begin, Cells &c) { // begin: the lane's first entry
  c.in = c.needed = 0u;
  unsigned n[CELLS], f[CELLS], past = 0u; // past: bits, `first` lies behind the last page
#pragma unroll
  for (int k = 0; k < CELLS; k++) {
    const unsigned cell = begin + k * 32;
    const bool in = cell < a.cells;
    c.in |= (in ? 1u : 0u) << k;
    c.row[k] = in ? a.by_per(cell) : 0u, c.at[k] = cell - c.row[k] * a.per;
    c.v[k] = in ? a.from[c.row[k] * a.from_stride + c.at[k]] : -1;
    n[k] = in ? (unsigned)min(max(a.length[c.row[k]], 0ll), a.max_seq) : 0u;
    const long long first = in && a.first ? a.first[c.row[k]] : 0ll;
    f[k] = (unsigned)min(max(first, 0ll), a.max_seq); // (from max_seq to `end`: the same page)
    past |= (first >= a.end ? 1u : 0u) << k;
  }
#pragma unroll
  for (int k = 0; k < CELLS; k++) {
    bool needed = n[k] && c.at[k] <= a.by_page(n[k] - 1); // entries of positions below the length
    if (a.first) needed = needed && ((!((past >> k) & 1u) && c.at[k] >= a.by_page(f[k])) || c.at[k] * (unsigned long long)a.page_size < a.sinks);
    c.needed |= (needed ? 1u : 0u) << k;
    if (!needed || (unsigned)c.v[k] >= a.num_pages) c.v[k] = -1;
  }
}
__device__ __forceinline__ void mark_pages(const Cells &c, uint32_t *bitmap) { // pages of neighbouring entries often share a word: one atomic for the warp
#pragma unroll
  for (int k = 0; k < CELLS; k++) {
    const int v = c.v[k];
    const unsigned have = __ballot_sync(0xffffffffu, v >= 0);
    if (!have) continue;
    const int lead = __ffs(have) - 1, w = __shfl_sync(0xffffffffu, v >> 5, lead);
    if (__all_sync(0xffffffffu, v < 0 || (v >> 5) == w)) {
      const unsigned bits = __reduce_or_sync(0xffffffffu, v >= 0 ? 1u << (v & 31) : 0u);
      if ((threadIdx.x & 31) == 0) atomicOr(bitmap + w, bits);
    } else if (v >= 0) atomicOr(bitmap + (v >> 5), 1u << (v & 31));
  }
}
__device__ __forceinline__ unsigned missing_cells(const Cells &c) { // of the warp
  unsigned n = 0;
#pragma unroll
  for (int k = 0; k < CELLS; k++) n += ((c.needed >> k) & 1u) && c.v[k] < 0;
  return __reduce_add_sync(0xffffffffu, n);
}
// list: the free pages from the rank `base` on; `at`: the rank of the warp's first missing entry; free_all: free pages there are
__device__ __forceinline__ void give_pages(const ReserveArgs &a, Cells &c, unsigned at, unsigned base, unsigned free_all, const int *list) {
  const unsigned below = (1u << (threadIdx.x & 31)) - 1u;
#pragma unroll
  for (int k = 0; k < CELLS; k++) {
    const bool none = ((c.needed >> k) & 1u) && c.v[k] < 0;
    const unsigned who = __ballot_sync(0xffffffffu, none);
    if (none) {
      const unsigned r = at + __popc(who & below);
      if (r < free_all) c.v[k] = list[r - base];
      else atomicMin(a.room + c.row[k], (long long)c.at[k] * a.page_size);
    }
    at += __popc(who);
    if ((c.in >> k) & 1u) a.to[c.row[k] * a.to_stride + c.at[k]] = c.v[k];
  }
}
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
  const unsigned x = lane < WARPS ? s_warp[lane] : 0u; // (up to 32 warps)
  const unsigned before = __reduce_add_sync(0xffffffffu, lane < warp ? x : 0u);
  total = __reduce_add_sync(0xffffffffu, x);
  __syncthreads();
  return before + inc - v;
}
// The bitmap in chunks of 256 words, a warp a chunk and a lane 8 neighbouring words of it (words behind the last page's are 0, and no page is free there).
constexpr unsigned CHUNK = 256, MOST_CHUNKS = (1u << 20) / 32 / CHUNK; // of RESERVE_MOST_PAGES
__device__ __forceinline__ uint32_t pages_of(const ReserveArgs &a, unsigned w) { // that there are of a word's 32
  return w * 32 + 32 <= a.num_pages ? 0xffffffffu : w * 32 < a.num_pages ? (1u << (a.num_pages & 31)) - 1u : 0u;
}
__device__ __forceinline__ void load_chunk(const ReserveArgs &a, const uint32_t *bitmap, unsigned chunk, uint32_t (&free)[8]) {
  const unsigned w = chunk * CHUNK + (threadIdx.x & 31) * 8;
  const uint4 x = *reinterpret_cast<const uint4 *>(bitmap + w), y = *reinterpret_cast<const uint4 *>(bitmap + w + 4);
  const uint32_t used[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
#pragma unroll
  for (int i = 0; i < 8; i++) free[i] = ~used[i];
  if ((chunk + 1) * (CHUNK * 32) > a.num_pages) // (the last one)
#pragma unroll
    for (int i = 0; i < 8; i++) free[i] &= pages_of(a, w + i);
}
template <int WARPS>
__device__ __forceinline__ unsigned count_free(const ReserveArgs &a, const uint32_t *bitmap, unsigned chunks, unsigned *s_chunk, unsigned *s_warp) { // s_chunk: free pages before each chunk
#pragma unroll 2
  for (unsigned k = threadIdx.x >> 5; k < chunks; k += WARPS) {
    uint32_t free[8];
    load_chunk(a, bitmap, k, free);
    unsigned n = 0;
#pragma unroll
    for (int i = 0; i < 8; i++) n += __popc(free[i]);
    n = __reduce_add_sync(0xffffffffu, n);
    if ((threadIdx.x & 31) == 0) s_chunk[k] = n;
  }
  __syncthreads();
  static_assert(MOST_CHUNKS <= 128 && WARPS >= 4, "a chunk a thread");
  unsigned all;
  const unsigned n = threadIdx.x < chunks ? s_chunk[threadIdx.x] : 0u, before = block_before<WARPS>(n, s_warp, all);
  if (threadIdx.x < chunks) s_chunk[threadIdx.x] = before;
  __syncthreads();
  return all;
}
// The free pages of ranks [first, first + n) into list: a word a thread, so that no thread has more than 32 pages to write (with a lane's 8 words as they are
// loaded above, the pages of a small cache were one lane's: 16 us for 4 rows of 64 entries).
template <int THREADS>
__device__ __forceinline__ void list_pages(const ReserveArgs &a, const uint32_t *bitmap, unsigned chunks, const unsigned *s_chunk, unsigned *s_warp, unsigned first, unsigned n, int *list) {
  constexpr unsigned GROUP = THREADS > CHUNK ? THREADS / CHUNK : 1, WORDS = THREADS > CHUNK ? 1 : CHUNK / THREADS; // chunks at a time, words of a thread
  unsigned k = 0; // the chunk of the first one: the last that begins at or before it
  for (unsigned end = chunks; end - k > 1;) {
    const unsigned mid = (k + end) / 2;
    if (s_chunk[mid] <= first) k = mid;
    else end = mid;
  }
  for (k = k / GROUP * GROUP; k < chunks && s_chunk[k] < first + n; k += GROUP) {
    unsigned before = s_chunk[k];
#pragma unroll
    for (unsigned x = 0; x < WORDS; x++) {
      const unsigned w = k * CHUNK + x * THREADS + threadIdx.x;
      uint32_t bits = w * 32 < a.num_pages ? ~bitmap[w] & pages_of(a, w) : 0u;
      unsigned sum, rank = before + block_before<THREADS / 32>(__popc(bits), s_warp, sum);
      for (; bits; bits &= bits - 1, rank++)
        if (rank >= first && rank < first + n) list[rank - first] = (int)(w * 32) + __ffs(bits) - 1;
      before += sum;
    }
  }
}

template <int THREADS> // CELLS entries each
__global__ void __launch_bounds__(THREADS, 1) kv_reserve_small_kernel(const ReserveArgs a) {
  constexpr int WARPS = THREADS / 32;
  extern __shared__ __align__(16) uint32_t bitmap[];
  __shared__ int s_list[THREADS * CELLS];
  __shared__ unsigned s_warp[WARPS], s_chunk[MOST_CHUNKS];
  const unsigned chunks = (a.num_pages + 32 * CHUNK - 1) / (32 * CHUNK), lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (unsigned i = threadIdx.x; i < chunks * CHUNK; i += THREADS) bitmap[i] = 0u;
  pdl_launch_dependents();
  pdl_wait();
  Cells c;
  load_cells(a, warp * (32 * CELLS) + lane, c);
  for (int b = threadIdx.x; b < a.batch; b += THREADS) a.room[b] = min(max(a.length[b], 0ll), a.max_seq);
  __syncthreads();
  mark_pages(c, bitmap);
  unsigned missing_all;
  const unsigned mine = missing_cells(c), before = block_before<WARPS>(lane == 0 ? mine : 0u, s_warp, missing_all); // (its barriers order the bitmap, too)
  const unsigned free_all = count_free<WARPS>(a, bitmap, chunks, s_chunk, s_warp);
  if (missing_all) {
    list_pages<THREADS>(a, bitmap, chunks, s_chunk, s_warp, 0u, missing_all, s_list);
    __syncthreads();
  }
  give_pages(a, c, __shfl_sync(0xffffffffu, before, 0), 0u, free_all, s_list);
  if (threadIdx.x == 0) *a.free = (long long)free_all - min(free_all, missing_all);
}

__global__ void __launch_bounds__(RESERVE_THREADS) kv_reserve_clear_kernel(const ReserveArgs a) {
  pdl_launch_dependents();
  pdl_wait();
  const unsigned words = (a.num_pages + 32 * CHUNK - 1) / (32 * CHUNK) * CHUNK;
  for (unsigned i = blockIdx.x * RESERVE_THREADS + threadIdx.x; i < words; i += gridDim.x * RESERVE_THREADS) a.bitmap[i] = 0u;
  for (unsigned b = blockIdx.x * RESERVE_THREADS + threadIdx.x; b < (unsigned)a.batch; b += gridDim.x * RESERVE_THREADS) a.room[b] = min(max(a.length[b], 0ll), a.max_seq);
}
__global__ void __launch_bounds__(RESERVE_THREADS) kv_reserve_mark_kernel(const ReserveArgs a) {
  __shared__ unsigned s_missing[RESERVE_THREADS / 32];
  const unsigned lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  pdl_launch_dependents();
  pdl_wait();
  Cells c;
  load_cells(a, blockIdx.x * (RESERVE_THREADS * CELLS) + warp * (32 * CELLS) + lane, c);
  mark_pages(c, a.bitmap);
  const unsigned n = missing_cells(c);
  if (lane == 0) s_missing[warp] = n;
  __syncthreads();
  if (threadIdx.x == 0) {
    unsigned all = 0;
#pragma unroll
    for (int w = 0; w < RESERVE_THREADS / 32; w++) all += s_missing[w];
    a.missing[blockIdx.x] = all;
  }
}
__global__ void __launch_bounds__(RESERVE_THREADS, 4) kv_reserve_give_kernel(const ReserveArgs a) {
  constexpr int WARPS = RESERVE_THREADS / 32;
  __shared__ int s_list[RESERVE_THREADS * CELLS];
  __shared__ unsigned s_warp[WARPS], s_chunk[MOST_CHUNKS];
  const unsigned lane = threadIdx.x & 31, warp = threadIdx.x >> 5, chunks = (a.num_pages + 32 * CHUNK - 1) / (32 * CHUNK);
  pdl_launch_dependents();
  pdl_wait();
  Cells c;
  load_cells(a, blockIdx.x * (RESERVE_THREADS * CELLS) + warp * (32 * CELLS) + lane, c);
  unsigned before = 0, all = 0;
  for (unsigned x = threadIdx.x; x < gridDim.x; x += RESERVE_THREADS) {
    const unsigned m = __ldcg(a.missing + x);
    all += m, before += x < blockIdx.x ? m : 0u;
  }
  unsigned here, missing_all, blocks_before, free_all = 0;
  const unsigned mine = missing_cells(c), at = __shfl_sync(0xffffffffu, block_before<WARPS>(lane == 0 ? mine : 0u, s_warp, here), 0);
  block_before<WARPS>(before, s_warp, blocks_before);
  block_before<WARPS>(all, s_warp, missing_all);
  if (here || blockIdx.x == 0) {
    free_all = count_free<WARPS>(a, a.bitmap, chunks, s_chunk, s_warp);
    list_pages<RESERVE_THREADS>(a, a.bitmap, chunks, s_chunk, s_warp, blocks_before, here, s_list);
    __syncthreads();
  }
  give_pages(a, c, blocks_before + at, blocks_before, free_all, s_list);
  if (blockIdx.x == 0 && threadIdx.x == 0) *a.free = (long long)free_all - min(free_all, missing_all);
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
  const int page = a.c.table[b * a.c.table_stride + pi];
  if (page < 0 || page >= a.c.num_pages) {
    atomicOr(&g_kv_plan_status, KV_NO_PAGE);
    return -1;
  }
  return (long long)page * a.page_size + (place - (long long)pi * a.page_size);
}

// Rows in the order of their sequences: every CTA adds up the counts (offsets in shared memory) and takes a run of tokens, each found by bisection. Bound by the
// chain counts, sums, page, stores: 200 sequences with 31000 tokens 4.7 us, a tenth of which its bytes take.
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
      place = first_place(a.pos, (long long)seq * a.pos_stride) + (t - s_off[seq]);
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
// reached, and goes on to where that one stands: the depth's logarithm of rounds (a walk from the root to every token would be a chain of as many loads as the
// tree is deep). 48 trees of up to 61 tokens 3.7 us, most of it the launch and two dependent loads.
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
  const long long pos = first_place(a.pos, (long long)b * a.pos_stride);
  if (i == 0) {
    a.p.offsets[b] = off, a.p.start[b] = a.pos[(long long)b * a.pos_stride];
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
// values of a head, KEEP_ROWS tokens at a time: all of them are read before one is written, and what a later batch reads lies behind what this one writes. Bound
// by the chain offsets, bits, pages, codes: 24 trees of up to 40 tokens, 8 heads of 128 in Q4_0, 5.1 us, in Q8_0 5.5.
constexpr int KEEP_WARPS = 4, KEEP_ROWS = 8;
template <int BITS, int HD>
__global__ void __launch_bounds__(KEEP_WARPS * 32) kv_keep_kernel(KvView c, xnq_kv_plan p, const long long *node, long long *pos_out) {
  using L = KvTile<BITS, HD>;
  constexpr int W = L::W, NB = L::NB;
  constexpr int K_ITEMS = 4 * W + NB / 2, V_ITEMS = 8 * W + NB, EACH = ((K_ITEMS > V_ITEMS ? K_ITEMS : V_ITEMS) + 31) / 32; // 32-bit words of a key, 16-bit halves of a value; with scales
  static_assert(K_ITEMS * 4 == L::RB + NB * 2 && V_ITEMS * 2 == L::RB + NB * 2, "a position's bytes");
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
  const int items = is_v ? V_ITEMS : K_ITEMS;
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
size_t reserve_bitmap_bytes(int64_t num_pages) { return (size_t)((num_pages + 32 * CHUNK - 1) / (32 * CHUNK)) * CHUNK * 4; }

} // namespace

int kv_plan_status(unsigned int *bits) {
  XNQ_CUDA(cudaMemcpyFromSymbol(bits, g_kv_plan_status, sizeof(*bits)));
  return XNQ_OK;
}
int kv_plan_init() {
  unsigned int zero = 0;
  XNQ_CUDA(cudaMemcpyToSymbol(g_kv_plan_status, &zero, sizeof(zero)));
  XNQ_CUDA(cudaFuncSetAttribute(kv_reserve_small_kernel<RESERVE_SMALL_THREADS>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)(RESERVE_MOST_PAGES / 8)));
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

size_t xnq_kv_reserve_workspace_bytes(int64_t batch, int64_t page_size, int64_t num_pages, int64_t max_seq) {
  if (batch < 0 || page_size < 1 || max_seq < 1 || num_pages < 1 || num_pages > RESERVE_MOST_PAGES) return 0;
  const int64_t cells = batch * ((max_seq + page_size - 1) / page_size);
  return cells <= RESERVE_SMALL ? 16 : reserve_bitmap_bytes(num_pages) + (size_t)(cells / (RESERVE_THREADS * CELLS) + 1) * 4;
}

int xnq_kv_reserve(int32_t *table, int64_t table_stride, const int32_t *from, int64_t from_stride, int64_t batch, int64_t page_size, int64_t num_pages, int64_t max_seq,
                   const long long *length, const long long *first, int64_t sinks, long long *room, long long *free_pages, void *workspace, size_t ws_bytes, void *stream) {
  clear_error();
  if (batch < 0 || batch > INT32_MAX || page_size < KV_TILE || page_size % KV_TILE || page_size > INT32_MAX || num_pages < 1 || max_seq < 1 || max_seq > INT32_MAX - KV_TILE || sinks < 0)
    return fail(XNQ_ERR_SHAPE, "kv_reserve: batch %lld, page_size %lld (a multiple of %d), num_pages %lld, max_seq %lld, sinks %lld", (long long)batch, (long long)page_size, KV_TILE,
                (long long)num_pages, (long long)max_seq, (long long)sinks);
  if (num_pages > RESERVE_MOST_PAGES) return fail(XNQ_ERR_UNSUPPORTED, "kv_reserve: %lld pages (up to %lld are served)", (long long)num_pages, RESERVE_MOST_PAGES);
  if (!free_pages || (batch && (!table || !from || !length || !room))) return fail(XNQ_ERR_NULL, "kv_reserve: NULL argument");
  const int64_t per = (max_seq + page_size - 1) / page_size, cells = batch * per;
  if (table_stride < per || from_stride < per) return fail(XNQ_ERR_SIZE, "kv_reserve: rows of %lld and %lld entries; %lld positions take %lld", (long long)table_stride, (long long)from_stride, (long long)max_seq, (long long)per);
  if (cells > INT32_MAX - RESERVE_SMALL) return fail(XNQ_ERR_SIZE, "kv_reserve: tables of %lld x %lld entries", (long long)batch, (long long)per);
  const size_t need = xnq_kv_reserve_workspace_bytes(batch, page_size, num_pages, max_seq);
  if (!workspace || ws_bytes < need) return fail(XNQ_ERR_SIZE, "kv_reserve: workspace has %zu bytes, needs %zu", ws_bytes, need);
  if (reinterpret_cast<uintptr_t>(workspace) & 15) return fail(XNQ_ERR_ALIGN, "kv_reserve: the workspace must be 16-byte aligned");
  uint8_t *const ws = static_cast<uint8_t *>(workspace);
  const ReserveArgs a{from, table, from_stride, table_stride, max_seq, per * page_size, length, first, room, free_pages, reinterpret_cast<uint32_t *>(ws),
                      reinterpret_cast<unsigned *>(ws + reserve_bitmap_bytes(num_pages)), (unsigned)num_pages, (unsigned)std::min<int64_t>(sinks, INT32_MAX), (unsigned)cells, (unsigned)per,
                      (unsigned)page_size, (int)batch, Divisor::of((unsigned)per), Divisor::of((unsigned)page_size)};
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (cells <= RESERVE_SMALL) {
    const size_t smem = reserve_bitmap_bytes(num_pages);
    if (cells <= 128 * CELLS && smem <= 16384) XNQ_CUDA(launch_pdl(kv_reserve_small_kernel<128>, dim3(1), dim3(128), smem, s, a));
    else XNQ_CUDA(launch_pdl(kv_reserve_small_kernel<RESERVE_SMALL_THREADS>, dim3(1), dim3(RESERVE_SMALL_THREADS), smem, s, a));
    count_launch();
    return XNQ_OK;
  }
  const dim3 block(RESERVE_THREADS), grid((unsigned)((cells + RESERVE_THREADS * CELLS - 1) / (RESERVE_THREADS * CELLS)));
  XNQ_CUDA(launch_pdl(kv_reserve_clear_kernel, dim3(32), block, 0, s, a));
  count_launch();
  XNQ_CUDA(launch_pdl(kv_reserve_mark_kernel, grid, block, 0, s, a));
  count_launch();
  XNQ_CUDA(launch_pdl(kv_reserve_give_kernel, grid, block, 0, s, a));
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
