// Attention over the quantized KV cache.
//
// ---- few query rows (a decode step, drafts) and f32 queries: kv_attend_split_kernel ----
//
//   s[j, r] = scale sum_blocks d_k[j, blk] (sum_i c_k[j, i] q[r, i] - z sum_i q[r, i])          z: the code of zero, 8 or 128
//   o[r, :] = sum_j p[j, r] d_v[j, blk] (c_v[j, :] - z) / sum_j p[j, r]                          p = 2^(s log2 e - reference)
//
// The codes are whole numbers and go to the tensor cores as they are, one matrix instruction (m16n8k16, f32 sums) for 16 positions (S) or 16 dims
// (O) by 8 query rows; scales meet the f32 sums (keys) or the weights (values). Bound by the cache's bytes, if unpacking stays cheap: a tile's 32
// positions are 4608 bytes, which an SM gets in 200 cycles. So no code is converted: masked out of its word, a nibble or byte in the low ten
// bits of a half is the f16 SUBNORMAL c 2^-24 (bits 4..7: 16 c 2^-24, the 16 undone in q or in the result), exact in the product; one shift and four masks a
// word of eight 4-bit codes. The -z term comes from the sums' start value (S) or from one more product, of the weights with -z (O).
//
// The rows of a KV head's query heads (and of a few tokens) are the 8 NT columns of a tile; a wider group takes several row tiles. The work is the
// flattened list of (sequence, KV head, row tile, tile of 32 positions), cut into equal runs, one a CTA, so that ragged batches balance. The four
// warps of a CTA take its tiles in turn, each with a ring of stages filled by cp.async and a running maximum and sum of its own; they meet in shared memory
// where the run leaves an item. An item that is cut goes through records in the workspace: its last CTA to arrive adds them, in the order of the
// parts, whoever came first.
//
// f32 queries (SPLIT): q and the weights are taken apart into two f16 each (22 bits), and the codes have their zero taken off first and are whole numbers in
// f16: a subnormal operand's products are summed with the bits that a number of 2^-14 would have, some 2^-18 of the score, and with many weights the two
// sums in O would cancel. The instruction's sums cut off what is too small for the larger summand, always downwards, so sixteen positions are summed by themselves and added to
// O by f32 additions: an output's error is 3e-7 to 5e-7 of its norm at any length (one sum through all of them: 5e-6 for 131072 positions of Q8_0;
// f32 products 9e-7). 16-bit queries: q is exact in f16 after a power of two a row, the weights are rounded to f16.
// Ranges: a row's reference lies 8 (8 bits: 11) below its maximum of the time and is renewed when a score passes it by more than 12 (14), so that nothing need
// be known of a tile's maximum beforehand; the values' scales are brought near one by a power of two a warp.
//
// Measured (bf16 queries, 32 heads over 8 of 128): 16 sequences of 8192 positions in Q4_0 blocks 43 us, 64 of 330 to 16384 in pages 140 us (4.2 TB/s of cache),
// one of 131072 47 us, of 512 10 us in a captured step; Q8_0, 16 of 8192, 66 us (4.3 TB/s). Few rows of many positions are bound by latency: a tile is one chain of 570
// instructions a warp, and with 12 warps an SM (128 registers and 16 warps were slower) issue, the ALU, tensor and memory pipes are each busy for less than half
// of the time. Few positions are bound by the chain of positions, first tile, a tile's arithmetic and the meeting of the parts.
#include <algorithm>
#include <cmath>

#include "xnq_kv_attend.cuh"
#include "xnq_quantize_act.cuh"

namespace xnq {
namespace {

__device__ unsigned int g_kv_attend_status;

constexpr int SPLIT_WARPS = 4, SPLIT_STAGES = 3, START_TILES = 12;
// What sequence b's queries see, as tiles [first, first + count).
struct Span {
  int first, count;
  long long pos;
};
__device__ __forceinline__ Span span_of(const AttendArgs &a, int b) {
  Span s;
  s.pos = a.pos[(long long)b * a.pos_stride];
  const long long hi = min(s.pos + a.seq - 1, a.c.max_seq - 1), p0 = max(s.pos, 0ll), lo = a.window ? max(p0 - a.window + 1, 0ll) : 0ll;
  s.first = (int)(min(lo, a.c.max_seq) / KV_TILE);
  s.count = hi < lo ? 0 : (int)(hi / KV_TILE) - s.first + 1;
  return s;
}
__device__ __forceinline__ void load8_any(const void *p, int dtype, long long at, float (&v)[8]) {
  if (dtype == XNQ_F32) load8(static_cast<const float *>(p) + at, v);
  else if (dtype == XNQ_F16) load8(static_cast<const __half *>(p) + at, v);
  else load8(static_cast<const __nv_bfloat16 *>(p) + at, v);
}
__device__ __forceinline__ void store_any(void *p, int dtype, long long at, float v) {
  if (dtype == XNQ_F32) static_cast<float *>(p)[at] = v;
  else if (dtype == XNQ_F16) static_cast<__half *>(p)[at] = __float2half_rn(v);
  else static_cast<__nv_bfloat16 *>(p)[at] = __float2bfloat16_rn(v);
}

template <int V> // 2 or 4 values
__device__ __forceinline__ void load_vec(const float *p, float (&v)[V]) {
  if (V == 4) {
    const float4 x = *reinterpret_cast<const float4 *>(p);
    v[0] = x.x, v[1] = x.y, v[V - 2] = x.z, v[V - 1] = x.w;
  } else {
    const float2 x = *reinterpret_cast<const float2 *>(p);
    v[0] = x.x, v[1] = x.y;
  }
}
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, const float (&c)[4]) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
}
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) { // d +=
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) { // of 16-bit values: lane (g, t) gives row g's columns 2 t, 2 t + 1 and gets column g's rows
  uint32_t d;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(v));
  return d;
}
template <int BITS, int HD, int NT>
struct SplitShape {
  static constexpr int R = 8 * NT;        // query rows of an item
  static constexpr int COL = HD + 4;      // floats from row to row of the accumulators in shared memory
  static constexpr int MERGE = SPLIT_WARPS * R * (COL + 2) * 4; // bytes
  // Ranges of the weights, 2^BELOW at a row's maximum when its reference was set and at most 2^OVER, and of the values' scales, 2^LEAST to 2^MOST before
  // they are brought near one, so that a weight times a scale stays below 2^16 and is 4 or more at the maximum: f16 holds it to its rounding
  // down to 2^-16 of that. Q8_0's scales are a sixteenth of Q4_0's for the same values.
  static constexpr float BELOW = BITS == 4 ? 8.f : 11.f, OVER = BITS == 4 ? 12.f : 14.f;
  static constexpr int LEAST = BITS == 4 ? -6 : -9, MOST = BITS == 4 ? 2 : 1;
};

// Parts of items in the workspace, two places a CTA: references [R], sums [R], accumulators [R][HD]. A cut item's ticket is that of the CTA which holds its
// first part.
constexpr int MAX_SPLIT_GRID = 148 * 4, RECORD_STRIDE = 16 * (128 + 2);
constexpr size_t RECORDS_BYTES = (size_t)MAX_SPLIT_GRID * 2 * RECORD_STRIDE * 4;

// A tile's copy into shared memory by one warp; null: zeros.
template <int BYTES>
__device__ __forceinline__ void copy_tile(uint32_t dst, const uint8_t *src, const uint8_t *some, int lane) {
  const uint32_t n = src ? 16u : 0u;
  const uint8_t *s = src ? src : some;
#pragma unroll
  for (int i = 0; i < (BYTES / 16 + 31) / 32; i++) {
    const int ch = i * 32 + lane;
    if (BYTES / 16 % 32 == 0 || ch < BYTES / 16)
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst + ch * 16), "l"(s + ch * 16), "r"(n) : "memory");
  }
}

// CTAs an SM that registers are to leave room for. f32 queries over 128 dims: with three, sums of their own spill (Q4_0, 131072 positions, 78 us against 70,
// 512 positions 12.7 against 10.7); over 64 dims two are slower (16 sequences of 8192 positions, Q8_0, 51 us against 49).
constexpr int split_ctas(int hd, int nt, bool split) { return nt == 1 && !(split && hd == 128) ? 3 : 2; }

template <int BITS, int HD, int NT, bool SPLIT>
__global__ void __launch_bounds__(SPLIT_WARPS * 32, split_ctas(HD, NT, SPLIT)) kv_attend_split_kernel(const AttendArgs a) {
  using L = KvTile<BITS, HD>;
  using P = SplitShape<BITS, HD, NT>;
  constexpr int NB = L::NB, W = L::W, R = P::R;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ long long s_sum[SPLIT_WARPS];
  __shared__ long long s_before;
  __shared__ int s_b, s_last;
  __shared__ Span s_span;
  __shared__ unsigned s_runs[4][SPLIT_WARPS];
  // Where an item's rows go; of an item and the next one: warp 0 writes the next one's while other warps still store this one's rows. Between an item and
  // the one after the next lie barriers that every warp reaches when it is done with the first.
  __shared__ long long s_row[2][R], s_lse_row[2][R];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  float *const merge = reinterpret_cast<float *>(smem + SPLIT_WARPS * SPLIT_STAGES * L::BYTES);
  float *const s_m = merge, *const s_l = merge + SPLIT_WARPS * R, *const s_acc = merge + 2 * SPLIT_WARPS * R;
  uint8_t *const ring = smem + warp * SPLIT_STAGES * L::BYTES;
  const uint32_t ring_addr = (uint32_t)__cvta_generic_to_shared(ring);
  pdl_launch_dependents();
  pdl_wait();

  // ---- this CTA's run of the flattened list: [t0, t1) of `total` tiles ----
  const int per_seq = a.c.kv_heads * a.row_tiles; // items of a sequence, all of its count of tiles
  const int batch = (int)a.batch;
  Span own{0, 0, 0}; // (most batches: the one look at the positions)
  if ((int)threadIdx.x < batch) own = span_of(a, threadIdx.x);
  const auto counted = [](int n) { return n ? n + (1ll << 40) : 0ll; }; // tiles, and above them sequences that have some
  long long mine = counted(own.count);
  bool look = (int)threadIdx.x < batch && (own.count == 0 || own.pos + a.seq > a.c.max_seq); // a sequence that sees nothing, or that lies past the cache
  for (int b = threadIdx.x + SPLIT_WARPS * 32; b < batch; b += SPLIT_WARPS * 32) {
    const Span sp = span_of(a, b);
    mine += counted(sp.count), look |= sp.count == 0 || sp.pos + a.seq > a.c.max_seq;
  }
#pragma unroll
  for (int o = 16; o >= 1; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
  if (lane == 0) s_sum[warp] = mine;
  look = __syncthreads_or(look);
  long long total = 0;
#pragma unroll
  for (int w = 0; w < SPLIT_WARPS; w++) total += s_sum[w];
  const long long items = (total >> 40) * per_seq;
  total = (total & ((1ll << 40) - 1)) * per_seq;
  // Short items go to CTAs of their own: a run shorter than a tile a warp only where the items are shorter too.
  const long long at_least = min((long long)SPLIT_WARPS, max(total / max(items, 1ll), 1ll));
  long long share = max((total + gridDim.x - 1) / gridDim.x, at_least);
  if (share > at_least) share = (share + SPLIT_WARPS - 1) / SPLIT_WARPS * SPLIT_WARPS; // as long for the warps, and fewer parts to join
  // A run that goes on into a second item pays for another start and end, about as long as START_TILES take: where a run of a few more tiles keeps every
  // CTA within one item, the items are rounded up to whole runs.
  bool whole_runs = false;
  {
    const long long more[4] = {share, share + max(share / 8, 1ll), share + max(share / 4, 2ll), share + max(share / 2, 3ll)};
    unsigned runs[4] = {0u, 0u, 0u, 0u};
    if (share <= 24) {
      for (int b = threadIdx.x; b < batch; b += SPLIT_WARPS * 32) {
        const unsigned n = (unsigned)(b == (int)threadIdx.x ? own.count : span_of(a, b).count);
#pragma unroll
        for (int k = 0; k < 4; k++) runs[k] += (n + (unsigned)more[k] - 1) / (unsigned)more[k];
      }
#pragma unroll
      for (int k = 0; k < 4; k++) runs[k] = __reduce_add_sync(0xffffffffu, runs[k]);
      if (lane == 0)
#pragma unroll
        for (int k = 0; k < 4; k++) s_runs[k][warp] = runs[k];
      __syncthreads();
#pragma unroll
      for (int k = 3; k >= 0; k--) {
        unsigned long long sum = 0;
#pragma unroll
        for (int w = 0; w < SPLIT_WARPS; w++) sum += s_runs[k][w];
        if (sum * per_seq <= gridDim.x) share = more[k], whole_runs = true, total = sum * per_seq * more[k];
      }
    }
  }
  // Else every item is as long in the list as its tiles and a start and end: with tiles alone the CTAs with many short items are the last (64 sequences of
  // 330 to 16384 positions: 149 us against 143).
  const int lead = whole_runs ? 0 : (int)min((long long)START_TILES, share / 2);
  if (lead) {
    total += items * lead;
    share = (total + gridDim.x - 1) / gridDim.x;
  }
  auto length = [&](int count) { return whole_runs ? (count + share - 1) / share * share : count ? (long long)count + lead : 0ll; }; // of an item in the list
  const long long t0 = blockIdx.x * share, t1 = min(total, t0 + share);

  if (look) // sequences that see nothing: rows of zeros
    for (int b = blockIdx.x; b < batch; b += gridDim.x) {
      const Span sp = span_of(a, b);
      if (threadIdx.x == 0 && sp.pos + a.seq > a.c.max_seq) atomicOr(&g_kv_attend_status, KV_PAST_ATTEND);
      if (sp.count) continue;
      for (long long i = threadIdx.x; i < a.seq * a.heads * HD; i += SPLIT_WARPS * 32) {
        const long long row = i / HD, s = row / a.heads;
        const int h = (int)(row - s * a.heads), d = (int)(i - row * HD);
        store_any(a.out.p, a.dtype, b * a.out.sb + s * a.out.ss + h * a.out.sh + d, 0.f);
        if (a.lse && d == 0) a.lse[(b * a.seq + s) * a.heads + h] = -INFINITY;
      }
    }
  if (t0 >= t1) return;
  // the sequence of tile t0: a scan of the lengths, a block of threads at a time
  if (threadIdx.x == 0) s_b = batch;
  long long before = 0;
  for (int base = 0; base < batch; base += SPLIT_WARPS * 32) {
    const Span sp = base == 0 ? own : base + (int)threadIdx.x < batch ? span_of(a, base + threadIdx.x) : Span{0, 0, 0};
    const long long n = length(sp.count) * per_seq;
    long long inc = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long up = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += up;
    }
    __syncthreads(); // s_sum has been read
    if (lane == 31) s_sum[warp] = inc;
    __syncthreads();
    long long here = before;
#pragma unroll
    for (int w = 0; w < SPLIT_WARPS; w++) {
      if (w < warp) here += s_sum[w];
      before += s_sum[w];
    }
    if (n && here + inc - n <= t0 && t0 < here + inc) s_b = base + threadIdx.x, s_before = here + inc - n, s_span = sp; // one thread
    if (before > t0) break;
  }
  __syncthreads();
  int b = s_b;
  if (b >= batch) return; // (only where pos changes under the kernel)
  long long item0 = s_before; // first tile of the item at hand in the flattened list
  Span sp = s_span;
  int item = (int)((t0 - item0) / length(sp.count)); // of the sequence: (KV head, row tile)
  item0 += item * length(sp.count);

  int turn = 0; // which of the two copies is the item's
  for (long long at = t0; at < t1;) {
    while (item == per_seq || sp.count == 0) { // on to the next sequence that has tiles
      item = 0;
      if (++b >= batch) return; // (only where pos changes under the kernel)
      sp = span_of(a, b);
    }
    const int kvh = item / a.row_tiles, rt = item - kvh * a.row_tiles;
    const int ta = (int)max(0ll, at - item0 - lead), tb = (int)min((long long)sp.count, t1 - item0 - lead); // tiles [ta, tb) of the item are this CTA's
    if (tb <= ta) { // (a run that ends or starts before the item's first tile)
      at = item0 + length(sp.count), item0 = at, item++;
      continue;
    }
    const int rows = (int)min((long long)R, a.seq * a.group - (long long)rt * R);

    // ---- start the ring: this warp's tiles are ta + warp, + 4, ...; lane i looks up the page of the i-th of a batch of 32 ----
    const int n_tiles = tb - ta > warp ? (tb - ta - warp + SPLIT_WARPS - 1) / SPLIT_WARPS : 0;
    const uint8_t *ahead = nullptr; // lane i's tile
    unsigned gone = 0;              // bit s: the tile in stage s has no page
    auto issue = [&](int i) {
      if (i < n_tiles) {
        if ((i & 31) == 0) {
          const int mine_i = i + lane;
          ahead = mine_i < n_tiles ? kv_tile_at(a.c, b, kvh, sp.first + ta + warp + mine_i * SPLIT_WARPS, L::BYTES) : nullptr;
        }
        const uint8_t *src = reinterpret_cast<const uint8_t *>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(ahead), i & 31));
        const int stage = i % SPLIT_STAGES;
        gone = (gone & ~(1u << stage)) | (src ? 0u : 1u << stage);
        copy_tile<L::BYTES>(ring_addr + stage * L::BYTES, src, a.c.pages, lane);
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
#pragma unroll
    for (int i = 0; i < SPLIT_STAGES - 1; i++) issue(i);

    // ---- the query rows as operands ----
    uint32_t qh[NT][NB][4], ql[SPLIT ? NT : 1][SPLIT ? NB : 1][4]; // [.. ][b][2 step + register]
    float start[SPLIT ? 1 : NT][SPLIT ? 1 : NB][4] = {}, factor[NT][2]; // of columns 2 t, 2 t + 1; start as the sums' registers are
    int lo[NT][2], hi[NT][2], lo_all = 0, hi_all = INT32_MAX, hi_any = -1, lo_any = INT32_MAX;
#pragma unroll
    for (int n = 0; n < NT; n++) {
      const int r = n * 8 + g; // this lane's row as an operand's column
      const long long row = (long long)rt * R + r, s = row / a.group;
      const int h = kvh * a.group + (int)(row - s * a.group);
      if (warp == 0 && t == 0) s_row[turn][r] = b * a.out.sb + s * a.out.ss + h * a.out.sh, s_lse_row[turn][r] = ((long long)b * a.seq + s) * a.heads + h;
      float v[NB][8], top = 0.f;
#pragma unroll
      for (int bl = 0; bl < NB; bl++) {
#pragma unroll
        for (int i = 0; i < 8; i++) v[bl][i] = 0.f;
        if (r < rows) load8_any(a.q.p, a.dtype, b * a.q.sb + s * a.q.ss + h * a.q.sh + bl * 32 + t * 8, v[bl]);
#pragma unroll
        for (int i = 0; i < 8; i++) top = fmaxf(top, fabsf(v[bl][i]));
      }
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      int e = top > 0.f && top < INFINITY ? 13 - ilogbf(top) : 0; // the largest |q| to [2^13, 2^14)
      e = max(-100, min(100, e));
      const float up = ldexpf(a.scale < 0.f ? -1.f : 1.f, e); // the scale's sign goes into q, so that the largest score is the largest sum
      float sum[NB];
#pragma unroll
      for (int bl = 0; bl < NB; bl++) {
        float hi_v[8], lo_v[8];
        sum[bl] = 0.f;
#pragma unroll
        for (int i = 0; i < 8; i++) {
          const float x = v[bl][i] * up;
          hi_v[i] = __half2float(__float2half_rn(x));
          lo_v[i] = SPLIT ? __half2float(__float2half_rn(x - hi_v[i])) : 0.f;
          sum[bl] += hi_v[i] + lo_v[i];
        }
        if (!SPLIT) {
          sum[bl] += __shfl_xor_sync(0xffffffffu, sum[bl], 1);
          sum[bl] += __shfl_xor_sync(0xffffffffu, sum[bl], 2);
        }
#pragma unroll
        for (int i = 0; i < 4; i++) { // pair i of a word: dims i and i + 4 (4 bits, the odd ones 16 times too large), or of word i / 2 bytes i % 2 and i % 2 + 2
          const int x = BITS == 4 ? i : (i >> 1) * 4 + (i & 1), y = BITS == 4 ? i + 4 : x + 2;
          const float down = !SPLIT && BITS == 4 && (i & 1) ? 0.0625f : 1.f;
          qh[n][bl][i] = pack_half2(hi_v[x] * down, hi_v[y] * down);
          if (SPLIT) ql[n][bl][i] = pack_half2(lo_v[x] * down, lo_v[y] * down);
        }
      }
      int l0, h0;
      seen_by(a, sp.pos, s, l0, h0);
      if (r >= rows) l0 = 0, h0 = INT32_MAX; // no row: its weights are thrown away
      else hi_any = max(hi_any, h0), lo_any = min(lo_any, l0);
      lo_all = max(lo_all, l0), hi_all = min(hi_all, h0);
      const float f = fmaxf(ldexpf(fabsf(a.scale) * LOG2E, (SPLIT ? 0 : 24) - e), LEAST_FACTOR);
#pragma unroll
      for (int c = 0; c < 2; c++) { // from the lane that holds row 2 t + c
        const int from = (2 * t + c) * 4;
        if (!SPLIT)
#pragma unroll
          for (int bl = 0; bl < NB; bl++)
            start[SPLIT ? 0 : n][SPLIT ? 0 : bl][c] = start[SPLIT ? 0 : n][SPLIT ? 0 : bl][c + 2] = __shfl_sync(0xffffffffu, sum[bl], from) * (-(float)L::ZERO / 16777216.f);
        factor[n][c] = __shfl_sync(0xffffffffu, f, from);
        lo[n][c] = __shfl_sync(0xffffffffu, l0, from), hi[n][c] = __shfl_sync(0xffffffffu, h0, from);
      }
    }
#pragma unroll
    for (int o = 4; o <= 16; o <<= 1) {
      lo_all = max(lo_all, __shfl_xor_sync(0xffffffffu, lo_all, o)), hi_all = min(hi_all, __shfl_xor_sync(0xffffffffu, hi_all, o));
      lo_any = min(lo_any, __shfl_xor_sync(0xffffffffu, lo_any, o)), hi_any = max(hi_any, __shfl_xor_sync(0xffffffffu, hi_any, o));
    }

    // ---- this warp's tiles ----
    float acc[NT][2 * NB][4], ref[NT][2], limit[NT][2], l[NT][2]; // limit: a score above it asks for another reference
#pragma unroll
    for (int n = 0; n < NT; n++) {
#pragma unroll
      for (int i = 0; i < 2 * NB; i++)
#pragma unroll
        for (int c = 0; c < 4; c++) acc[n][i][c] = 0.f;
      ref[n][0] = ref[n][1] = 0.f, limit[n][0] = limit[n][1] = -INFINITY, l[n][0] = l[n][1] = 0.f;
    }
    int k = 0;                 // the values' scales are taken times 2^k
    bool k_set = false;
    float d_most = 0.f;        // more than this: another k
    for (int i = 0; i < n_tiles; i++) {
      issue(i + SPLIT_STAGES - 1);
      asm volatile("cp.async.wait_group %0;" ::"n"(SPLIT_STAGES - 1) : "memory");
      __syncwarp();
      const int stage = i % SPLIT_STAGES;
      const uint8_t *tile = ring + stage * L::BYTES;
      const int j0 = (sp.first + ta + warp + i * SPLIT_WARPS) * KV_TILE;
      const bool masked = j0 < lo_all || j0 + KV_TILE - 1 > hi_all;
      if ((gone >> stage) & 1) { // no page: not attended to
        if (lane == 0) atomicOr(&g_kv_attend_status, KV_NO_PAGE);
        __syncwarp();
        continue;
      }
      if (j0 > hi_any || j0 + KV_TILE - 1 < lo_any) { // (other row tiles of the sequence see it)
        __syncwarp();
        continue;
      }
      // scores: registers [group of 16][n][c]; c 0, 1: position g, 2, 3: g + 8 of the group; columns 2 t + (c & 1)
      float s[2][NT][4];
#pragma unroll
      for (int u = 0; u < 2; u++) {
        uint32_t w[2][W];
        uint32_t dk[2][NB / 2];
#pragma unroll
        for (int e = 0; e < 2; e++) {
          const int row = u * 16 + e * 8 + g;
          if (W == 2) {
            const uint2 x = *reinterpret_cast<const uint2 *>(tile + L::k_word(row, t, 0));
            w[e][0] = x.x, w[e][1] = x.y;
          } else {
#pragma unroll
            for (int q4 = 0; q4 < W; q4 += 4) {
              const uint4 x = *reinterpret_cast<const uint4 *>(tile + L::k_word(row, t, q4));
              w[e][q4] = x.x, w[e][q4 + 1] = x.y, w[e][q4 + 2] = x.z, w[e][q4 + 3] = x.w;
            }
          }
#pragma unroll
          for (int q2 = 0; q2 < NB / 2; q2 += 2) {
            if (NB == 4) {
              const uint2 x = *reinterpret_cast<const uint2 *>(tile + L::k_scale(row, 0));
              dk[e][0] = x.x, dk[e][NB / 2 - 1] = x.y;
            } else dk[e][0] = *reinterpret_cast<const uint32_t *>(tile + L::k_scale(row, 0));
          }
        }
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
          for (int c = 0; c < 4; c++) s[u][n][c] = 0.f;
#pragma unroll
        for (int bl = 0; bl < NB; bl++) {
          const float d0 = bl & 1 ? __high2float(as_half2(dk[0][bl / 2])) : __low2float(as_half2(dk[0][bl / 2]));
          const float d1 = bl & 1 ? __high2float(as_half2(dk[1][bl / 2])) : __low2float(as_half2(dk[1][bl / 2]));
          uint32_t op[2][4];
#pragma unroll
          for (int step = 0; step < 2; step++)
#pragma unroll
            for (int e = 0; e < 2; e++) {
              const uint32_t x = BITS == 4 ? w[e][bl] : w[e][2 * bl + step];
              const int i0 = BITS == 4 ? 2 * step : 0;
              op[step][e] = SPLIT ? signed_pair<BITS>(x, i0) : code_pair<BITS>(x, i0), op[step][e + 2] = SPLIT ? signed_pair<BITS>(x, i0 + 1) : code_pair<BITS>(x, i0 + 1);
            }
#pragma unroll
          for (int n = 0; n < NT; n++) {
            float d[4];
            mma(d, op[0], qh[n][bl][0], qh[n][bl][1], start[SPLIT ? 0 : n][SPLIT ? 0 : bl]);
            mma(d, op[1], qh[n][bl][2], qh[n][bl][3]);
            if (SPLIT) {
              mma(d, op[0], ql[SPLIT ? n : 0][SPLIT ? bl : 0][0], ql[SPLIT ? n : 0][SPLIT ? bl : 0][1]);
              mma(d, op[1], ql[SPLIT ? n : 0][SPLIT ? bl : 0][2], ql[SPLIT ? n : 0][SPLIT ? bl : 0][3]);
            }
            s[u][n][0] += d0 * d[0], s[u][n][1] += d0 * d[1], s[u][n][2] += d1 * d[2], s[u][n][3] += d1 * d[3];
          }
        }
      }
      // the values' scales: half2 of a pair of positions [group][pair t or t + 4][block]
      uint32_t dv[2][2][NB];
#pragma unroll
      for (int u = 0; u < 2; u++)
#pragma unroll
        for (int e = 0; e < 2; e++) {
          const int pair = u * 8 + e * 4 + t;
          if (NB == 4) {
            const uint4 x = *reinterpret_cast<const uint4 *>(tile + L::v_scale(pair, 0));
            dv[u][e][0] = x.x, dv[u][e][1] = x.y, dv[u][e][NB - 2] = x.z, dv[u][e][NB - 1] = x.w;
          } else {
            const uint2 x = *reinterpret_cast<const uint2 *>(tile + L::v_scale(pair, 0));
            dv[u][e][0] = x.x, dv[u][e][1] = x.y;
          }
        }
      if (masked) {
        // What no row sees may be anything: zeros. What some row sees and another does not must not reach the other as 0 times infinity: such a scale is taken
        // as zero, and the results of the rows that see it are made NaN.
        unsigned bad = 0; // positions
#pragma unroll
        for (int u = 0; u < 2; u++)
#pragma unroll
          for (int e = 0; e < 2; e++) {
            const int in = u * 16 + e * 8 + 2 * t, j = j0 + in;
            const uint32_t keep = (j >= lo_any && j <= hi_any ? 0xffffu : 0u) | (j + 1 >= lo_any && j + 1 <= hi_any ? 0xffff0000u : 0u);
#pragma unroll
            for (int bl = 0; bl < NB; bl++) {
              uint32_t x = dv[u][e][bl] & keep;
              if ((x & 0x7c00u) == 0x7c00u) x &= 0xffff0000u, bad |= 1u << in;
              if ((x & 0x7c000000u) == 0x7c000000u) x &= 0xffffu, bad |= 2u << in;
              dv[u][e][bl] = x;
            }
          }
        bad = __reduce_or_sync(0xffffffffu, bad);
        if (bad) {
#pragma unroll
          for (int n = 0; n < NT; n++)
#pragma unroll
            for (int c = 0; c < 2; c++) {
              const int first = max(lo[n][c] - j0, 0), last = min(hi[n][c] - j0, 31);
              if (first <= last && (bad >> first) << (31 - last + first)) {
#pragma unroll
                for (int x = 0; x < 2 * NB; x++) acc[n][x][c] = acc[n][x][c + 2] = NAN;
              }
            }
        }
      }
      if (masked) {
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
          for (int u = 0; u < 2; u++)
#pragma unroll
            for (int c = 0; c < 4; c++) {
              const int j = j0 + u * 16 + (c >> 1) * 8 + g;
              if (j < lo[n][c & 1] || j > hi[n][c & 1]) s[u][n][c] = -INFINITY;
            }
      }
      // One vote a tile: a score over its limit, or a scale over the others' range. Where scales are taken as they are: one of two or more, seen in the union
      // of the bits; else the largest of this lane's. (With a vote that was always taken there, and Q8_0's range as Q4_0's: 64 sequences of 4096
      // positions, Q8_0, 242 us with values of 0.3 and 135 with values of 0.7; now 137 and 138, and 214 with values of 0.05.)
      auto largest = [&]() {
        __half2 d_top = __float2half2_rn(0.f);
#pragma unroll
        for (int u = 0; u < 2; u++)
#pragma unroll
          for (int e = 0; e < 2; e++)
#pragma unroll
            for (int bl = 0; bl < NB; bl++) d_top = __hmax2(d_top, __habs2(as_half2(dv[u][e][bl])));
        return fmaxf(__low2float(d_top), __high2float(d_top));
      };
      bool look = !k_set;
      {
        uint32_t bits = 0;
#pragma unroll
        for (int u = 0; u < 2; u++)
#pragma unroll
          for (int e = 0; e < 2; e++)
#pragma unroll
            for (int bl = 0; bl < NB; bl++) bits |= dv[u][e][bl];
        look |= (bits & 0x40004000u) != 0;
      }
      if (k != 0) look |= largest() > d_most;
      float top[NT][2];
#pragma unroll
      for (int n = 0; n < NT; n++)
#pragma unroll
        for (int c = 0; c < 2; c++) {
          const float x = fmaxf(fmaxf(s[0][n][c], s[0][n][c + 2]), fmaxf(s[1][n][c], s[1][n][c + 2]));
          top[n][c] = x == -INFINITY ? x : x * factor[n][c];
          look |= top[n][c] > limit[n][c];
        }
      if (__any_sync(0xffffffffu, look)) {
        float d_max = largest(), o_by = 1.f;
#pragma unroll
        for (int o = 16; o >= 1; o >>= 1) d_max = fmaxf(d_max, __shfl_xor_sync(0xffffffffu, d_max, o));
        if (d_max > 0.f && (d_max > d_most || !k_set)) {
          const int k_new = scale_shift(d_max, P::LEAST, P::MOST);
          o_by = k_set ? ldexpf(1.f, k_new - k) : 0.f;
          k = k_new, k_set = true, d_most = ldexpf(1.f, P::MOST - k);
        }
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
          for (int c = 0; c < 2; c++) {
#pragma unroll
            for (int o = 4; o <= 16; o <<= 1) top[n][c] = fmaxf(top[n][c], __shfl_xor_sync(0xffffffffu, top[n][c], o));
            float by = 1.f;
            if (top[n][c] > limit[n][c]) {
              const float to = top[n][c] - P::BELOW;
              by = limit[n][c] == -INFINITY ? 0.f : exp2_approx(ref[n][c] - to);
              ref[n][c] = to, limit[n][c] = to + P::OVER, l[n][c] *= by;
            }
            const float a_by = by * o_by;
#pragma unroll
            for (int x = 0; x < 2 * NB; x++) acc[n][x][c] *= a_by, acc[n][x][c + 2] *= a_by;
          }
      }
      if (k != 0) {
#pragma unroll
        for (int u = 0; u < 2; u++)
#pragma unroll
          for (int e = 0; e < 2; e++)
#pragma unroll
            for (int bl = 0; bl < NB; bl++) dv[u][e][bl] = raise_pair(dv[u][e][bl], k);
      }
      uint32_t ph[2][NT][2], pl[2][SPLIT ? NT : 1][2]; // weights of positions (2 t, 2 t + 1), (+ 8) of the group, query row g
#pragma unroll
      for (int u = 0; u < 2; u++)
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
          for (int e = 0; e < 2; e++) {
            const float p0 = exp2_approx(fmaf(s[u][n][2 * e], factor[n][0], -ref[n][0])), p1 = exp2_approx(fmaf(s[u][n][2 * e + 1], factor[n][1], -ref[n][1]));
            l[n][0] += p0, l[n][1] += p1;
            const uint32_t h2 = pack_half2(p0, p1);
            ph[u][n][e] = transpose8x8(h2);
            if (SPLIT) pl[u][SPLIT ? n : 0][e] = transpose8x8(pack_half2(p0 - __low2float(as_half2(h2)), p1 - __high2float(as_half2(h2))));
          }
      // values
      const uint32_t z0 = BITS == 4 ? 0x80088008u : 0x80808080u, z1 = 0x80808080u, minus_zero[4] = {z0, z1, z0, z1}; // -z of an operand's even and odd dims
#pragma unroll
      for (int u = 0; u < 2; u++) {
        uint32_t w[2][W];
#pragma unroll
        for (int e = 0; e < 2; e++) {
          const int pair = u * 8 + e * 4 + t;
          if (W == 2) {
            const uint2 x = *reinterpret_cast<const uint2 *>(tile + L::v_word(pair, g, 0));
            w[e][0] = x.x, w[e][1] = x.y;
          } else {
#pragma unroll
            for (int q4 = 0; q4 < W; q4 += 4) {
              const uint4 x = *reinterpret_cast<const uint4 *>(tile + L::v_word(pair, g, q4));
              w[e][q4] = x.x, w[e][q4 + 1] = x.y, w[e][q4 + 2] = x.z, w[e][q4 + 3] = x.w;
            }
          }
        }
#pragma unroll
        for (int bl = 0; bl < NB; bl++) {
          uint32_t op[2][4]; // dims 4 g (rows 0..7) and 4 g + 1 (rows 8..15) of the block, then 4 g + 2 and 4 g + 3
#pragma unroll
          for (int half = 0; half < 2; half++)
#pragma unroll
            for (int e = 0; e < 2; e++) {
              const uint32_t x = BITS == 4 ? w[e][bl] : w[e][2 * bl + half];
              const int i0 = BITS == 4 ? 2 * half : 0;
              op[half][2 * e] = SPLIT ? signed_pair<BITS>(x, i0) : code_pair<BITS>(x, i0);
              op[half][2 * e + 1] = SPLIT ? signed_pair<BITS>(x, i0 + 1) : code_pair<BITS>(x, i0 + 1);
            }
#pragma unroll
          for (int n = 0; n < NT; n++) {
            uint32_t bh[2], bl2[2];
#pragma unroll
            for (int e = 0; e < 2; e++) {
              const __half2 ph2 = as_half2(ph[u][n][e]), d2 = as_half2(dv[u][e][bl]);
              if (!SPLIT) {
                bh[e] = as_u32(__hmul2(ph2, d2));
              } else {
                const __half2 pl2 = as_half2(pl[u][SPLIT ? n : 0][e]);
                const float p0 = __low2float(ph2) + __low2float(pl2), p1 = __high2float(ph2) + __high2float(pl2);
                const float x0 = p0 * __low2float(d2), x1 = p1 * __high2float(d2);
                bh[e] = pack_half2(x0, x1);
                bl2[e] = pack_half2(x0 - __low2float(as_half2(bh[e])), x1 - __high2float(as_half2(bh[e])));
              }
            }
#pragma unroll
            for (int half = 0; half < 2; half++) {
              if (!SPLIT) {
                mma(acc[n][2 * bl + half], op[half], bh[0], bh[1]);
                mma(acc[n][2 * bl + half], minus_zero, bh[0], bh[1]);
              } else { // summed by itself, and added as f32 rounds
                const float zero[4] = {};
                float part[4];
                mma(part, op[half], bl2[0], bl2[1], zero);
                mma(part, op[half], bh[0], bh[1]);
#pragma unroll
                for (int c = 0; c < 4; c++) acc[n][2 * bl + half][c] += part[c];
              }
            }
          }
        }
      }
      __syncwarp(); // the stage is free
    }
    asm volatile("cp.async.wait_all;" ::: "memory");

    // ---- the warps meet ----
    __syncthreads(); // (of the item before, everything in s_m, s_l and s_acc has been read)
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
      for (int c = 0; c < 2; c++) {
        const int col = n * 8 + 2 * t + c;
        float sum = l[n][c];
#pragma unroll
        for (int o = 4; o <= 16; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (g == 0) s_m[warp * R + col] = limit[n][c] == -INFINITY ? -INFINITY : ref[n][c], s_l[warp * R + col] = sum;
        const float down = ldexpf(1.f, -k);
#pragma unroll
        for (int bl = 0; bl < NB; bl++) {
          float4 v;
          const float *x = acc[n][2 * bl], *y = acc[n][2 * bl + 1];
          if (SPLIT) v = make_float4(x[c] * down, x[c + 2] * down, y[c] * down, y[c + 2] * down);
          else { // codes came as c 2^-24, those of the odd dims 16 times as much with 4 bits
            const float one = 16777216.f * down, odd = BITS == 4 ? 1048576.f * down : one;
            v = make_float4(x[c] * one, x[c + 2] * odd, y[c] * one, y[c + 2] * odd);
          }
          *reinterpret_cast<float4 *>(s_acc + (warp * R + col) * P::COL + bl * 32 + g * 4) = v;
        }
      }
    __syncthreads();
    // A warp takes a row at a time, a lane HD / 32 neighbouring dims of it.
    constexpr int V = HD / 32;
    const bool whole = ta == 0 && tb == sp.count;
    auto put = [&](int r, float m_all, float l_all, float (&v)[V]) { // a finished row
      const float by = l_all > 0.f ? 1.f / l_all : l_all; // 0: nothing seen, zeros; NaN stays
#pragma unroll
      for (int i = 0; i < V; i++) v[i] *= by;
      store_vec<V>(a.out.p, a.dtype, s_row[turn][r] + lane * V, v);
      if (a.lse && lane == 0) a.lse[s_lse_row[turn][r]] = l_all > 0.f ? (m_all + log2f(l_all)) * LN2 : l_all == 0.f ? -INFINITY : l_all;
    };
    float *const rec = a.records + (blockIdx.x * 2 + (ta == 0 ? 1 : 0)) * (long long)RECORD_STRIDE;
    for (int r = warp; r < rows; r += SPLIT_WARPS) {
      float m_all = -INFINITY, l_all = 0.f, v[V] = {};
#pragma unroll
      for (int w = 0; w < SPLIT_WARPS; w++) m_all = fmaxf(m_all, s_m[w * R + r]);
#pragma unroll
      for (int w = 0; w < SPLIT_WARPS; w++) {
        const float mw = s_m[w * R + r];
        const float by = mw == -INFINITY ? 0.f : exp2_approx(mw - m_all);
        l_all += by * s_l[w * R + r];
        float x[V];
        load_vec<V>(s_acc + (w * R + r) * P::COL + lane * V, x);
#pragma unroll
        for (int i = 0; i < V; i++) v[i] += by * x[i];
      }
      if (whole) put(r, m_all, l_all, v);
      else {
        if (lane == 0) rec[r] = m_all, rec[R + r] = l_all;
        store_vec<V>(rec, XNQ_F32, 2 * R + r * HD + lane * V, v);
      }
    }
    if (!whole) {
      const long long c_first = (item0 + lead) / share; // the CTAs that hold parts of the item: c_first .. c_first + others
      const int others = (int)((item0 + lead + sp.count - 1) / share - c_first);
      __syncthreads();
      if (threadIdx.x == 0) {
        __threadfence(); // the CTA's parts, which the barrier has ordered before, become visible before the count does
        s_last = atomicInc(a.tickets + c_first, (unsigned)others) == (unsigned)others;
        __threadfence();
      }
      __syncthreads();
      // All parts are there: added in the order of their places, PARTS in flight.
      auto join = [&](auto in_flight) {
        constexpr int PARTS = decltype(in_flight)::value;
        const float *const part0 = a.records + (c_first * 2 + 1) * RECORD_STRIDE; // the first lies in its CTA's second place, the others in the first ones
        for (int r = warp; r < rows; r += SPLIT_WARPS) {
          float m_all = -INFINITY, l_all = 0.f, v[V] = {};
          for (int c = 0; c <= others; c += PARTS) {
            float mp[PARTS], lp[PARTS], x[PARTS][V], m_new = m_all;
#pragma unroll
            for (int i = 0; i < PARTS; i++) {
              const float *p = part0 + (long long)(min(c + i, others) * 2 - (c + i ? 1 : 0)) * RECORD_STRIDE;
              mp[i] = __ldcg(p + r), lp[i] = __ldcg(p + R + r);
              load_vec_cg<V>(p + 2 * R + r * HD + lane * V, x[i]);
            }
#pragma unroll
            for (int i = 0; i < PARTS; i++) m_new = fmaxf(m_new, mp[i]);
            const float old = m_all == -INFINITY ? 0.f : exp2_approx(m_all - m_new);
            l_all *= old;
#pragma unroll
            for (int k2 = 0; k2 < V; k2++) v[k2] *= old;
#pragma unroll
            for (int i = 0; i < PARTS; i++) {
              const float by = c + i > others || mp[i] == -INFINITY ? 0.f : exp2_approx(mp[i] - m_new);
              if (c + i <= others) {
                l_all += by * lp[i];
#pragma unroll
                for (int k2 = 0; k2 < V; k2++) v[k2] += by * x[i][k2];
              }
            }
            m_all = m_new;
          }
          put(r, m_all, l_all, v);
        }
      };
      if (s_last) {
        if (others < 16) join(std::integral_constant<int, 8>{});
        else join(std::integral_constant<int, 20>{}); // 131072 positions of one sequence, 55 parts: 46.7 us against 48.2 (twenty for few parts: more code to fetch, 0.6 us at 512)
      }
    }
    if (whole_runs) return; // one item a CTA
    at = item0 + length(sp.count), item0 = at;
    item++, turn ^= 1;
  }
}

int g_sms[64]; // of the devices that xnq_init has seen

template <int BITS, int HD, int NT, bool SPLIT>
struct SplitLaunch {
  static constexpr size_t smem() { return SPLIT_WARPS * SPLIT_STAGES * KvTile<BITS, HD>::BYTES + SplitShape<BITS, HD, NT>::MERGE; }
  static inline int per_sm = 0;
  static int init() {
    XNQ_CUDA(cudaFuncSetAttribute(kv_attend_split_kernel<BITS, HD, NT, SPLIT>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem()));
    int n = 0;
    XNQ_CUDA(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kv_attend_split_kernel<BITS, HD, NT, SPLIT>, SPLIT_WARPS * 32, smem()));
    per_sm = std::max(1, std::min(n, 4));
    return XNQ_OK;
  }
};
// Query rows of a KV head to an item of the split kernel: 8 or 16. Sixteen read a tile half as often and take 1.3 to 1.6 times as long for
// it, with two CTAs an SM instead of three. Where the items fill the GPU that gains (16 rows, 64 sequences of 4096 positions and 8 KV heads: 131 us against 145,
// Q8_0 184 against 252), unless the second half of the last sixteen is empty (4 bits, 24 rows: 229 against 204). Where they do not, items of 8 go to more SMs
// and are done sooner (16 rows of one sequence of 8192: 37 us against 25, of 512: 22 against 16).
int split_nt(int bits, int64_t rows, int64_t heads, int sms) {
  const int64_t eights = (rows + 7) / 8;
  return eights == 1 || heads * eights <= sms || (bits == 4 && eights == 3) ? 1 : 2;
}
// 16-bit query rows of a KV head from which the kernel for many rows takes them, whose time hardly depends on their number up to 128. Below it they keep this
// kernel's scores, exact products of the codes, where the other's keys are rounded to 16 bits (an error of 1e-4 of a row's log sum), also where the other is
// sooner. 8 KV heads, us, this kernel against that: Q4_0, 32 rows, one sequence of 8192 27 against 28, of 32768 52 against 52, 16 sequences of 8192 123 against
// 129; 64 rows, 36 against 32, 78 against 52, 219 against 131. Q8_0, 16 rows, 29 against 28, 47 against 50, 98 against 135; 64 rows, 46 against 32, 92 against
// 54, 309 against 136.
constexpr int64_t PROMPT_ROWS = 64;

template <int BITS, int HD, int NT, bool SPLIT>
int run_split(AttendArgs a, int sms, cudaStream_t s) {
  const int64_t rows = a.seq * a.group;
  a.row_tiles = (int)((rows + 8 * NT - 1) / (8 * NT));
  using Launch = SplitLaunch<BITS, HD, NT, SPLIT>;
  // no more CTAs than the longest caches could fill
  const int64_t most = a.batch * a.c.kv_heads * a.row_tiles * ((a.c.max_seq + KV_TILE - 1) / KV_TILE);
  const int64_t grid = std::max<int64_t>(1, std::min<int64_t>(std::min(sms * Launch::per_sm, MAX_SPLIT_GRID), std::max<int64_t>(most, a.batch)));
  XNQ_CUDA(launch_pdl(kv_attend_split_kernel<BITS, HD, NT, SPLIT>, dim3((unsigned)grid), dim3(SPLIT_WARPS * 32), Launch::smem(), s, a));
  count_launch();
  return XNQ_OK;
}

template <typename F>
int for_each_split(F f) { // f<BITS, HD, NT, SPLIT>()
  int rc = XNQ_OK;
  auto one = [&](auto l) {
    if (rc == XNQ_OK) rc = f(l);
  };
  one(SplitLaunch<4, 64, 1, false>{}), one(SplitLaunch<4, 64, 2, false>{}), one(SplitLaunch<4, 64, 1, true>{}), one(SplitLaunch<4, 64, 2, true>{});
  one(SplitLaunch<4, 128, 1, false>{}), one(SplitLaunch<4, 128, 2, false>{}), one(SplitLaunch<4, 128, 1, true>{}), one(SplitLaunch<4, 128, 2, true>{});
  one(SplitLaunch<8, 64, 1, false>{}), one(SplitLaunch<8, 64, 2, false>{}), one(SplitLaunch<8, 64, 1, true>{}), one(SplitLaunch<8, 64, 2, true>{});
  one(SplitLaunch<8, 128, 1, false>{}), one(SplitLaunch<8, 128, 2, false>{}), one(SplitLaunch<8, 128, 1, true>{}), one(SplitLaunch<8, 128, 2, true>{});
  return rc;
}

template <int BITS, int HD>
int run_attend(const AttendArgs &a, int sms, cudaStream_t s) {
  const bool one = split_nt(BITS, a.seq * a.group, a.batch * a.c.kv_heads, sms) == 1;
  if (a.dtype == XNQ_F32) return one ? run_split<BITS, HD, 1, true>(a, sms, s) : run_split<BITS, HD, 2, true>(a, sms, s);
  return one ? run_split<BITS, HD, 1, false>(a, sms, s) : run_split<BITS, HD, 2, false>(a, sms, s);
}

} // namespace

int kv_attend_status(unsigned int *bits) {
  unsigned int prompt = 0;
  XNQ_CUDA(cudaMemcpyFromSymbol(bits, g_kv_attend_status, sizeof(*bits)));
  const int rc = kv_prompt_status(&prompt);
  *bits |= prompt;
  return rc;
}
int kv_attend_init(int device) {
  unsigned int zero = 0;
  XNQ_CUDA(cudaMemcpyToSymbol(g_kv_attend_status, &zero, sizeof(zero)));
  if (device < 64) XNQ_CUDA(cudaDeviceGetAttribute(&g_sms[device], cudaDevAttrMultiProcessorCount, device));
  const int rc = kv_prompt_init(device);
  return rc != XNQ_OK ? rc : for_each_split([](auto l) { return decltype(l)::init(); });
}

} // namespace xnq

using namespace xnq;

extern "C" {

size_t xnq_kv_attend_workspace_bytes(int64_t batch, int64_t seq, int heads, int kv_heads, int head_dim) {
  if (batch <= 0 || seq <= 0 || heads < 1 || kv_heads < 1 || heads % kv_heads || (head_dim != 64 && head_dim != 128)) return 0;
  // (for the kernel for many rows at its most: a part for every SM)
  return KV_TICKET_BYTES + std::max(RECORDS_BYTES, seq * (heads / kv_heads) >= PROMPT_ROWS ? kv_prompt_parts_bytes(head_dim) : 0);
}

int xnq_kv_attend(const xnq_kv_cache *cache, const xnq_rows *q, const xnq_rows *out, float *lse, int64_t batch, int64_t seq, int heads, const long long *pos,
                  int pos_stride, float scale, int causal, int64_t window, void *workspace, size_t ws_bytes, void *stream) {
  clear_error();
  AttendArgs a{};
  int rc = kv_view("kv_attend", cache, batch, &a.c);
  if (rc != XNQ_OK) return rc;
  if (!q || !out || !pos) return fail(XNQ_ERR_NULL, "kv_attend: NULL argument");
  if (seq < 0 || seq > INT32_MAX || heads < 1 || heads > 65535 || heads % cache->kv_heads || pos_stride < 0 || pos_stride > 1 || window < 0)
    return fail(XNQ_ERR_SHAPE, "kv_attend: seq %lld, heads %d over %d, pos_stride %d (0 or 1), window %lld", (long long)seq, heads, cache->kv_heads, pos_stride, (long long)window);
  if (!std::isfinite(scale)) return fail(XNQ_ERR_SHAPE, "kv_attend: the scale is not a finite number");
  if (batch == 0 || seq == 0) return XNQ_OK;
  if ((rc = kv_rows("kv_attend", "q", q, &a.q)) != XNQ_OK || (rc = kv_rows("kv_attend", "out", out, &a.out)) != XNQ_OK) return rc;
  if (out->dtype != q->dtype) return fail(XNQ_ERR_DTYPE, "kv_attend: q has type %d, out %d", q->dtype, out->dtype);
  const size_t need = xnq_kv_attend_workspace_bytes(batch, seq, heads, cache->kv_heads, cache->head_dim);
  if (!workspace || ws_bytes < need) return fail(XNQ_ERR_SIZE, "kv_attend: workspace has %zu bytes, needs %zu (zero it once after allocating)", ws_bytes, need);
  if (reinterpret_cast<uintptr_t>(workspace) & 15) return fail(XNQ_ERR_ALIGN, "kv_attend: the workspace must be 16-byte aligned");
  int device = 0;
  XNQ_CUDA(cudaGetDevice(&device));
  const int sms = device < 64 ? g_sms[device] : 0;
  if (!sms) return fail(XNQ_ERR_UNSUPPORTED, "kv_attend: xnq_init has not run for device %d", device);
  a.lse = lse, a.batch = batch, a.seq = seq, a.heads = heads, a.group = heads / cache->kv_heads, a.dtype = q->dtype;
  a.pos_stride = pos_stride, a.causal = causal, a.pos = pos, a.scale = scale, a.window = std::min<int64_t>(window, INT32_MAX);
  a.tickets = static_cast<unsigned int *>(workspace);
  a.records = reinterpret_cast<float *>(static_cast<uint8_t *>(workspace) + KV_TICKET_BYTES);
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int bits = kv_bits(cache->ggml_dtype);
  if (q->dtype != XNQ_F32 && seq * a.group >= PROMPT_ROWS) return launch_kv_prompt(a, bits, cache->head_dim, sms, s);
  if (bits == 4) return cache->head_dim == 64 ? run_attend<4, 64>(a, sms, s) : run_attend<4, 128>(a, sms, s);
  return cache->head_dim == 64 ? run_attend<8, 64>(a, sms, s) : run_attend<8, 128>(a, sms, s);
}

} // extern "C"
