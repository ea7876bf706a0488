// What the kernels of attention over the quantized KV cache share.
#pragma once

#include "xnq_kv_cache.cuh"

namespace xnq {

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
// What scores are multiplied by is no less: a hidden position's is -inf, whose product with a factor that has sunk to zero is not. (Scores of the
// operands, below 2^45, times this are nothing, as those of a scale of 0 are.)
constexpr float LEAST_FACTOR = 1e-30f;

struct AttendArgs {
  KvView c;
  KvRows q, out;
  float *lse; // [batch, seq, heads], or null
  long long batch, seq, window;
  int heads, group, dtype, pos_stride, causal; // group: query heads of a KV head
  const long long *pos;
  float scale;
  int row_tiles, splits;  // tiles of query rows of a KV head; CTAs that share a row tile's positions (many rows)
  unsigned int *tickets;  // KV_TICKETS words, zero between calls
  float *records;         // parts of rows
  // What the kernels look at in their second form (MORE): first positions that stay visible, and packed tokens (offsets null: none).
  long long sinks, tokens;
  const long long *offsets, *position, *start;
  const uint32_t *sees, *nodes; // null: no trees
  int words, clear;             // words of a token's bits; rows behind the last sequence: zeros
  long long rows_from, rows_to; // this launch's sequences: those with that many query rows of a KV head, [from, to)
};

// Workspace: the tickets, at one place whatever the call, then the parts.
constexpr int KV_TICKETS = 1024;
constexpr size_t KV_TICKET_BYTES = KV_TICKETS * 4;
static_assert(KV_TICKET_BYTES == XNQ_KV_WORKSPACE_ZEROED, "what a caller zeroes");
constexpr unsigned KV_WAIT = 8; // status: a wait of the kernel for many rows expired (with the bits of xnq_kv_cache.cuh)

// xnq_kv_prompt.cu: many 16-bit query rows
int kv_prompt_init(int device);
int kv_prompt_status(unsigned int *bits);
size_t kv_prompt_parts_bytes(int head_dim, bool packed);
int launch_kv_prompt(const AttendArgs &a, bool more, int bits, int head_dim, int sms, cudaStream_t s);

#ifdef __CUDACC__
// positions [lo, hi] that the query at token s of a sequence at `pos` sees
__device__ __forceinline__ void seen_by(const AttendArgs &a, long long pos, long long s, int &lo, int &hi) {
  const long long p = pos + s;
  const long long h = p < 0 ? -1 : min(a.causal ? p : pos + a.seq - 1, a.c.max_seq - 1);
  const long long l = a.window ? max(p - a.window + 1, 0ll) : 0ll;
  hi = (int)h, lo = (int)min(l, a.c.max_seq);
}
// What a sequence's queries are, and which tiles of the cache they see between them: the first `head` and `count - head` more, `gap` tiles on.
struct Sequence {
  long long pos, first_row; // place of its first token; its first row among all tokens
  int seq, head, gap, count;
  bool here;                // of this launch
  __device__ __forceinline__ int tile(int i) const { return i < head ? i : i + gap; }
};
// tiles of what tokens [s0, s1] of the sequence see
__device__ __forceinline__ void tiles_seen(const AttendArgs &a, Sequence &x, long long s0, long long s1) {
  const long long end = a.sees || !a.causal ? x.pos + x.seq - 1 : x.pos + s1, hi = min(end, a.c.max_seq - 1);
  const long long p0 = max(a.sees ? x.pos : x.pos + s0, 0ll), lo = a.window ? min(max(p0 - a.window + 1, 0ll), a.c.max_seq) : 0ll;
  const int first = (int)(lo / KV_TILE);
  x.head = hi < 0 ? 0 : min((int)((min(a.sinks, hi + 1) + KV_TILE - 1) / KV_TILE), first);
  x.gap = first - x.head;
  x.count = x.head + (hi < lo ? 0 : (int)(hi / KV_TILE) - first + 1);
}
__device__ __forceinline__ Sequence sequence_of(const AttendArgs &a, int b) {
  Sequence x;
  if (a.offsets) {
    x.pos = first_place(a.start, b), x.first_row = a.offsets[b], x.seq = (int)(a.offsets[b + 1] - x.first_row);
    const long long rows = (long long)x.seq * a.group;
    x.here = rows >= a.rows_from && rows < a.rows_to;
  } else x.pos = first_place(a.pos, (long long)b * a.pos_stride), x.first_row = b * a.seq, x.seq = (int)a.seq, x.here = true;
  x.head = x.gap = x.count = 0;
  if (x.here && x.seq > 0) tiles_seen(a, x, 0, x.seq - 1);
  return x;
}
// What one of a sequence's tokens sees: positions [lo, hi], the first `sinks` up to hi, and tokens of its tree (whose first is at place pos).
struct Sight {
  int lo, hi;
  bool none; // no token: sees nothing, and must not be looked at either
};
__device__ __forceinline__ Sight sight_of(const AttendArgs &a, const Sequence &x, long long s) {
  const long long p = a.offsets ? a.position[x.first_row + s] : x.pos + s;
  const long long h = p < 0 ? -1 : min(a.sees ? x.pos - 1 : a.causal ? p : x.pos + x.seq - 1, a.c.max_seq - 1);
  const long long l = a.window ? min(max(p - a.window + 1, 0ll), a.c.max_seq) : 0ll;
  return Sight{(int)l, (int)h, p < 0};
}
__device__ __forceinline__ uint32_t bits_between(int from, int to) { // bits [from, to] of 32
  from = max(from, 0), to = min(to, 31);
  return from <= to ? (0xffffffffu >> (31 - to + from)) << from : 0u;
}
__device__ __forceinline__ uint32_t bits_at(const uint32_t *row, int words, int off) { // 32 bits from bit `off` on (it may be negative, or past the row)
  if (off <= -32 || off >= words * 32) return 0u;
  if (off < 0) return row[0] << -off;
  const int w = off >> 5;
  return __funnelshift_r(row[w], w + 1 < words ? row[w + 1] : 0u, off & 31);
}
// of the 32 positions from j0 on; row: the token's bits
__device__ __forceinline__ uint32_t seen_in_tile(const AttendArgs &a, const Sight &v, const uint32_t *row, long long pos, int j0) {
  uint32_t m = bits_between(v.lo - j0, v.hi - j0) | bits_between(-j0, (int)min(a.sinks - 1, (long long)v.hi) - j0);
  if (row && j0 + KV_TILE > pos) m |= bits_at(row, a.words, (int)(j0 - pos));
  return m;
}
// whether every one of some tokens sees all of a tile: lo and hi are the largest and the smallest of theirs
__device__ __forceinline__ bool all_seen(const AttendArgs &a, int lo, int hi, int j0) { return j0 + KV_TILE - 1 <= hi && (j0 >= lo || j0 + KV_TILE <= a.sinks); }
// Rows behind the last sequence: zeros. By every block of a launch.
__device__ __forceinline__ void clear_behind(const AttendArgs &a, int head_dim) {
  const int chunks = a.heads * (head_dim * (a.dtype == XNQ_F32 ? 4 : 2) / 16), each = chunks / a.heads;
  for (long long t = a.offsets[a.batch] + blockIdx.x; t < a.tokens; t += gridDim.x)
    for (int i = threadIdx.x; i < chunks; i += blockDim.x) {
      const int h = i / each, x = i - h * each;
      const long long row = t * a.out.ss + h * a.out.sh;
      uint8_t *const p = static_cast<uint8_t *>(a.out.p) + row * (a.dtype == XNQ_F32 ? 4 : 2) + x * 16;
      *reinterpret_cast<uint4 *>(p) = make_uint4(0u, 0u, 0u, 0u);
      if (a.lse && x == 0) a.lse[t * a.heads + h] = -INFINITY;
    }
}
__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ __half2 as_half2(uint32_t v) { return *reinterpret_cast<const __half2 *>(&v); }
__device__ __forceinline__ uint32_t as_u32(__half2 v) { return *reinterpret_cast<const uint32_t *>(&v); }
__device__ __forceinline__ float exp2_approx(float x) { // 2^x within 2 ulp
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
template <int V> // 2 or 4 values
__device__ __forceinline__ void load_vec_cg(const float *p, float (&v)[V]) {
  if (V == 4) {
    const float4 x = __ldcg(reinterpret_cast<const float4 *>(p));
    v[0] = x.x, v[1] = x.y, v[V - 2] = x.z, v[V - 1] = x.w;
  } else {
    const float2 x = __ldcg(reinterpret_cast<const float2 *>(p));
    v[0] = x.x, v[1] = x.y;
  }
}
template <int V>
__device__ __forceinline__ void store_vec(void *p, int dtype, long long at, const float (&v)[V]) {
  if (dtype == XNQ_F32) {
    float *q = static_cast<float *>(p) + at;
    if (V == 4) *reinterpret_cast<float4 *>(q) = make_float4(v[0], v[1], v[V - 2], v[V - 1]);
    else *reinterpret_cast<float2 *>(q) = make_float2(v[0], v[1]);
    return;
  }
  uint32_t w[V / 2];
#pragma unroll
  for (int i = 0; i < V / 2; i++) {
    if (dtype == XNQ_F16) {
      const __half2 h = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t *>(&h);
    } else {
      const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t *>(&h);
    }
  }
  uint16_t *q = static_cast<uint16_t *>(p) + at;
  if (V == 4) *reinterpret_cast<uint2 *>(q) = make_uint2(w[0], w[V / 2 - 1]);
  else *reinterpret_cast<uint32_t *>(q) = w[0];
}
// Pair i of a word's codes (16 bits apart) as f16 subnormals, c 2^-24; 4 bits: 16 times that where i is odd.
template <int BITS>
__device__ __forceinline__ uint32_t code_pair(uint32_t w, int i) {
  if (BITS == 4) return (i & 2 ? w >> 8 : w) & (i & 1 ? 0x00f000f0u : 0x000f000fu);
  return (i & 1 ? w >> 8 : w) & 0x00ff00ffu;
}
template <int BITS>
__device__ __forceinline__ uint32_t signed_pair(uint32_t w, int i) { // the same pair as the whole numbers that it stands for
  if (BITS == 4) {
    const uint32_t m = code_pair<4>(w, i) | 0x64006400u; // 1024 + c, or 1024 + 16 c
    return as_u32(i & 1 ? __hfma2(as_half2(m), __float2half2_rn(0.0625f), __float2half2_rn(-72.f)) : __hsub2(as_half2(m), __float2half2_rn(1032.f)));
  }
  return as_u32(__hsub2(as_half2(code_pair<8>(w, i) | 0x64006400u), __float2half2_rn(1152.f)));
}
// How much the scales of a run of blocks, the largest of which is `top`, are raised (a power of two): not at all from 2^least to 2^most
__device__ __forceinline__ int scale_shift(float top, int least, int most) {
  const int e = top > 0.f && top < INFINITY ? ilogbf(top) : 0;
  return e >= most || e < least ? -e : 0;
}
__device__ __forceinline__ uint32_t raise_pair(uint32_t d, int k) { // two scales times 2^k, -15 <= k <= 24
  const __half2 by = __float2half2_rn(ldexpf(1.f, min(k, 15))), by2 = __float2half2_rn(ldexpf(1.f, max(k - 15, 0))); // 2^24 is past f16
  return as_u32(__hmul2(__hmul2(as_half2(d), by), by2));
}
#endif

} // namespace xnq
