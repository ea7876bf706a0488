// The quantized KV cache is written (quantized as it is stored, after an optional rotary embedding of q and k) and read back.
//
// Both kernels are bound by their bytes: one pass, each value read once and written once.
//
// Store: a thread takes 8 consecutive dims of a PAIR of positions (2 i, 2 i + 1) that share the words of V's codes, so a pair is stored in whole words;
// where only one of the two is new, the other half of a word is left alone (2-byte stores). Four neighbouring threads hold a block of 32. A warp stays with
// its pair (a query's position) and goes over heads, so that sequence, page and rotation are looked up once; few positions are shared by several
// warps (`slices`). Read back: a warp takes a tile of a head, keys or values, in the order of its words. (A thread a unit of 8 dims, each with its own
// divisions of 64-bit indexes: 8 x 4096 tokens with rotation and their read-back 354 us, read-back of 16 x 8192 positions 211 us.)
#include <algorithm>
#include <type_traits>

#include "xnq_kv_attend.cuh"
#include "xnq_quantize_act.cuh"

namespace xnq {
namespace {

__device__ unsigned int g_kv_store_status;

struct RopeArgs {
  const float *cos, *sin; // [rows][head_dim / 2]
  long long rows;
  KvRows q, q_out;
  int heads, q_out_dtype;
};

template <typename T>
__device__ __forceinline__ void store8(T *p, const float (&v)[8]);
template <>
__device__ __forceinline__ void store8<float>(float *p, const float (&v)[8]) {
  *reinterpret_cast<float4 *>(p) = make_float4(v[0], v[1], v[2], v[3]);
  *reinterpret_cast<float4 *>(p + 4) = make_float4(v[4], v[5], v[6], v[7]);
}
template <>
__device__ __forceinline__ void store8<__half>(__half *p, const float (&v)[8]) {
  __half2 h[4];
#pragma unroll
  for (int i = 0; i < 4; i++) h[i] = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
  *reinterpret_cast<uint4 *>(p) = *reinterpret_cast<const uint4 *>(h);
}
template <>
__device__ __forceinline__ void store8<__nv_bfloat16>(__nv_bfloat16 *p, const float (&v)[8]) {
  __nv_bfloat162 h[4];
#pragma unroll
  for (int i = 0; i < 4; i++) h[i] = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
  *reinterpret_cast<uint4 *>(p) = *reinterpret_cast<const uint4 *>(h);
}

template <typename T>
__device__ __forceinline__ void store4(T *p, const float (&v)[4]);
template <>
__device__ __forceinline__ void store4<float>(float *p, const float (&v)[4]) {
  *reinterpret_cast<float4 *>(p) = make_float4(v[0], v[1], v[2], v[3]);
}
template <>
__device__ __forceinline__ void store4<__half>(__half *p, const float (&v)[4]) {
  const __half2 h[2] = {__floats2half2_rn(v[0], v[1]), __floats2half2_rn(v[2], v[3])};
  *reinterpret_cast<uint2 *>(p) = *reinterpret_cast<const uint2 *>(h);
}
template <>
__device__ __forceinline__ void store4<__nv_bfloat16>(__nv_bfloat16 *p, const float (&v)[4]) {
  const __nv_bfloat162 h[2] = {__floats2bfloat162_rn(v[0], v[1]), __floats2bfloat162_rn(v[2], v[3])};
  *reinterpret_cast<uint2 *>(p) = *reinterpret_cast<const uint2 *>(h);
}
__device__ __forceinline__ float widen(float v) { return v; }
__device__ __forceinline__ float widen(__half v) { return __half2float(v); }
__device__ __forceinline__ float widen(__nv_bfloat16 v) { return __bfloat162float(v); }
template <int N> // 1, 2 or 4 words at p, or 8 in two fours
__device__ __forceinline__ void load_words(const uint8_t *p, const uint8_t *p2, uint32_t (&w)[N]) {
  if (N == 1) w[0] = *reinterpret_cast<const uint32_t *>(p);
  else if (N == 2) {
    const uint2 x = *reinterpret_cast<const uint2 *>(p);
    w[0] = x.x, w[N - 1] = x.y;
  } else {
    const uint4 x = *reinterpret_cast<const uint4 *>(p);
    w[0] = x.x, w[1 % N] = x.y, w[2 % N] = x.z, w[3 % N] = x.w;
    if (N == 8) {
      const uint4 y = *reinterpret_cast<const uint4 *>(p2);
      w[4 % N] = y.x, w[5 % N] = y.y, w[6 % N] = y.z, w[7 % N] = y.w;
    }
  }
}

// One block of 32 in four neighbouring lanes, 8 values each: the arithmetic of BlockQ4_0::from_float and BlockQ8_0::from_float
// (k_quants.rs:235-270, 636-661), every operation rounded for itself, but for Q8_0's scale: max|x| times the f32 nearest 1 / 127, which is what torch makes of
// a division by 127 on a GPU, where the file's quantizer (and the one of this library's activations) divides. The two differ in the scale's last f32 bit and, by that,
// in codes where x / scale is a half: 5 of 100000 bf16 values, 7 of a million f16 ones, one in four million f32 ones, by one, to the other side of the tie. No f16
// scale differs where x is f16 or bf16, one in a few million where it is f32. The codes come back unsigned: 4 bits, eight nibbles in lo; 8 bits, code + 128.
struct Codes8 {
  uint32_t lo, hi;
  __half d;
};
template <int BITS>
__device__ __forceinline__ Codes8 quantize8(const float (&v)[8]) {
  Codes8 o;
  if (BITS == 8) {
    float amax = 0.f;
#pragma unroll
    for (int i = 0; i < 8; i++) amax = fmaxf(amax, fabsf(v[i])); // a NaN is passed over
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
    const float d = __fmul_rn(amax, 1.0f / 127.0f), id = d != 0.f ? __fdiv_rn(1.0f, d) : 0.f;
    int q[8];
#pragma unroll
    for (int i = 0; i < 8; i++) q[i] = round_away(__fmul_rn(v[i], id));
    o.lo = pack_sat_i8(q[0], q[1], pack_sat_i8(q[2], q[3], 0u)) ^ 0x80808080u;
    o.hi = pack_sat_i8(q[4], q[5], pack_sat_i8(q[6], q[7], 0u)) ^ 0x80808080u;
    o.d = __float2half_rn(d);
    return o;
  }
  // the first value of the largest magnitude; a NaN is passed over
  float mx = -INFINITY, mn = INFINITY;
#pragma unroll
  for (int i = 0; i < 8; i++) mx = fmaxf(mx, v[i]), mn = fminf(mn, v[i]);
#pragma unroll
  for (int off = 1; off <= 2; off <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, off)), mn = fminf(mn, __shfl_xor_sync(0xffffffffu, mn, off));
  float m = mx >= -mn ? mx : mn;
  if (mx == -INFINITY && mn == INFINITY) m = 0.f; // NaN alone
  if (__any_sync(0xffffffffu, mx == -mn && mx > 0.f)) { // both signs: whichever comes first
    int at = 64; // twice the place, and the sign; 64: none of this thread's
    const int t = threadIdx.x & 3;
#pragma unroll
    for (int i = 7; i >= 0; i--)
      if (fabsf(v[i]) == mx) at = 2 * (t * 8 + i) + (v[i] < 0.f);
    at = min(at, __shfl_xor_sync(0xffffffffu, at, 1));
    at = min(at, __shfl_xor_sync(0xffffffffu, at, 2));
    if (mx == -mn && mx > 0.f) m = at & 1 ? mn : mx;
  }
  const float d = __fmul_rn(m, -0.125f), id = d != 0.f ? __frcp_rn(d) : 0.f; // (the quotients by -8 and of 1 by d, as IEEE rounds them)
  uint32_t w = 0;
#pragma unroll
  for (int i = 0; i < 8; i++) { // trunc, saturated to 0 .. 15, NaN: 0; behind 2^23 a float's last bits are the number
    const float y = fminf(fmaxf(__fadd_rn(__fmul_rn(v[i], id), 8.5f), 0.f), 15.5f);
    w += __float_as_uint(__fadd_rz(y, 8388608.f)) << (4 * i);
  }
  w -= 0xfb000000u; // the sum of 0x4b000000 << 4 i
  o.lo = w, o.hi = 0u, o.d = __float2half_rn(d);
  return o;
}

__device__ __forceinline__ float rope_of(float x, float other, float c, float s, bool upper) { // rotate-half: x's half of the pair
  return upper ? __fadd_rn(__fmul_rn(x, c), __fmul_rn(other, s)) : __fsub_rn(__fmul_rn(x, c), __fmul_rn(other, s));
}
// this thread's 8 values of a head rotated; its partner, half a head away, holds the other half of the pairs
template <int HD>
__device__ __forceinline__ void rope8(float (&v)[8], const float (&c)[8], const float (&s)[8], bool upper) {
#pragma unroll
  for (int i = 0; i < 8; i++) v[i] = rope_of(v[i], __shfl_xor_sync(0xffffffffu, v[i], HD / 16), c[i], s[i], upper);
}
template <int HD>
__device__ __forceinline__ void load_tables(const RopeArgs &r, long long pos, int l, bool valid, float (&c)[8], float (&s)[8]) {
#pragma unroll
  for (int i = 0; i < 8; i++) c[i] = s[i] = 0.f;
  if (!valid) return;
  load8(r.cos + pos * (HD / 2) + (l & (HD / 16 - 1)) * 8, c);
  load8(r.sin + pos * (HD / 2) + (l & (HD / 16 - 1)) * 8, s);
}

struct PackedRows { // of a plan: where each token goes, and the position that it is rotated at
  const long long *slot, *position;
};

struct StoreUnits { // warps: [0, kv) store keys and values, the rest rotate queries
  unsigned kv, all, pairs, kv_slices, q_slices;
  unsigned each; // packed: tokens of a warp that stores keys and values
};

// PACKED: the tokens of all sequences one after the other (seq: how many). A warp has a token, and the next one with it where the two share a pair.
template <int BITS, int HD, typename T, bool ROPE, bool PACKED>
// Four blocks an SM: with the 120 registers that it would take, and two blocks, 8 x 4096 bf16 tokens with rotation took half as long again.
__global__ void __launch_bounds__(256, 4) kv_store_kernel(KvView c, KvRows k, KvRows v, RopeArgs r, StoreUnits un, long long seq, const long long *pos_p, int pos_stride, PackedRows pk) {
  using L = KvTile<BITS, HD>;
  constexpr int LANES = HD / 8, ROWS = 32 / LANES; // threads of a head's row, rows of a warp
  const int lane = threadIdx.x & 31, l = lane % LANES, sub = lane / LANES;
  unsigned u = blockIdx.x * 8 + (threadIdx.x >> 5);
  pdl_launch_dependents();
  pdl_wait();
  if (u >= un.all) return;
  if (ROPE && u >= un.kv) { // queries
    u -= un.kv;
    const unsigned bs = u / un.q_slices, slice = u - bs * un.q_slices, b = PACKED ? 0u : bs / (unsigned)seq, s = bs - b * (unsigned)seq;
    const long long p = PACKED ? pk.position[s] : pos_p[(long long)b * pos_stride] + s;
    const bool valid = p >= 0 && p < r.rows;
    // A lane takes four dims and their partners half a head on; U rows are on their way at a time. (16-bit types: with eight dims, 252 us instead of 157 for
    // 8 x 4096 tokens. PACKED with eight rows: registers spilled, 33000 tokens of 32 sequences 267 us instead of 162.)
    constexpr int E = 4, QL = HD / 2 / E, QROWS = 32 / QL, U = sizeof(T) == 2 && !PACKED ? 8 : 4;
    using Raw = typename std::conditional<sizeof(T) == 2, uint2, uint4>::type;
    const int ql = lane % QL, qsub = lane / QL;
    float cs[E], sn[E];
#pragma unroll
    for (int i = 0; i < E; i += 4) {
      float4 x = make_float4(0.f, 0.f, 0.f, 0.f), y = x;
      if (valid) x = *reinterpret_cast<const float4 *>(r.cos + p * (HD / 2) + ql * E + i), y = *reinterpret_cast<const float4 *>(r.sin + p * (HD / 2) + ql * E + i);
      cs[i] = x.x, cs[i + 1] = x.y, cs[i + 2] = x.z, cs[i + 3] = x.w, sn[i] = y.x, sn[i + 1] = y.y, sn[i + 2] = y.z, sn[i + 3] = y.w;
    }
    const T *src = static_cast<const T *>(r.q.p) + b * r.q.sb + s * r.q.ss + ql * E;
    const long long dst = b * r.q_out.sb + s * r.q_out.ss + ql * E;
    for (int base = slice * QROWS + qsub; base < r.heads; base += un.q_slices * QROWS * U) {
      Raw lo[U], hi[U];
#pragma unroll
      for (int k = 0; k < U; k++) {
        const int h = base + k * un.q_slices * QROWS;
        lo[k] = hi[k] = Raw{};
        if (valid && h < r.heads) lo[k] = *reinterpret_cast<const Raw *>(src + h * r.q.sh), hi[k] = *reinterpret_cast<const Raw *>(src + h * r.q.sh + HD / 2);
      }
#pragma unroll
      for (int k = 0; k < U; k++) {
        const int h = base + k * un.q_slices * QROWS;
        if (h >= r.heads) break;
        const long long at = dst + h * r.q_out.sh;
        const T *x = reinterpret_cast<const T *>(&lo[k]), *y = reinterpret_cast<const T *>(&hi[k]);
        float a[E], z[E];
#pragma unroll
        for (int i = 0; i < E; i++) {
          const float u0 = widen(x[i]), u1 = widen(y[i]);
          a[i] = rope_of(u0, u1, cs[i], sn[i], false), z[i] = rope_of(u1, u0, cs[i], sn[i], true);
        }
        if (r.q_out_dtype == XNQ_F32) store4(static_cast<float *>(r.q_out.p) + at, a), store4(static_cast<float *>(r.q_out.p) + at + HD / 2, z);
        else if (r.q_out_dtype == XNQ_F16) store4(static_cast<__half *>(r.q_out.p) + at, a), store4(static_cast<__half *>(r.q_out.p) + at + HD / 2, z);
        else store4(static_cast<__nv_bfloat16 *>(r.q_out.p) + at, a), store4(static_cast<__nv_bfloat16 *>(r.q_out.p) + at + HD / 2, z);
      }
    }
    return;
  }
  const unsigned bp = u / un.kv_slices, slice = u - bp * un.kv_slices, b = PACKED ? 0u : bp / un.pairs;
  const auto put = [&](long long token) { // PACKED: of all tokens
    long long p0, s0; // the pair's even position and its token
    bool has[2], past = false;
    uint8_t *tile0; // head 0's
    int row;
    float cs[2][8], sn[2][8];
    if constexpr (PACKED) {
      const long long at = pk.slot[token], before = token > 0 ? pk.slot[token - 1] : -1, after = token + 1 < seq ? pk.slot[token + 1] : -1;
      if (at < 0 || ((at & 1) && before == at - 1)) return; // no token, or the one before has taken it along
      has[0] = !(at & 1), has[1] = (at & 1) || after == at + 1;
      s0 = token - (at & 1);
      if (ROPE) {
#pragma unroll
        for (int e = 0; e < 2; e++) {
          const long long turn = has[e] ? pk.position[s0 + e] : 0;
          if (has[e] && turn >= r.rows) has[e] = false, past = true;
          load_tables<HD>(r, turn, l, has[e], cs[e], sn[e]);
        }
      }
      const long long size = (long long)c.page_tiles * KV_TILE, page = at / size;
      const int in = (int)(at - page * size);
      row = in % KV_TILE & ~1;
      if (page >= c.num_pages) return; // (the plan is another cache's)
      tile0 = c.pages + page * c.page_bytes + (long long)(in / KV_TILE) * L::BYTES;
    } else {
      const long long first = pos_p[(long long)b * pos_stride];
      p0 = ((first >> 1) + (bp - b * un.pairs)) * 2, s0 = p0 - first;
#pragma unroll
      for (int e = 0; e < 2; e++) {
        const long long p = p0 + e, s = s0 + e;
        has[e] = s >= 0 && s < seq && p >= 0;
        if (has[e] && (p >= c.max_seq || (ROPE && p >= r.rows))) has[e] = false, past = true;
      }
    }
    if (past && lane == 0) atomicOr(&g_kv_store_status, KV_PAST_STORE);
    if (!has[0] && !has[1]) return;
    if constexpr (!PACKED) {
      tile0 = kv_tile_at(c, (int)b, 0, (int)(p0 / KV_TILE), L::BYTES);
      if (!tile0) {
        if (lane == 0) atomicOr(&g_kv_store_status, KV_NO_PAGE);
        return;
      }
      row = (int)p0 % KV_TILE;
    }
    const int pair = row / 2, blk = l / 4, t = l % 4;
    if constexpr (ROPE && !PACKED) load_tables<HD>(r, p0, l, has[0], cs[0], sn[0]), load_tables<HD>(r, p0 + 1, l, has[1], cs[1], sn[1]);
    const T *const kp = static_cast<const T *>(k.p) + b * k.sb + s0 * k.ss + l * 8, *const vp = static_cast<const T *>(v.p) + b * v.sb + s0 * v.ss + l * 8;
    auto row_of = [&](int x, float (&val)[2][8]) { // rows 0 .. KV - 1: keys, the next KV: values
      const bool is_v = x >= c.kv_heads, in = x < 2 * c.kv_heads;
      const T *p = is_v ? vp + (x - c.kv_heads) * v.sh : kp + x * k.sh;
      const long long ss = is_v ? v.ss : k.ss;
#pragma unroll
      for (int e = 0; e < 2; e++) {
#pragma unroll
        for (int i = 0; i < 8; i++) val[e][i] = 0.f;
        if (in && has[e]) load8(p + e * ss, val[e]);
      }
    };
    for (int base = slice * ROWS; base < 2 * c.kv_heads; base += un.kv_slices * ROWS) {
      const int x = base + sub;
      const bool is_v = x >= c.kv_heads;
      float val[2][8];
      row_of(x, val);
      Codes8 q[2];
#pragma unroll
      for (int e = 0; e < 2; e++) {
        if (ROPE) { // values keep theirs; the shuffles want every lane
          float y[8];
#pragma unroll
          for (int i = 0; i < 8; i++) y[i] = val[e][i];
          rope8<HD>(y, cs[e], sn[e], l >= HD / 16);
#pragma unroll
          for (int i = 0; i < 8; i++) val[e][i] = is_v ? val[e][i] : y[i];
        }
        q[e] = quantize8<BITS>(val[e]);
      }
      if (x >= 2 * c.kv_heads) continue;
      uint8_t *tile = tile0 + (is_v ? x - c.kv_heads : x) * c.head_bytes;
      if (!is_v) {
#pragma unroll
        for (int e = 0; e < 2; e++) {
          if (!has[e]) continue;
          if (BITS == 4) *reinterpret_cast<uint32_t *>(tile + L::k_word(row + e, t, blk)) = q[e].lo;
          else *reinterpret_cast<uint2 *>(tile + L::k_word(row + e, t, 2 * blk)) = make_uint2(q[e].lo, q[e].hi);
          if (t == 0) *reinterpret_cast<__half *>(tile + L::k_scale(row + e, blk)) = q[e].d;
        }
        continue;
      }
      constexpr int G = BITS / 4; // words a granule of four dims takes
#pragma unroll
      for (int half = 0; half < 2; half++) { // dims 8 t + 4 half ..: chunk g = 2 t + half
#pragma unroll
        for (int j = 0; j < G; j++) {
          uint32_t g[2];
#pragma unroll
          for (int e = 0; e < 2; e++) {
            const uint32_t w = BITS == 4 ? q[e].lo : (half ? q[e].hi : q[e].lo);
            g[e] = (BITS == 4 ? w >> (16 * half) : w >> (16 * j)) & 0xffffu;
          }
          uint8_t *at = tile + L::v_word(pair, 2 * t + half, G * blk + j);
          if (has[0] && has[1]) *reinterpret_cast<uint32_t *>(at) = g[0] | (g[1] << 16);
          else *reinterpret_cast<uint16_t *>(at + (has[0] ? 0 : 2)) = (uint16_t)(has[0] ? g[0] : g[1]);
        }
      }
      if (t == 0) {
        __half *at = reinterpret_cast<__half *>(tile + L::v_scale(pair, blk));
        if (has[0] && has[1]) *reinterpret_cast<__half2 *>(at) = __halves2half2(q[0].d, q[1].d);
        else at[has[0] ? 0 : 1] = has[0] ? q[0].d : q[1].d;
      }
    }
  };
  if constexpr (PACKED) {
    for (unsigned k = 0; k < un.each && bp * un.each + k < seq; k++) put(bp * un.each + k);
  } else put(0);
}

__device__ __forceinline__ float2 pair_values(uint32_t codes, __half2 d) { // two codes as whole numbers in f16, two scales: the exact products
  const float2 c = __half22float2(as_half2(codes)), s = __half22float2(d);
  return make_float2(c.x * s.x, c.y * s.y);
}

// k_out, v_out [batch, kv_heads, n, head_dim]: positions start .. start + n - 1. Positions outside [0, max_seq) or without a page: zeros.
template <int BITS, int HD, typename T>
__global__ void __launch_bounds__(256) kv_load_kernel(KvView c, T *k_out, T *v_out, unsigned units, unsigned tiles, long long n, const long long *start_p, int start_stride,
                                                      long long start0) {
  using L = KvTile<BITS, HD>;
  constexpr int NB = L::NB, W = L::W;
  const int lane = threadIdx.x & 31;
  const unsigned u = blockIdx.x * 8 + (threadIdx.x >> 5); // (b, head, K or V, tile)
  pdl_launch_dependents();
  pdl_wait();
  if (u >= units) return;
  const unsigned bh = u / tiles, b = bh / (2 * c.kv_heads);
  const int kh = (int)(bh - b * (2 * c.kv_heads)), head = kh >> 1;
  const long long first = start_p ? start_p[(long long)b * start_stride] : start0;
  const long long tile_i = (first >> 5) + (u - bh * tiles), j0 = tile_i * KV_TILE; // positions j0 .. j0 + 31, of which [lo, hi) are asked for
  static_assert(KV_TILE == 32, "a shift");
  const int lo = (int)max(first - j0, 0ll), hi = (int)min(first + n - j0, (long long)KV_TILE);
  if (lo >= hi) return;
  const int there = (int)min(max(c.max_seq - j0, 0ll), (long long)KV_TILE); // positions of the tile that the cache has
  const uint8_t *tile = j0 >= 0 && there > 0 ? kv_tile_at(c, (int)b, head, (int)tile_i, L::BYTES) : nullptr;
  if (lane == 0) {
    if (j0 >= 0 && there < hi) atomicOr(&g_kv_store_status, KV_PAST_STORE);
    if (j0 >= 0 && there > 0 && !tile) atomicOr(&g_kv_store_status, KV_NO_PAGE);
  }
  T *const out = (kh & 1 ? v_out : k_out) + (((long long)b * c.kv_heads + head) * n + (j0 - first)) * HD;
  if (!(kh & 1)) { // keys: a lane takes the chunk of 8 dims of every block of a row
#pragma unroll
    for (int it = 0; it < 4; it++) {
      const int row = it * 8 + lane / 4, t = lane % 4;
      if (row < lo || row >= hi) continue;
      const bool ok = tile && row < there;
      uint32_t w[W], d[NB / 2];
#pragma unroll
      for (int i = 0; i < W; i++) w[i] = 0u;
#pragma unroll
      for (int i = 0; i < NB / 2; i++) d[i] = 0u;
      if (ok) {
        load_words<W>(tile + L::k_word(row, t, 0), W == 8 ? tile + L::k_word(row, t, 4) : nullptr, w);
        load_words<NB / 2>(tile + L::k_scale(row, 0), nullptr, d);
      }
#pragma unroll
      for (int bl = 0; bl < NB; bl++) {
        const __half2 d2 = bl & 1 ? __high2half2(as_half2(d[bl / 2])) : __low2half2(as_half2(d[bl / 2]));
        float v[8];
#pragma unroll
        for (int i = 0; i < 4; i++) { // dims (i, i + 4), or (0, 2), (1, 3), (4, 6), (5, 7)
          const float2 x = pair_values(signed_pair<BITS>(BITS == 4 ? w[bl] : w[2 * bl + i / 2], BITS == 4 ? i : i & 1), d2);
          const int y = BITS == 4 ? i : (i >> 1) * 4 + (i & 1), z = BITS == 4 ? i + 4 : y + 2;
          v[y] = x.x, v[z] = x.y;
        }
        store8(out + (long long)row * HD + bl * 32 + t * 8, v);
      }
    }
    return;
  }
#pragma unroll
  for (int it = 0; it < 4; it++) { // values: a lane takes the chunk of 4 dims of every block of a pair of positions
    const int pair = it * 4 + lane / 8, g = lane % 8;
    if (2 * pair + 1 < lo || 2 * pair >= hi) continue;
    uint32_t w[W], d[NB];
#pragma unroll
    for (int i = 0; i < W; i++) w[i] = 0u;
#pragma unroll
    for (int i = 0; i < NB; i++) d[i] = 0u;
    if (tile && 2 * pair < there) {
      load_words<W>(tile + L::v_word(pair, g, 0), W == 8 ? tile + L::v_word(pair, g, 4) : nullptr, w);
      load_words<NB>(tile + L::v_scale(pair, 0), nullptr, d);
    }
    const bool odd = 2 * pair + 1 < there;
#pragma unroll
    for (int bl = 0; bl < NB; bl++) {
      float v[2][4];
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const float2 x = pair_values(signed_pair<BITS>(BITS == 4 ? w[bl] : w[2 * bl + i / 2], BITS == 4 ? i : i & 1), as_half2(d[bl]));
        v[0][i] = x.x, v[1][i] = odd ? x.y : 0.f;
      }
#pragma unroll
      for (int e = 0; e < 2; e++) {
        const int row = 2 * pair + e;
        if (row >= lo && row < hi) store4(out + (long long)row * HD + bl * 32 + g * 4, v[e]);
      }
    }
  }
}

// Warps that share a position's rows: as many as it takes to fill the GPU (148 SMs of 32 warps), a row group each at most.
unsigned slices_for(int64_t positions, int64_t groups) { return (unsigned)std::max<int64_t>(1, std::min<int64_t>(groups, 4736 / std::max<int64_t>(positions, 1))); }

template <int BITS, int HD, typename T, bool PACKED>
int run_store(const KvView &c, const KvRows &k, const KvRows &v, const RopeArgs &r, int64_t batch, int64_t seq, const long long *pos, int pos_stride, const PackedRows &pk, cudaStream_t s) {
  constexpr int ROWS = 32 / (HD / 8);
  StoreUnits un{};
  // Packed: two tokens a warp where there are enough of them, mostly one pair and a token that the one before has taken along.
  un.each = PACKED && seq >= 2 * 4736 ? 2 : 1;
  const int64_t pairs = PACKED ? (seq + un.each - 1) / un.each : seq / 2 + 1; // that `seq` positions may touch
  un.pairs = (unsigned)pairs;
  un.kv_slices = slices_for(batch * pairs, (2 * c.kv_heads + ROWS - 1) / ROWS);
  const int64_t kv = batch * pairs * un.kv_slices;
  int64_t all = kv;
  if (r.cos && r.q.p) {
    constexpr int QROWS = 32 / (HD / 8);
    un.q_slices = slices_for(batch * seq, (r.heads + QROWS - 1) / QROWS);
    all += batch * seq * un.q_slices;
  }
  if (all > INT32_MAX) return fail(XNQ_ERR_SIZE, "kv_store: %lld x %lld tokens are more than one launch takes", (long long)batch, (long long)seq);
  un.kv = (unsigned)kv, un.all = (unsigned)all;
  const dim3 grid((unsigned)((all + 7) / 8)), block(256);
  if (r.cos) XNQ_CUDA(launch_pdl(kv_store_kernel<BITS, HD, T, true, PACKED>, grid, block, 0, s, c, k, v, r, un, seq, pos, pos_stride, pk));
  else XNQ_CUDA(launch_pdl(kv_store_kernel<BITS, HD, T, false, PACKED>, grid, block, 0, s, c, k, v, r, un, seq, pos, pos_stride, pk));
  count_launch();
  return XNQ_OK;
}
template <int BITS, int HD, typename T>
int run_load(const KvView &c, void *k, void *v, int64_t batch, int64_t n, const long long *start, int start_stride, int64_t start0, cudaStream_t s) {
  const int64_t tiles = start || start0 % KV_TILE ? (n + KV_TILE - 2) / KV_TILE + 1 : (n + KV_TILE - 1) / KV_TILE; // that n positions may touch
  const int64_t units = batch * 2 * c.kv_heads * tiles;
  if (units > INT32_MAX) return fail(XNQ_ERR_SIZE, "kv_load: %lld x %lld positions are more than one launch takes", (long long)batch, (long long)n);
  XNQ_CUDA(launch_pdl(kv_load_kernel<BITS, HD, T>, dim3((unsigned)((units + 7) / 8)), dim3(256), 0, s, c, static_cast<T *>(k), static_cast<T *>(v), (unsigned)units, (unsigned)tiles, n,
                      start, start_stride, start0));
  count_launch();
  return XNQ_OK;
}

} // namespace

int kv_rows(const char *who, const char *what, const xnq_rows *x, KvRows *out) {
  if (!x || !x->data) return fail(XNQ_ERR_NULL, "%s: %s is NULL", who, what);
  if (!is_float_dtype(x->dtype)) return fail(XNQ_ERR_DTYPE, "%s: %s of type %d (f32, f16 and bf16 are served)", who, what, x->dtype);
  const int64_t e = 16 / type_size(x->dtype);
  if ((reinterpret_cast<uintptr_t>(x->data) & 15) || x->stride_b % e || x->stride_s % e || x->stride_h % e)
    return fail(XNQ_ERR_ALIGN, "%s: the rows of %s must be 16-byte aligned", who, what);
  *out = KvRows{x->data, x->stride_b, x->stride_s, x->stride_h};
  return XNQ_OK;
}

int kv_view(const char *who, const xnq_kv_cache *c, int64_t batch, KvView *v) {
  if (!c || !c->pages) return fail(XNQ_ERR_NULL, "%s: the cache is NULL", who);
  const int bits = kv_bits(c->ggml_dtype);
  if (!bits) return fail(XNQ_ERR_DTYPE, "%s: a cache holds Q4_0 (2) or Q8_0 (8), not %d", who, c->ggml_dtype);
  if (c->head_dim != 64 && c->head_dim != 128) return fail(XNQ_ERR_UNSUPPORTED, "%s: head_dim %d (64 and 128 are served)", who, c->head_dim);
  if (c->kv_heads < 1 || c->kv_heads > 65535 || c->page_size < KV_TILE || c->page_size % KV_TILE || c->page_size > INT32_MAX || c->num_pages < 1 || c->max_seq < 1 ||
      c->max_seq > INT32_MAX - KV_TILE || batch < 0 || batch > INT32_MAX)
    return fail(XNQ_ERR_SHAPE, "%s: batch %lld, kv_heads %d, page_size %lld (a multiple of %d), num_pages %lld, max_seq %lld", who, (long long)batch, c->kv_heads,
                (long long)c->page_size, KV_TILE, (long long)c->num_pages, (long long)c->max_seq);
  if (c->page_table ? (c->table_stride < 0 || (c->max_seq + c->page_size - 1) / c->page_size > c->table_stride) : (c->max_seq > c->page_size || batch > c->num_pages))
    return fail(XNQ_ERR_SIZE, "%s: %lld positions of %lld sequences do not fit %lld pages of %lld positions%s", who, (long long)c->max_seq, (long long)batch,
                (long long)(c->page_table ? c->table_stride : c->num_pages), (long long)c->page_size, c->page_table ? " a sequence" : " (one a sequence)");
  if (reinterpret_cast<uintptr_t>(c->pages) & 15) return fail(XNQ_ERR_ALIGN, "%s: the pages must be 16-byte aligned", who);
  const long long tile = (long long)kv_tile_bytes(bits, c->head_dim), tiles = c->page_size / KV_TILE;
  *v = KvView{static_cast<uint8_t *>(c->pages), c->page_table, c->table_stride, c->num_pages, tile * tiles * c->kv_heads, tile * tiles, c->max_seq, (int)tiles, c->kv_heads};
  return XNQ_OK;
}
namespace {
// rows and rotation of a store
int store_args(const xnq_rows *k, const xnq_rows *v, const xnq_kv_rope *rope, KvRows *kr, KvRows *vr, RopeArgs *r) {
  int rc;
  if ((rc = kv_rows("kv_store", "k", k, kr)) != XNQ_OK || (rc = kv_rows("kv_store", "v", v, vr)) != XNQ_OK) return rc;
  if (v->dtype != k->dtype) return fail(XNQ_ERR_DTYPE, "kv_store: k has type %d, v %d", k->dtype, v->dtype);
  if (!rope) return XNQ_OK;
  if (!rope->cos_table || !rope->sin_table) return fail(XNQ_ERR_NULL, "kv_store: a rotation without tables");
  if (rope->table_rows < 1 || rope->heads < 0 || rope->heads > 65535) return fail(XNQ_ERR_SHAPE, "kv_store: tables of %lld rows, %d heads", (long long)rope->table_rows, rope->heads);
  if ((reinterpret_cast<uintptr_t>(rope->cos_table) | reinterpret_cast<uintptr_t>(rope->sin_table)) & 15) return fail(XNQ_ERR_ALIGN, "kv_store: the tables must be 16-byte aligned");
  r->cos = rope->cos_table, r->sin = rope->sin_table, r->rows = rope->table_rows, r->heads = rope->heads;
  if (rope->heads) {
    if ((rc = kv_rows("kv_store", "q", &rope->q, &r->q)) != XNQ_OK || (rc = kv_rows("kv_store", "q_out", &rope->q_out, &r->q_out)) != XNQ_OK) return rc;
    if (rope->q.dtype != k->dtype) return fail(XNQ_ERR_DTYPE, "kv_store: k has type %d, q %d", k->dtype, rope->q.dtype);
    r->q_out_dtype = rope->q_out.dtype;
  }
  return XNQ_OK;
}
} // namespace
int kv_store_status(unsigned int *bits) {
  XNQ_CUDA(cudaMemcpyFromSymbol(bits, g_kv_store_status, sizeof(*bits)));
  return XNQ_OK;
}
int kv_store_init() {
  unsigned int zero = 0;
  XNQ_CUDA(cudaMemcpyToSymbol(g_kv_store_status, &zero, sizeof(zero)));
  return XNQ_OK;
}

} // namespace xnq

using namespace xnq;

extern "C" {

size_t xnq_kv_page_bytes(int ggml_dtype, int kv_heads, int head_dim, int64_t page_size) {
  const int bits = kv_bits(ggml_dtype);
  if (!bits || kv_heads < 1 || kv_heads > 65535 || (head_dim != 64 && head_dim != 128) || page_size < KV_TILE || page_size % KV_TILE || page_size > INT32_MAX) return 0;
  return kv_tile_bytes(bits, head_dim) * (size_t)(page_size / KV_TILE) * kv_heads;
}

int xnq_kv_store(const xnq_kv_cache *cache, const xnq_rows *k, const xnq_rows *v, int64_t batch, int64_t seq, const long long *pos, int pos_stride,
                 const xnq_kv_rope *rope, void *stream) {
  clear_error();
  KvView c;
  int rc = kv_view("kv_store", cache, batch, &c);
  if (rc != XNQ_OK) return rc;
  if (!k || !v || !pos) return fail(XNQ_ERR_NULL, "kv_store: NULL argument");
  if (seq < 0 || seq > INT32_MAX || pos_stride < 0 || pos_stride > 1) return fail(XNQ_ERR_SHAPE, "kv_store: seq %lld, pos_stride %d (0 or 1)", (long long)seq, pos_stride);
  if (batch == 0 || seq == 0) return XNQ_OK;
  KvRows kr, vr;
  RopeArgs r{};
  if ((rc = store_args(k, v, rope, &kr, &vr, &r)) != XNQ_OK) return rc;
  return kv_dispatch(kv_bits(cache->ggml_dtype), cache->head_dim, k->dtype, [&](auto f) {
    return run_store<f.BITS, f.HD, typename decltype(f)::T, false>(c, kr, vr, r, batch, seq, pos, pos_stride, PackedRows{}, static_cast<cudaStream_t>(stream));
  });
}

int xnq_kv_store_packed(const xnq_kv_cache *cache, const xnq_rows *k, const xnq_rows *v, const xnq_kv_plan *plan, const xnq_kv_rope *rope, void *stream) {
  clear_error();
  KvView c;
  int rc = kv_plan_check("kv_store", plan);
  if (rc != XNQ_OK || (rc = kv_view("kv_store", cache, plan->batch, &c)) != XNQ_OK) return rc;
  if (!k || !v) return fail(XNQ_ERR_NULL, "kv_store: NULL argument");
  if (plan->tokens == 0) return XNQ_OK;
  KvRows kr, vr;
  RopeArgs r{};
  if ((rc = store_args(k, v, rope, &kr, &vr, &r)) != XNQ_OK) return rc;
  kr.sb = vr.sb = r.q.sb = r.q_out.sb = 0;
  return kv_dispatch(kv_bits(cache->ggml_dtype), cache->head_dim, k->dtype, [&](auto f) {
    return run_store<f.BITS, f.HD, typename decltype(f)::T, true>(c, kr, vr, r, 1, plan->tokens, nullptr, 0, PackedRows{plan->slot, plan->position}, static_cast<cudaStream_t>(stream));
  });
}

int xnq_kv_load(const xnq_kv_cache *cache, int64_t batch, const long long *start_dev, int start_stride, int64_t start, int64_t n, int out_dtype, void *k_out,
                void *v_out, void *stream) {
  clear_error();
  KvView c;
  int rc = kv_view("kv_load", cache, batch, &c);
  if (rc != XNQ_OK) return rc;
  if (!is_float_dtype(out_dtype)) return fail(XNQ_ERR_DTYPE, "kv_load: results of type %d (f32, f16 and bf16 are served)", out_dtype);
  if (n < 0 || n > INT32_MAX || start_stride < 0 || start_stride > 1 || (!start_dev && (start < 0 || start + n > cache->max_seq)))
    return fail(XNQ_ERR_SHAPE, "kv_load: positions %lld .. + %lld of %lld, start_stride %d (0 or 1)", (long long)start, (long long)n, (long long)cache->max_seq, start_stride);
  if (batch == 0 || n == 0) return XNQ_OK;
  if (!k_out || !v_out) return fail(XNQ_ERR_NULL, "kv_load: NULL argument");
  if ((reinterpret_cast<uintptr_t>(k_out) | reinterpret_cast<uintptr_t>(v_out)) & 15) return fail(XNQ_ERR_ALIGN, "kv_load: results must be 16-byte aligned");
  return kv_dispatch(kv_bits(cache->ggml_dtype), cache->head_dim, out_dtype, [&](auto f) {
    return run_load<f.BITS, f.HD, typename decltype(f)::T>(c, k_out, v_out, batch, n, start_dev, start_stride, start, static_cast<cudaStream_t>(stream));
  });
}

} // extern "C"
