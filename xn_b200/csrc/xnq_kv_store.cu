// The quantized KV cache is written (quantized as it is stored, after an optional rotary embedding of q and k) and read back.
//
// Both kernels are bound by their bytes: one pass, each value read once and written once. A thread takes 8 consecutive dims of a PAIR of
// positions (2 i, 2 i + 1) that share the words of V's codes, so a pair is stored in whole words; where only one of the two is new, the other
// half of a word is left alone (2-byte stores). Four neighbouring threads hold a block of 32.
#include "xnq_kv_cache.cuh"
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

// One block of 32 in four neighbouring lanes, 8 values each: the arithmetic of BlockQ4_0::from_float and BlockQ8_0::from_float
// (k_quants.rs:235-270, 636-661), every operation rounded for itself, but for Q8_0's scale: max|x| times the f32 nearest 1 / 127, where the file's quantizer
// divides by 127 (the two differ in the scale's last f32 bit, one f16 scale in some 4000 and one code at a tie). The codes come back unsigned: 4 bits, eight
// nibbles in lo; 8 bits, code + 128.
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
  float amax = 0.f, mx = 0.f; // the first value of the largest magnitude; a NaN is passed over
#pragma unroll
  for (int i = 0; i < 8; i++)
    if (amax < fabsf(v[i])) amax = fabsf(v[i]), mx = v[i];
  const int t = threadIdx.x & 3;
#pragma unroll
  for (int off = 1; off <= 2; off <<= 1) {
    const float oa = __shfl_xor_sync(0xffffffffu, amax, off), om = __shfl_xor_sync(0xffffffffu, mx, off);
    if (oa > amax || (oa == amax && (t & off))) amax = oa, mx = om; // of equals the lower lane's
  }
  const float d = __fdiv_rn(mx, -8.0f), id = d != 0.f ? __fdiv_rn(1.0f, d) : 0.f;
  uint32_t w = 0;
#pragma unroll
  for (int i = 0; i < 8; i++) w |= (uint32_t)min(max(__float2int_rz(__fadd_rn(__fmul_rn(v[i], id), 8.5f)), 0), 15) << (4 * i);
  o.lo = w, o.hi = 0u, o.d = __float2half_rn(d);
  return o;
}

__device__ __forceinline__ float rope_of(float x, float other, float c, float s, bool upper) { // rotate-half: x's half of the pair
  return upper ? __fadd_rn(__fmul_rn(x, c), __fmul_rn(other, s)) : __fsub_rn(__fmul_rn(x, c), __fmul_rn(other, s));
}
// this thread's 8 values of a head rotated; its partner, half a head away, holds the other half of the pairs
template <int HD>
__device__ __forceinline__ void rope8(float (&v)[8], const RopeArgs &r, long long pos, int l, bool valid) {
  const bool upper = l >= HD / 16;
  float c[8], s[8];
#pragma unroll
  for (int i = 0; i < 8; i++) c[i] = s[i] = 0.f;
  if (valid) {
    load8(r.cos + pos * (HD / 2) + (l & (HD / 16 - 1)) * 8, c);
    load8(r.sin + pos * (HD / 2) + (l & (HD / 16 - 1)) * 8, s);
  }
#pragma unroll
  for (int i = 0; i < 8; i++) {
    const float other = __shfl_xor_sync(0xffffffffu, v[i], HD / 16);
    v[i] = rope_of(v[i], other, c[i], s[i], upper);
  }
}

// Blocks [0, kv_blocks) store keys and values, the rest rotate queries. Whole warps work or leave together.
template <int BITS, int HD, typename T, bool ROPE>
__global__ void __launch_bounds__(256) kv_store_kernel(KvView c, KvRows k, KvRows v, RopeArgs r, long long batch, long long seq, const long long *pos_p, int pos_stride,
                                                       long long kv_blocks) {
  using L = KvTile<BITS, HD>;
  constexpr int LANES = HD / 8; // threads of a head's row
  pdl_launch_dependents();
  pdl_wait();
  const int l = threadIdx.x % LANES;
  if (blockIdx.x >= kv_blocks) { // queries
    const long long u = (long long)(blockIdx.x - kv_blocks) * (256 / LANES) + threadIdx.x / LANES; // row (b, s, head)
    const bool in = u < batch * seq * r.heads;
    const long long bs = in ? u / r.heads : 0, b = bs / seq, s = bs - b * seq;
    const int h = in ? (int)(u - bs * r.heads) : 0;
    const long long p = pos_p[b * pos_stride] + s;
    const bool valid = in && p >= 0 && p < r.rows;
    float x[8] = {};
    if (valid) load8(static_cast<const T *>(r.q.p) + b * r.q.sb + s * r.q.ss + h * r.q.sh + l * 8, x);
    rope8<HD>(x, r, p, l, valid);
    const long long at = b * r.q_out.sb + s * r.q_out.ss + h * r.q_out.sh + l * 8;
    if (!in) return;
    if (r.q_out_dtype == XNQ_F32) store8(static_cast<float *>(r.q_out.p) + at, x);
    else if (r.q_out_dtype == XNQ_F16) store8(static_cast<__half *>(r.q_out.p) + at, x);
    else store8(static_cast<__nv_bfloat16 *>(r.q_out.p) + at, x);
    return;
  }
  const long long pairs = seq / 2 + 1; // pairs that `seq` positions may touch
  const long long u = (long long)blockIdx.x * (256 / LANES) + threadIdx.x / LANES; // (b, pair, K or V, head)
  const bool in = u < batch * pairs * 2 * c.kv_heads;
  const long long bp = in ? u / (2 * c.kv_heads) : 0, b = bp / pairs;
  const int kh = in ? (int)(u - bp * (2 * c.kv_heads)) : 0;
  const bool is_v = kh >= c.kv_heads;
  const int head = is_v ? kh - c.kv_heads : kh;
  const long long first = pos_p[b * pos_stride];
  const long long p0 = ((first >> 1) + (bp - b * pairs)) * 2; // the pair's even position
  const KvRows &x = is_v ? v : k;
  bool has[2];
  float val[2][8];
#pragma unroll
  for (int e = 0; e < 2; e++) {
    const long long p = p0 + e, s = p - first;
    has[e] = in && s >= 0 && s < seq && p >= 0;
    if (has[e] && (p >= c.max_seq || (ROPE && p >= r.rows))) {
      has[e] = false;
      if (l == 0) atomicOr(&g_kv_store_status, KV_PAST_STORE);
    }
#pragma unroll
    for (int i = 0; i < 8; i++) val[e][i] = 0.f;
    if (has[e]) load8(static_cast<const T *>(x.p) + b * x.sb + s * x.ss + head * x.sh + l * 8, val[e]);
  }
  Codes8 q[2];
#pragma unroll
  for (int e = 0; e < 2; e++) {
    if (ROPE) { // values keep theirs; the shuffles want every lane
      float t[8];
#pragma unroll
      for (int i = 0; i < 8; i++) t[i] = val[e][i];
      rope8<HD>(t, r, p0 + e, l, has[e]);
#pragma unroll
      for (int i = 0; i < 8; i++) val[e][i] = is_v ? val[e][i] : t[i];
    }
    q[e] = quantize8<BITS>(val[e]);
  }
  if (!has[0] && !has[1]) return;
  uint8_t *tile = kv_tile_at(c, (int)b, head, (int)(p0 / KV_TILE), L::BYTES);
  if (!tile) {
    if (l == 0) atomicOr(&g_kv_store_status, KV_NO_PAGE);
    return;
  }
  const int row = (int)(p0 % KV_TILE), pair = row / 2, blk = l / 4, t = l % 4;
  if (!is_v) {
#pragma unroll
    for (int e = 0; e < 2; e++) {
      if (!has[e]) continue;
      if (BITS == 4) *reinterpret_cast<uint32_t *>(tile + L::k_word(row + e, t, blk)) = q[e].lo;
      else *reinterpret_cast<uint2 *>(tile + L::k_word(row + e, t, 2 * blk)) = make_uint2(q[e].lo, q[e].hi);
      if (t == 0) *reinterpret_cast<__half *>(tile + L::k_scale(row + e, blk)) = q[e].d;
    }
    return;
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
#pragma unroll
    for (int e = 0; e < 2; e++)
      if (has[e]) at[e] = q[e].d;
  }
}

// k_out, v_out [batch, kv_heads, n, head_dim]: positions start .. start + n - 1. Positions outside [0, max_seq) or without a page: zeros.
template <int BITS, int HD, typename T>
__global__ void __launch_bounds__(256) kv_load_kernel(KvView c, T *k_out, T *v_out, long long batch, long long n, const long long *start_p, int start_stride,
                                                      long long start0) {
  using L = KvTile<BITS, HD>;
  constexpr int LANES = HD / 8;
  pdl_launch_dependents();
  pdl_wait();
  const int l = threadIdx.x % LANES, blk = l / 4, t = l % 4;
  const long long pairs = n / 2 + 1;
  const long long u = (long long)blockIdx.x * (256 / LANES) + threadIdx.x / LANES; // (b, K or V, head, pair)
  if (u >= batch * 2 * c.kv_heads * pairs) return;
  const long long bk = u / pairs, b = bk / (2 * c.kv_heads);
  const int kh = (int)(bk - b * (2 * c.kv_heads));
  const bool is_v = kh >= c.kv_heads;
  const int head = is_v ? kh - c.kv_heads : kh;
  const long long first = start_p ? start_p[b * start_stride] : start0;
  const long long p0 = ((first >> 1) + (u - bk * pairs)) * 2;
  T *out = (is_v ? v_out : k_out) + (b * c.kv_heads + head) * n * HD + l * 8;
  uint8_t *tile = nullptr;
  if (p0 >= 0 && p0 < c.max_seq) {
    tile = kv_tile_at(c, (int)b, head, (int)(p0 / KV_TILE), L::BYTES);
    if (!tile && l == 0) atomicOr(&g_kv_store_status, KV_NO_PAGE);
  }
  const int row = (int)(p0 % KV_TILE), pair = row / 2;
  uint32_t w[2][2] = {}; // [position][lo, hi]: codes as the quantizer made them
  float d[2] = {};
  if (tile) {
    if (!is_v) {
#pragma unroll
      for (int e = 0; e < 2; e++) {
        if (BITS == 4) w[e][0] = *reinterpret_cast<const uint32_t *>(tile + L::k_word(row + e, t, blk));
        else {
          const uint2 x = *reinterpret_cast<const uint2 *>(tile + L::k_word(row + e, t, 2 * blk));
          w[e][0] = x.x, w[e][1] = x.y;
        }
        d[e] = __half2float(*reinterpret_cast<const __half *>(tile + L::k_scale(row + e, blk)));
      }
    } else {
      constexpr int G = BITS / 4;
#pragma unroll
      for (int half = 0; half < 2; half++)
#pragma unroll
        for (int j = 0; j < G; j++) {
          const uint32_t x = *reinterpret_cast<const uint32_t *>(tile + L::v_word(pair, 2 * t + half, G * blk + j));
          const int at = BITS == 4 ? 0 : half, sh = BITS == 4 ? 16 * half : 16 * j;
          w[0][at] |= (x & 0xffffu) << sh, w[1][at] |= (x >> 16) << sh;
        }
      const __half2 s = *reinterpret_cast<const __half2 *>(tile + L::v_scale(pair, blk));
      d[0] = __low2float(s), d[1] = __high2float(s);
    }
  }
#pragma unroll
  for (int e = 0; e < 2; e++) {
    const long long p = p0 + e, s = p - first;
    if (s < 0 || s >= n) continue;
    const bool ok = tile && p < c.max_seq;
    if (!ok && p >= c.max_seq && l == 0) atomicOr(&g_kv_store_status, KV_PAST_STORE);
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; i++) {
      const int code = BITS == 4 ? (int)(w[e][0] >> (4 * i)) & 15 : (int)(w[e][i / 4] >> (8 * (i % 4))) & 255;
      v[i] = ok ? d[e] * (float)(code - L::ZERO) : 0.f;
    }
    store8(out + s * HD, v);
  }
}

template <int BITS, int HD, typename T>
int run_store(const KvView &c, const KvRows &k, const KvRows &v, const RopeArgs &r, int64_t batch, int64_t seq, const long long *pos, int pos_stride, cudaStream_t s) {
  const int64_t rows_per_block = 256 / (HD / 8);
  const int64_t kv = (batch * (seq / 2 + 1) * 2 * c.kv_heads + rows_per_block - 1) / rows_per_block;
  const int64_t q = r.cos && r.q.p ? (batch * seq * r.heads + rows_per_block - 1) / rows_per_block : 0;
  if (kv + q > INT32_MAX) return fail(XNQ_ERR_SIZE, "kv_store: %lld x %lld tokens are more than one launch takes", (long long)batch, (long long)seq);
  const dim3 grid((unsigned)(kv + q)), block(256);
  if (r.cos) XNQ_CUDA(launch_pdl(kv_store_kernel<BITS, HD, T, true>, grid, block, 0, s, c, k, v, r, batch, seq, pos, pos_stride, kv));
  else XNQ_CUDA(launch_pdl(kv_store_kernel<BITS, HD, T, false>, grid, block, 0, s, c, k, v, r, batch, seq, pos, pos_stride, kv));
  count_launch();
  return XNQ_OK;
}
template <int BITS, int HD, typename T>
int run_load(const KvView &c, void *k, void *v, int64_t batch, int64_t n, const long long *start, int start_stride, int64_t start0, cudaStream_t s) {
  const int64_t rows_per_block = 256 / (HD / 8);
  const int64_t blocks = (batch * 2 * c.kv_heads * (n / 2 + 1) + rows_per_block - 1) / rows_per_block;
  if (blocks > INT32_MAX) return fail(XNQ_ERR_SIZE, "kv_load: %lld x %lld positions are more than one launch takes", (long long)batch, (long long)n);
  XNQ_CUDA(launch_pdl(kv_load_kernel<BITS, HD, T>, dim3((unsigned)blocks), dim3(256), 0, s, c, static_cast<T *>(k), static_cast<T *>(v), batch, n, start, start_stride, start0));
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
  if ((rc = kv_rows("kv_store", "k", k, &kr)) != XNQ_OK || (rc = kv_rows("kv_store", "v", v, &vr)) != XNQ_OK) return rc;
  if (v->dtype != k->dtype) return fail(XNQ_ERR_DTYPE, "kv_store: k has type %d, v %d", k->dtype, v->dtype);
  RopeArgs r{};
  if (rope) {
    if (!rope->cos_table || !rope->sin_table) return fail(XNQ_ERR_NULL, "kv_store: a rotation without tables");
    if (rope->table_rows < 1 || rope->heads < 0 || rope->heads > 65535) return fail(XNQ_ERR_SHAPE, "kv_store: tables of %lld rows, %d heads", (long long)rope->table_rows, rope->heads);
    if ((reinterpret_cast<uintptr_t>(rope->cos_table) | reinterpret_cast<uintptr_t>(rope->sin_table)) & 15) return fail(XNQ_ERR_ALIGN, "kv_store: the tables must be 16-byte aligned");
    r.cos = rope->cos_table, r.sin = rope->sin_table, r.rows = rope->table_rows, r.heads = rope->heads;
    if (rope->heads) {
      if ((rc = kv_rows("kv_store", "q", &rope->q, &r.q)) != XNQ_OK || (rc = kv_rows("kv_store", "q_out", &rope->q_out, &r.q_out)) != XNQ_OK) return rc;
      if (rope->q.dtype != k->dtype) return fail(XNQ_ERR_DTYPE, "kv_store: k has type %d, q %d", k->dtype, rope->q.dtype);
      r.q_out_dtype = rope->q_out.dtype;
    }
  }
  return kv_dispatch(kv_bits(cache->ggml_dtype), cache->head_dim, k->dtype, [&](auto f) {
    return run_store<f.BITS, f.HD, typename decltype(f)::T>(c, kr, vr, r, batch, seq, pos, pos_stride, static_cast<cudaStream_t>(stream));
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
