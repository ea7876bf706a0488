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
};

// Workspace: the tickets, at one place whatever the call, then the parts.
constexpr int KV_TICKETS = 1024;
constexpr size_t KV_TICKET_BYTES = KV_TICKETS * 4;
static_assert(KV_TICKET_BYTES == XNQ_KV_WORKSPACE_ZEROED, "what a caller zeroes");
constexpr unsigned KV_WAIT = 8; // status: a wait of the kernel for many rows expired (with the bits of xnq_kv_cache.cuh)

// xnq_kv_prompt.cu: many 16-bit query rows
int kv_prompt_init(int device);
int kv_prompt_status(unsigned int *bits);
size_t kv_prompt_parts_bytes(int head_dim);
int launch_kv_prompt(const AttendArgs &a, int bits, int head_dim, int sms, cudaStream_t s);

#ifdef __CUDACC__
// positions [lo, hi] that the query at token s of a sequence at `pos` sees
__device__ __forceinline__ void seen_by(const AttendArgs &a, long long pos, long long s, int &lo, int &hi) {
  const long long p = pos + s;
  const long long h = p < 0 ? -1 : min(a.causal ? p : pos + a.seq - 1, a.c.max_seq - 1);
  const long long l = a.window ? max(p - a.window + 1, 0ll) : 0ll;
  hi = (int)h, lo = (int)min(l, a.c.max_seq);
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
