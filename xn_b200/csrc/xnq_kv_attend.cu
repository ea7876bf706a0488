// Attention over the quantized KV cache.
#include <cmath>

#include "xnq_kv_cache.cuh"

namespace xnq {
namespace {

__device__ unsigned int g_kv_attend_status;

struct AttendArgs {
  KvView c;
  KvRows q, out;
  float *lse; // [batch, seq, heads], or null
  long long batch, seq;
  int heads, pos_stride, causal;
  const long long *pos;
  float scale;
  long long window;
};

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void from_float(float *p, float v) { *p = v; }
__device__ __forceinline__ void from_float(__half *p, float v) { *p = __float2half_rn(v); }
__device__ __forceinline__ void from_float(__nv_bfloat16 *p, float v) { *p = __float2bfloat16_rn(v); }

// One warp per query row; a lane holds one dim of every block of 32.
template <int BITS, int HD, typename T>
__global__ void __launch_bounds__(128) kv_attend_rows_kernel(AttendArgs a) {
  using L = KvTile<BITS, HD>;
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const long long row = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (row >= a.batch * a.seq * a.heads) return;
  const long long bs = row / a.heads, b = bs / a.seq, s = bs - b * a.seq;
  const int h = (int)(row - bs * a.heads), kvh = h / (a.heads / a.c.kv_heads);
  const long long first = a.pos[b * a.pos_stride], p = first + s;
  long long hi = a.causal ? p : first + a.seq - 1, lo = a.window ? p - a.window + 1 : 0;
  if (lo < 0) lo = 0;
  if (hi >= a.c.max_seq) {
    hi = a.c.max_seq - 1;
    if (lane == 0) atomicOr(&g_kv_attend_status, KV_PAST_ATTEND);
  }
  if (p < 0) hi = -1;
  float q[L::NB], acc[L::NB], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int i = 0; i < L::NB; i++) {
    q[i] = to_float(static_cast<const T *>(a.q.p)[b * a.q.sb + s * a.q.ss + h * a.q.sh + i * 32 + lane]) * a.scale;
    acc[i] = 0.f;
  }
  for (long long j = lo; j <= hi; j++) {
    const uint8_t *tile = kv_tile_at(a.c, (int)b, kvh, (int)(j / KV_TILE), L::BYTES);
    if (!tile) {
      if (lane == 0) atomicOr(&g_kv_attend_status, KV_NO_PAGE);
      continue;
    }
    const int r = (int)(j % KV_TILE);
    float d = 0.f;
#pragma unroll
    for (int i = 0; i < L::NB; i++) {
      const float sc = __half2float(*reinterpret_cast<const __half *>(tile + L::k_scale(r, i)));
      int code;
      if (BITS == 4) code = *reinterpret_cast<const uint32_t *>(tile + L::k_word(r, lane / 8, i)) >> (4 * (lane & 7)) & 15;
      else code = *reinterpret_cast<const uint32_t *>(tile + L::k_word(r, lane / 8, 2 * i + (lane & 7) / 4)) >> (8 * (lane & 3)) & 255;
      d += q[i] * (sc * (float)(code - L::ZERO));
    }
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) d += __shfl_xor_sync(0xffffffffu, d, o);
    const float mn = fmaxf(m, d), corr = m == -INFINITY ? 0.f : expf(m - mn), w = expf(d - mn);
    l = l * corr + w;
    m = mn;
#pragma unroll
    for (int i = 0; i < L::NB; i++) {
      const float sc = __half2float(*reinterpret_cast<const __half *>(tile + L::v_scale(r / 2, i) + 2 * (r & 1)));
      int code;
      if (BITS == 4) code = *reinterpret_cast<const uint32_t *>(tile + L::v_word(r / 2, lane / 4, i)) >> (16 * (r & 1) + 4 * (lane & 3)) & 15;
      else code = *reinterpret_cast<const uint32_t *>(tile + L::v_word(r / 2, lane / 4, 2 * i + (lane & 3) / 2)) >> (16 * (r & 1) + 8 * (lane & 1)) & 255;
      acc[i] = acc[i] * corr + w * (sc * (float)(code - L::ZERO));
    }
  }
  T *o = static_cast<T *>(a.out.p) + b * a.out.sb + s * a.out.ss + h * a.out.sh;
#pragma unroll
  for (int i = 0; i < L::NB; i++) from_float(o + i * 32 + lane, l > 0.f ? acc[i] / l : 0.f);
  if (a.lse && lane == 0) a.lse[row] = l > 0.f ? m + logf(l) : -INFINITY;
}

template <int BITS, int HD, typename T>
int run_attend(const AttendArgs &a, cudaStream_t s) {
  const long long blocks = (a.batch * a.seq * a.heads + 3) / 4;
  if (blocks > INT32_MAX) return fail(XNQ_ERR_SIZE, "kv_attend: too many rows");
  XNQ_CUDA(launch_pdl(kv_attend_rows_kernel<BITS, HD, T>, dim3((unsigned)blocks), dim3(128), 0, s, a));
  count_launch();
  return XNQ_OK;
}

} // namespace

int kv_attend_status(unsigned int *bits) {
  XNQ_CUDA(cudaMemcpyFromSymbol(bits, g_kv_attend_status, sizeof(*bits)));
  return XNQ_OK;
}
int kv_attend_init(int) {
  unsigned int zero = 0;
  XNQ_CUDA(cudaMemcpyToSymbol(g_kv_attend_status, &zero, sizeof(zero)));
  return XNQ_OK;
}

} // namespace xnq

using namespace xnq;

extern "C" {

size_t xnq_kv_attend_workspace_bytes(int64_t batch, int64_t seq, int heads, int kv_heads, int head_dim) {
  if (batch <= 0 || seq <= 0 || heads < 1 || kv_heads < 1 || heads % kv_heads || (head_dim != 64 && head_dim != 128)) return 0;
  return 16;
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
  if (batch == 0 || seq == 0) return XNQ_OK;
  if ((rc = kv_rows("kv_attend", "q", q, &a.q)) != XNQ_OK || (rc = kv_rows("kv_attend", "out", out, &a.out)) != XNQ_OK) return rc;
  if (out->dtype != q->dtype) return fail(XNQ_ERR_DTYPE, "kv_attend: q has type %d, out %d", q->dtype, out->dtype);
  if (!std::isfinite(scale)) return fail(XNQ_ERR_SHAPE, "kv_attend: the scale is not a finite number");
  const size_t need = xnq_kv_attend_workspace_bytes(batch, seq, heads, cache->kv_heads, cache->head_dim);
  if (!workspace || ws_bytes < need) return fail(XNQ_ERR_SIZE, "kv_attend: workspace has %zu bytes, needs %zu (zero it once after allocating)", ws_bytes, need);
  if (reinterpret_cast<uintptr_t>(workspace) & 15) return fail(XNQ_ERR_ALIGN, "kv_attend: the workspace must be 16-byte aligned");
  a.lse = lse, a.batch = batch, a.seq = seq, a.heads = heads, a.pos_stride = pos_stride, a.causal = causal, a.pos = pos, a.scale = scale, a.window = window;
  return kv_dispatch(kv_bits(cache->ggml_dtype), cache->head_dim, q->dtype,
                     [&](auto f) { return run_attend<f.BITS, f.HD, typename decltype(f)::T>(a, static_cast<cudaStream_t>(stream)); });
}

} // extern "C"
