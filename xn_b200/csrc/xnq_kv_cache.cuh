// The quantized KV cache: how a page's bytes are laid out, and where a position's page is. Shared by the kernels that write it, read it
// back and attend over it.
//
// A page holds `page_size` positions (a multiple of 32) of every KV head: [kv_heads][page_size / 32] tiles, so that the tiles of a head are
// one run of memory. A TILE is 32 positions of one head, keys and values with their scales, in one piece (4608 bytes for 4-bit codes and
// head_dim 128), which one warp copies and consumes:
//   K codes [32 rows]       row r: RB bytes            K scales f16 [32 rows][NB]
//   V codes [16 pairs]      pair p: 2 RB bytes         V scales f16 [16 pairs][NB][2]
// with NB = head_dim / 32 blocks a row and RB code bytes a row. The codes are unsigned (0..15 for Q4_0, the int8 code + 128 for Q8_0) and lie
// in the order in which the lanes of an m16n8k16 matrix instruction take them as its first operand, so that a lane's words are ONE 8- or
// 16-byte load and unpacking is a mask (and a shift) a register, with no exchange between lanes:
//   K  rows of the operand are positions: lane (g, t) = (lane / 4, lane % 4) of row g takes the dims 8 t .. 8 t + 7 of every block.
//      Word i of chunk t: Q4_0 block i's eight nibbles; Q8_0 four bytes, words 2 b and 2 b + 1 block b's.
//   V  rows of the operand are dims, so its registers pair up POSITIONS: lane (g, t) takes the dims 4 g .. 4 g + 3 of every block at positions
//      2 t, 2 t + 1 (pair t). Word i of chunk g: the even position's 16 bits below the odd one's; Q4_0 block i's four nibbles, Q8_0 two
//      bytes, words 2 b and 2 b + 1 block b's.
// The chunks of a row or pair are rotated (K: Q8_0 with head_dim 128; V: always) so that the lanes of a shared-memory phase meet every bank once.
#pragma once

#include "xnq_common.cuh"

namespace xnq {

constexpr int KV_TILE = 32; // positions of a tile

template <int BITS_, int HD_>
struct KvTile {
  static constexpr int BITS = BITS_, HD = HD_, NB = HD / 32, RB = HD * BITS / 8;
  static constexpr int W = NB * BITS / 4; // words of a lane's chunk of a row (K) or pair (V)
  static constexpr int K_SCALES = KV_TILE * RB, V_CODES = K_SCALES + KV_TILE * NB * 2, V_SCALES = V_CODES + KV_TILE * RB, BYTES = V_SCALES + KV_TILE * NB * 2;
  static constexpr int ZERO = BITS == 4 ? 8 : 128; // the code that stands for 0
  // byte offsets in the tile
  __host__ __device__ static constexpr int k_word(int row, int t, int i) {
    return W == 8 ? row * RB + ((i >> 2) ^ (row & 1)) * 64 + t * 16 + (i & 3) * 4 : row * RB + t * (W * 4) + i * 4;
  }
  __host__ __device__ static constexpr int k_scale(int row, int b) { return K_SCALES + (row * NB + b) * 2; }
  __host__ __device__ static constexpr int v_word(int pair, int g, int i) {
    return V_CODES + (W == 2 ? pair * (2 * RB) + ((g + 4 * ((pair >> 1) & 1)) & 7) * 8 + i * 4
                             : pair * (2 * RB) + (i >> 2) * 128 + ((g + 2 * (pair & 3)) & 7) * 16 + (i & 3) * 4);
  }
  __host__ __device__ static constexpr int v_scale(int pair, int b) { return V_SCALES + (pair * NB + b) * 4; } // two f16: the pair's
};

inline size_t kv_tile_bytes(int bits, int head_dim) { return (size_t)KV_TILE * 2 * (head_dim * bits / 8 + head_dim / 16); }
inline int kv_bits(int ggml_dtype) { return ggml_dtype == XNQ_Q4_0 ? 4 : (ggml_dtype == XNQ_Q8_0 ? 8 : 0); }

// What the kernels get of a cache.
struct KvView {
  uint8_t *pages;
  const int *table; // null: sequence b is page b
  long long table_stride, num_pages, page_bytes, head_bytes; // head_bytes: a head's tiles of one page
  long long max_seq;
  int page_tiles; // tiles of a head in a page
  int kv_heads;
};
struct KvRows { // [batch, seq, heads, head_dim] of a float type; strides in elements, head_dim contiguous, every row 16-byte aligned
  void *p;
  long long sb, ss, sh;
};
int kv_rows(const char *who, const char *what, const xnq_rows *x, KvRows *out);
// calls f with a KvForm of the cache's format and head_dim and of a float type
template <int BITS_, int HD_, typename T_>
struct KvForm {
  static constexpr int BITS = BITS_, HD = HD_;
  using T = T_;
};
template <int BITS, int HD, typename F>
int kv_dispatch_type(int dtype, F f) {
  if (dtype == XNQ_F32) return f(KvForm<BITS, HD, float>{});
  if (dtype == XNQ_F16) return f(KvForm<BITS, HD, __half>{});
  return f(KvForm<BITS, HD, __nv_bfloat16>{});
}
template <typename F>
int kv_dispatch(int bits, int head_dim, int dtype, F f) {
  if (bits == 4) return head_dim == 64 ? kv_dispatch_type<4, 64>(dtype, f) : kv_dispatch_type<4, 128>(dtype, f);
  return head_dim == 64 ? kv_dispatch_type<8, 64>(dtype, f) : kv_dispatch_type<8, 128>(dtype, f);
}

int kv_view(const char *who, const xnq_kv_cache *c, int64_t batch, KvView *v); // checks the descriptor

// status bits (xnq_device_status bits 27 and up): a position past the cache was asked for, by a store or load (1) or by attention (2); a page table's
// entry was outside the cache (4)
constexpr unsigned KV_PAST_STORE = 1, KV_PAST_ATTEND = 2, KV_NO_PAGE = 4;

#ifdef __CUDACC__
// The tile of (sequence, head) that holds positions 32 * tile .. ; null where the page table has no page there.
__device__ __forceinline__ uint8_t *kv_tile_at(const KvView &c, int b, int head, int tile, int tile_bytes) {
  long long page = b;
  int in = tile;
  if (c.table) {
    const int pi = tile / c.page_tiles;
    in = tile - pi * c.page_tiles;
    page = __ldg(c.table + b * c.table_stride + pi);
    if (page < 0 || page >= c.num_pages) return nullptr;
  }
  return c.pages + page * c.page_bytes + head * c.head_bytes + (long long)in * tile_bytes;
}
#endif

} // namespace xnq
