// Tiled attention of prompt portions over a cache in 4 bits: the blocks of attention_prefill.hip (see there for the
// method) with another way of getting a tile of keys and values into LDS.  A lane asks for its pieces of eight codes two
// tiles ahead of the one being multiplied, 4 bytes of codes and a step of 2 where the other cache has 16, and turns
// them into bfloat16 values one tile ahead, exactly (cache_int4.h says why that is no rounding); what follows is the same
// code, so that this attention is that one over a cache of these values.
#include <math.h>

#include "common.h"
#include "pagedserve_hip.h"

#include "attention_prefill_block.h"

template <int NDB, int KS, int QW = 2, int KR = 1>
__global__ __launch_bounds__(64 * QW * KS) void attention_prefill_int4_kernel(
    const bf16_t* __restrict__ q, int64_t q_stride, const uint8_t* __restrict__ k_pool,
    const uint8_t* __restrict__ v_pool, bf16_t* __restrict__ out, int64_t out_stride,
    const int* __restrict__ tile_item, const int* __restrict__ tile_q0,
    const int* __restrict__ cu_tokens, const int* __restrict__ kv_lens,
    const int* __restrict__ tables, int table_width, int heads, int kv_heads, int page_size,
    int page_shift, int num_pages, float scale, int window, const AttnExtras extra) {
  __shared__ PrefillLds<NDB, KS, QW, KR> lds;
  attention_prefill_block<NDB, KS, QW, KR, Int4Pages>(lds, blockIdx.x, blockIdx.y, q, q_stride, k_pool, v_pool, out,
                                                      out_stride, tile_item, tile_q0, cu_tokens, kv_lens, tables,
                                                      table_width, heads, kv_heads, page_size, page_shift,
                                                      num_pages, scale, window, extra);
}

extern "C" int ps_attention_prefill_int4(const void* q, int64_t q_stride, const void* k_pool, const void* v_pool,
                                         void* out, int64_t out_stride, const int* tile_item, const int* tile_q0,
                                         int tiles, const int* cu_tokens, const int* kv_lens, const int* tables,
                                         int table_width, int heads, int kv_heads, int head_dim, int page_size,
                                         int num_pages, float scale, int window, int max_kv_len, int query_tile,
                                         const float* sink, float softcap, void* stream) {
  const char* who = "ps_attention_prefill_int4";
  PS_REQUIRE(tiles >= 0 && heads > 0 && kv_heads > 0 && page_size > 0 && num_pages > 0 && table_width > 0,
             "%s: bad sizes", who);
  PS_REQUIRE(heads % kv_heads == 0, "%s: heads (%d) must be a multiple of kv_heads (%d)", who, heads, kv_heads);
  PS_REQUIRE(head_dim > 0 && head_dim % 16 == 0 && head_dim <= 256,
             "%s: head_dim %d must be a multiple of 16 up to 256", who, head_dim);
  PS_REQUIRE(page_size % 8 == 0 && page_size <= (1 << 20),
             "%s: pages of a cache in 4 bits hold a multiple of 8 keys, not %d", who, page_size);
  PS_REQUIRE(tiles <= 65535, "%s: too many tiles (%d)", who, tiles);
  PS_REQUIRE(query_tile == AP_QUERIES || (query_tile == AP_QUERIES / 2 && head_dim <= 128) ||
                 (query_tile == AP_QUERIES * 2 && head_dim <= AP_LARGE_HEAD_DIM),
             "%s: tiles of %d, (head sizes up to 128) %d or (head sizes up to %d) %d queries, not %d", who,
             AP_QUERIES, AP_QUERIES / 2, AP_LARGE_HEAD_DIM, AP_QUERIES * 2, query_tile);
  PS_REQUIRE((int64_t)num_pages * kv_heads * page_size < ((int64_t)1 << 32),
             "%s: a pool of %d pages x %d heads x %d keys has 2^32 key rows or more", who, num_pages, kv_heads, page_size);
  PS_REQUIRE(scale > 0.f, "%s: the score scale must be positive, got %g", who, scale);
  PS_REQUIRE(table_width <= AP_TABLE_MAX, "%s: block tables of %d pages exceed the %d that a tile keeps", who,
             table_width, AP_TABLE_MAX);
  PS_REQUIRE((q_stride % 8) == 0 && ((uintptr_t)q % 16) == 0 && (out_stride % 4) == 0 && ((uintptr_t)out % 8) == 0,
             "%s: q and out rows must allow 16- and 8-byte accesses", who);
  if (tiles == 0) return 0;
  int page_shift = -1;
  if ((page_size & (page_size - 1)) == 0) {
    page_shift = 0;
    while ((1 << page_shift) < page_size) ++page_shift;
  }
  hipStream_t s = (hipStream_t)stream;
  const AttnExtras extra = {sink, nullptr, 0, softcap, nullptr, 1.f};
  dim3 grid(heads, tiles);
  // four waves along the keys where few blocks see many keys, as for the other cache
  const bool wide = (int64_t)tiles * heads <= ps_compute_units() * 2 && (max_kv_len <= 0 || max_kv_len >= 512);
#define PS_LAUNCH_P4(THREADS, ...)                                                                              \
  hipLaunchKernelGGL((attention_prefill_int4_kernel<__VA_ARGS__>), grid, dim3(THREADS), 0, s, (const bf16_t*)q, \
                     q_stride, (const uint8_t*)k_pool, (const uint8_t*)v_pool, (bf16_t*)out, out_stride,        \
                     tile_item, tile_q0, cu_tokens, kv_lens, tables, table_width, heads, kv_heads, page_size,   \
                     page_shift, num_pages, scale, window, extra)
#define PS_TILES_P4(NDB)                                      \
  case NDB:                                                   \
    if (query_tile == AP_QUERIES * 2) {                       \
      if constexpr (NDB <= AP_LARGE_HEAD_DIM / 16) PS_LAUNCH_P4(256, NDB, 1, 4, 2); \
    } else if (query_tile != AP_QUERIES) {                    \
      if constexpr (NDB <= 8) PS_LAUNCH_P4(256, NDB, 4, 1);   \
    } else if (NDB <= 8 && wide) {                            \
      if constexpr (NDB <= 8) PS_LAUNCH_P4(512, NDB, 4);      \
    } else {                                                  \
      PS_LAUNCH_P4(256, NDB, 2);                              \
    }                                                         \
    break
  switch (head_dim / 16) {
    PS_TILES_P4(1);
    PS_TILES_P4(2);
    PS_TILES_P4(3);
    PS_TILES_P4(4);
    PS_TILES_P4(5);
    PS_TILES_P4(6);
    PS_TILES_P4(7);
    PS_TILES_P4(8);
    PS_TILES_P4(9);
    PS_TILES_P4(10);
    PS_TILES_P4(11);
    PS_TILES_P4(12);
    PS_TILES_P4(13);
    PS_TILES_P4(14);
    PS_TILES_P4(15);
    default: PS_LAUNCH_P4(256, 16, 2);
  }
#undef PS_TILES_P4
#undef PS_LAUNCH_P4
  PS_CHECK_LAUNCH("ps_attention_prefill_int4");
  return 0;
}
