// Tiled attention of prompt portions over a cache in 4 bits: the blocks of attention_prefill.hip (see there for the
// method) with another way of getting a tile of keys and values into LDS.  A thread asks for a quarter of a key's (or a
// value's) row of codes, 4 bytes of each group, two tiles ahead of the one being multiplied, and turns them into bfloat16
// values one tile ahead, exactly (cache_int4.h says why that is no rounding); what follows is the same code, so that this
// attention is that one over a cache of these values.
//
// Bound: the vector instructions of the conversion (3.5 to a value: four bits to a float, one product, half a packing;
// every block converts what it reads) come on top of those of the softmax, which bound the other cache's kernel.  So a
// block multiplies what it has converted with as many queries as its registers allow: 128 rows, of one head, or of two
// that share a key/value head, where the blocks fill the units.  2 x 4,096 tokens of 12 heads of 64: 108 us, 478 TFLOP/s
// (the other cache 85); 4,096 of 16 heads of 128 141 us, 487 TFLOP/s (64 rows: 184); 16 heads of 128 behind 5,000 keys,
// 962 tokens, 98 us, 415 TFLOP/s, by pairs of heads and 112 by one (the other cache 90).
//
// Where the blocks are fewer than the compute units, keys are cut into ranges, whose records a second launch joins: 512
// tokens of 12 heads behind 3,500 keys 29 us (the other cache, without ranges, 40), 64 of 8 heads of 128 behind 8,000
// 23.6 (117), 1,024 of 8 heads of 256 40 (48).
//
// Keys whose page the table does not name are masked, and values that are no number stay in their own dimensions: both
// are looked for by a bit to a block, and cost the blocks without any 0 to 3 % (2 x 1,024 tokens of 12 heads of 64 21.1 and
// 21.6 us, 4,096 of 16 heads of 128 level).
//
// Blocks of 64 rows: 8 waves, four along the keys, for heads of up to 128 (16 heads of 128: 4,096 tokens 180 us, of four
// waves, two along the keys, 258), but many blocks of smaller heads, whose four waves fit a unit more often (2 x 4,096 tokens of 12
// heads of 64 122 us), and heads beyond 128, whose accumulators take the registers of eight.
#include <math.h>

#include "common.h"
#include "pagedserve_hip.h"

#include "attention_prefill_block.h"

template <int NDB, int KS, int QW, int KR, int HP>
__global__ __launch_bounds__(64 * QW * KS) void attention_prefill_int4_kernel(
    const bf16_t* __restrict__ q, int64_t q_stride, const uint8_t* __restrict__ k_pool,
    const uint8_t* __restrict__ v_pool, bf16_t* __restrict__ out, int64_t out_stride,
    const int* __restrict__ tile_item, const int* __restrict__ tile_q0,
    const int* __restrict__ cu_tokens, const int* __restrict__ kv_lens,
    const int* __restrict__ tables, int table_width, int heads, int kv_heads, int page_size,
    int page_shift, int num_pages, float scale, int window, const AttnExtras extra, int ranges, float* sums,
    float* states) {
  __shared__ PrefillLds<NDB, KS, QW, KR> lds;
  attention_prefill_block<NDB, KS, QW, KR, Int4Pages, HP>(lds, blockIdx.x, blockIdx.y, q, q_stride, k_pool, v_pool, out,
                                                     out_stride, tile_item, tile_q0, cu_tokens, kv_lens, tables,
                                                     table_width, heads, kv_heads, page_size, page_shift,
                                                     num_pages, scale, window, extra,
                                                     PrefillRange{(int)blockIdx.z, ranges, sums, states});
}

// The records of a tile's queries joined: four dimensions of a query to a thread.
__global__ __launch_bounds__(256) void attention_prefill_int4_join_kernel(
    const float* __restrict__ sums, const float* __restrict__ states, bf16_t* __restrict__ out, int64_t out_stride,
    const int* __restrict__ tile_item, const int* __restrict__ tile_q0, const int* __restrict__ cu_tokens, int heads,
    int head_dim, int query_tile, int ranges) {
  const int head = blockIdx.x, item = tile_item[blockIdx.y], q0 = tile_q0[blockIdx.y];
  const int tok0 = cu_tokens[item] + q0, left = cu_tokens[item + 1] - tok0;
  const int rows = left < query_tile ? left : query_tile;
  const int quads = head_dim / 4, i = blockIdx.z * 256 + threadIdx.x;
  if (i >= rows * quads) return;
  const int row = i / quads, d = (i - row * quads) * 4;
  const int64_t first = ((int64_t)blockIdx.y * heads + head) * ranges * query_tile + row;
  float m = -INFINITY;
  for (int r = 0; r < ranges; ++r) m = fmaxf(m, states[(first + (int64_t)r * query_tile) * 2]);
  float total = 0.f, x[4] = {0.f, 0.f, 0.f, 0.f};
  for (int r = 0; r < ranges; ++r) {
    const int64_t record = first + (int64_t)r * query_tile;
    const float2 state = *reinterpret_cast<const float2*>(states + record * 2);
    const float4 v = *reinterpret_cast<const float4*>(sums + record * head_dim + d);
    // (a range without keys: a maximum of -inf, sums of 0; a maximum that is no number stays one in its sums)
    const float c = state.x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(state.x - m);
    total = fmaf(state.y, c, total);
    x[0] = fmaf(v.x, c, x[0]);
    x[1] = fmaf(v.y, c, x[1]);
    x[2] = fmaf(v.z, c, x[2]);
    x[3] = fmaf(v.w, c, x[3]);
  }
  const float inv = total == 0.f ? 0.f : 1.f / total;        // (a query that sees nothing: zeros)
  *reinterpret_cast<uint2*>(out + (tok0 + row) * out_stride + (int64_t)head * head_dim + d) =
      make_uint2(pack2_bf16(x[0] * inv, x[1] * inv), pack2_bf16(x[2] * inv, x[3] * inv));
}

extern "C" int ps_attention_prefill_int4(const void* q, int64_t q_stride, const void* k_pool, const void* v_pool,
                                         void* out, int64_t out_stride, const int* tile_item, const int* tile_q0,
                                         int tiles, const int* cu_tokens, const int* kv_lens, const int* tables,
                                         int table_width, int heads, int kv_heads, int head_dim,
                                         int page_size, int num_pages, float scale, int window, int max_kv_len,
                                         int query_tile, const float* sink, float softcap, int block_heads,
                                         int ranges, float* partial, int64_t partial_floats, void* stream) {
  const char* who = "ps_attention_prefill_int4";
  PS_REQUIRE(tiles >= 0 && heads > 0 && kv_heads > 0 && page_size > 0 && num_pages > 0 && table_width > 0,
             "%s: bad sizes", who);
  PS_REQUIRE(heads % kv_heads == 0, "%s: heads (%d) must be a multiple of kv_heads (%d)", who, heads, kv_heads);
  PS_REQUIRE(head_dim > 0 && head_dim % 16 == 0 && head_dim <= 256,
             "%s: head_dim %d must be a multiple of 16 up to 256", who, head_dim);
  PS_REQUIRE(page_size % 8 == 0 && page_size <= (1 << 20),
             "%s: pages of a cache in 4 bits hold a multiple of 8 keys, not %d", who, page_size);
  PS_REQUIRE(tiles <= 65535, "%s: too many tiles (%d)", who, tiles);
  PS_REQUIRE(query_tile == AP_QUERIES || (query_tile == AP_QUERIES * 2 && head_dim <= 128),
             "%s: tiles of %d or, head sizes up to 128, %d queries, not %d", who, AP_QUERIES, AP_QUERIES * 2, query_tile);
  PS_REQUIRE(block_heads == 1 || (block_heads == 2 && heads / kv_heads % 2 == 0 && query_tile == AP_QUERIES &&
                                  head_dim > 64 && head_dim <= 128),
             "%s: %d heads to a block (two of one key/value head, head sizes from 65 to 128, tiles of %d queries)", who,
             block_heads, AP_QUERIES);
  PS_REQUIRE((int64_t)num_pages * kv_heads * page_size < ((int64_t)1 << 32),
             "%s: a pool of %d pages x %d heads x %d keys has 2^32 key rows or more", who, num_pages, kv_heads, page_size);
  PS_REQUIRE(scale > 0.f, "%s: the score scale must be positive, got %g", who, scale);
  PS_REQUIRE(table_width <= AP_TABLE_MAX, "%s: block tables of %d pages exceed the %d that a tile keeps", who,
             table_width, AP_TABLE_MAX);
  PS_REQUIRE((q_stride % 8) == 0 && ((uintptr_t)q % 16) == 0 && (out_stride % 4) == 0 && ((uintptr_t)out % 8) == 0,
             "%s: q and out rows must allow 16- and 8-byte accesses", who);
  PS_REQUIRE(ranges >= 1 && ranges <= 64, "%s: 1 to 64 ranges of keys, not %d", who, ranges);
  const int64_t records = (int64_t)tiles * heads * ranges * query_tile;
  PS_REQUIRE(ranges == 1 || tiles == 0 ||
                 (partial != nullptr && (uintptr_t)partial % 16 == 0 && partial_floats >= records * (head_dim + 2)),
             "%s: %d ranges need %lld floats of scratch from a multiple of 16 bytes on, not %lld", who, ranges,
             (long long)(records * (head_dim + 2)), (long long)partial_floats);
  if (tiles == 0) return 0;
  int page_shift = -1;
  if ((page_size & (page_size - 1)) == 0) {
    page_shift = 0;
    while ((1 << page_shift) < page_size) ++page_shift;
  }
  hipStream_t s = (hipStream_t)stream;
  const AttnExtras extra = {sink, nullptr, 0, softcap, nullptr, 1.f};
  const dim3 grid(heads / block_heads, tiles, ranges);
  float* states = ranges > 1 ? partial + records * head_dim : nullptr;
  // head sizes up to 64: four waves along the keys where few blocks see many keys, as for the other cache
  const bool wide = (int64_t)tiles * heads * ranges <= ps_compute_units() * 2 && (max_kv_len <= 0 || max_kv_len >= 512);
#define PS_LAUNCH_P4(NDB, KS, QW, KR, HP)                                                                            \
  hipLaunchKernelGGL((attention_prefill_int4_kernel<NDB, KS, QW, KR, HP>), grid, dim3(64 * KS * QW), 0, s, (const bf16_t*)q, \
                     q_stride, (const uint8_t*)k_pool, (const uint8_t*)v_pool, (bf16_t*)out, out_stride,        \
                     tile_item, tile_q0, cu_tokens, kv_lens, tables, table_width, heads, kv_heads, page_size,   \
                     page_shift, num_pages, scale, window, extra, ranges, partial, states)
#define PS_TILES_P4(NDB)                                                   \
  case NDB:                                                                \
    if constexpr (NDB <= 4) {                                              \
      if (query_tile == AP_QUERIES * 2) PS_LAUNCH_P4(NDB, 1, 4, 2, 1);     \
      else if (wide) PS_LAUNCH_P4(NDB, 4, 2, 1, 1);                        \
      else PS_LAUNCH_P4(NDB, 2, 2, 1, 1);                                  \
    } else if constexpr (NDB <= 8) {                                       \
      if (query_tile == AP_QUERIES * 2) PS_LAUNCH_P4(NDB, 2, 4, 1, 1);     \
      else if (block_heads == 2) PS_LAUNCH_P4(NDB, 2, 4, 1, 2);            \
      else PS_LAUNCH_P4(NDB, 4, 2, 1, 1);                                  \
    } else {                                                               \
      PS_LAUNCH_P4(NDB, 2, 2, 1, 1);                                       \
    }                                                                      \
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
    default: PS_LAUNCH_P4(16, 2, 2, 1, 1);
  }
#undef PS_TILES_P4
#undef PS_LAUNCH_P4
  PS_CHECK_LAUNCH("ps_attention_prefill_int4");
  if (ranges > 1) {
    hipLaunchKernelGGL(attention_prefill_int4_join_kernel,
                       dim3(heads, tiles, (query_tile * (head_dim / 4) + 255) / 256), dim3(256), 0, s,
                       partial, states, (bf16_t*)out, out_stride, tile_item, tile_q0, cu_tokens, heads, head_dim, query_tile, ranges);
    PS_CHECK_LAUNCH("ps_attention_prefill_int4(join)");
  }
  return 0;
}
