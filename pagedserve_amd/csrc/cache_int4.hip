// The step's keys and values into their pages as 4-bit codes, and back (see cache_int4.h for the form).
//
// Four lanes share a row of a head: 8 dimensions of each of its G groups to a lane, which are 4 G bytes side by side in
// the page for keys and for values alike, so that a row comes by loads of 16 bytes and leaves by stores of 4 G.  The
// extremes over a group are two exchanges among the four lanes.  Keys and values are two halves of one grid.  Where there
// are many tokens a block of one wave takes 16 of them of one head: neighbouring tokens lie side by side in the page, and the lines
// of 128 bytes that they share are written by one compute unit.
//
// Of 2 x 1,024 tokens, 25 heads of 64, bfloat16: stored in 7.6 us (2.2 TB/s of all bytes), read back in 6.5 (2.6 TB/s); 8,192
// tokens, 8 heads of 128: 16.9 and 16.8 us; 8 tokens of 12 heads: 2.9 and 2.9.  What bounds it is the trip position ->
// block table -> page -> row, which all waves make at the same time.  (Blocks of two and four waves: the same within 3 %;
// with 16 lanes to a group, a byte each, 20 and 13.9 us, 47 and 35.)
#include <math.h>

#include "cache_int4.h"
#include "pagedserve_hip.h"

// Where a token's row lies: its page and its place there, or page -1 where the block table has none.
struct Int4Place {
  int page, within;
};
__device__ inline Int4Place int4_place(const int* __restrict__ tok_item, const int* __restrict__ tok_pos,
                                       const int* __restrict__ tables, int table_width, int t, int page_size,
                                       int num_pages) {
  const int pos = tok_pos[t];
  const int* table = tables + (int64_t)tok_item[t] * table_width;
  const int logical = pos / page_size;
  if (pos < 0 || logical >= table_width) return {-1, 0};
  const int page = table[logical];
  return {page >= 0 && page < num_pages ? page : -1, pos - logical * page_size};
}

// A row's 8 dimensions from d0 on as numbers, zeros behind the last; WIDE: by loads of 16 bytes.
template <bool WIDE, typename T>
__device__ inline void int4_load8(const T* __restrict__ row, int d0, int head_dim, float* x) {
  // (every load is made, from the row's last dimensions where there are none: one in a branch is waited for in it)
  const bool inside = d0 < head_dim;
  if constexpr (WIDE && sizeof(T) == 2) {
    const uint4 raw = *reinterpret_cast<const uint4*>(row + (inside ? d0 : head_dim - 8));
    const uint32_t words[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = __uint_as_float(inside ? words[i] << 16 : 0u);
      x[2 * i + 1] = __uint_as_float(inside ? words[i] & 0xffff0000u : 0u);
    }
  } else if constexpr (WIDE) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float4 part = *reinterpret_cast<const float4*>(row + (inside ? d0 : head_dim - 8) + 4 * i);
      x[4 * i] = inside ? part.x : 0.f;
      x[4 * i + 1] = inside ? part.y : 0.f;
      x[4 * i + 2] = inside ? part.z : 0.f;
      x[4 * i + 3] = inside ? part.w : 0.f;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float value = to_float(row[d0 + i < head_dim ? d0 + i : head_dim - 1]);
      x[i] = d0 + i < head_dim ? value : 0.f;
    }
  }
}

template <bool WIDE, typename T>
__device__ inline void int4_store8(T* __restrict__ row, int d0, int head_dim, const float* x) {
  if constexpr (WIDE) {
    if (d0 >= head_dim) return;
    if constexpr (sizeof(T) == 2) {
      *reinterpret_cast<uint4*>(row + d0) =
          make_uint4(pack2_bf16(x[0], x[1]), pack2_bf16(x[2], x[3]), pack2_bf16(x[4], x[5]), pack2_bf16(x[6], x[7]));
    } else {
      *reinterpret_cast<float4*>(row + d0) = make_float4(x[0], x[1], x[2], x[3]);
      *reinterpret_cast<float4*>(row + d0 + 4) = make_float4(x[4], x[5], x[6], x[7]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (d0 + i < head_dim) row[d0 + i] = from_float<T>(x[i]);
  }
}

// The token and head of four lanes: 2^token_shift tokens by 16 >> token_shift heads to a block.
__device__ inline void int4_row_of(int token_shift, int& t, int& head) {
  const int local = threadIdx.x >> 2;
  t = (blockIdx.x << token_shift) + (local & ((1 << token_shift) - 1));
  head = blockIdx.y * (16 >> token_shift) + (local >> token_shift);
}

template <typename T, int G, bool WIDE>
__global__ __launch_bounds__(64) void kv_write_int4_kernel(
    const T* __restrict__ k, const T* __restrict__ v, int64_t k_stride, int64_t v_stride,
    uint8_t* __restrict__ k_pool, uint8_t* __restrict__ v_pool, const int* __restrict__ tok_item,
    const int* __restrict__ tok_pos, const int* __restrict__ tables, int table_width, int tokens, int kv_heads,
    int head_dim, int page_size, int num_pages, int token_shift) {
  const bool values = blockIdx.z != 0;
  const int c = threadIdx.x & 3;
  int t, head;
  int4_row_of(token_shift, t, head);
  if (t >= tokens || head >= kv_heads) return;               // (whole groups of four lanes)
  const T* row = (values ? v + t * v_stride : k + t * k_stride) + (int64_t)head * head_dim;
  float x[G][8];
#pragma unroll
  for (int g = 0; g < G; ++g) int4_load8<WIDE>(row, g * PS_INT4_GROUP + 8 * c, head_dim, x[g]);
  const Int4Place place = int4_place(tok_item, tok_pos, tables, table_width, t, page_size, num_pages);
  if (place.page < 0) return;
  uint32_t words[G], steps[(G + 1) / 2];
  int4_code_row<G, sizeof(T) == 2>(x, values, words, steps);
  uint8_t* page = (values ? v_pool : k_pool) + int4_page_at(place.page, kv_heads, head, page_size, G);
  int4_store_row<G>(page, page_size, place.within, c, words, steps);
}

template <typename T, int G, bool WIDE>
__global__ __launch_bounds__(64) void kv_read_int4_kernel(
    const uint8_t* __restrict__ k_pool, const uint8_t* __restrict__ v_pool, T* __restrict__ k, T* __restrict__ v,
    int64_t k_stride, int64_t v_stride, const int* __restrict__ tok_item, const int* __restrict__ tok_pos,
    const int* __restrict__ tables, int table_width, int tokens, int kv_heads, int head_dim, int page_size,
    int num_pages, int token_shift) {
  const bool values = blockIdx.z != 0;
  const int c = threadIdx.x & 3;
  int t, head;
  int4_row_of(token_shift, t, head);
  if (t >= tokens || head >= kv_heads) return;
  const Int4Place place = int4_place(tok_item, tok_pos, tables, table_width, t, page_size, num_pages);
  if (place.page < 0) return;
  const uint8_t* page = (values ? v_pool : k_pool) + int4_page_at(place.page, kv_heads, head, page_size, G);
  uint32_t words[G], steps[(G + 1) / 2];
  int4_load_words<G>(page + place.within * (16 * G) + c * (4 * G), words);
  const uint8_t* from = page + page_size * (16 * G) + place.within * (2 * G);
  if constexpr (G % 2 == 0) {
    int4_load_words<G / 2>(from, steps);
  } else {
#pragma unroll
    for (int g = 0; g < G; ++g) {
      const uint32_t bits = reinterpret_cast<const uint16_t*>(from)[g];
      steps[g / 2] = g % 2 ? steps[g / 2] | bits << 16 : bits;
    }
  }
  if (values) int4_turn_bytes<G, true>(words);
  T* row = (values ? v + t * v_stride : k + t * k_stride) + (int64_t)head * head_dim;
#pragma unroll
  for (int g = 0; g < G; ++g) {
    const float step = __uint_as_float(steps[g / 2] >> (16 * (g % 2)) << 16);
    float x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = (float)((int)(words[g] >> (4 * i) & 15u) - 8) * step;
    int4_store8<WIDE>(row, g * PS_INT4_GROUP + 8 * c, head_dim, x);
  }
}

static int check_int4_rows(const char* who, int64_t k_stride, int64_t v_stride, int table_width, int tokens,
                           int kv_heads, int head_dim, int page_size, int num_pages, int dtype) {
  PS_REQUIRE(tokens >= 0 && kv_heads > 0 && page_size > 0 && num_pages > 0 && table_width > 0, "%s: bad sizes", who);
  PS_REQUIRE(head_dim > 0 && head_dim <= 256, "%s: head_dim %d must lie in 1..256", who, head_dim);
  PS_REQUIRE(page_size % 8 == 0, "%s: pages of a cache in 4 bits hold a multiple of 8 keys, not %d", who, page_size);
  PS_REQUIRE(page_size <= (1 << 20), "%s: pages of %d keys are too large", who, page_size);
  PS_REQUIRE(kv_heads <= 65535, "%s: too many heads (%d)", who, kv_heads);
  PS_REQUIRE(k_stride >= (int64_t)kv_heads * head_dim && v_stride >= (int64_t)kv_heads * head_dim,
             "%s: row stride too small", who);
  PS_REQUIRE(dtype == PS_F32 || dtype == PS_BF16, "%s: unknown dtype %d", who, dtype);
  return 0;
}

// Whether rows allow accesses of 16 bytes.
static bool int4_wide(const void* k, const void* v, int64_t k_stride, int64_t v_stride, int head_dim, int dtype) {
  const int64_t lane = dtype == PS_F32 ? 4 : 8;
  return head_dim % 8 == 0 && k_stride % lane == 0 && v_stride % lane == 0 && ((uintptr_t)k | (uintptr_t)v) % 16 == 0;
}
// Tokens of a block, as a power of two.
static int int4_token_shift(int tokens) { return tokens >= 64 ? 4 : 0; }

#define PS_OF_WIDTH(LAUNCH, T, G)  \
  if (wide) LAUNCH(T, G, true);    \
  else LAUNCH(T, G, false);        \
  break
#define PS_OF_GROUPS(LAUNCH, T)               \
  switch (int4_groups(head_dim)) {            \
    case 1: PS_OF_WIDTH(LAUNCH, T, 1);        \
    case 2: PS_OF_WIDTH(LAUNCH, T, 2);        \
    case 3: PS_OF_WIDTH(LAUNCH, T, 3);        \
    case 4: PS_OF_WIDTH(LAUNCH, T, 4);        \
    case 5: PS_OF_WIDTH(LAUNCH, T, 5);        \
    case 6: PS_OF_WIDTH(LAUNCH, T, 6);        \
    case 7: PS_OF_WIDTH(LAUNCH, T, 7);        \
    default: PS_OF_WIDTH(LAUNCH, T, 8);       \
  }

extern "C" int ps_kv_write_int4(const void* k, const void* v, int64_t k_stride, int64_t v_stride, void* k_pool,
                                void* v_pool, const int* tok_item, const int* tok_pos, const int* tables,
                                int table_width, int tokens, int kv_heads, int head_dim, int page_size,
                                int num_pages, int dtype, void* stream) {
  if (check_int4_rows("ps_kv_write_int4", k_stride, v_stride, table_width, tokens, kv_heads, head_dim, page_size,
                      num_pages, dtype))
    return 1;
  PS_REQUIRE(((uintptr_t)k_pool | (uintptr_t)v_pool) % 16 == 0, "%s: pools must begin at multiples of 16 bytes", "ps_kv_write_int4");
  if (tokens == 0) return 0;
  const bool wide = int4_wide(k, v, k_stride, v_stride, head_dim, dtype);
  const int shift = int4_token_shift(tokens), per_block = 16 >> shift;
  const dim3 grid((tokens + (1 << shift) - 1) >> shift, (kv_heads + per_block - 1) / per_block, 2);
  hipStream_t s = (hipStream_t)stream;
#define PS_LAUNCH_W4(T, G, WIDE)                                                                                          \
  hipLaunchKernelGGL((kv_write_int4_kernel<T, G, WIDE>), grid, dim3(64), 0, s, (const T*)k, (const T*)v, k_stride, v_stride, \
                     (uint8_t*)k_pool, (uint8_t*)v_pool, tok_item, tok_pos, tables, table_width, tokens, kv_heads, \
                     head_dim, page_size, num_pages, shift)
  if (dtype == PS_F32) {
    PS_OF_GROUPS(PS_LAUNCH_W4, float)
  } else {
    PS_OF_GROUPS(PS_LAUNCH_W4, bf16_t)
  }
#undef PS_LAUNCH_W4
  PS_CHECK_LAUNCH("ps_kv_write_int4");
  return 0;
}

extern "C" int ps_kv_read_int4(const void* k_pool, const void* v_pool, void* k, void* v, int64_t k_stride,
                               int64_t v_stride, const int* tok_item, const int* tok_pos, const int* tables,
                               int table_width, int tokens, int kv_heads, int head_dim, int page_size, int num_pages,
                               int dtype, void* stream) {
  if (check_int4_rows("ps_kv_read_int4", k_stride, v_stride, table_width, tokens, kv_heads, head_dim, page_size,
                      num_pages, dtype))
    return 1;
  PS_REQUIRE(((uintptr_t)k_pool | (uintptr_t)v_pool) % 16 == 0, "%s: pools must begin at multiples of 16 bytes", "ps_kv_read_int4");
  if (tokens == 0) return 0;
  const bool wide = int4_wide(k, v, k_stride, v_stride, head_dim, dtype);
  const int shift = int4_token_shift(tokens), per_block = 16 >> shift;
  const dim3 grid((tokens + (1 << shift) - 1) >> shift, (kv_heads + per_block - 1) / per_block, 2);
  hipStream_t s = (hipStream_t)stream;
#define PS_LAUNCH_R4(T, G, WIDE)                                                                                        \
  hipLaunchKernelGGL((kv_read_int4_kernel<T, G, WIDE>), grid, dim3(64), 0, s, (const uint8_t*)k_pool, (const uint8_t*)v_pool, \
                     (T*)k, (T*)v, k_stride, v_stride, tok_item, tok_pos, tables, table_width, tokens, kv_heads,   \
                     head_dim, page_size, num_pages, shift)
  if (dtype == PS_F32) {
    PS_OF_GROUPS(PS_LAUNCH_R4, float)
  } else {
    PS_OF_GROUPS(PS_LAUNCH_R4, bf16_t)
  }
#undef PS_LAUNCH_R4
  PS_CHECK_LAUNCH("ps_kv_read_int4");
  return 0;
}
