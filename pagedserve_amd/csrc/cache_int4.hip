// The step's keys and values into their pages as 4-bit codes, and back (see cache_int4.h for the form).
//
// 16 lanes take one group of one head of one token: two neighbouring dimensions to a lane, which are one
// byte of the page, and the extremes over the group are four exchanges within a row of lanes.  Keys and values are two
// halves of one grid.  What bounds both is the trip: position -> block table -> page.
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

template <typename T>
__global__ __launch_bounds__(256) void kv_write_int4_kernel(
    const T* __restrict__ k, const T* __restrict__ v, int64_t k_stride, int64_t v_stride,
    uint8_t* __restrict__ k_pool, uint8_t* __restrict__ v_pool, const int* __restrict__ tok_item,
    const int* __restrict__ tok_pos, const int* __restrict__ tables, int table_width, int kv_heads, int head_dim,
    int groups, int page_size, int num_pages) {
  const int t = blockIdx.x;
  const bool values = blockIdx.z != 0;
  const int unit = blockIdx.y * 16 + threadIdx.x / 16;      // which group of which head
  const int n = threadIdx.x & 15;
  if (unit >= kv_heads * groups) return;                     // (whole rows of lanes)
  const int head = unit / groups, g = unit - head * groups;
  const Int4Place place = int4_place(tok_item, tok_pos, tables, table_width, t, page_size, num_pages);
  if (place.page < 0) return;
  const T* row = (values ? v + t * v_stride : k + t * k_stride) + (int64_t)head * head_dim;
  const int d0 = g * PS_INT4_GROUP + 2 * n;
  const float a = d0 < head_dim ? to_float(row[d0]) : 0.f;
  const float b = d0 + 1 < head_dim ? to_float(row[d0 + 1]) : 0.f;
  const float high = lanes_max<16>(fmaxf(a, b));
  const float low = -lanes_max<16>(fmaxf(-a, -b));
  // (a maximum passes over a NaN: what is not finite is counted apart)
  const bool finite = fabsf(a) < INFINITY && fabsf(b) < INFINITY;
  const bool all_finite = lanes_max<16>(finite ? 0.f : 1.f) == 0.f;
  const float step = all_finite ? int4_step(high, low) : __uint_as_float(0x7fc00000u);
  int codes = 0x88;
  if (all_finite && step != 0.f) codes = int4_code(a, step) | int4_code(b, step) << 4;
  uint8_t* page = (values ? v_pool : k_pool) + int4_page_at(place.page, kv_heads, head, page_size, groups);
  const int at = values ? int4_value_byte(16 * g + n, groups) : int4_key_word(4 * g + (n >> 2), groups) + (n & 3);
  page[place.within * 16 * groups + at] = (uint8_t)codes;
  if (n == 0)
    reinterpret_cast<uint16_t*>(page + page_size * 16 * groups)[place.within * groups + g] =
        (uint16_t)(__float_as_uint(step) >> 16);
}

template <typename T>
__global__ __launch_bounds__(256) void kv_read_int4_kernel(
    const uint8_t* __restrict__ k_pool, const uint8_t* __restrict__ v_pool, T* __restrict__ k, T* __restrict__ v,
    int64_t k_stride, int64_t v_stride, const int* __restrict__ tok_item, const int* __restrict__ tok_pos,
    const int* __restrict__ tables, int table_width, int kv_heads, int head_dim, int groups, int page_size,
    int num_pages) {
  const int t = blockIdx.x;
  const bool values = blockIdx.z != 0;
  const int unit = blockIdx.y * 16 + threadIdx.x / 16;
  const int n = threadIdx.x & 15;
  if (unit >= kv_heads * groups) return;
  const int head = unit / groups, g = unit - head * groups;
  const Int4Place place = int4_place(tok_item, tok_pos, tables, table_width, t, page_size, num_pages);
  if (place.page < 0) return;
  const uint8_t* page = (values ? v_pool : k_pool) + int4_page_at(place.page, kv_heads, head, page_size, groups);
  const int at = values ? int4_value_byte(16 * g + n, groups) : int4_key_word(4 * g + (n >> 2), groups) + (n & 3);
  const int codes = page[place.within * 16 * groups + at];
  const uint32_t bits =
      reinterpret_cast<const uint16_t*>(page + page_size * 16 * groups)[place.within * groups + g];
  const float step = __uint_as_float(bits << 16);
  T* row = (values ? v + t * v_stride : k + t * k_stride) + (int64_t)head * head_dim;
  const int d0 = g * PS_INT4_GROUP + 2 * n;
  if (d0 < head_dim) row[d0] = from_float<T>((float)((codes & 15) - 8) * step);
  if (d0 + 1 < head_dim) row[d0 + 1] = from_float<T>((float)((codes >> 4) - 8) * step);
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

extern "C" int ps_kv_write_int4(const void* k, const void* v, int64_t k_stride, int64_t v_stride, void* k_pool,
                                void* v_pool, const int* tok_item, const int* tok_pos, const int* tables,
                                int table_width, int tokens, int kv_heads, int head_dim, int page_size,
                                int num_pages, int dtype, void* stream) {
  if (check_int4_rows("ps_kv_write_int4", k_stride, v_stride, table_width, tokens, kv_heads, head_dim, page_size,
                      num_pages, dtype))
    return 1;
  if (tokens == 0) return 0;
  const int groups = int4_groups(head_dim);
  const dim3 grid(tokens, (kv_heads * groups + 15) / 16, 2);
  hipStream_t s = (hipStream_t)stream;
#define PS_LAUNCH_W4(T)                                                                                         \
  hipLaunchKernelGGL(kv_write_int4_kernel<T>, grid, dim3(256), 0, s, (const T*)k, (const T*)v, k_stride, v_stride, \
                     (uint8_t*)k_pool, (uint8_t*)v_pool, tok_item, tok_pos, tables, table_width, kv_heads, head_dim, \
                     groups, page_size, num_pages)
  if (dtype == PS_F32) PS_LAUNCH_W4(float);
  else PS_LAUNCH_W4(bf16_t);
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
  if (tokens == 0) return 0;
  const int groups = int4_groups(head_dim);
  const dim3 grid(tokens, (kv_heads * groups + 15) / 16, 2);
  hipStream_t s = (hipStream_t)stream;
#define PS_LAUNCH_R4(T)                                                                                     \
  hipLaunchKernelGGL(kv_read_int4_kernel<T>, grid, dim3(256), 0, s, (const uint8_t*)k_pool, (const uint8_t*)v_pool, \
                     (T*)k, (T*)v, k_stride, v_stride, tok_item, tok_pos, tables, table_width, kv_heads, head_dim, \
                     groups, page_size, num_pages)
  if (dtype == PS_F32) PS_LAUNCH_R4(float);
  else PS_LAUNCH_R4(bf16_t);
#undef PS_LAUNCH_R4
  PS_CHECK_LAUNCH("ps_kv_read_int4");
  return 0;
}
