// Attention of single tokens over a cache in 4 bits (see cache_int4.h for its form).
//
// One block per (token, head, range of keys), four waves.  LPK lanes share a key: a lane holds eight dimensions of the
// query and takes one 32-bit word of the key's codes, the step of its group and four bytes of the value's codes.  A group's
// step is a factor of the whole partial sum, so a product costs a conversion of the code and one multiply-add.  Every
// group of lanes keeps a softmax state of its own (running maximum in units of log 2, sum and accumulators in
// float), merged at the end over the wave and the block; ranges leave records that a second launch merges.
#include <math.h>

#include "attention_decode_block.h"
#include "cache_int4.h"
#include "pagedserve_hip.h"

struct Int4Lds {
  __attribute__((aligned(16))) float acc[4][256];
  float ml[4][2];
};

template <typename T, int LPK>
__global__ __launch_bounds__(256) void attention_decode_int4_kernel(
    const T* __restrict__ q, int64_t q_stride, const uint8_t* __restrict__ k_pool,
    const uint8_t* __restrict__ v_pool, T* __restrict__ out, int64_t out_stride, float* __restrict__ partial,
    const int* __restrict__ tok_list, const int* __restrict__ tok_item, const int* __restrict__ tok_pos,
    const int* __restrict__ tables, int table_width, int heads, int kv_heads, int head_dim, int page_size,
    int num_pages, float scale_log2, int window, int splits, const float* __restrict__ sink, float softcap) {
  constexpr int KEYS = 64 / LPK;      // keys of one load of a wave
  constexpr int UNROLL = 4;
  constexpr int TURN = 4 * KEYS * UNROLL;
  __shared__ Int4Lds lds;
  const int n = blockIdx.x, head = blockIdx.y, split = blockIdx.z;
  const int t = tok_list ? tok_list[n] : n;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int group = lane / LPK;
  const int groups = int4_groups(head_dim);
  const int kv_head = head / (heads / kv_heads);
  const int pos = tok_pos[t];
  const int* table = tables + (int64_t)(tok_item ? tok_item[t] : t) * table_width;
  // the lane's dimensions: word w of the key
  const int w = lane % LPK;
  const bool has_word = w < 4 * groups;
  const int word = has_word ? w : 0;
  const int key_at = int4_key_word(word, groups);
  float query[8];
  float query_sum = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int d = 8 * w + i;
    query[i] = d < head_dim ? to_float(q[t * q_stride + (int64_t)head * head_dim + d]) : 0.f;
    query_sum += query[i];
  }

  // (a token in front of its context sees nothing, and reads no entry of the table)
  const int first = pos < 0 ? 0 : first_visible_key(pos, window);
  int end = pos + 1;
  if (end > (int64_t)table_width * page_size) end = table_width * page_size;
  int begin = first;
  if (splits > 1) {
    const int chunk = ((end - first + splits - 1) / splits + TURN - 1) / TURN * TURN;
    begin = first + split * chunk;
    if (begin + chunk < end) end = begin + chunk;
  }

  float m = -INFINITY, l = 0.f;
  float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  if (sink != nullptr && split == 0 && wave == 0 && group == 0) {
    m = sink[head] * 1.4426950408889634f;     // a score without key or value starts one state
    l = 1.f;
  }
  for (int base = begin + wave * KEYS * UNROLL; base < end; base += TURN) {
    uint32_t codes[UNROLL], value[UNROLL][4], k_step[UNROLL], v_step[UNROLL];
    bool valid[UNROLL];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      const int key = base + u * KEYS + group;
      const int safe = key < end ? key : end - 1;
      const int logical = safe / page_size;
      const int page = table[logical];
      valid[u] = key < end && page >= 0 && page < num_pages;
      // (a place that exists, whatever the key: what is loaded from it counts only where the key is valid)
      const int within = safe - logical * page_size;
      const int64_t at = int4_page_at(valid[u] ? page : 0, kv_heads, kv_head, page_size, groups);
      const uint8_t* kp = k_pool + at;
      const uint8_t* vp = v_pool + at;
      const int row = within * 16 * groups;
      const int steps = page_size * 16 * groups + 2 * (within * groups + (word >> 2));
      codes[u] = *reinterpret_cast<const uint32_t*>(kp + row + key_at);
      k_step[u] = *reinterpret_cast<const uint16_t*>(kp + steps);
#pragma unroll
      for (int b = 0; b < 4; ++b) value[u][b] = vp[row + int4_value_byte(4 * word + b, groups)];
      v_step[u] = *reinterpret_cast<const uint16_t*>(vp + steps);
    }
    float s[UNROLL];
    float m_new = m;
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      float dot = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) dot = fmaf(query[i], (float)((int)(codes[u] >> (4 * i) & 15) - 8), dot);
      dot = has_word ? dot * __uint_as_float(k_step[u] << 16) : 0.f;
      dot = lanes_sum<(LPK <= 16 ? LPK : 16)>(dot);
      if (LPK > 16) dot += __shfl_xor(dot, 16, 64);
      float score = dot * scale_log2;
      if (softcap > 0.f) score = capped_score_as<T>(score, softcap * 1.4426950408889634f);
      // (a maximum passes over a NaN: infinity makes as much of the sums)
      s[u] = valid[u] ? (score == score ? score : INFINITY) : -INFINITY;
      m_new = fmaxf(m_new, s[u]);
    }
    if (m_new != -INFINITY) {
      const float correction = m == -INFINITY ? 0.f : exp2_fast<T>(m - m_new);
      l *= correction;
#pragma unroll
      for (int i = 0; i < 8; ++i) acc[i] *= correction;
#pragma unroll
      for (int u = 0; u < UNROLL; ++u) {
        const float p = exp2_fast<T>(s[u] - m_new);
        l += p;
        // (a masked key's step may be anything, also NaN)
        const float weight = valid[u] ? p * __uint_as_float(v_step[u] << 16) : 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i)
          acc[i] = fmaf(weight, (float)((int)(value[u][i >> 1] >> (4 * (i & 1)) & 15) - 8), acc[i]);
      }
      m = m_new;
    }
  }
  const float wave_m = groups_max<LPK>(m);
  const float share = m == -INFINITY ? 0.f : exp2_fast<T>(m - wave_m);
  l = groups_sum<LPK>(l * share);
#pragma unroll
  for (int i = 0; i < 8; ++i) acc[i] = groups_sum<LPK>(acc[i] * share);
  if (group == 0 && has_word) {
#pragma unroll
    for (int i = 0; i < 8; ++i) lds.acc[wave][8 * w + i] = acc[i];
  }
  if (lane == 0) {
    lds.ml[wave][0] = wave_m;
    lds.ml[wave][1] = l;
  }
  __syncthreads();
  const int d = threadIdx.x;
  if (d >= head_dim) return;
  float block_m = -INFINITY;
#pragma unroll
  for (int i = 0; i < 4; ++i) block_m = fmaxf(block_m, lds.ml[i][0]);
  float sum = 0.f, total = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float m_i = lds.ml[i][0];
    const float c = m_i == -INFINITY ? 0.f : exp2_fast<T>(m_i - block_m);
    total += lds.ml[i][1] * c;
    sum += lds.acc[i][d] * c;
  }
  if (splits == 1) {
    // (a token that sees nothing: zeros)
    out[t * out_stride + (int64_t)head * head_dim + d] = from_float<T>(total == 0.f ? 0.f : sum / total);
    return;
  }
  float* record = partial + (((int64_t)n * heads + head) * splits + split) * (head_dim + 2);
  record[d] = sum;
  if (d == 0) {
    record[head_dim] = block_m;
    record[head_dim + 1] = total;
  }
}

// The records of a token's ranges joined: a block per (token, head), a thread per dimension.
template <typename T>
__global__ __launch_bounds__(256) void attention_decode_int4_merge_kernel(const float* __restrict__ partial,
                                                                          const int* __restrict__ tok_list, int heads,
                                                                          int head_dim, int splits,
                                                                          T* __restrict__ out, int64_t out_stride) {
  const int n = blockIdx.x, head = blockIdx.y, d = threadIdx.x;
  const int stride = head_dim + 2;
  const float* records = partial + ((int64_t)n * heads + head) * splits * stride;
  float m = -INFINITY;
  for (int s = 0; s < splits; ++s) m = fmaxf(m, records[s * stride + head_dim]);
  float sum = 0.f, total = 0.f;
  for (int s = 0; s < splits; ++s) {
    const float m_s = records[s * stride + head_dim];
    const float c = m_s == -INFINITY ? 0.f : exp2_fast<T>(m_s - m);
    total += records[s * stride + head_dim + 1] * c;
    if (d < head_dim) sum += records[s * stride + d] * c;
  }
  const int t = tok_list ? tok_list[n] : n;
  if (d < head_dim)
    out[t * out_stride + (int64_t)head * head_dim + d] = from_float<T>(total == 0.f ? 0.f : sum / total);
}

extern "C" int ps_attention_decode_int4(const void* q, int64_t q_stride, const void* k_pool, const void* v_pool,
                                        void* out, int64_t out_stride, float* partial, int64_t partial_floats,
                                        const int* tok_list, const int* tok_item, const int* tok_pos,
                                        const int* tables, int table_width, int count, int heads, int kv_heads,
                                        int head_dim, int page_size, int num_pages, float scale, int window,
                                        int splits, const float* sink, float softcap, int dtype, void* stream) {
  PS_REQUIRE(count >= 0 && heads > 0 && kv_heads > 0 && page_size > 0 && num_pages > 0 && table_width > 0,
             "ps_attention_decode_int4: bad sizes");
  PS_REQUIRE(heads % kv_heads == 0 && heads <= 65535,
             "ps_attention_decode_int4: heads (%d) must be a multiple of kv_heads (%d), 65535 at most", heads, kv_heads);
  PS_REQUIRE(head_dim > 0 && head_dim <= 256, "ps_attention_decode_int4: head_dim %d must lie in 1..256", head_dim);
  PS_REQUIRE(page_size % 8 == 0 && page_size <= (1 << 20),
             "ps_attention_decode_int4: pages of a cache in 4 bits hold a multiple of 8 keys, not %d", page_size);
  PS_REQUIRE((int64_t)table_width * page_size < ((int64_t)1 << 31),
             "ps_attention_decode_int4: block tables of %d pages of %d keys", table_width, page_size);
  PS_REQUIRE(splits >= 1 && splits <= 64, "ps_attention_decode_int4: 1 to 64 ranges, not %d", splits);
  PS_REQUIRE(dtype == PS_F32 || dtype == PS_BF16, "ps_attention_decode_int4: unknown dtype %d", dtype);
  PS_REQUIRE(splits == 1 || (partial != nullptr &&
                             partial_floats >= (int64_t)count * heads * splits * (head_dim + 2)),
             "ps_attention_decode_int4: %lld floats of scratch are too few for %d ranges", (long long)partial_floats,
             splits);
  if (count == 0) return 0;
  hipStream_t s = (hipStream_t)stream;
  const dim3 grid(count, heads, splits);
#define PS_LAUNCH_D4(T, LPK)                                                                                        \
  hipLaunchKernelGGL((attention_decode_int4_kernel<T, LPK>), grid, dim3(256), 0, s, (const T*)q, q_stride,          \
                     (const uint8_t*)k_pool, (const uint8_t*)v_pool, (T*)out, out_stride, partial, tok_list, tok_item, \
                     tok_pos, tables, table_width, heads, kv_heads, head_dim, page_size, num_pages,                 \
                     scale * 1.4426950408889634f, window, splits, sink, softcap)
#define PS_LAUNCH_D4T(T)                      \
  do {                                        \
    if (head_dim <= 32) PS_LAUNCH_D4(T, 4);   \
    else if (head_dim <= 64) PS_LAUNCH_D4(T, 8);   \
    else if (head_dim <= 128) PS_LAUNCH_D4(T, 16); \
    else PS_LAUNCH_D4(T, 32);                 \
  } while (0)
  if (dtype == PS_F32) PS_LAUNCH_D4T(float);
  else PS_LAUNCH_D4T(bf16_t);
#undef PS_LAUNCH_D4T
#undef PS_LAUNCH_D4
  PS_CHECK_LAUNCH("ps_attention_decode_int4");
  if (splits > 1) {
    if (dtype == PS_F32)
      hipLaunchKernelGGL(attention_decode_int4_merge_kernel<float>, dim3(count, heads), dim3(256), 0, s, partial,
                         tok_list, heads, head_dim, splits, (float*)out, out_stride);
    else
      hipLaunchKernelGGL(attention_decode_int4_merge_kernel<bf16_t>, dim3(count, heads), dim3(256), 0, s, partial,
                         tok_list, heads, head_dim, splits, (bf16_t*)out, out_stride);
    PS_CHECK_LAUNCH("ps_attention_decode_int4(merge)");
  }
  return 0;
}
