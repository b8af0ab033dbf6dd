// Attention of single tokens over a cache in 4 bits (see cache_int4.h for its form).
//
// bfloat16 queries run on the matrix cores.  A block takes a token, up to 16 heads that share a key/value head, and a range
// of keys; a wave takes 32 keys at a time, with a softmax state of its own, and nothing passes through LDS before the waves'
// states meet at the end:
//
//   scores   S[key][head] = K Q^T, v_mfma_f32_16x16x32_bf16 twice for 16 keys each, a product per group of 32 dimensions.
//            A lane holds 8 dimensions of one key: one word of its codes.  Shifted and joined to the bits of 16.0 a code
//            is the bfloat16 number 16 + code, two of them with two instructions; that is 24 more than it stands for, and
//            the sum starts from -24 times the sum of the group's queries.  The group's step multiplies the sum, in
//            float: the codes themselves never become scaled values, and nothing is rounded.
//   softmax  a lane has the scores of 8 keys of one head.  The reference of the exponentials is raised only where a
//            score passes it by more than 2^8, so that most tiles need no exchange between lanes and no rescaling.
//   values   O^T[dimension][head] = V^T P^T over the 32 keys, which are the lane's own 8 and those of three others: no
//            exchange here either.  The weights are multiplied by the group's step before they are rounded to bfloat16 (2^-9 of
//            each on average); the codes are 16 + code again, and a product of ones with the same weights gives what
//            is to be taken off, 24 times, at the end.
//
// Bound by memory where there are blocks enough (4.5 bits a value), else by the trip block table -> codes: a tile's codes
// are asked for a tile ahead, its table entries, which are the same for a wave and come through the scalar unit, two.
//
// float queries, and scales that are not positive, take the kernel on the vector unit: LPK lanes share a key, a lane holds
// eight dimensions of the query and takes one word of the key's codes; a conversion of the code and a multiply-add to a
// product, all in float.
#include <math.h>

#include "attention_decode_block.h"
#include "cache_int4.h"
#include "pagedserve_hip.h"

typedef __attribute__((__vector_size__(8 * sizeof(__bf16)))) __bf16 int4_bf16x8;
typedef float int4_f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t int4_u32x4 __attribute__((ext_vector_type(4)));

#define I4_TILE 32           // keys of a wave at a time
#define I4_HEADS 16          // heads of a block, at most
#define I4_OFFSET 24.f       // what a code is held as, less what it stands for
#define I4_SLACK 8.f         // how far (in units of log 2) a score may pass the exponentials' reference

// Words of W consecutive bytes (a power of two) at a multiple of W.
template <int W>
__device__ inline void int4_load(const uint8_t* p, uint32_t* words) {
  if constexpr (W == 1) words[0] = *p;
  else if constexpr (W == 2) words[0] = *reinterpret_cast<const uint16_t*>(p);
  else if constexpr (W == 4) words[0] = *reinterpret_cast<const uint32_t*>(p);
  else if constexpr (W == 8) {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    words[0] = v.x;
    words[1] = v.y;
  } else {
#pragma unroll
    for (int i = 0; i < W / 16; ++i) {
      const uint4 v = *reinterpret_cast<const uint4*>(p + 16 * i);
      words[4 * i] = v.x;
      words[4 * i + 1] = v.y;
      words[4 * i + 2] = v.z;
      words[4 * i + 3] = v.w;
    }
  }
}
// The largest power of two that divides n, 16 at most.
constexpr int int4_piece(int n) { return n % 16 == 0 ? 16 : n % 8 == 0 ? 8 : n % 4 == 0 ? 4 : n % 2 == 0 ? 2 : 1; }

// Nibbles i and i + 4 of a word as the bfloat16 numbers 16 + nibble, in the low and the high half.
template <int I>
__device__ inline uint32_t int4_pair(uint32_t word) {
  const uint32_t at = I == 0 ? word << 3 : word >> (4 * I - 3);
  return (at & 0x00780078u) | 0x41804180u;
}

// What a wave loads of 32 keys.  Lane (16 c + n): keys n and 16 + n, words c G ..; of keys 4 c .. + 3 and 16 + 4 c .. + 3 their
// bytes n G .. and all their steps.
template <int G>
struct Int4Keys {
  uint32_t codes[2][G], steps[2][2 * G];
};
template <int G>
struct Int4Values {
  static constexpr int PIECE = G % 4 == 0 ? 4 : G % 2 == 0 ? 2 : 1;       // bytes of a load
  uint32_t codes[8][G / PIECE], steps[2][2 * G];
};
__device__ inline float int4_step_at(const uint32_t* steps, int i) {
  return __uint_as_float(i & 1 ? steps[i / 2] & 0xffff0000u : steps[i / 2] << 16);
}

struct Int4Decode {
  const bf16_t* q;
  int64_t q_stride;
  const uint8_t* k_pool;
  const uint8_t* v_pool;
  bf16_t* out;
  int64_t out_stride;
  float* partial;
  const int* tok_list;
  const int* tok_item;
  const int* tok_pos;
  const int* tables;
  int table_width, heads, kv_heads, parts, block_heads, head_dim, page_size, page_shift, num_pages, window, splits, wide_q;
  float scale_log2, softcap_log2;
  const float* sink;
};

// EVEN: 16 keys from a multiple of 16 on lie in one page (else 8 from a multiple of 8), whose place the scalar unit
// works out for the wave.
// dynamic LDS: the waves' maxima and sums [WAVES][16] each, the block's maxima [16], the waves' accumulators
// [WAVES][heads of the block][32 G]
template <int G, int WAVES, bool EVEN>
__global__ __launch_bounds__(64 * WAVES) void attention_decode_int4_heads_kernel(const Int4Decode a) {
  extern __shared__ __attribute__((aligned(16))) float lds[];
  float* s_m = lds;
  float* s_l = lds + WAVES * I4_HEADS;
  float* s_block = lds + 2 * WAVES * I4_HEADS;
  float* s_acc = s_block + I4_HEADS;
  const int index = blockIdx.x, split = blockIdx.z;
  const int kv_head = blockIdx.y / a.parts, part = blockIdx.y - kv_head * a.parts;
  const int t = a.tok_list ? a.tok_list[index] : index;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n = lane & 15, c = lane >> 4;
  const int pos = a.tok_pos[t];
  const int* table = a.tables + (int64_t)(a.tok_item ? a.tok_item[t] : t) * a.table_width;
  const int kv_group = a.heads / a.kv_heads;
  const int head0 = kv_head * kv_group + part * a.block_heads;
  const int left = kv_group - part * a.block_heads, count = left < a.block_heads ? left : a.block_heads;

  const int first = pos < 0 ? 0 : first_visible_key(pos, a.window);
  const int64_t room = (int64_t)a.table_width * a.page_size;
  const int end_key = pos + 1 < room ? pos + 1 : (int)room;
  int begin = first & ~(I4_TILE - 1), end = end_key;
  if (a.splits > 1) {
    int chunk = (end - begin + a.splits - 1) / a.splits;
    chunk = (chunk + I4_TILE * WAVES - 1) / (I4_TILE * WAVES) * (I4_TILE * WAVES);
    begin += split * chunk;
    if (begin + chunk < end) end = begin + chunk;
  }

  // the pages of a tile's units of 8 (EVEN: 16) keys, and which of them exist
  constexpr int UNITS = EVEN ? 2 : 4, UNIT = I4_TILE / UNITS;
  struct Entries {
    int page[UNITS];
  };
  auto logical_of = [&](int key) { return a.page_shift >= 0 ? key >> a.page_shift : key / a.page_size; };
  auto unit_key = [&](int base, int u) { return base + UNIT * u < end ? base + UNIT * u : (end - 1) & ~(UNIT - 1); };
  auto ask = [&](int base) {
    Entries e;
#pragma unroll
    for (int u = 0; u < UNITS; ++u) e.page[u] = scalar_load(table + logical_of(unit_key(base, u)));
    return e;
  };
  auto units_of = [&](const Entries& e) {
    unsigned units = 0;
#pragma unroll
    for (int u = 0; u < UNITS; ++u) units |= (unsigned)((unsigned)e.page[u] < (unsigned)a.num_pages) << u;
    return units;
  };
  const int64_t page_bytes = (int64_t)a.page_size * (18 * G);
  // a unit's first row of codes, and of steps, in bytes from the pool's beginning
  auto places = [&](const Entries& e, int base, int u, int64_t& code_at, int64_t& step_at) {
    const int key = unit_key(base, u);
    const int within = key - logical_of(key) * a.page_size;
    const int page = (unsigned)e.page[u] < (unsigned)a.num_pages ? e.page[u] : 0;     // a place that exists
    const int64_t at = ((int64_t)page * a.kv_heads + kv_head) * page_bytes;
    code_at = at + within * (16 * G);
    step_at = at + (int64_t)a.page_size * (16 * G) + within * (2 * G);
  };
  // where a lane's rows lie within its unit; `half`: which of two units of 8
  const int key_row = EVEN ? n : n & 7, value_row = EVEN ? 4 * c : 4 * (c & 1);
  const uint32_t key_lane = key_row * (16 * G) + c * (4 * G), value_lane = value_row * (16 * G) + n * G;
  const uint32_t step_lane = value_row * (2 * G);
  auto load_keys = [&](Int4Keys<G>& keys, const Entries& e, int base) {
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      int64_t code_at, step_at;
      const uint8_t *codes, *steps;
      if constexpr (EVEN) {
        places(e, base, s, code_at, step_at);
        codes = a.k_pool + code_at;
        steps = a.k_pool + step_at;
      } else {
        int64_t code_2, step_2;
        places(e, base, 2 * s, code_at, step_at);
        places(e, base, 2 * s + 1, code_2, step_2);
        codes = a.k_pool + (n & 8 ? code_2 : code_at);
        steps = a.k_pool + (c & 2 ? step_2 : step_at);
      }
      constexpr int W = int4_piece(4 * G), SW = int4_piece(8 * G);
#pragma unroll
      for (int i = 0; i < 4 * G; i += W) int4_load<W>(codes + key_lane + i, keys.codes[s] + i / 4);
#pragma unroll
      for (int i = 0; i < 8 * G; i += SW) int4_load<SW>(steps + step_lane + i, keys.steps[s] + i / 4);
    }
  };
  auto load_values = [&](Int4Values<G>& values, const Entries& e, int base) {
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      int64_t code_at, step_at;
      const uint8_t *codes, *steps;
      if constexpr (EVEN) {
        places(e, base, s, code_at, step_at);
        codes = a.v_pool + code_at;
        steps = a.v_pool + step_at;
      } else {
        int64_t code_2, step_2;
        places(e, base, 2 * s, code_at, step_at);
        places(e, base, 2 * s + 1, code_2, step_2);
        codes = a.v_pool + (c & 2 ? code_2 : code_at);
        steps = a.v_pool + (c & 2 ? step_2 : step_at);
      }
      constexpr int W = Int4Values<G>::PIECE, SW = int4_piece(8 * G);
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int i = 0; i < G / W; ++i) int4_load<W>(codes + value_lane + r * (16 * G) + i * W, values.codes[4 * s + r] + i);
#pragma unroll
      for (int i = 0; i < 8 * G; i += SW) int4_load<SW>(steps + step_lane + i, values.steps[s] + i / 4);
    }
  };

  int base = begin + wave * I4_TILE;
  Int4Keys<G> keys;
  Int4Values<G> values;
  Entries entries = {};
  unsigned units = 0;
  if (base < end) {
    entries = ask(base);
    units = units_of(entries);
    load_keys(keys, entries, base);
    load_values(values, entries, base);
    if (base + I4_TILE * WAVES < end) entries = ask(base + I4_TILE * WAVES);
  }

  // the queries, column n of the products: dimensions 32 g + 8 c + (0, 4, 1, 5, ..), the order of a word's nibbles
  int4_bf16x8 query[G];
  int4_f32x4 start[G];
#pragma unroll
  for (int g = 0; g < G; ++g) {
    uint32_t raw[4] = {0u, 0u, 0u, 0u};
    const int d0 = 32 * g + 8 * c;
    if (n < count) {
      const bf16_t* from = a.q + t * a.q_stride + (int64_t)(head0 + n) * a.head_dim + d0;
      if (a.wide_q) {
        if (d0 < a.head_dim) {
          const uint4 v = *reinterpret_cast<const uint4*>(from);
          raw[0] = v.x;
          raw[1] = v.y;
          raw[2] = v.z;
          raw[3] = v.w;
        }
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (d0 + i < a.head_dim) raw[i / 2] |= (uint32_t)from[i].bits << (16 * (i & 1));
      }
    }
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) sum += __uint_as_float(raw[i] << 16) + __uint_as_float(raw[i] & 0xffff0000u);
    sum = halves_sum(xor_sum<16>(sum)) * -I4_OFFSET;
    start[g] = int4_f32x4{sum, sum, sum, sum};
    const int4_u32x4 pairs = {(raw[0] & 0xffffu) | raw[2] << 16, raw[0] >> 16 | (raw[2] & 0xffff0000u),
                              (raw[1] & 0xffffu) | raw[3] << 16, raw[1] >> 16 | (raw[3] & 0xffff0000u)};
    query[g] = __builtin_bit_cast(int4_bf16x8, pairs);
  }

  float m = -INFINITY, reference = 0.f, l = 0.f;
  int4_f32x4 acc[G][2];
#pragma unroll
  for (int g = 0; g < G; ++g) acc[g][0] = acc[g][1] = int4_f32x4{0.f, 0.f, 0.f, 0.f};
  // -24 in all places
  const int4_bf16x8 offsets =
      __builtin_bit_cast(int4_bf16x8, (int4_u32x4){0xc1c0c1c0u, 0xc1c0c1c0u, 0xc1c0c1c0u, 0xc1c0c1c0u});

  // scores of the lane's 8 keys: 4 c .. + 3 and 16 + 4 c .. + 3, head n; unscaled
  auto score = [&](float (&s)[8]) {
#pragma unroll
    for (int sub = 0; sub < 2; ++sub)
#pragma unroll
      for (int g = 0; g < G; ++g) {
        const uint32_t w = keys.codes[sub][g];
        const int4_u32x4 row = {int4_pair<0>(w), int4_pair<1>(w), int4_pair<2>(w), int4_pair<3>(w)};
        const int4_f32x4 dot = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(int4_bf16x8, row), query[g],
                                                                       start[g], 0, 0, 0);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float step = int4_step_at(keys.steps[sub], r * G + g);
          s[4 * sub + r] = g == 0 ? dot[r] * step : fmaf(dot[r], step, s[4 * sub + r]);
        }
      }
  };
  // their weights, and the state that these are relative to
  auto weigh = [&](float (&s)[8]) {
    float high = fmaxf(fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3])), fmaxf(fmaxf(s[4], s[5]), fmaxf(s[6], s[7])));
    if (__builtin_amdgcn_ballot_w64(high > m + I4_SLACK)) {
      const float m_new = fmaxf(m, halves_max(xor_max<16>(high)));
      reference = m_new == -INFINITY ? 0.f : m_new;
      const float correction = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - reference);
      m = m_new;
      l *= correction;
#pragma unroll
      for (int g = 0; g < G; ++g)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          acc[g][0][r] *= correction;
          acc[g][1][r] *= correction;
        }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      s[i] = __builtin_amdgcn_exp2f(s[i] - reference);
      l += s[i];
    }
  };
  auto mix = [&](const float (&p)[8], const bool whole, const unsigned seen) {
    // two keys' codes side by side, of as many groups as a half word has bytes
    constexpr int PIECE = Int4Values<G>::PIECE, BYTES = PIECE >= 2 ? 2 : 1;
#pragma unroll
    for (int g0 = 0; g0 < G; g0 += BYTES) {
      uint32_t both[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t lo = values.codes[2 * j][g0 / PIECE], hi = values.codes[2 * j + 1][g0 / PIECE];
        both[j] = __builtin_amdgcn_perm(hi, lo, PIECE == 4 && (g0 & 2) ? 0x07060302u : 0x05040100u);
      }
#pragma unroll
      for (int b = 0; b < BYTES; ++b) {
        const int g = g0 + b;
        int4_u32x4 weights, low, high;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          float w[2];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int i = 2 * j + h;
            w[h] = p[i] * int4_step_at(values.steps[i >> 2], (i & 3) * G + g);
            // (what a masked key's step is, nobody knows)
            if (!whole) w[h] = seen >> i & 1u ? w[h] : 0.f;
          }
          weights[j] = pack2_bf16(w[0], w[1]);
          low[j] = b == 0 ? int4_pair<0>(both[j]) : int4_pair<2>(both[j]);
          high[j] = b == 0 ? int4_pair<1>(both[j]) : int4_pair<3>(both[j]);
        }
        const int4_bf16x8 column = __builtin_bit_cast(int4_bf16x8, weights);
        const int4_f32x4 shifted[2] = {__builtin_amdgcn_mfma_f32_16x16x32_bf16(offsets, column, acc[g][0], 0, 0, 0),
                                       __builtin_amdgcn_mfma_f32_16x16x32_bf16(offsets, column, acc[g][1], 0, 0, 0)};
        acc[g][0] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(int4_bf16x8, low), column, shifted[0], 0, 0, 0);
        acc[g][1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(int4_bf16x8, high), column, shifted[1], 0, 0, 0);
      }
    }
  };

  // The keys of the next tile are asked for when this one's scores are made, its values when these are used: each then has
  // the other half of the work to arrive in, and one set of registers serves.
  while (base < end) {
    const int after = base + I4_TILE * WAVES;
    const bool whole = base >= first && base + I4_TILE <= end && units == (1u << UNITS) - 1;
    float s[8];
    score(s);
    if (after < end) load_keys(keys, entries, after);
#pragma unroll
    for (int i = 0; i < 8; ++i) s[i] *= a.scale_log2;
    if (a.softcap_log2 > 0.f) {
#pragma unroll
      for (int i = 0; i < 8; ++i) s[i] = capped_score_fast(s[i], a.softcap_log2);
    }
    if (whole) {
      weigh(s);
      mix(s, true, 0);
    } else {
      unsigned seen = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int within = 16 * (i >> 2) + 4 * c + (i & 3);
        const bool visible = base + within >= first && base + within < end && (units >> (within / UNIT) & 1u);
        seen |= (unsigned)visible << i;
        s[i] = visible ? s[i] : -INFINITY;
      }
      weigh(s);
      mix(s, false, seen);
    }
    if (after < end) {
      units = units_of(entries);
      load_values(values, entries, after);
      if (after + I4_TILE * WAVES < end) entries = ask(after + I4_TILE * WAVES);
    }
    base = after;
  }

  // the waves' states meet: maxima first, then sums and accumulators scaled to the block's
  l = halves_sum(xor_sum<16>(l));
  if (c == 0) s_m[wave * I4_HEADS + n] = m;
  __syncthreads();
  float block_m = -INFINITY;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) block_m = fmaxf(block_m, s_m[w * I4_HEADS + n]);
  const bool sinks = a.sink != nullptr && split == 0 && n < count;
  const float sink = sinks ? a.sink[head0 + n] * 1.4426950408889634f : -INFINITY;
  block_m = fmaxf(block_m, sink);
  const float share = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - block_m);
  if (c == 0) {
    s_l[wave * I4_HEADS + n] = l * share + (wave == 0 && sinks ? __builtin_amdgcn_exp2f(sink - block_m) : 0.f);
    if (wave == 0) s_block[n] = block_m;
  }
  if (n < count) {
    float* mine = s_acc + (wave * count + n) * (32 * G);
#pragma unroll
    for (int g = 0; g < G; ++g)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        *reinterpret_cast<float2*>(mine + 32 * g + 2 * (4 * c + r)) = make_float2(acc[g][0][r] * share, acc[g][1][r] * share);
  }
  __syncthreads();
  for (int i = threadIdx.x; i < count * (32 * G); i += 64 * WAVES) {
    const int h = i / (32 * G), d = i - h * (32 * G);
    if (d >= a.head_dim) continue;
    float sum = 0.f, total = 0.f;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      sum += s_acc[(w * count + h) * (32 * G) + d];
      total += s_l[w * I4_HEADS + h];
    }
    const int head = head0 + h;
    if (a.splits == 1) {
      // (a token that sees nothing: zeros)
      a.out[t * a.out_stride + (int64_t)head * a.head_dim + d] = float_to_bf16(total == 0.f ? 0.f : sum / total);
      continue;
    }
    float* record = a.partial + (((int64_t)index * a.heads + head) * a.splits + split) * (a.head_dim + 2);
    record[d] = sum;
    if (d == 0) {
      record[a.head_dim] = s_block[h];
      record[a.head_dim + 1] = total;
    }
  }
}

template <int G>
static void launch_heads(const Int4Decode& a, int count, int waves, hipStream_t s) {
  const dim3 grid(count, a.kv_heads * a.parts, a.splits);
  const int bytes = (I4_HEADS + waves * (2 * I4_HEADS + a.block_heads * 32 * G)) * 4;      // 64 KB at most
  const bool even = a.page_size % 16 == 0;
#define PS_LAUNCH_H4(WAVES, EVEN) \
  hipLaunchKernelGGL((attention_decode_int4_heads_kernel<G, WAVES, EVEN>), grid, dim3(64 * WAVES), bytes, s, a)
  if constexpr (G <= 4) {
    if (waves == 8) {
      if (even) PS_LAUNCH_H4(8, true);
      else PS_LAUNCH_H4(8, false);
      return;
    }
  }
  if (even) PS_LAUNCH_H4(4, true);
  else PS_LAUNCH_H4(4, false);
#undef PS_LAUNCH_H4
}

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
  if (dtype == PS_BF16 && scale > 0.f) {
    const int kv_group = heads / kv_heads, groups = int4_groups(head_dim);
    // heads of more than 128 dimensions: eight to a block, whose accumulators then meet in 32 KB of LDS
    const int most = groups > 4 ? I4_HEADS / 2 : I4_HEADS;
    const int block_heads = kv_group < most ? kv_group : most;
    int page_shift = -1;
    if ((page_size & (page_size - 1)) == 0) {
      page_shift = 0;
      while ((1 << page_shift) < page_size) ++page_shift;
    }
    const bool wide_q = head_dim % 8 == 0 && q_stride % 8 == 0 && (uintptr_t)q % 16 == 0;
    const Int4Decode a{(const bf16_t*)q, q_stride, (const uint8_t*)k_pool, (const uint8_t*)v_pool, (bf16_t*)out, out_stride,
                       partial, tok_list, tok_item, tok_pos, tables, table_width, heads, kv_heads,
                       (kv_group + block_heads - 1) / block_heads, block_heads, head_dim, page_size, page_shift, num_pages, window, splits,
                       wide_q, scale * 1.4426950408889634f, softcap * 1.4426950408889634f, sink};
    const int64_t blocks = (int64_t)count * kv_heads * a.parts;
    const int waves = splits == 1 && blocks <= ps_compute_units() && groups <= 4 && block_heads * groups <= 32 ? 8 : 4;
    switch (groups) {
      case 1: launch_heads<1>(a, count, waves, s); break;
      case 2: launch_heads<2>(a, count, waves, s); break;
      case 3: launch_heads<3>(a, count, waves, s); break;
      case 4: launch_heads<4>(a, count, waves, s); break;
      case 5: launch_heads<5>(a, count, waves, s); break;
      case 6: launch_heads<6>(a, count, waves, s); break;
      case 7: launch_heads<7>(a, count, waves, s); break;
      default: launch_heads<8>(a, count, waves, s); break;
    }
  } else if (dtype == PS_F32) PS_LAUNCH_D4T(float);
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
