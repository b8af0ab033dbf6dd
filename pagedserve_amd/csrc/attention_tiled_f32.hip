// Paged attention of items with several tokens (prompt portions) in true 32-bit.
//
// A block of four waves per (32 queries, head); the waves take the request's keys 32 at a time in turn, each
// with a softmax of its own that runs online in float with the library's expf (reference:
// src/kernels/triton_paged_attention.py:219-223,275-331), and the four results are merged through LDS at the end.
// Scores and weighted values are v_mfma_f32_32x32x2_f32: true 32-bit products and sums.
//
// The scores are made transposed (keys x queries), so that a lane holds 16 keys of one query: the softmax
// needs one exchange with the lane of the other half, its correction is one factor per lane, and the
// probabilities are, where they lie, the operand of the product with the values (also transposed:
// dimensions x queries), since instruction e takes keys 8 (e / 4) + e % 4 + {0, 4} from the lane halves.
// Keys and values come straight from their pages into registers, a row of a key in pieces of 16 bytes,
// a value 128 bytes of a row at a time; the next tile's keys are on their way during softmax and values,
// its values during the scores.
//
// What bounds it: a tile of 32 x 32 at 64 dimensions is 64 matrix instructions of 64 cycles beside some 800
// others, 4.5 us for a wave alone on its SIMD; a portion of a few hundred tokens is a dozen blocks per head, so
// that what counts is the longest chain.  With tiles of 64 queries, plain multiply-adds and one run over the
// keys per block a portion of 300 tokens at 12 heads of 64 took 55 us, now 17; 512 tokens 86 and 21, 2 x 1,024
// tokens 179 and 64 (a third of the time the matrix cores are busy).
//
// The tiles are those of the bfloat16 kernel (`tile_item`, `tile_q0`: the item of each tile and its first query within
// the item's tokens of this step), of 32 queries or of 64, which are two blocks or one (ops/kernels.py says where), and so
// are the rules: query i of an
// item whose cached length after the step is L and which brings n tokens stands at position
// L - n + i and sees keys first_visible_key(position, window) .. position.
//
// Over a cache in 4 bits (cache_int4.h) a lane reads its key's whole row of codes, 16 bytes a group, and of a value the
// byte of its dimension in every group, with the keys' steps; they become floats, exactly, where they are multiplied:
// 2 x 1,024 tokens of 12 heads of 64 65 us (floats 59), 512 behind 3,500 keys 163 (126), 512 of 16 heads of 128 over 4
// behind 2,000 153 (138); token by token 370, 618 and 982.
//
// Head sizes that are multiples of 4 up to 128; others stay with the one-wave-per-token
// kernel.
#include <math.h>

#include "cache_int4.h"
#include "common.h"
#include "pagedserve_hip.h"

#define AF_TILE 64       // queries of a listed tile
#define AF_ROWS 32       // queries of a block, and keys per turn of a wave's loop
#define AF_WAVES 4
#define AF_MAX_DIM 128

typedef __attribute__((__vector_size__(4 * sizeof(float)))) float af_f32x4;
typedef __attribute__((__vector_size__(16 * sizeof(float)))) float af_f32x16;

// What the pools hold: floats, or bytes of codes and steps.
template <bool INT4>
struct AfPool {
  typedef float Element;
};
template <>
struct AfPool<true> {
  typedef uint8_t Element;
};

// DF: 32 head dimensions each; RAGGED: the head size is not 32 DF; PAIRS: one block takes the 64 queries of a tile,
// two waves to 32 of them; `parts`: else, blocks to a listed tile (of 32 queries each); INT4: a cache in 4 bits
// (over codes heads of 65 to 96 dimensions get registers for two waves to a SIMD, eight fewer than they would take: 2 x 1,024
// tokens of 12 heads of 96 95 us, with one wave 109)
template <int DF, bool RAGGED, bool PAIRS, bool INT4>
__global__ __launch_bounds__(64 * AF_WAVES, INT4 && DF == 3 ? 2 : 1) void attention_tiled_f32_kernel(
    const float* __restrict__ q, int64_t q_stride, const typename AfPool<INT4>::Element* __restrict__ k_pool,
    const typename AfPool<INT4>::Element* __restrict__ v_pool, float* __restrict__ out, int64_t out_stride,
    const int* __restrict__ tile_item, const int* __restrict__ tile_q0,
    const int* __restrict__ cu_tokens, const int* __restrict__ kv_lens,
    const int* __restrict__ tables, int table_width, int heads, int kv_heads, int head_dim,
    int page_size, int num_pages, float scale, int window, int parts, const AttnExtras extra) {
  constexpr int STEPS = 4 * DF;                 // pieces of 2 x 4 dimensions of a score
  constexpr int STRIDE = 32 * DF + 4;           // floats from query to query of a wave's result
  __shared__ __attribute__((aligned(16))) float s_out[AF_WAVES * AF_ROWS * STRIDE];
  __shared__ float s_max[AF_WAVES * AF_ROWS], s_sum[AF_WAVES * AF_ROWS];

  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int column = lane & 31;                 // the lane's query, and its key when keys are read
  const int half = lane >> 5;
  // (the lists begin with the tiles that see the most keys, and so do the blocks, the later half of a tile first: with the
  // longest at the end prompts of 500, 20, 35, 800 and 64 tokens at 16 heads of 64 take 56 us, this way 40)
  const int index = blockIdx.x;
  const int tile_index = index / (parts * heads);
  const int part = parts - 1 - (index - tile_index * parts * heads) / heads;   // which 32 queries of the listed tile
  const int head = index % heads;
  const int kv_head = head / (heads / kv_heads);

  const int item = tile_item[tile_index];
  const int tile_q = tile_q0[tile_index];
  const int tok0 = cu_tokens[item];
  const int count = cu_tokens[item + 1] - tok0;
  const int start = kv_lens[item] - count;      // position of the portion's first token
  const int* table = tables + (int64_t)item * table_width;
  constexpr int TURNS = PAIRS ? 2 : AF_WAVES;   // waves that share the keys of 32 queries
  const int turn = PAIRS ? wave & 1 : wave;     // which of them this one is
  const int first_q = tile_q + part * AF_ROWS;  // of the block
  if (first_q >= count) return;                 // (the whole block)
  const int q0 = PAIRS ? first_q + (wave >> 1) * AF_ROWS : first_q;
  const int last_q = q0 + AF_ROWS - 1 < count ? q0 + AF_ROWS - 1 : count - 1;
  const int key_begin = first_visible_key(start + q0, window);
  const int key_end = q0 < count ? start + last_q + 1 : key_begin;

  const int q_pos = q0 + column < count ? start + q0 + column : -1;
  const int q_first = q_pos < 0 ? 0 : first_visible_key(q_pos, window);

  // the lane's query: dimensions 8 s + 4 half ..; rows beyond the item's tokens are zeros and never stored
  af_f32x4 query[STEPS];
#pragma unroll
  for (int s = 0; s < STEPS; ++s) {
    const int dim = 8 * s + 4 * half;
    query[s] = af_f32x4{0.f, 0.f, 0.f, 0.f};
    if (q_pos >= 0 && (!RAGGED || dim < head_dim))
      query[s] = *reinterpret_cast<const af_f32x4*>(q + (int64_t)(tok0 + q0 + column) * q_stride +
                                                    (int64_t)head * head_dim + dim);
  }

  // The page of key k0 + column as the table names it (read without a branch: a wait for it then leaves the
  // loads behind it on their way), and the first value of the key's row in the pools, or -1.
  auto page_of = [&](int k0) {
    const int logical = (k0 + column) / page_size;
    return table[logical < table_width ? logical : table_width - 1];
  };
  // (of codes: the first byte of the key's row of codes, and how far behind it the key's steps lie)
  auto row_of = [&](int k0, int page, int& to_steps) -> int64_t {
    const int key = k0 + column;
    const int logical = key / page_size, within = key - logical * page_size;
    const bool there = key < key_end && logical < table_width && page >= 0 && page < num_pages;
    if constexpr (INT4) {
      to_steps = page_size * (16 * DF) - (there ? within * (14 * DF) : 0);
      const int64_t row = int4_page_at(page, kv_heads, kv_head, page_size, DF) + within * (16 * DF);
      return there ? row : -1;
    }
    const int64_t row = (((int64_t)page * kv_heads + kv_head) * page_size + within) * head_dim;
    return there ? row : -1;
  };
  af_f32x4 key_values[INT4 ? 1 : STEPS];
  float values[DF][16];
  // a key's words and its steps; of 16 values a byte per group and the steps
  constexpr int BYTES = DF == 3 ? 3 : 1, STEP_WORDS = DF == 4 ? 2 : DF == 3 ? 3 : 1;
  uint4 key_codes[INT4 ? DF : 1];
  uint32_t key_steps[INT4 ? STEP_WORDS : 1];
  uint32_t value_codes[INT4 ? 16 : 1][BYTES], value_steps[INT4 ? 16 : 1][STEP_WORDS];
  auto load_steps = [&](const uint8_t* from, uint32_t (&words)[STEP_WORDS]) {
    if constexpr (DF == 4) {
      const uint2 both = *reinterpret_cast<const uint2*>(from);
      words[0] = both.x;
      words[1] = both.y;
    } else if constexpr (DF == 2) {
      words[0] = *reinterpret_cast<const uint32_t*>(from);
    } else {
#pragma unroll
      for (int g = 0; g < DF; ++g) words[g] = reinterpret_cast<const uint16_t*>(from)[g];
    }
  };
  auto step_of = [&](const uint32_t (&words)[STEP_WORDS], int g) {
    if constexpr (DF % 2 == 1) return __uint_as_float(words[g] << 16);
    else return __uint_as_float(g % 2 ? words[g / 2] & 0xffff0000u : words[g / 2] << 16);
  };
  // (rows that are not there are read from the pool's first row and not used)
  auto load_keys = [&](int64_t row, int to_steps) {
    const auto* source = k_pool + (row < 0 ? 0 : row);
    if constexpr (INT4) {
#pragma unroll
      for (int g = 0; g < DF; ++g) key_codes[g] = reinterpret_cast<const uint4*>(source)[g];
      load_steps(source + to_steps, key_steps);
    } else {
#pragma unroll
      for (int s = 0; s < STEPS; ++s) {
        const int dim = 8 * s + 4 * half;
        key_values[s] = *reinterpret_cast<const af_f32x4*>(source + (!RAGGED || dim < head_dim ? dim : 0));
      }
    }
  };
  // the key's dimensions 8 s + 4 half .. + 3
  auto key_piece = [&](int s) -> af_f32x4 {
    if constexpr (INT4) {
      const int g = s / 4, w = (s % 4) * DF + g;
      const uint32_t words[4] = {key_codes[w / 4].x, key_codes[w / 4].y, key_codes[w / 4].z, key_codes[w / 4].w};
      const uint32_t codes = words[w % 4] >> (16 * half);
      const float step = step_of(key_steps, g), base = -8.f * step;
      af_f32x4 piece;
#pragma unroll
      for (int i = 0; i < 4; ++i) piece[i] = fmaf((float)(codes >> (4 * i) & 15u), step, base);
      return piece;
    } else {
      return key_values[s];
    }
  };
  auto load_values = [&](int64_t row, int to_steps) {
    const int64_t from = row < 0 ? 0 : row;
    const int low = (int)from, high = (int)(from >> 32);
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      // key 8 (e / 4) + e % 4 for the lower half of the lanes, four further on for the upper one
      const int key = (e >> 2) * 8 + (e & 3);
      const int low_0 = __builtin_amdgcn_readlane(low, key), low_1 = __builtin_amdgcn_readlane(low, key + 4);
      const int high_0 = __builtin_amdgcn_readlane(high, key), high_1 = __builtin_amdgcn_readlane(high, key + 4);
      const int64_t base = ((int64_t)(half ? high_1 : high_0) << 32) | (unsigned int)(half ? low_1 : low_0);
      if constexpr (INT4) {
        const int steps_0 = __builtin_amdgcn_readlane(to_steps, key), steps_1 = __builtin_amdgcn_readlane(to_steps, key + 4);
        const uint8_t* bytes = v_pool + base + (column >> 1) * DF;
        if constexpr (DF == 4) value_codes[e][0] = *reinterpret_cast<const uint32_t*>(bytes);
        else if constexpr (DF == 2) value_codes[e][0] = *reinterpret_cast<const uint16_t*>(bytes);
        else
#pragma unroll
          for (int g = 0; g < DF; ++g) value_codes[e][g] = bytes[g];
        load_steps(v_pool + base + (half ? steps_1 : steps_0), value_steps[e]);
      } else {
#pragma unroll
        for (int f = 0; f < DF; ++f) {
          const int dim = 32 * f + column;
          values[f][e] = v_pool[base + (!RAGGED || dim < head_dim ? dim : 0)];
        }
      }
    }
  };
  // A value that is no number must not reach the queries that do not see its key: their weight of 0 would still make it one.
  // It is 0 in the product, and the largest magnitude of all steps, as a number of its bits, says at the end that there was one.
  typedef uint16_t two __attribute__((ext_vector_type(2)));
  two largest = {0, 0};
  auto convert_values = [&]() {
    if constexpr (INT4) {
#pragma unroll
      for (int e = 0; e < 16; ++e)
#pragma unroll
        for (int w = 0; w < STEP_WORDS; ++w)
          largest = __builtin_elementwise_max(largest, __builtin_bit_cast(two, value_steps[e][w] & 0x7fff7fffu));
#pragma unroll
      for (int e = 0; e < 16; ++e)
#pragma unroll
        for (int f = 0; f < DF; ++f) {
          const uint32_t code = value_codes[e][DF == 3 ? f : 0] >> ((DF == 3 ? 0 : 8 * f) + 4 * (column & 1)) & 15u;
          const float step = step_of(value_steps[e], f);
          values[f][e] = ((float)code - 8.f) * (step == step ? step : 0.f);
        }
    }
  };

  // (a sink is a score without key or value: it starts the denominator, in one lane half of one wave)
  const bool starts = turn == 0 && extra.sink != nullptr;
  float run_max = starts ? extra.sink[head] : -INFINITY;
  float run_sum = starts && half == 0 ? 1.f : 0.f;     // of the lane's own keys
  af_f32x16 acc[DF];
#pragma unroll
  for (int f = 0; f < DF; ++f)
#pragma unroll
    for (int e = 0; e < 16; ++e) acc[f][e] = 0.f;

  int k0 = key_begin + turn * AF_ROWS;
  if (k0 < key_end) {
    constexpr int TURN = TURNS * AF_ROWS;
    int to_steps = 0, next_to_steps = 0;
    int64_t row = row_of(k0, page_of(k0), to_steps);
    load_keys(row, to_steps);
    int next_page = page_of(k0 + TURN);
    load_values(row, to_steps);
    for (; k0 < key_end; k0 += TURN) {
      // two chains of half the length: no instruction waits for the one before, half the rounding
      af_f32x16 sums[2];
#pragma unroll
      for (int e = 0; e < 16; ++e) sums[0][e] = sums[1][e] = 0.f;
#pragma unroll
      for (int s = 0; s < STEPS; ++s) {
        af_f32x4 piece = key_piece(s);
        if (RAGGED && 8 * s + 4 * half >= head_dim) piece = af_f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < 4; ++i)
          sums[i & 1] = __builtin_amdgcn_mfma_f32_32x32x2f32(piece[i], query[s][i], sums[i & 1], 0, 0, 0);
      }
      const int64_t next_row = row_of(k0 + TURN, next_page, next_to_steps);
      load_keys(next_row, next_to_steps);
      next_page = page_of(k0 + 2 * TURN);
      __builtin_amdgcn_sched_barrier(0);   // (these loads stay in front of the softmax)

      // the lane's 16 scores: query `column`, keys k0 + 8 (e / 4) + 4 half + e % 4
      const unsigned long long there = __ballot(row >= 0);
      float p[16];
#pragma unroll
      for (int e = 0; e < 16; ++e) p[e] = (sums[0][e] + sums[1][e]) * scale;
      if (extra.softcap > 0.f) {
#pragma unroll
        for (int e = 0; e < 16; ++e) p[e] = capped_score(p[e], extra.softcap);
      }
      const unsigned int mine = (unsigned int)(there >> (4 * half));
      float tile_max = -INFINITY;
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int offset = (e >> 2) * 8 + (e & 3);
        const int key = k0 + 4 * half + offset;
        const bool visible = ((mine >> offset) & 1u) != 0 && key <= q_pos && key >= q_first;
        p[e] = visible ? p[e] : -INFINITY;
        tile_max = fmaxf(tile_max, p[e]);
      }
      if (extra.logistic != nullptr) {
        const float shift = extra.logistic[head];
#pragma unroll
        for (int e = 0; e < 16; ++e) p[e] = 1.0f / (1.0f + expf(-(p[e] + shift)));   // 0 where p is -inf
      } else {
        tile_max = fmaxf(tile_max, __shfl_xor(tile_max, 32));
        const float new_max = fmaxf(run_max, tile_max);
        // new_max is -inf only while no key has been visible: zeros then
        const float base = new_max == -INFINITY ? 0.f : new_max;
        const float correction = expf(run_max - base);
        float tile_sum = 0.f;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          p[e] = expf(p[e] - base);
          tile_sum += p[e];
        }
        run_sum = run_sum * correction + tile_sum;
        run_max = new_max;
#pragma unroll
        for (int f = 0; f < DF; ++f)
#pragma unroll
          for (int e = 0; e < 16; ++e) acc[f][e] *= correction;
      }
      convert_values();
      if (there != ~0ull) {
        // (nothing of rows that are not there: a weight of zero would keep what is not a number)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const bool here = ((mine >> ((e >> 2) * 8 + (e & 3))) & 1u) != 0;
#pragma unroll
          for (int f = 0; f < DF; ++f) values[f][e] = here ? values[f][e] : 0.f;
        }
      }
#pragma unroll
      for (int e = 0; e < 16; ++e)
#pragma unroll
        for (int f = 0; f < DF; ++f)
          acc[f] = __builtin_amdgcn_mfma_f32_32x32x2f32(values[f][e], p[e], acc[f], 0, 0, 0);
      load_values(next_row, next_to_steps);
      row = next_row;
    }
  }

  // ---- the four waves' results: dimension 32 f + 8 (e / 4) + 4 half + e % 4 of query `column`
  run_sum += __shfl_xor(run_sum, 32);
  float* mine = s_out + (wave * AF_ROWS + column) * STRIDE;
#pragma unroll
  for (int f = 0; f < DF; ++f)
#pragma unroll
    for (int g = 0; g < 4; ++g)
      *reinterpret_cast<float4*>(mine + 32 * f + 8 * g + 4 * half) =
          make_float4(acc[f][4 * g], acc[f][4 * g + 1], acc[f][4 * g + 2], acc[f][4 * g + 3]);
  if constexpr (INT4) {
    if (__builtin_expect(__builtin_amdgcn_ballot_w64(largest.x > 0x7f80 || largest.y > 0x7f80) != 0, 0)) {
      // The steps of the wave's values once more: the sums of a query that sees one which is no number are none in its
      // group's dimensions.
      uint32_t bad = 0;
#pragma unroll 1
      for (int from = key_begin + turn * AF_ROWS; from < key_end; from += TURNS * AF_ROWS) {
        int to_steps = 0;
        const int64_t row = row_of(from, page_of(from), to_steps);
        const uint16_t* at = reinterpret_cast<const uint16_t*>(v_pool + (row < 0 ? 0 : row) + to_steps);
        uint32_t found = 0;
#pragma unroll
        for (int g = 0; g < DF; ++g) found |= (uint32_t)(row >= 0 && (at[g] & 0x7fffu) > 0x7f80u) << g;
        uint32_t left = (uint32_t)__builtin_amdgcn_ballot_w64(found != 0);      // (both halves ask for the same keys)
        while (left != 0) {
          const int i = __builtin_ctz(left);
          left &= left - 1;
          const uint32_t groups = __builtin_amdgcn_readlane(found, i);
          bad |= from + i <= q_pos && from + i >= q_first ? groups : 0u;
        }
      }
      const float none = __uint_as_float(0x7fc00000u);
#pragma unroll 1
      for (int f = 0; f < DF; ++f) {
        if ((bad >> f & 1u) == 0) continue;
#pragma unroll
        for (int g = 0; g < 4; ++g)
          *reinterpret_cast<float4*>(mine + 32 * f + 8 * g + 4 * half) = make_float4(none, none, none, none);
      }
    }
  }
  if (half == 0) {
    s_max[wave * AF_ROWS + column] = run_max;
    s_sum[wave * AF_ROWS + column] = run_sum;
  }
  __syncthreads();
  // eight threads to a query, four where the block has 64 of them
  constexpr int SHARE = PAIRS ? 4 : 8;
  const int row = tid / SHARE;
  const int first = PAIRS ? (row >> 5) * 2 * AF_ROWS + (row & 31) : row;   // the query in its first wave's results
  if (first_q + row >= count) return;
  float total_max = -INFINITY;
#pragma unroll
  for (int w = 0; w < TURNS; ++w) total_max = fmaxf(total_max, s_max[w * AF_ROWS + first]);
  float factor[TURNS], total = 0.f;
#pragma unroll
  for (int w = 0; w < TURNS; ++w) {
    const float wave_max = s_max[w * AF_ROWS + first];
    factor[w] = wave_max == -INFINITY ? 0.f : expf(wave_max - total_max);
    total += s_sum[w * AF_ROWS + first] * factor[w];
  }
  if (extra.logistic != nullptr) {
#pragma unroll
    for (int w = 0; w < TURNS; ++w) factor[w] = 1.f;
    total = extra.logistic_norm;
  }
  const float inverse = (total != 0.f ? 1.f / total : 0.f) * gate_factor(extra, tok0 + first_q + row, head);
  float* to = out + (int64_t)(tok0 + first_q + row) * out_stride + (int64_t)head * head_dim;
#pragma unroll
  for (int v = 0; v < 8 * DF / SHARE; ++v) {
    const int dim = 4 * (tid % SHARE) + 4 * SHARE * v;
    if (RAGGED && dim >= head_dim) continue;
    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < TURNS; ++w) {
      const float4 value = *reinterpret_cast<const float4*>(s_out + (w * AF_ROWS + first) * STRIDE + dim);
      sum.x = fmaf(factor[w], value.x, sum.x);
      sum.y = fmaf(factor[w], value.y, sum.y);
      sum.z = fmaf(factor[w], value.z, sum.z);
      sum.w = fmaf(factor[w], value.w, sum.w);
    }
    *reinterpret_cast<float4*>(to + dim) =
        make_float4(sum.x * inverse, sum.y * inverse, sum.z * inverse, sum.w * inverse);
  }
}

extern "C" int ps_attention_tiled_f32_supported(int head_dim) {
  return head_dim >= 4 && head_dim <= AF_MAX_DIM && head_dim % 4 == 0;
}

extern "C" int ps_attention_tiled_f32_tile() { return AF_TILE; }

#define PS_LAUNCH_AF_FORM(DF, RAGGED, PAIRS, INT4)                                                \
  hipLaunchKernelGGL((attention_tiled_f32_kernel<DF, RAGGED, PAIRS, INT4>), dim3((unsigned)blocks), \
                     dim3(64 * AF_WAVES), 0, s, (const float*)q, q_stride,                        \
                     (const AfPool<INT4>::Element*)k_pool, (const AfPool<INT4>::Element*)v_pool,  \
                     (float*)out, out_stride, tile_item, tile_q0, cu_tokens, kv_lens, tables,     \
                     table_width, heads, kv_heads, head_dim, page_size, num_pages, scale, window, parts, extra)
#define PS_LAUNCH_AF_DF(DF, INT4)                                                                 \
  do {                                                                                            \
    if (head_dim == 32 * DF && paired) PS_LAUNCH_AF_FORM(DF, false, true, INT4);                  \
    else if (head_dim == 32 * DF) PS_LAUNCH_AF_FORM(DF, false, false, INT4);                      \
    else if (paired) PS_LAUNCH_AF_FORM(DF, true, true, INT4);                                     \
    else PS_LAUNCH_AF_FORM(DF, true, false, INT4);                                                \
  } while (0)
#define PS_LAUNCH_AF(INT4)                    \
  switch ((head_dim + 31) / 32) {             \
    case 1: PS_LAUNCH_AF_DF(1, INT4); break;  \
    case 2: PS_LAUNCH_AF_DF(2, INT4); break;  \
    case 3: PS_LAUNCH_AF_DF(3, INT4); break;  \
    default: PS_LAUNCH_AF_DF(4, INT4); break; \
  }

extern "C" int ps_attention_tiled_f32(const void* q, int64_t q_stride, const void* k_pool,
                                      const void* v_pool, void* out, int64_t out_stride,
                                      const int* tile_item, const int* tile_q0, int tiles,
                                      const int* cu_tokens, const int* kv_lens, const int* tables,
                                      int table_width, int heads, int kv_heads, int head_dim,
                                      int page_size, int num_pages, float scale, int window,
                                      const float* sink, const float* gate, int64_t gate_ld,
                                      float softcap, const float* logistic, float logistic_norm,
                                      int query_tile, int paired, void* stream) {
  PS_REQUIRE(tiles >= 0 && heads > 0 && kv_heads > 0 && page_size > 0 && num_pages > 0 &&
                 table_width > 0,
             "ps_attention_tiled_f32: bad sizes");
  PS_REQUIRE(ps_attention_tiled_f32_supported(head_dim),
             "ps_attention_tiled_f32: head_dim %d must be a multiple of 4 up to %d "
             "(ps_attention_rowwise takes every size)", head_dim, AF_MAX_DIM);
  PS_REQUIRE(heads % kv_heads == 0,
             "ps_attention_tiled_f32: heads (%d) must be a multiple of kv_heads (%d)", heads, kv_heads);
  PS_REQUIRE(scale > 0.f, "ps_attention_tiled_f32: the score scale must be positive, got %g", scale);
  PS_REQUIRE((q_stride % 4) == 0 && (out_stride % 4) == 0 && ((uintptr_t)q % 16) == 0 &&
                 ((uintptr_t)out % 16) == 0 && ((uintptr_t)k_pool % 16) == 0 &&
                 ((uintptr_t)v_pool % 16) == 0,
             "ps_attention_tiled_f32: rows of q, out and the pools must allow 16-byte accesses");
  PS_REQUIRE(query_tile == AF_TILE || query_tile == AF_ROWS,
             "ps_attention_tiled_f32: tiles of %d or %d queries, not %d", AF_TILE, AF_ROWS, query_tile);
  PS_REQUIRE(!paired || query_tile == AF_TILE, "ps_attention_tiled_f32: one block takes a tile of %d queries, not of %d",
             AF_TILE, query_tile);
  const int parts = paired ? 1 : query_tile / AF_ROWS;
  const int64_t blocks = (int64_t)tiles * heads * parts;
  PS_REQUIRE(blocks < ((int64_t)1 << 31), "ps_attention_tiled_f32: too many blocks");
  if (blocks == 0) return 0;
  hipStream_t s = (hipStream_t)stream;
  const AttnExtras extra = {sink, gate, gate_ld, softcap, logistic, logistic_norm};
  PS_LAUNCH_AF(false);
  PS_CHECK_LAUNCH("ps_attention_tiled_f32");
  return 0;
}

extern "C" int ps_attention_tiled_f32_int4(const void* q, int64_t q_stride, const void* k_pool, const void* v_pool,
                                           void* out, int64_t out_stride, const int* tile_item, const int* tile_q0,
                                           int tiles, const int* cu_tokens, const int* kv_lens, const int* tables,
                                           int table_width, int heads, int kv_heads, int head_dim, int page_size,
                                           int num_pages, float scale, int window, const float* sink, float softcap,
                                           int query_tile, int paired, void* stream) {
  const char* who = "ps_attention_tiled_f32_int4";
  PS_REQUIRE(tiles >= 0 && heads > 0 && kv_heads > 0 && page_size > 0 && num_pages > 0 && table_width > 0,
             "%s: bad sizes", who);
  PS_REQUIRE(ps_attention_tiled_f32_supported(head_dim), "%s: head_dim %d must be a multiple of 4 up to %d", who, head_dim,
             AF_MAX_DIM);
  PS_REQUIRE(heads % kv_heads == 0, "%s: heads (%d) must be a multiple of kv_heads (%d)", who, heads, kv_heads);
  PS_REQUIRE(page_size % 8 == 0 && page_size <= (1 << 20),
             "%s: pages of a cache in 4 bits hold a multiple of 8 keys, not %d", who, page_size);
  PS_REQUIRE(scale > 0.f, "%s: the score scale must be positive, got %g", who, scale);
  PS_REQUIRE(q_stride % 4 == 0 && out_stride % 4 == 0 &&
                 ((uintptr_t)q | (uintptr_t)out | (uintptr_t)k_pool | (uintptr_t)v_pool) % 16 == 0,
             "%s: rows of q, out and the pools must allow 16-byte accesses", who);
  PS_REQUIRE(query_tile == AF_TILE || (query_tile == AF_ROWS && !paired),
             "%s: tiles of %d (paired or not) or %d queries, not %d", who, AF_TILE, AF_ROWS, query_tile);
  const int parts = paired ? 1 : query_tile / AF_ROWS;
  const int64_t blocks = (int64_t)tiles * heads * parts;
  PS_REQUIRE(blocks < ((int64_t)1 << 31), "%s: too many blocks", who);
  if (blocks == 0) return 0;
  hipStream_t s = (hipStream_t)stream;
  const AttnExtras extra = {sink, nullptr, 0, softcap, nullptr, 1.f};
  PS_LAUNCH_AF(true);
  PS_CHECK_LAUNCH(who);
  return 0;
}
