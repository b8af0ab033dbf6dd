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
//            each on average); the codes are 16 + code again, and a product of -24 in all places with the same weights
//            comes first, in every tile, and takes off what that is too much.
//
// Bound by memory where there are blocks enough (4.5 bits a value), else by the trip block table -> codes: a tile's codes
// are asked for one tile ahead (Int4Stage), its table entries, which are the same for a wave and come through the scalar
// unit, two.  32 requests over 8,192 keys, 12 heads of 64: 51 to 54 us, 4.2 to 4.4 TB/s, 85 to 90 % of a large copy's rate
// (64: 92 us, 4.9 TB/s); 64 over 768 to 1,024, 25 heads that share no keys: 29.4 to 31 us, 3.4 TB/s; 24 over up to 6,000,
// 16 heads of 128 over 2: 16.1 us; 1 over 900: 5.0 us and 2.0 for the merge.  Storing the tokens' own rows as a decode step
// does (under the profiler, beside the same without): 32 over 8,192 53.6 and 52.5 us, 64 over 768 to 1,024 of 25 heads 34.1 and
// 31.3, 1 over 900 6.1 and 4.9.
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
#define I4_OWN 80            // words for a token's own rows: 8 of codes and 1 of steps to a group, up to a multiple of 64 bytes
#define I4_SLACK 8.f         // how far (in units of log 2) a score may pass the exponentials' reference

// Reads from LDS, at constant distances from an address, that have arrived when they return.  (Written as assembly: the
// compiler would wait for every load on its way to LDS before a read of its own.)
typedef __attribute__((address_space(3))) void* int4_lds_ptr;
typedef const __attribute__((address_space(1))) void* int4_global_ptr;
typedef uint32_t int4_u32x2 __attribute__((ext_vector_type(2)));
#define I4_READ2(OP, X, Y, AT, A, B)                                                                              \
  asm volatile(OP " %0, %2 offset:%3\n\t" OP " %1, %2 offset:%4\n\ts_waitcnt lgkmcnt(0)"                           \
               : "=&v"(X), "=&v"(Y)                                                                               \
               : "v"(AT), "n"(A), "n"(B)                                                                          \
               : "memory")
#define I4_READ8(OP, X, AT, D, SUB)                                                                               \
  asm volatile(OP " %0, %8 offset:%9\n\t" OP " %1, %8 offset:%10\n\t" OP " %2, %8 offset:%11\n\t" OP              \
                  " %3, %8 offset:%12\n\t" OP " %4, %8 offset:%13\n\t" OP " %5, %8 offset:%14\n\t" OP             \
                  " %6, %8 offset:%15\n\t" OP " %7, %8 offset:%16\n\ts_waitcnt lgkmcnt(0)"                       \
               : "=&v"(X[0]), "=&v"(X[1]), "=&v"(X[2]), "=&v"(X[3]), "=&v"(X[4]), "=&v"(X[5]), "=&v"(X[6]),       \
                 "=&v"(X[7])                                                                                      \
               : "v"(AT), "n"(0), "n"(D), "n"(2 * (D)), "n"(3 * (D)), "n"(SUB), "n"((SUB) + (D)),                 \
                 "n"((SUB) + 2 * (D)), "n"((SUB) + 3 * (D))                                                       \
               : "memory")
// BYTES at `at` and at `at` + SUB, into words of two rows.
template <int BYTES, int SUB, int FROM = 0>
__device__ inline void int4_read_pair(uint32_t at, uint32_t* first, uint32_t* second) {
  if constexpr (BYTES - FROM >= 16 && BYTES % 16 == 0) {
    int4_u32x4 x, y;
    I4_READ2("ds_read_b128", x, y, at, FROM, SUB + FROM);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      first[FROM / 4 + i] = x[i];
      second[FROM / 4 + i] = y[i];
    }
    int4_read_pair<BYTES, SUB, FROM + 16>(at, first, second);
  } else if constexpr (BYTES - FROM >= 8 && BYTES % 8 == 0) {
    int4_u32x2 x, y;
    I4_READ2("ds_read_b64", x, y, at, FROM, SUB + FROM);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      first[FROM / 4 + i] = x[i];
      second[FROM / 4 + i] = y[i];
    }
    int4_read_pair<BYTES, SUB, FROM + 8>(at, first, second);
  } else if constexpr (BYTES - FROM >= 4) {
    I4_READ2("ds_read_b32", first[FROM / 4], second[FROM / 4], at, FROM, SUB + FROM);
    int4_read_pair<BYTES, SUB, FROM + 4>(at, first, second);
  }
}

// Nibbles i and i + 4 of a word as the bfloat16 numbers 16 + nibble, in the low and the high half.  (mask and sixteens:
// 0x00780078 and 0x41804180 in registers; written out, they would cost an instruction more.)
template <int I>
__device__ inline uint32_t int4_pair(uint32_t word, uint32_t mask, uint32_t sixteens) {
  const uint32_t at = I == 0 ? word << 3 : word >> (4 * I - 3);
  return (at & mask) | sixteens;
}

// The largest of three, in one instruction (the library's maxima quiet every operand first).
__device__ inline float int4_max3(float x, float y, float z) {
  float high;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(high) : "v"(x), "v"(y), "v"(z));
  return high;
}

// A tile of 32 keys in LDS: the rows of the keys' codes, those of the values', the keys' steps and the values'.  It comes there
// from the pages by loads that pass no register: 16 bytes of codes, 4 of steps to a lane.
template <int G>
struct Int4Stage {
  static constexpr int CODES = I4_TILE * 16 * G;               // bytes of the keys' codes, and of the values'
  static constexpr int STEPS = I4_TILE * 2 * G;                // bytes of the keys' steps, and of the values'
  static constexpr int STEP_LOADS = (2 * STEPS + 255) / 256;
  static constexpr int LOADS = G + STEP_LOADS;                 // instructions of a wave
  static constexpr int BYTES = 2 * CODES + 256 * STEP_LOADS;
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
  const bf16_t* new_k;         // the tokens' own rows, stored first (STORES)
  const bf16_t* new_v;
  int64_t new_k_stride, new_v_stride;
};

// EVEN: pages of a power of two, 16 or more: 16 keys from a multiple of 16 on lie in one page (else 8 from a multiple of 8), whose
// place the scalar unit works out for the wave.
// STORES: a token's own key and value are stored first.  The wave whose tile holds them works out their codes, which go to LDS,
// from where they replace what that tile's loads have found in their place, and at the end to the page, for later calls.
//
// dynamic LDS: the waves' maxima and sums [WAVES][16] each, the block's maxima [16], the token's own rows, then the waves'
// pairs of tiles, in whose place the accumulators [WAVES][heads of the block][32 G] meet at the end
// (registers for five waves to a SIMD of heads up to 64 and for four of heads up to 96, a few less than some forms take by
// themselves: pages of 24, 64 requests of 25 heads of 64 over 1,024 keys 44.2 -> 43.0 us, 48 of 20 heads of 96 over 2,000
// 71 -> 63; where that would spill, heads up to 64 that store over such pages, they take what they take)
template <int G, int WAVES, bool EVEN, bool STORES>
__global__ __launch_bounds__(64 * WAVES, G == 2 && (EVEN || !STORES) ? 5 : G == 3 ? 4 : 1) void
attention_decode_int4_heads_kernel(const Int4Decode a) {
  typedef Int4Stage<G> Stage;
  extern __shared__ __attribute__((aligned(1024))) float lds[];
  float* s_m = lds;
  float* s_l = lds + WAVES * I4_HEADS;
  float* s_block = lds + 2 * WAVES * I4_HEADS;
  uint32_t* s_own = reinterpret_cast<uint32_t*>(s_block + I4_HEADS);      // codes of key and value, then their steps
  float* s_acc = s_block + I4_HEADS + I4_OWN;
  unsigned char* stages = reinterpret_cast<unsigned char*>(s_acc);      // (the accumulators come when no tile is left)
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

  uint32_t raw_query[G][4];
#pragma unroll
  for (int g = 0; g < G; ++g) {
    uint32_t (&raw)[4] = raw_query[g];
    raw[0] = raw[1] = raw[2] = raw[3] = 0u;
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
  }

  const int first = pos < 0 ? 0 : first_visible_key(pos, a.window);
  const int64_t room = (int64_t)a.table_width * a.page_size;
  const int end_key = pos < 0 ? 0 : pos < room ? pos + 1 : (int)room;
  int begin = first & ~(I4_TILE - 1), end = end_key;
  if (a.splits > 1) {
    int chunk = (end - begin + a.splits - 1) / a.splits;
    chunk = (chunk + I4_TILE * WAVES - 1) / (I4_TILE * WAVES) * (I4_TILE * WAVES);
    begin += split * chunk;
    if (begin + chunk < end) end = begin + chunk;
  }

  // the token's own rows, by the wave whose tile holds them: 8 dimensions to a lane, of the key and then of the value
  const bool own = STORES && pos >= begin && pos < end;
  const bool mine = own && wave == (pos - begin) / I4_TILE % WAVES;
  float row[1][8];
  if (STORES && mine && lane < 8 * G) {
    const bool is_value = lane >= 4 * G;
    const bf16_t* from = (is_value ? a.new_v + t * a.new_v_stride : a.new_k + t * a.new_k_stride) + (int64_t)kv_head * a.head_dim;
    const int d0 = 8 * (lane % (4 * G));
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float value = to_float(from[d0 + i < a.head_dim ? d0 + i : a.head_dim - 1]);
      row[0][i] = d0 + i < a.head_dim ? value : 0.f;
    }
  }

  // the pages of a tile's units of 8 (EVEN: 16) keys, and which of them exist
  constexpr int UNITS = EVEN ? 2 : 4, UNIT = I4_TILE / UNITS;
  struct Entries {
    int page[UNITS];
  };
  auto logical_of = [&](int key) { return EVEN ? key >> a.page_shift : key / a.page_size; };
  auto unit_key = [&](int base, int u) { return base + UNIT * u < end ? base + UNIT * u : (end - 1) & ~(UNIT - 1); };
  auto ask = [&](int base) __attribute__((always_inline)) {
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
  const uint64_t page_stride = (uint64_t)a.kv_heads * (unsigned)a.page_size * (18 * G);
  const int64_t head_at = (int64_t)kv_head * a.page_size * (18 * G), steps_at = (int64_t)a.page_size * (16 * G);
  // a unit's first row of codes, and of steps, in bytes from the pool's beginning
  struct Places {
    int64_t codes[UNITS], steps[UNITS];
  };
  auto places = [&](const Entries& e, int base) __attribute__((always_inline)) {
    Places at;
#pragma unroll
    for (int u = 0; u < UNITS; ++u) {
      const int key = unit_key(base, u);
      const int within = EVEN ? key & (a.page_size - 1) : key - logical_of(key) * a.page_size;
      const unsigned page = (unsigned)e.page[u] < (unsigned)a.num_pages ? e.page[u] : 0u;     // a place that exists
      const int64_t first_byte = (int64_t)((uint64_t)page * page_stride) + head_at;
      at.codes[u] = first_byte + within * (16 * G);
      at.steps[u] = first_byte + steps_at + within * (2 * G);
    }
    return at;
  };
  auto of_unit = [&](const int64_t (&at)[UNITS], int u) __attribute__((always_inline)) {
    // (by masks: differences are the scalar unit's, and a selection would keep the array in memory)
    int64_t found = at[0];
#pragma unroll
    for (int i = 1; i < UNITS; ++i) found += (at[i] - at[0]) & -(int64_t)(u == i);
    return found;
  };
  unsigned char* pair = stages + wave * (2 * Stage::BYTES);
  auto issue = [&](int slot, const Entries& e, int base) __attribute__((always_inline)) {
    const Places at = places(e, base);
    unsigned char* stage = pair + slot * Stage::BYTES;
#pragma unroll
    for (int j = 0; j < G; ++j) {
      const int piece = j * 64 + lane;
      const bool is_value = piece >= 32 * G;
      const int p = is_value ? piece - 32 * G : piece;
      const int key = p / G, within = p - key * G;
      const uint8_t* from = (is_value ? a.v_pool : a.k_pool) + of_unit(at.codes, key / UNIT) +
                            ((key % UNIT) * (16 * G) + within * 16);
      __builtin_amdgcn_global_load_lds((int4_global_ptr)from, (int4_lds_ptr)(stage + j * 1024), 16, 0, 0);
    }
#pragma unroll
    for (int j = 0; j < Stage::STEP_LOADS; ++j) {
      const int word = j * 64 + lane < 32 * G ? j * 64 + lane : 32 * G - 1;      // (what is left over repeats the last one)
      const bool is_value = word >= 16 * G;
      const int p = is_value ? word - 16 * G : word;
      constexpr int UNIT_WORDS = UNIT * G / 2;
      const uint8_t* from =
          (is_value ? a.v_pool : a.k_pool) + of_unit(at.steps, p / UNIT_WORDS) + 4 * (p % UNIT_WORDS);
      __builtin_amdgcn_global_load_lds((int4_global_ptr)from, (int4_lds_ptr)(stage + 2 * Stage::CODES + j * 256), 4, 0, 0);
    }
  };

  // one tile is on its way while one is worked on; the table's entries are asked for one tile earlier still
  int base = begin + wave * I4_TILE, ahead = base;
  constexpr int STRIDE = I4_TILE * WAVES;
  Entries entries = {};
  unsigned exist = 0;         // which units of the tiles on their way have a page, four bits a tile, the nearest lowest
  int on_way = 0;
  auto send = [&](int slot) __attribute__((always_inline)) {
    exist |= units_of(entries) << (4 * on_way);
    issue(slot, entries, ahead);
    ++on_way;
    ahead += STRIDE;
    if (ahead < end) entries = ask(ahead);
  };
  if (base < end) {
    entries = ask(base);
    send(0);
  }

  if (STORES && mine && lane < 8 * G) {
    uint32_t word[1], step[1];
    int4_code_row<1, true>(row, false, word, step);            // (a group to four lanes)
    const int g = lane % (4 * G) / 4, quarter = lane & 3;
    unsigned char* at = reinterpret_cast<unsigned char*>(s_own);
    if (lane < 4 * G) {
      s_own[quarter * G + g] = word[0];
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) at[16 * G + (4 * quarter + i) * G + g] = (unsigned char)(word[0] >> (8 * i));
    }
    if (quarter == 0) reinterpret_cast<uint16_t*>(at + 32 * G)[lane / 4] = (uint16_t)step[0];
  }

  // the queries, column n of the products: dimensions 32 g + 8 c + (0, 4, 1, 5, ..), the order of a word's nibbles
  int4_bf16x8 query[G];
  int4_f32x4 start[G];
#pragma unroll
  for (int g = 0; g < G; ++g) {
    const uint32_t (&raw)[4] = raw_query[g];
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
  uint32_t mask = 0x00780078u, sixteens = 0x41804180u;
  asm volatile("" : "+s"(mask));
  asm volatile("" : "+v"(sixteens));
  // -24 in all places
  const int4_bf16x8 offsets =
      __builtin_bit_cast(int4_bf16x8, (int4_u32x4){0xc1c0c1c0u, 0xc1c0c1c0u, 0xc1c0c1c0u, 0xc1c0c1c0u});

  // Lane (16 c + n) reads the words c G .. of keys n and 16 + n, and of keys 4 c .. + 3 and 16 + 4 c .. + 3 the bytes n G .. of
  // the values and all steps.
  const uint32_t pair_at = (uint32_t)(uintptr_t)(int4_lds_ptr)pair;
  const uint32_t key_lane = n * (16 * G) + c * (4 * G), value_lane = Stage::CODES + 4 * c * (16 * G) + n * G;
  const uint32_t step_lane = 2 * Stage::CODES + 4 * c * (2 * G);
  // scores of those 8 keys, head n; unscaled
  auto score = [&](float (&s)[8], uint32_t stage) {
    uint32_t codes[2][G], steps[2][2 * G];
    int4_read_pair<4 * G, 256 * G>(stage + key_lane, codes[0], codes[1]);
    int4_read_pair<8 * G, 32 * G>(stage + step_lane, steps[0], steps[1]);
#pragma unroll
    for (int sub = 0; sub < 2; ++sub)
#pragma unroll
      for (int g = 0; g < G; ++g) {
        const uint32_t w = codes[sub][g];
        const int4_u32x4 row = {int4_pair<0>(w, mask, sixteens), int4_pair<1>(w, mask, sixteens),
                                int4_pair<2>(w, mask, sixteens), int4_pair<3>(w, mask, sixteens)};
        const int4_f32x4 dot = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(int4_bf16x8, row), query[g],
                                                                       start[g], 0, 0, 0);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float step = int4_step_at(steps[sub], r * G + g);
          s[4 * sub + r] = g == 0 ? dot[r] * step : fmaf(dot[r], step, s[4 * sub + r]);
        }
      }
  };
  // their weights, and the state that these are relative to; capped scores are scaled already
  const float factor = a.softcap_log2 > 0.f ? 1.f : a.scale_log2;
  auto weigh = [&](float (&s)[8]) {
    const float high = int4_max3(int4_max3(s[0], s[1], s[2]), int4_max3(s[3], s[4], s[5]), int4_max3(s[6], s[7], s[7])) * factor;
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
    float unit = factor;
    if (__builtin_amdgcn_ballot_w64(fabsf(reference) > 1048576.f)) {
      // (of such a product the part that rounding takes is an exponent of its own: all are rounded as the reference was)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        s[i] *= factor;
        asm volatile("" : "+v"(s[i]));
      }
      unit = 1.f;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      s[i] = __builtin_amdgcn_exp2f(fmaf(s[i], unit, -reference));
      l += s[i];
    }
  };
  auto mix = [&](const float (&p)[8], uint32_t stage) {
    // two keys' codes side by side, of as many groups as a half word has bytes
    constexpr int PIECE = G % 4 == 0 ? 4 : G % 2 == 0 ? 2 : 1, BYTES = PIECE >= 2 ? 2 : 1;
    uint32_t steps[2][2 * G];
    int4_read_pair<8 * G, 32 * G>(stage + Stage::STEPS + step_lane, steps[0], steps[1]);
    uint32_t codes[8];
#pragma unroll
    for (int g0 = 0; g0 < G; g0 += BYTES) {
      if (g0 % PIECE == 0) {
        if constexpr (PIECE == 4) I4_READ8("ds_read_b32", codes, stage + value_lane + g0, 16 * G, 256 * G);
        else if constexpr (PIECE == 2) I4_READ8("ds_read_u16", codes, stage + value_lane + g0, 16 * G, 256 * G);
        else I4_READ8("ds_read_u8", codes, stage + value_lane + g0, 16 * G, 256 * G);
      }
      uint32_t both[4];
#pragma unroll
      for (int j = 0; j < 4; ++j)
        both[j] = __builtin_amdgcn_perm(codes[2 * j + 1], codes[2 * j], PIECE == 4 && (g0 & 2) ? 0x07060302u : 0x05040100u);
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
            w[h] = p[i] * int4_step_at(steps[i >> 2], (i & 3) * G + g);
          }
          weights[j] = pack2_bf16(w[0], w[1]);
          low[j] = b == 0 ? int4_pair<0>(both[j], mask, sixteens) : int4_pair<2>(both[j], mask, sixteens);
          high[j] = b == 0 ? int4_pair<1>(both[j], mask, sixteens) : int4_pair<3>(both[j], mask, sixteens);
        }
        const int4_bf16x8 column = __builtin_bit_cast(int4_bf16x8, weights);
        const int4_f32x4 shifted[2] = {__builtin_amdgcn_mfma_f32_16x16x32_bf16(offsets, column, acc[g][0], 0, 0, 0),
                                       __builtin_amdgcn_mfma_f32_16x16x32_bf16(offsets, column, acc[g][1], 0, 0, 0)};
        acc[g][0] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(int4_bf16x8, low), column, shifted[0], 0, 0, 0);
        acc[g][1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(int4_bf16x8, high), column, shifted[1], 0, 0, 0);
      }
    }
  };

  int slot = 0;
  while (base < end) {
    // the stage that was read last is filled again
    if (ahead < end) send(slot ^ 1);
    // the loads of this tile have landed; those behind it are on their way
    if (on_way == 2) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(Stage::LOADS) : "memory");
    else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    const unsigned units = exist & 15u;
    const bool whole = base >= first && base + I4_TILE <= end && units == (1u << UNITS) - 1;
    const uint32_t stage = pair_at + slot * Stage::BYTES;
    if (STORES && own && base <= pos && pos < base + I4_TILE) {
      unsigned char* at = pair + slot * Stage::BYTES;
      const int within = pos - base;
      int lane = threadIdx.x & 63;
      asm volatile("" : "+v"(lane));       // (worked out here, once: kept through the loop it takes a register too many)
      if (lane < 8 * G)
        reinterpret_cast<uint32_t*>(at + (lane >= 4 * G ? Stage::CODES : 0) + within * (16 * G))[lane % (4 * G)] = s_own[lane];
      if (lane < 2 * G)
        reinterpret_cast<uint16_t*>(at + 2 * Stage::CODES + (lane >= G ? Stage::STEPS : 0) + within * (2 * G))[lane % G] =
            reinterpret_cast<const uint16_t*>(s_own + 8 * G)[lane];
    }
    float s[8];
    score(s, stage);
    if (a.softcap_log2 > 0.f) {
#pragma unroll
      for (int i = 0; i < 8; ++i) s[i] = capped_score_fast(s[i] * a.scale_log2, a.softcap_log2);
    }
    if (!whole) {
      auto visible = [&](int within) {
        return (base + within >= first) & (base + within < end) & ((units >> (within / UNIT) & 1u) != 0);
      };
#pragma unroll
      for (int i = 0; i < 8; ++i) s[i] = visible(16 * (i >> 2) + 4 * c + (i & 3)) ? s[i] : -INFINITY;
      // nobody knows what a masked key's steps are, and 0 times a NaN is none: the values' steps become 0 where they lie
      if (lane < I4_TILE && !visible(lane)) {
        uint16_t* steps = reinterpret_cast<uint16_t*>(pair + slot * Stage::BYTES + 2 * Stage::CODES + Stage::STEPS) + lane * G;
#pragma unroll
        for (int g = 0; g < G; ++g) steps[g] = 0;
      }
    }
    weigh(s);
    mix(s, stage);
    base += STRIDE;
    exist >>= 4;
    --on_way;
    slot ^= 1;
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
    s_l[wave * I4_HEADS + n] = l * share + (wave == 0 && sink != -INFINITY ? __builtin_amdgcn_exp2f(sink - block_m) : 0.f);
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
  if (STORES && mine) {
    // the codes to their page (here, where nothing waits for that)
    const int logical = logical_of(pos), within = pos - logical * a.page_size;
    const int page = scalar_load(table + logical);
    if ((unsigned)page < (unsigned)a.num_pages) {
      const int64_t at = int4_page_at(page, a.kv_heads, kv_head, a.page_size, G);
      if (lane < 8 * G)
        reinterpret_cast<uint32_t*>((uint8_t*)(lane >= 4 * G ? a.v_pool : a.k_pool) + at + within * (16 * G))[lane % (4 * G)] =
            s_own[lane];
      if (lane < 2 * G)
        reinterpret_cast<uint16_t*>((uint8_t*)(lane >= G ? a.v_pool : a.k_pool) + at + a.page_size * (16 * G) +
                                    within * (2 * G))[lane % G] = reinterpret_cast<const uint16_t*>(s_own + 8 * G)[lane];
    }
  }
}

// (beyond the 64 KB that a kernel may ask for without saying so)
static void int4_allow_lds(const void* kernel, int bytes) {
  if (bytes > 64 * 1024)
    (void)hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
}

template <int G>
static void launch_heads(const Int4Decode& a, int count, int waves, hipStream_t s) {
  const dim3 grid(count, a.kv_heads * a.parts, a.splits);
  // A pair of tiles to a wave.  (Three or four leave room for fewer blocks on a unit, which weighs more: 64 requests of 25 heads over
  // 1,024 keys 32.7 us with two, 34.0 with three and 36.4 with four, 128 of 12 over 1,000 29.7, 32.0 and 33.2; 64 of 32 heads
  // of 128 over 8 and 1,500 keys 28.8 with two, 32 with three; 48 of 20 heads of 96 over 2,000 53 and 63.)
  const int pairs = waves * 2 * Int4Stage<G>::BYTES, meet = waves * a.block_heads * 32 * G * 4;
  const int bytes = (I4_HEADS + waves * 2 * I4_HEADS + I4_OWN) * 4 + (pairs > meet ? pairs : meet);
  const bool even = a.page_size >= 16 && a.page_shift >= 0;
#define PS_LAUNCH_H4S(WAVES, EVEN, STORES)                                                                          \
  do {                                                                                                              \
    int4_allow_lds(reinterpret_cast<const void*>(attention_decode_int4_heads_kernel<G, WAVES, EVEN, STORES>), bytes); \
    hipLaunchKernelGGL((attention_decode_int4_heads_kernel<G, WAVES, EVEN, STORES>), grid, dim3(64 * WAVES), bytes, s, a); \
  } while (0)
#define PS_LAUNCH_H4E(WAVES, EVEN)                                  \
  do {                                                              \
    if (a.new_k != nullptr) PS_LAUNCH_H4S(WAVES, EVEN, true);       \
    else PS_LAUNCH_H4S(WAVES, EVEN, false);                         \
  } while (0)
#define PS_LAUNCH_H4(WAVES)                \
  do {                                     \
    if (even) PS_LAUNCH_H4E(WAVES, true);  \
    else PS_LAUNCH_H4E(WAVES, false);      \
  } while (0)
  if constexpr (G <= 4) {
    if (waves == 8) {
      PS_LAUNCH_H4(8);
      return;
    }
  }
  PS_LAUNCH_H4(4);
#undef PS_LAUNCH_H4S
#undef PS_LAUNCH_H4E
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
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int d = 8 * w + i;
    query[i] = d < head_dim ? to_float(q[t * q_stride + (int64_t)head * head_dim + d]) : 0.f;
  }

  // (a token in front of its context sees nothing, and reads no entry of the table)
  const int first = pos < 0 ? 0 : first_visible_key(pos, window);
  int end = pos < 0 ? 0 : pos < (int64_t)table_width * page_size ? pos + 1 : table_width * page_size;
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

// The records of a token's ranges joined, a wave per (token, head): lane s fetches maximum and sum of range s (64 at most),
// and with them the first eight ranges' values leave, so that a merge of eight is one trip to memory.  A lane owns dimensions
// lane, lane + 64, .. (DIMS of them).
template <typename T, int DIMS>
__global__ __launch_bounds__(64) void attention_decode_int4_merge_kernel(const float* __restrict__ partial,
                                                                         const int* __restrict__ tok_list, int heads,
                                                                         int head_dim, int splits,
                                                                         T* __restrict__ out, int64_t out_stride) {
  const int n = blockIdx.x, head = blockIdx.y, lane = threadIdx.x;
  const int stride = head_dim + 2;
  const float* records = partial + ((int64_t)n * heads + head) * splits * stride;
  const int own = lane < splits ? lane : 0;
  float m = records[own * stride + head_dim], l = records[own * stride + head_dim + 1];
  float part[8][DIMS], value[DIMS];
  auto ask = [&](int from) {
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
      for (int k = 0; k < DIMS; ++k)
        part[j][k] = records[(from + j < splits ? from + j : 0) * stride + (64 * k + lane < head_dim ? 64 * k + lane : 0)];
  };
  ask(0);
  const int t = tok_list ? tok_list[n] : n;
  if (lane >= splits) {
    m = -INFINITY;
    l = 0.f;
  }
  const float high = wave_max(m);
  const float weight = m == -INFINITY ? 0.f : exp2_fast<T>(m - high);
  const float total = wave_sum(l * weight);
#pragma unroll
  for (int k = 0; k < DIMS; ++k) value[k] = 0.f;
  for (int from = 0; from < splits; from += 8) {
    if (from > 0) ask(from);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float w = read_lane(weight, (from + j) & 63);        // (0 for ranges beyond the last)
#pragma unroll
      for (int k = 0; k < DIMS; ++k) value[k] = from + j < splits ? fmaf(part[j][k], w, value[k]) : value[k];
    }
  }
#pragma unroll
  for (int k = 0; k < DIMS; ++k) {
    const int d = 64 * k + lane;
    if (d < head_dim)
      out[t * out_stride + (int64_t)head * head_dim + d] = from_float<T>(total == 0.f ? 0.f : value[k] / total);
  }
}

extern "C" int ps_attention_decode_int4(const void* q, int64_t q_stride, const void* new_k, const void* new_v,
                                        int64_t new_k_stride, int64_t new_v_stride, const void* k_pool,
                                        const void* v_pool, void* out, int64_t out_stride, float* partial,
                                        int64_t partial_floats, const int* tok_list, const int* tok_item,
                                        const int* tok_pos, const int* tables, int table_width, int count, int heads,
                                        int kv_heads, int head_dim, int page_size, int num_pages, float scale, int window,
                                        int splits, const float* sink, float softcap, int dtype, void* stream) {
  PS_REQUIRE(count >= 0 && heads > 0 && kv_heads > 0 && page_size > 0 && num_pages > 0 && table_width > 0,
             "ps_attention_decode_int4: bad sizes");
  PS_REQUIRE(heads % kv_heads == 0 && heads <= 65535,
             "ps_attention_decode_int4: heads (%d) must be a multiple of kv_heads (%d), 65535 at most", heads, kv_heads);
  PS_REQUIRE(head_dim > 0 && head_dim <= 256, "ps_attention_decode_int4: head_dim %d must lie in 1..256", head_dim);
  PS_REQUIRE(page_size % 8 == 0 && page_size <= (1 << 20),
             "ps_attention_decode_int4: pages of a cache in 4 bits hold a multiple of 8 keys, not %d", page_size);
  PS_REQUIRE((int64_t)table_width * page_size < ((int64_t)1 << 30),
             "ps_attention_decode_int4: block tables of %d pages of %d keys", table_width, page_size);
  PS_REQUIRE(splits >= 1 && splits <= 64, "ps_attention_decode_int4: 1 to 64 ranges, not %d", splits);
  PS_REQUIRE(dtype == PS_F32 || dtype == PS_BF16, "ps_attention_decode_int4: unknown dtype %d", dtype);
  PS_REQUIRE(splits == 1 || (partial != nullptr &&
                             partial_floats >= (int64_t)count * heads * splits * (head_dim + 2)),
             "ps_attention_decode_int4: %lld floats of scratch are too few for %d ranges", (long long)partial_floats,
             splits);
  PS_REQUIRE((new_k == nullptr) == (new_v == nullptr) &&
                 (new_k == nullptr || (dtype == PS_BF16 && scale > 0.f && tok_item == nullptr && tok_list == nullptr)),
             "ps_attention_decode_int4: rows to be stored are keys and values in bfloat16, a request's to a token, under a "
             "positive scale");
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
                       (kv_group + block_heads - 1) / block_heads, block_heads, head_dim, page_size, page_shift,
                       num_pages, window, splits,
                       wide_q, scale * 1.4426950408889634f, softcap * 1.4426950408889634f, sink,
                       (const bf16_t*)new_k, (const bf16_t*)new_v, new_k_stride, new_v_stride};
    const int64_t blocks = (int64_t)count * kv_heads * a.parts;
    int waves = splits == 1 && blocks <= ps_compute_units() && groups <= 4 && block_heads * groups <= 32 ? 8 : 4;
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
#define PS_LAUNCH_M4(T, DIMS)                                                                                      \
  hipLaunchKernelGGL((attention_decode_int4_merge_kernel<T, DIMS>), dim3(count, heads), dim3(64), 0, s, partial, \
                     tok_list, heads, head_dim, splits, (T*)out, out_stride)
#define PS_LAUNCH_M4T(T)                        \
  do {                                          \
    if (head_dim <= 64) PS_LAUNCH_M4(T, 1);     \
    else if (head_dim <= 128) PS_LAUNCH_M4(T, 2); \
    else PS_LAUNCH_M4(T, 4);                    \
  } while (0)
    if (dtype == PS_F32) PS_LAUNCH_M4T(float);
    else PS_LAUNCH_M4T(bf16_t);
#undef PS_LAUNCH_M4T
#undef PS_LAUNCH_M4
    PS_CHECK_LAUNCH("ps_attention_decode_int4(merge)");
  }
  return 0;
}
