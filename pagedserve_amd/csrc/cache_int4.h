// Keys and values held in 4 bits: the form of a page, and what a code stands for.
//
// 32 consecutive head dimensions of one key (or value) of one head are a group with one step d; the
// last group of a head may be shorter and is filled up with zeros.  An element x is held as
//   code = clamp(rint(x / d), -8, 7) + 8,  and stands for (code - 8) d.
// With e the element of largest magnitude (the positive one where both signs have it), d = -e / 8
// rounded to five significant bits, ties to even: e itself is code 0 up to that rounding, all sixteen codes are
// used, and (code - 8) d, three bits times five, is a bfloat16 number without rounding, so that
// attention over this cache is attention over a bfloat16 cache which holds these values.  (Root mean
// square error of normal values 8.62 % of theirs, 8.60 % with the step unrounded; codes -7 .. 7 of the magnitude 9.7 %.)
// A step that is still below the normal floats becomes 0, and the group zeros; a group that holds an infinity or a NaN
// gets a NaN for its step and is NaN as a whole, as a cache in the model's type would show it.
//
// A page of one head: the codes of its keys, 16 G bytes each (G groups), then their steps, G bfloat16
// each: 18 G bytes a key, 4.5 bits a value.  Pages hold a multiple of 8 keys, so both parts begin at multiples of
// 16 bytes.  Within a key's row the 32-bit word c G + g (c = 0..3) holds dimensions 32 g + 8 c .. + 7,
// the lowest bits first; within a value's row byte n G + g (n = 0..15) holds dimensions 32 g + 2 n
// and the next.  So lane c of four that share a key finds its operands of all groups' products over dimensions side by
// side, and lane n of sixteen its dimensions of all groups, which are rows of the products over keys.
#pragma once

#include "common.h"

#define PS_INT4_GROUP 32

__host__ __device__ inline int int4_groups(int head_dim) { return (head_dim + PS_INT4_GROUP - 1) / PS_INT4_GROUP; }
__host__ __device__ inline int int4_row_bytes(int groups) { return 18 * groups; }

// Where the page of a head begins in its pool, in bytes.
__device__ inline int64_t int4_page_at(int page, int kv_heads, int kv_head, int page_size, int groups) {
  return ((int64_t)page * kv_heads + kv_head) * page_size * int4_row_bytes(groups);
}

// The word of a key's row with dimensions 8 w .. 8 w + 7 (w = 4 g + c), counted in bytes from the row's first.
__device__ inline int int4_key_word(int w, int groups) { return 4 * ((w & 3) * groups + (w >> 2)); }
// The byte of a value's row with dimensions 2 b and 2 b + 1 (b = 16 g + n).
__device__ inline int int4_value_byte(int b, int groups) { return (b & 15) * groups + (b >> 4); }

// The step of a group from its largest and its smallest element.
__device__ inline float int4_step(float high, float low) {
  const float e = high >= -low ? high : low;
  const uint32_t bits = __float_as_uint(e * -0.125f);
  uint32_t size = bits & 0x7fffffffu;
  size = (size + 0x3ffffu + ((size >> 19) & 1u)) & ~0x7ffffu;       // five significant bits, ties to even
  if (size > 0x7df80000u) size = 0x7df80000u;                       // 31/16 2^124, eight times which is a finite float
  if (size < 0x00800000u) size = 0x00800000u;
  // (from 2^-123 (1 - 2^-6) on, five bits make an eighth of it the smallest normal float)
  return fabsf(e) < __uint_as_float(0x01fc0000u) ? 0.f : __uint_as_float(size | (bits & 0x80000000u));
}

// The codes of eight numbers, less 8, under a step other than 0; BF16: numbers of 8 significant bits.
//
// The product with the step's reciprocal, which may be off in its last place, is x / d but for some last places.  Of
// numbers of 8 bits the quotient lies a 2^9th of itself or more from a half or on it: one correction by the remainder
// makes it exact there, and rounding it gives the code.  (Not where the remainder is below the normal floats.)  Else the
// whole number nearest to the product is taken, and the remainder of that, at most about half a step, is exact (a
// multiple of the last place of x or of d, whichever is lower, and within 24 bits of it) and decides, ties to even.
template <bool BF16>
__device__ inline void int4_codes(const float* x, float step, float* codes) {
  const float inverse = __builtin_amdgcn_rcpf(step), half = fabsf(step) * 0.5f;
  if (BF16 && half >= 7.8886091e-31f) {       // 2^-100
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float ratio = x[i] * inverse;
      codes[i] = rintf(fmaf(fmaf(-ratio, step, x[i]), inverse, ratio));
    }
  } else {
    float rest[8], most = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      codes[i] = rintf(x[i] * inverse);
      rest[i] = fmaf(-codes[i], step, x[i]);
      most = fmaxf(most, fabsf(rest[i]));
    }
    if (most >= half) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const bool odd = fabsf(fmaf(-2.f, rintf(codes[i] * 0.5f), codes[i])) == 1.f;
        const bool off = (fabsf(rest[i]) > half) | ((fabsf(rest[i]) == half) & odd);
        const float by = (rest[i] > 0.f) == (step > 0.f) ? 1.f : -1.f;
        codes[i] += off ? by : 0.f;
      }
    }
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) codes[i] = fminf(fmaxf(codes[i], -8.f), 7.f);
}

// The quarter of a value's row holds byte i of group g's word as its byte i G + g: from the words of the groups, and back.
template <int G, bool BACK>
__device__ inline void int4_turn_bytes(uint32_t* words) {
  uint32_t turned[G];
#pragma unroll
  for (int g = 0; g < G; ++g) turned[g] = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int g = 0; g < G; ++g) {
      const int at = i * G + g;
      if (BACK) turned[g] |= (words[at / 4] >> (8 * (at % 4)) & 0xffu) << (8 * i);
      else turned[at / 4] |= (words[g] >> (8 * i) & 0xffu) << (8 * (at % 4));
    }
#pragma unroll
  for (int g = 0; g < G; ++g) words[g] = turned[g];
}

// N words from or to an address that is a multiple of the largest power of two in 4 N bytes, 16 at most.
template <int N>
__device__ inline void int4_load_words(const uint8_t* from, uint32_t* words) {
  if constexpr (N % 4 == 0) {
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {
      const uint4 v = reinterpret_cast<const uint4*>(from)[i];
      words[4 * i] = v.x;
      words[4 * i + 1] = v.y;
      words[4 * i + 2] = v.z;
      words[4 * i + 3] = v.w;
    }
  } else if constexpr (N % 2 == 0) {
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
      const uint2 v = reinterpret_cast<const uint2*>(from)[i];
      words[2 * i] = v.x;
      words[2 * i + 1] = v.y;
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) words[i] = reinterpret_cast<const uint32_t*>(from)[i];
  }
}
template <int N>
__device__ inline void int4_store_words(uint8_t* to, const uint32_t* words) {
  if constexpr (N % 4 == 0) {
#pragma unroll
    for (int i = 0; i < N / 4; ++i)
      reinterpret_cast<uint4*>(to)[i] = make_uint4(words[4 * i], words[4 * i + 1], words[4 * i + 2], words[4 * i + 3]);
  } else if constexpr (N % 2 == 0) {
#pragma unroll
    for (int i = 0; i < N / 2; ++i) reinterpret_cast<uint2*>(to)[i] = make_uint2(words[2 * i], words[2 * i + 1]);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) reinterpret_cast<uint32_t*>(to)[i] = words[i];
  }
}

// What lane c of four that share a row holds of it: the words of its codes in the page's order and the row's steps (the
// lane's 8 dimensions of each group in x; BF16: numbers of 8 bits).
template <int G, bool BF16>
__device__ inline void int4_code_row(const float (&x)[G][8], bool values, uint32_t (&words)[G],
                                     uint32_t (&steps)[(G + 1) / 2]) {
#pragma unroll
  for (int g = 0; g < G; ++g) {
    float high = x[g][0], low = x[g][0], finite = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      high = fmaxf(high, x[g][i]);
      low = fminf(low, x[g][i]);
      finite = fmaf(x[g][i], 0.f, finite);                   // (NaN by an infinity or a NaN, which an extreme passes over)
    }
    high = lanes_max<4>(high);
    low = -lanes_max<4>(-low);
    const bool all_finite = lanes_max<4>(finite == 0.f ? 0.f : 1.f) == 0.f;
    const float step = all_finite ? int4_step(high, low) : __uint_as_float(0x7fc00000u);
    words[g] = 0x88888888u;
    if (all_finite && step != 0.f) {
      float codes[8];
      int4_codes<BF16>(x[g], step, codes);
      uint32_t halves[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        // four codes less 8 as the digits of a number to the base of 16, and 8 to each
        float digits = 0.f;
#pragma unroll
        for (int i = 3; i >= 0; --i) digits = fmaf(digits, 16.f, codes[4 * h + i]);
        halves[h] = (uint32_t)(digits + 34952.f);
      }
      words[g] = halves[0] | halves[1] << 16;
    }
    const uint32_t bits = __float_as_uint(step) >> 16;
    steps[g / 2] = g % 2 ? steps[g / 2] | bits << 16 : bits;
  }
  if (values) int4_turn_bytes<G, false>(words);
}

// That into place `within` of a page.
template <int G>
__device__ inline void int4_store_row(uint8_t* page, int page_size, int within, int c, const uint32_t (&words)[G],
                                      const uint32_t (&steps)[(G + 1) / 2]) {
  int4_store_words<G>(page + within * (16 * G) + c * (4 * G), words);
  if (c == 0) {
    uint8_t* to = page + page_size * (16 * G) + within * (2 * G);
    if constexpr (G % 2 == 0) {
      int4_store_words<G / 2>(to, steps);
    } else {
#pragma unroll
      for (int g = 0; g < G; ++g) reinterpret_cast<uint16_t*>(to)[g] = (uint16_t)(steps[g / 2] >> (16 * (g % 2)));
    }
  }
}
