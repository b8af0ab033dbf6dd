// Keys and values held in 4 bits: the form of a page, and what a code stands for.
//
// 32 consecutive head dimensions of one key (or value) of one head are a group with one step d; the
// last group of a head may be shorter and is filled up with zeros.  An element x is held as
//   code = clamp(rint(x / d), -8, 7) + 8,  and stands for (code - 8) d.
// With e the element of largest magnitude (the positive one where both signs have it), d = -e / 8
// rounded to five significant bits, ties to even: e itself is code 0 up to that rounding, all sixteen codes are
// used, and (code - 8) d, three bits times five, is a bfloat16 number without rounding, so that
// attention over this cache is attention over a bfloat16 cache which holds these values.  (Root mean
// square error of normal values 8.62 % of theirs, 8.60 % with the step unrounded; codes -7 .. 7 of the magnitude 9.7 %.)  A step that is still
// below the normal floats becomes 0, and the group zeros; a group that holds an infinity or a NaN
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
