// Log probabilities of given tokens, with the row's entropy, the token's rank and the most likely alternatives.
//
//   logprob = x_t - lse,  lse = M + log Z,  M = max x,  Z = sum e^(x - M)
//   entropy = log Z - T / Z,  T = sum (x - M) e^(x - M)
//   rank    = the number of logits above x_t, or equal to it at a lower id
//   alternatives: the `top` highest logits, the lower id first among equals
//
// A block reads its part of a row once.  Every thread keeps a running maximum with the sums scaled to it (in float),
// the count for the rank and where its own highest logit lies.  The `top`-th highest of the threads' highest logits, T,
// bounds the alternatives from below, and at most `top` threads have any logit that reaches it: these alone read
// their share again (out of the cache) and hand what reaches T to one wave, which sorts.  So alternatives cost no
// second pass over the row.  Logits and ids are compared as one 64-bit number, in which no two are equal: a row of
// equal logits is no special case, and the results do not depend on the order in which candidates arrive.
//
// Long rows are cut into parts (also where few rows would leave most units idle), whose records a second launch joins.
#include <math.h>

#include "common.h"
#include "pagedserve_hip.h"

#define LP_THREADS 512
#define LP_WAVES (LP_THREADS / PS_WAVE)
#define LP_MAX_TOP 32
#define LP_CANDIDATES 4096                                   // what LDS holds of them
#define LP_SHARE (LP_CANDIDATES / LP_MAX_TOP)                // logits of one thread, at most
#define LP_PART (LP_SHARE * LP_THREADS)                      // so no part can have more candidates than LDS holds
#define LP_MAX_PARTS 64

// A logit and its id as one number: higher for a higher logit, then for a lower id.
__device__ inline uint64_t lp_key(float x, int id) {
  const uint32_t bits = __float_as_uint(x + 0.f);            // (-0 is 0)
  const uint32_t ordered = bits & 0x80000000u ? ~bits : bits | 0x80000000u;
  return (uint64_t)ordered << 32 | (uint32_t)~id;
}
__device__ inline int lp_id(uint64_t key) { return (int)~(uint32_t)key; }
__device__ inline float lp_logit(uint64_t key) {
  const uint32_t ordered = (uint32_t)(key >> 32);
  return __uint_as_float(ordered & 0x80000000u ? ordered & 0x7fffffffu : ~ordered);
}

__device__ inline uint64_t lp_exchange(uint64_t v, int offset) { return __shfl_xor((unsigned long long)v, offset, 64); }

// The wave's 64 numbers, highest first.
__device__ inline uint64_t lp_sort(uint64_t v, int lane) {
#pragma unroll
  for (int size = 2; size <= 64; size *= 2)
#pragma unroll
    for (int offset = size / 2; offset > 0; offset /= 2) {
      const uint64_t other = lp_exchange(v, offset);
      const bool keep_high = ((lane & offset) == 0) == ((lane & size) == 0);
      v = (v > other) == keep_high ? v : other;
    }
  return v;
}
// The 64 highest of two sorted 64, sorted.
__device__ inline uint64_t lp_join(uint64_t a, uint64_t b, int lane) {
  const uint64_t back = __shfl((unsigned long long)b, 63 - lane, 64);
  uint64_t v = a > back ? a : back;
#pragma unroll
  for (int offset = 32; offset > 0; offset /= 2) {
    const uint64_t other = lp_exchange(v, offset);
    v = (v > other) == ((lane & offset) == 0) ? v : other;
  }
  return v;
}

// A part's sums: maximum, sum and weighted sum (in units of log 2, scaled to the maximum), logits ahead of the token.
struct LpSums {
  float m, z, t;
  int ahead;
};
__device__ inline LpSums lp_add(const LpSums a, const LpSums b) {
  const float m = fmaxf(a.m, b.m);
  LpSums out{m, 0.f, 0.f, a.ahead + b.ahead};
  // (a state without a finite maximum has sums of 0, or of no number)
  const float da = a.m == -INFINITY ? 0.f : (a.m - m) * 1.4426950408889634f;
  const float db = b.m == -INFINITY ? 0.f : (b.m - m) * 1.4426950408889634f;
  const float ca = exp2f(da), cb = exp2f(db);
  out.z = a.z * ca + b.z * cb;
  out.t = ca * fmaf(a.z, fmaxf(da, -200.f), a.t) + cb * fmaf(b.z, fmaxf(db, -200.f), b.t);
  return out;
}

__device__ inline LpSums lp_wave_sums(LpSums s) {
#pragma unroll
  for (int offset = 1; offset < 64; offset *= 2) {
    const LpSums other{__shfl_xor(s.m, offset, 64), __shfl_xor(s.z, offset, 64), __shfl_xor(s.t, offset, 64),
                       __shfl_xor(s.ahead, offset, 64)};
    s = lp_add(s, other);
  }
  return s;
}

struct LpOut {
  float* logprobs;
  float* entropy;
  int* ranks;
  int* top_ids;
  float* top_logprobs;
  int top;
};

// What a row's sums and its highest logits come to; one wave.
__device__ inline void lp_finish(const LpSums s, uint64_t best, int row, int token, int vocab, float given,
                                 const LpOut out, int lane) {
  const float log_z = logf(s.z);
  if (lane == 0) {
    const bool is_token = token >= 0 && token < vocab;
    if (out.logprobs)
      out.logprobs[row] = is_token ? (given - s.m) - log_z : token == -1 ? 0.f : __uint_as_float(0x7fc00000u);
    if (out.entropy) out.entropy[row] = log_z - 0.6931471805599453f * (s.t / s.z);
    if (out.ranks) out.ranks[row] = is_token ? s.ahead : -1;
  }
  if (lane < out.top) {
    const bool found = best != 0;
    if (out.top_ids) out.top_ids[(int64_t)row * out.top + lane] = found ? lp_id(best) : -1;
    if (out.top_logprobs)
      out.top_logprobs[(int64_t)row * out.top + lane] =
          found ? (lp_logit(best) - s.m) - log_z : __uint_as_float(0x7fc00000u);
  }
}

// floats of one part's record: sums, then `top` numbers of 64 bits
__host__ __device__ inline int lp_record(int top) { return 4 + 2 * top; }

template <typename T>
__global__ __launch_bounds__(LP_THREADS) void logprobs_kernel(const T* __restrict__ logits, int64_t ld, int vocab,
                                                              const int* __restrict__ tokens, const LpOut out,
                                                              int parts, int part_size, float* __restrict__ partial) {
  __shared__ uint64_t s_lists[LP_WAVES / 2][64];
  __shared__ uint64_t s_found[LP_CANDIDATES];
  __shared__ uint64_t s_bound;
  __shared__ int s_count;
  __shared__ LpSums s_sums[LP_WAVES];
  const int row = blockIdx.x, part = blockIdx.y;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const T* x = logits + row * ld;
  const int begin = part * part_size;
  const int end = begin + part_size < vocab ? begin + part_size : vocab;
  const int token = tokens ? tokens[row] : -1;
  const bool is_token = token >= 0 && token < vocab;
  const float given = is_token ? to_float(x[token]) : 0.f;
  if (threadIdx.x == 0) s_count = 0;

  LpSums s{-INFINITY, 0.f, 0.f, 0};
  uint64_t best = 0;
  for (int i = begin + threadIdx.x; i < end; i += LP_THREADS) {
    const float v = to_float(x[i]);
    if (is_token) s.ahead += v > given || (v == given && i < token);
    const uint64_t key = lp_key(v, i);
    if (v == v && key > best) best = key;
    const float m = fmaxf(s.m, v);
    const float reference = m == -INFINITY ? 0.f : m;
    const float down = s.m == -INFINITY ? 0.f : (s.m - reference) * 1.4426950408889634f;
    const float c = exp2f(down);
    const float d = (v - reference) * 1.4426950408889634f;
    const float e = exp2f(d);
    s.t = c * fmaf(s.z, fmaxf(down, -200.f), s.t) + e * fmaxf(d, -200.f);
    s.z = s.z * c + e;
    s.m = m;
  }
  s = lp_wave_sums(s);
  if (lane == 0) s_sums[wave] = s;
  if (out.top > 0) {
    uint64_t list = lp_sort(best, lane);
#pragma unroll
    for (int half = LP_WAVES / 2; half > 0; half /= 2) {
      if (wave >= half && wave < 2 * half) s_lists[wave - half][lane] = list;
      __syncthreads();
      if (wave < half) list = lp_join(list, s_lists[wave][lane], lane);
      __syncthreads();
    }
    if (wave == 0 && lane == out.top - 1) s_bound = list;
    __syncthreads();
    const uint64_t bound = s_bound;
    if (best != 0 && best >= bound) {
      for (int i = begin + threadIdx.x; i < end; i += LP_THREADS) {
        const float v = to_float(x[i]);
        const uint64_t key = lp_key(v, i);
        if (v == v && key >= bound) s_found[atomicAdd(&s_count, 1)] = key;
      }
    }
  }
  __syncthreads();
  if (wave > 0) return;
  s = lane < LP_WAVES ? s_sums[lane] : LpSums{-INFINITY, 0.f, 0.f, 0};
  s = lp_wave_sums(s);
  uint64_t list = 0;
  const int count = s_count;
  for (int at = 0; at < count; at += 64) {
    const uint64_t more = lp_sort(at + lane < count ? s_found[at + lane] : 0, lane);
    list = at == 0 ? more : lp_join(list, more, lane);
  }
  if (parts == 1) {
    lp_finish(s, list, row, token, vocab, given, out, lane);
    return;
  }
  float* record = partial + ((int64_t)row * parts + part) * lp_record(out.top);
  if (lane == 0) {
    record[0] = s.m;
    record[1] = s.z;
    record[2] = s.t;
    record[3] = __uint_as_float(s.ahead);
  }
  if (lane < out.top) {
    record[4 + 2 * lane] = __uint_as_float((uint32_t)list);
    record[5 + 2 * lane] = __uint_as_float((uint32_t)(list >> 32));
  }
}

template <typename T>
__global__ __launch_bounds__(64) void logprobs_join_kernel(const T* __restrict__ logits, int64_t ld, int vocab,
                                                           const int* __restrict__ tokens, const LpOut out, int parts,
                                                           const float* __restrict__ partial) {
  const int row = blockIdx.x, lane = threadIdx.x;
  const int token = tokens ? tokens[row] : -1;
  const float given = token >= 0 && token < vocab ? to_float(logits[row * ld + token]) : 0.f;
  const float* records = partial + (int64_t)row * parts * lp_record(out.top);
  LpSums s{-INFINITY, 0.f, 0.f, 0};
  if (lane < parts) {
    const float* r = records + lane * lp_record(out.top);
    s = LpSums{r[0], r[1], r[2], (int)__float_as_uint(r[3])};
  }
  s = lp_wave_sums(s);
  uint64_t list = 0;
  if (out.top > 0) {
    for (int p = 0; p < parts; ++p) {
      const float* r = records + p * lp_record(out.top) + 4;
      uint64_t more = 0;
      if (lane < out.top) more = __float_as_uint(r[2 * lane]) | (uint64_t)__float_as_uint(r[2 * lane + 1]) << 32;
      list = p == 0 ? more : lp_join(list, more, lane);
    }
  }
  lp_finish(s, list, row, token, vocab, given, out, lane);
}

// Parts of a row: as many as LDS holds the candidates of, and for few rows more.
static int lp_parts(int rows, int vocab) {
  const int least = (vocab + LP_PART - 1) / LP_PART;
  int wanted = ps_compute_units() / (rows > 0 ? rows : 1);
  const int most = (vocab + 4095) / 4096;
  if (wanted > most) wanted = most;
  if (wanted > 16) wanted = 16;
  return wanted > least ? wanted : least;
}

extern "C" int64_t ps_logprob_scratch(int rows, int vocab, int top) {
  if (rows <= 0 || vocab <= 0 || top < 0 || top > LP_MAX_TOP) return 0;
  const int parts = lp_parts(rows, vocab);
  return parts == 1 ? 0 : (int64_t)rows * parts * lp_record(top);
}

extern "C" int ps_token_logprobs(const void* logits, int64_t ld, int rows, int vocab, const int* tokens,
                                 float* logprobs, float* entropy, int* ranks, int* top_ids, float* top_logprobs,
                                 int top, float* partial, int64_t partial_floats, int dtype, void* stream) {
  const char* who = "ps_token_logprobs";
  PS_REQUIRE(rows >= 0 && vocab > 0 && ld >= vocab, "%s: bad sizes", who);
  PS_REQUIRE(dtype == PS_F32 || dtype == PS_BF16, "%s: unknown dtype %d", who, dtype);
  PS_REQUIRE(top >= 0 && top <= LP_MAX_TOP && top <= vocab, "%s: 0 to %d alternatives out of a vocabulary of %d, not %d",
             who, LP_MAX_TOP, vocab, top);
  PS_REQUIRE((int64_t)vocab <= (int64_t)LP_PART * LP_MAX_PARTS, "%s: a vocabulary of %d is too large", who, vocab);
  if (rows == 0) return 0;
  const int parts = lp_parts(rows, vocab);
  PS_REQUIRE(parts == 1 || (partial != nullptr && partial_floats >= ps_logprob_scratch(rows, vocab, top)),
             "%s: %lld floats of scratch are too few", who, (long long)partial_floats);
  const int part_size = (vocab + parts - 1) / parts;
  const LpOut out{logprobs, entropy, ranks, top_ids, top_logprobs, top};
  hipStream_t s = (hipStream_t)stream;
#define PS_LAUNCH_LP(T)                                                                                          \
  do {                                                                                                           \
    hipLaunchKernelGGL(logprobs_kernel<T>, dim3(rows, parts), dim3(LP_THREADS), 0, s, (const T*)logits, ld, vocab, \
                       tokens, out, parts, part_size, partial);                                                  \
    if (parts > 1)                                                                                               \
      hipLaunchKernelGGL(logprobs_join_kernel<T>, dim3(rows), dim3(64), 0, s, (const T*)logits, ld, vocab, tokens, \
                         out, parts, partial);                                                                   \
  } while (0)
  if (dtype == PS_F32) PS_LAUNCH_LP(float);
  else PS_LAUNCH_LP(bf16_t);
#undef PS_LAUNCH_LP
  PS_CHECK_LAUNCH(who);
  return 0;
}
