// Log probabilities of given tokens, with the row's entropy, the token's rank and the most likely alternatives.
//
//   logprob = x_t - lse,  lse = M + log Z,  M = max x,  Z = sum e^(x - M)
//   entropy = log Z - T / Z,  T = sum (x - M) e^(x - M)
//   rank    = the number of logits above x_t, or equal to it at a lower id
//   alternatives: the `top` highest logits, the lower id first among equals
//
// A block reads its part of a row once, 16 bytes to a load.  Every thread keeps a running maximum with the sums scaled to it
// (in float), the count for the rank and where its own highest logit lies.  The `top`-th highest of the threads' highest
// logits, T, bounds the alternatives from below, and about `top` threads have any logit that reaches it: the shares of
// these are read again (out of the cache), a share by a wave, and what reaches T goes to one wave, which sorts.  So
// alternatives cost no second pass over the row.  Logits and ids are compared as one 64-bit number, in which no two are
// equal: a row of equal logits costs a second round for that bound, no more, and the results do not depend on the order in
// which candidates arrive.
//
// Long rows are cut into parts, whose records a second launch joins.
//
// Bound by memory where there are rows enough: 512 float rows of 50,257 with 20 alternatives in 25.3 us, 4.1 TB/s, 83 % of a
// large copy's rate (without alternatives 22.6); by the chain of maxima, bound, candidates and the joining launch where
// there are few: 8 rows with 5 alternatives 7.1 + 4.3 us.
#include <math.h>

#include "common.h"
#include "pagedserve_hip.h"

#define LP_THREADS 512
#define LP_WAVES (LP_THREADS / PS_WAVE)
#define LP_AHEAD 4                                           // loads of a thread at a time
#define LP_MAX_TOP 32
#define LP_CANDIDATES 4096                                   // what LDS holds of them
#define LP_SHARE 120                                         // logits of one thread, at most, but for two at the edges
#define LP_PART (LP_SHARE * LP_THREADS)
#define LP_OWNERS 33                                         // threads whose shares are read again
static_assert((LP_SHARE + 2) * LP_OWNERS <= LP_CANDIDATES && LP_MAX_TOP <= LP_OWNERS, "no part has more candidates than LDS holds");
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

// The word of lane (l ^ OFFSET): within rows of 16 lanes by the vector unit, between rows and halves by their swaps.
template <int OFFSET>
__device__ inline uint32_t lp_other(uint32_t v, int lane) {
  if constexpr (OFFSET == 1) return __builtin_amdgcn_update_dpp(0, v, 0xB1, 0xF, 0xF, true);
  else if constexpr (OFFSET == 2) return __builtin_amdgcn_update_dpp(0, v, 0x4E, 0xF, 0xF, true);
  else if constexpr (OFFSET == 4) return __builtin_amdgcn_ds_swizzle(v, 0x101F);
  else if constexpr (OFFSET == 8) return __builtin_amdgcn_update_dpp(0, v, 0x128, 0xF, 0xF, true);
  else if constexpr (OFFSET == 16) {
    const auto both = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    return lane & 16 ? both[0] : both[1];
  } else {
    const auto both = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return lane & 32 ? both[0] : both[1];
  }
}
template <int OFFSET>
__device__ inline uint32_t lp_exchange(uint32_t v, int lane) { return lp_other<OFFSET>(v, lane); }
template <int OFFSET>
__device__ inline uint64_t lp_exchange(uint64_t v, int lane) {
  return (uint64_t)lp_other<OFFSET>((uint32_t)(v >> 32), lane) << 32 | lp_other<OFFSET>((uint32_t)v, lane);
}
// Rounds of comparisons at falling distances: lanes of `high_first` runs keep the higher number in front.
template <int OFFSET, typename N>
__device__ inline N lp_merge(N v, int lane, bool high_first) {
  const N other = lp_exchange<OFFSET>(v, lane);
  v = (v > other) == (((lane & OFFSET) == 0) == high_first) ? v : other;
  if constexpr (OFFSET > 1) v = lp_merge<OFFSET / 2>(v, lane, high_first);
  return v;
}
// The wave's 64 numbers, highest first.
template <typename N>
__device__ inline N lp_sort(N v, int lane) {
  v = lp_merge<1>(v, lane, (lane & 2) == 0);
  v = lp_merge<2>(v, lane, (lane & 4) == 0);
  v = lp_merge<4>(v, lane, (lane & 8) == 0);
  v = lp_merge<8>(v, lane, (lane & 16) == 0);
  v = lp_merge<16>(v, lane, (lane & 32) == 0);
  return lp_merge<32>(v, lane, true);
}
// The 64 highest of two sorted 64, sorted.
template <typename N>
__device__ inline N lp_join(N a, N b, int lane) {
  N back;
  if constexpr (sizeof(N) == 8) back = __shfl((unsigned long long)b, 63 - lane, 64);
  else back = __shfl(b, 63 - lane, 64);
  return lp_merge<32>(a > back ? a : back, lane, true);
}

// The waves' sorted lists joined; wave 0 has the 64 highest of all.
template <int HALF, typename N>
__device__ inline N lp_block_join(N list, N (&lists)[HALF][64], int wave, int lane) {
#pragma unroll
  for (int half = HALF; half > 0; half /= 2) {
    if (wave >= half && wave < 2 * half) lists[wave - half][lane] = list;
    __syncthreads();
    if (wave < half) list = lp_join(list, lists[wave][lane], lane);
    __syncthreads();
  }
  return list;
}

// A part's sums: maximum, sum and weighted sum (in units of log 2, scaled to the maximum), logits ahead of the token.
struct LpSums {
  float m, z, t;
  int ahead;
};
// Those of all lanes (a lane without any: minus infinity and zeros), in every lane.
__device__ inline LpSums lp_wave_sums(const LpSums s) {
  const float m = wave_max(s.m);
  // (a state without a finite maximum has sums of 0, or of no number)
  const float down = s.m == -INFINITY ? 0.f : (s.m - m) * 1.4426950408889634f;
  const float c = __builtin_amdgcn_exp2f(down);
  const float z = s.z * c, t = c * fmaf(s.z, fmaxf(down, -200.f), s.t);
  int ahead = s.ahead;
#pragma unroll
  for (int offset = 1; offset < 64; offset *= 2) ahead += __shfl_xor(ahead, offset, 64);
  return LpSums{m, wave_sum(z), wave_sum(t), ahead};
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

// What lies in one load of 16 bytes.
template <typename T>
struct LpVector {
  static constexpr int COUNT = 16 / sizeof(T);
  uint4 raw;
  __device__ inline void load(const T* p) { raw = *reinterpret_cast<const uint4*>(p); }
  __device__ inline float at(int i) const {
    const uint32_t words[4] = {raw.x, raw.y, raw.z, raw.w};
    if constexpr (sizeof(T) == 4) return __uint_as_float(words[i]);
    else return __uint_as_float(i & 1 ? words[i / 2] & 0xffff0000u : words[i / 2] << 16);
  }
};

// The next float below (of a number; minus infinity and NaN stay).
__device__ inline float lp_below(float x) {
  const uint32_t bits = __float_as_uint(x);
  if (!(x > -INFINITY)) return x;
  if ((bits & 0x7fffffffu) == 0) return __uint_as_float(0x80000001u);
  return __uint_as_float(bits & 0x80000000u ? bits + 1 : bits - 1);
}

template <typename T>
__global__ __launch_bounds__(LP_THREADS) void logprobs_kernel(const T* __restrict__ logits, int64_t ld, int vocab,
                                                              const int* __restrict__ tokens, const LpOut out,
                                                              int parts, int part_size, float* __restrict__ partial) {
  typedef LpVector<T> Vector;
  constexpr int V = Vector::COUNT, AHEAD = LP_AHEAD;
  __shared__ uint32_t s_highs[LP_WAVES / 2][64];
  __shared__ uint64_t s_lists[LP_WAVES / 2][64];
  __shared__ uint64_t s_found[LP_CANDIDATES];
  __shared__ uint64_t s_bound;
  __shared__ int s_count, s_owners;
  __shared__ int s_owner[LP_OWNERS];
  __shared__ LpSums s_sums[LP_WAVES];
  const int row = blockIdx.x, part = blockIdx.y;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const T* x = logits + row * ld;
  const int begin = part * part_size;
  const int end = begin + part_size < vocab ? begin + part_size : vocab;
  // a few logits in front of the first whole 16 bytes, the vectors, a few behind
  const int off = (int)((reinterpret_cast<uintptr_t>(x + begin) & 15) / sizeof(T));
  const int lead = off == 0 ? 0 : (V - off < end - begin ? V - off : end - begin);
  const int first = begin + lead;
  const int vectors = end > first ? (end - first) / V : 0;
  const int behind = first + vectors * V;
  const int token = tokens ? tokens[row] : -1;
  const bool is_token = token >= 0 && token < vocab;
  const float given = is_token ? to_float(x[token]) : 0.f;
  // (more likely than the token: above it; equal to it, which is above the next float below, at a lower id)
  const float above = is_token ? given : INFINITY, equal = is_token ? lp_below(given) : INFINITY;
  const bool lowest = is_token && given == -INFINITY;
  if (tid == 0) s_count = s_owners = 0;

  LpSums s{-INFINITY, 0.f, 0.f, 0};
  int best_id = 0x7fffffff;
  auto add = [&](float v) {
    const float d = (v - s.m) * 1.4426950408889634f;
    const float e = __builtin_amdgcn_exp2f(d);
    s.z += e;
    s.t = fmaf(e, fmaxf(d, -200.f), s.t);
  };
  auto raise = [&](float m) {      // to a maximum above the one so far
    const float down = s.m == -INFINITY ? 0.f : (s.m - m) * 1.4426950408889634f;
    const float c = __builtin_amdgcn_exp2f(down);
    s.t = c * fmaf(s.z, fmaxf(down, -200.f), s.t);
    s.z *= c;
    s.m = m;
  };
  auto take_one = [&](int i) {
    const float v = to_float(x[i]);
    s.ahead += v > (i < token ? equal : above);
    if (v > s.m || (v == -INFINITY && best_id == 0x7fffffff)) {
      if (v > s.m) raise(v);
      best_id = i;
    }
    if (s.m != -INFINITY || v != v) add(v);
  };
  if (tid < lead) take_one(begin + tid);
  for (int at = tid; at < vectors; at += AHEAD * LP_THREADS) {
    Vector in[AHEAD];
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      const int j = at + u * LP_THREADS;
      in[u].load(x + first + (int64_t)(j < vectors ? j : at) * V);
    }
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      const int j = at + u * LP_THREADS;
      if (j >= vectors) break;
      const int id = first + j * V;
      float high = in[u].at(0);
#pragma unroll
      for (int i = 1; i < V; ++i) high = fmaxf(high, in[u].at(i));
      if (high > s.m) {
        raise(high);
#pragma unroll
        for (int i = V - 1; i >= 0; --i)
          if (in[u].at(i) == high) best_id = id + i;
      }
      if (is_token) {
        // (one bound for a vector but for the one that the token lies in)
        const float bound = id < token ? equal : above;
        const bool split = id < token && token < id + V;
#pragma unroll
        for (int i = 0; i < V; ++i) s.ahead += in[u].at(i) > (split && id + i >= token ? above : bound);
      }
      if (s.m == -INFINITY) {
        // nothing but minus infinity so far, or NaN
#pragma unroll
        for (int i = V - 1; i >= 0; --i) {
          if (in[u].at(i) != in[u].at(i)) s.z = in[u].at(i);
          else if (best_id > id + i) best_id = id + i;
        }
      } else {
#pragma unroll
        for (int i = 0; i < V; ++i) add(in[u].at(i));
      }
    }
  }
  if (behind + tid < end) take_one(behind + tid);
  uint64_t best = best_id == 0x7fffffff ? 0 : lp_key(s.m, best_id);
  if (lowest) {
    // every token in front that is a number is as likely; (rare: counted apart)
    s.ahead = 0;
    for (int i = begin + tid; i < end; i += LP_THREADS) {
      const float v = to_float(x[i]);
      s.ahead += v > given || (v == given && i < token);
    }
  }
  s = lp_wave_sums(s);
  if (lane == 0) s_sums[wave] = s;
  if (out.top > 0) {
    // the bound by the logits alone, and who reaches it: `top` threads, more only where logits are equal there
    uint32_t high = lp_sort((uint32_t)(best >> 32), lane);
    high = lp_block_join(high, s_highs, wave, lane);
    if (wave == 0 && lane == out.top - 1) s_bound = (uint64_t)high << 32;
    __syncthreads();
    if (best != 0 && best >= s_bound) {
      const int slot = atomicAdd(&s_owners, 1);
      if (slot < LP_OWNERS) s_owner[slot] = tid;
    }
    __syncthreads();
    if (s_owners > LP_OWNERS) {
      // many equal ones: by logits and ids, of which no two are equal, it is `top` threads at most
      uint64_t list = lp_sort(best, lane);
      list = lp_block_join(list, s_lists, wave, lane);
      if (wave == 0 && lane == out.top - 1) s_bound = list;
      if (tid == 0) s_owners = 0;
      __syncthreads();
      if (best != 0 && best >= s_bound) s_owner[atomicAdd(&s_owners, 1)] = tid;
      __syncthreads();
    }
    const uint64_t bound = s_bound;
    const int owners = s_owners;
    for (int w = wave; w < owners; w += LP_WAVES) {
      const int owner = s_owner[w];
      auto offer = [&](float v, int id) {
        const uint64_t key = lp_key(v, id);
        if (v == v && key >= bound) s_found[atomicAdd(&s_count, 1)] = key;
      };
      const int j = owner + lane * LP_THREADS;
      if (j < vectors) {
        Vector in;
        in.load(x + first + (int64_t)j * V);
#pragma unroll
        for (int i = 0; i < V; ++i) offer(in.at(i), first + j * V + i);
      }
      if (lane == 62 && owner < lead) offer(to_float(x[begin + owner]), begin + owner);
      if (lane == 63 && behind + owner < end) offer(to_float(x[behind + owner]), behind + owner);
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

// The records of a row's parts: eight waves join the parts' alternatives, a part after the other each, then with each other.
template <typename T>
__global__ __launch_bounds__(512) void logprobs_join_kernel(const T* __restrict__ logits, int64_t ld, int vocab,
                                                                   const int* __restrict__ tokens, const LpOut out,
                                                                   int parts, const float* __restrict__ partial) {
  constexpr int WAVES = 8;
  __shared__ uint64_t s_lists[WAVES / 2][64];
  const int row = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int token = tokens ? tokens[row] : -1;
  const float given = token >= 0 && token < vocab ? to_float(logits[row * ld + token]) : 0.f;
  const float* records = partial + (int64_t)row * parts * lp_record(out.top);
  uint64_t list = 0;
  if (out.top > 0) {
    for (int p = wave; p < parts; p += WAVES) {
      const float* r = records + p * lp_record(out.top) + 4;
      uint64_t more = 0;
      if (lane < out.top) more = __float_as_uint(r[2 * lane]) | (uint64_t)__float_as_uint(r[2 * lane + 1]) << 32;
      list = p == wave ? more : lp_join(list, more, lane);
    }
    list = lp_block_join(list, s_lists, wave, lane);
  }
  if (wave > 0) return;
  LpSums s{-INFINITY, 0.f, 0.f, 0};
  if (lane < parts) {
    const float* r = records + lane * lp_record(out.top);
    s = LpSums{r[0], r[1], r[2], (int)__float_as_uint(r[3])};
  }
  lp_finish(lp_wave_sums(s), list, row, token, vocab, given, out, lane);
}

// Parts of a row: at least as many as LDS holds the candidates of, and where the rows leave most units idle as many as come
// to a block per unit, of 4,096 logits or more, 16 at most.  (One unit takes in some 30 GB/s: 8 rows of 50,257 in 13 parts and in
// one, with 5 alternatives 10.7 and 14.6 us, without 5.8 and 11.3; 64 rows in 4 parts 13.2 and 16.3; 256 rows in 2
// parts 22.4 and 20.7.)
static int lp_parts(int rows, int vocab) {
  const int least = (vocab - 1) / LP_PART + 1;
  int wanted = ps_compute_units() / (rows > 0 ? rows : 1);
  if (wanted > vocab / 4096 + 1) wanted = vocab / 4096 + 1;
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
  PS_REQUIRE(rows >= 0 && vocab > 0 && (ld >= vocab || ld == 0), "%s: bad sizes", who);     // (0: one row for all tokens)
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
#define PS_LAUNCH_LP(T)                                                                                           \
  do {                                                                                                            \
    hipLaunchKernelGGL((logprobs_kernel<T>), dim3(rows, parts), dim3(LP_THREADS), 0, s, (const T*)logits, ld,    \
                       vocab, tokens, out, parts, part_size, partial);                                            \
    if (parts > 1)                                                                                                \
      hipLaunchKernelGGL(logprobs_join_kernel<T>, dim3(rows), dim3(512), 0, s, (const T*)logits, ld, vocab,       \
                         tokens, out, parts, partial);                                                            \
  } while (0)
  if (dtype == PS_F32) PS_LAUNCH_LP(float);
  else PS_LAUNCH_LP(bf16_t);
#undef PS_LAUNCH_LP
  PS_CHECK_LAUNCH(who);
  return 0;
}
