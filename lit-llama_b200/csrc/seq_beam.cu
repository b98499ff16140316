// Beam search's selection: of a group's beams and the vocabulary the `count` largest of
//
//   value[w, v] = score[w] + x[w, v] - log sum_u exp x[w, u],    ties to the lowest w V + v
//
// Within a beam the order is that of its logits, so one pass over them gives the sum and each part's `count` largest, as keys of 64 bits: the logit as an integer of
// the same order, and what is left to the lowest index.  A block holds its part in registers, bf16 as it lies.  Its threads, by fours where few are wanted, have a largest
// value each; the count-th largest of these is a bound that at least `count` entries reach and few more (18 for 16 of 8192 at random), so these are found without a
// sort, and ranked by counting.  Where more than a list holds reach it, entries alike, keys take the place of values in the same steps: then they are all in `count`
// threads' entries.  A second launch, a block for a group of beams, does the same with the beams' parts, by values in 64 bits.  Scores and logits of different beams
// may be neighbours, or alike: where values are closer than what f32 has lost of their sums, these are formed again as whole numbers, which no order of the terms changes.
//
// A beam whose score or log-probabilities are no numbers (a score of -inf, a logit that is NaN or +inf, none above -inf) is out: its values are -inf.
//
// What bounds it: for many rows the latency of a block's steps (its loads, bound, sums, what reaches the bound, ranks) with four blocks on an SM, and an exponential for every
// logit: 48 x 8 beams of 100003 bf16, 16 of each group: 29 us for the parts, 2.7 TB/s, and 13 for the second launch by themselves; a call 36 where L2 has the logits, as it has
// those that a model's last product has just written, 56 where it has not.  Few beams: the two launches, 4 of 32000 in 4.5 and 5.9 us.
// (Parts of 8192 entries 32 us; keys of 64 bits compared throughout 94; blocks that stay and load the next part ahead 40, as fewer have room.)
#include <algorithm>

#include "seq_rows.cuh"

namespace b2l {
namespace beam {

constexpr int THREADS = 256, MOST_COUNT = 64, MOST_BEAMS = 64, LIST = 4096;
constexpr int MOST_VOCAB = 1 << 30;                          // places in a row, and behind it as far as a part goes, are 32-bit integers

struct Key { unsigned long long hi; uint32_t lo, beam; };    // larger first, then the lowest `lo`
__device__ __forceinline__ bool before(const Key& x, const Key& y) { return x.hi > y.hi || (x.hi == y.hi && x.lo < y.lo); }
// a float or double as an unsigned integer of the same order, never 0 for a number
__device__ __forceinline__ uint32_t ordered(float x) {
  const uint32_t u = __float_as_uint(x + 0.f);               // no -0
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float unordered(uint32_t u) { return __uint_as_float(u & 0x80000000u ? u & 0x7fffffffu : ~u); }
__device__ __forceinline__ unsigned long long ordered(double x) {
  const unsigned long long u = (unsigned long long)__double_as_longlong(x + 0.0);
  return u >> 63 ? ~u : u | 1ull << 63;
}
__device__ __forceinline__ double unordered(unsigned long long u) { return __longlong_as_double((long long)(u >> 63 ? u & ~(1ull << 63) : ~u)); }

// threads whose largest keys are compared as one: with few to find 4, so that 64 keys are compared with each other
__device__ __forceinline__ int lanes_of(int count) { return count <= 16 ? 4 : 1; }

struct Select {
  const void* logits;
  const float* scores;
  long long ld;                                              // between a beam's rows
  int groups, beams, vocab, count, splits;
  unsigned long long* keys;                                  // [rows][splits][count]
  double* sums;                                              // [rows][splits], of exp(x - largest)
  float* tops;                                               // [rows][splits]; +inf: a logit is NaN or +inf
  float* values;
  int *from, *tokens;
  int bf16;
};

// A block's entries as they lie: 16 bytes of a row at a time, -inf where there is none
template <typename act_t, int VECS> struct Entries;
template <int VECS> struct Entries<float, VECS> {
  float x[4 * VECS];
  __device__ __forceinline__ void load(const float* row, int at, int n) { rows::load<float, VECS>(row, at, n, -INFINITY, x); }
  __device__ __forceinline__ float operator[](int i) const { return x[i]; }
  __device__ __forceinline__ float top() const {             // NaN if one is
    float m = x[0];
#pragma unroll
    for (int i = 1; i < 4 * VECS; ++i) asm("max.NaN.f32 %0, %0, %1;" : "+f"(m) : "f"(x[i]));
    return m;
  }
};
template <int VECS> struct Entries<__nv_bfloat16, VECS> {
  uint32_t w[4 * VECS];
  __device__ __forceinline__ void load(const __nv_bfloat16* row, int at, int n) {
    if (rows::inside<__nv_bfloat16, VECS>(at, n)) {
#pragma unroll
      for (int v = 0; v < VECS; ++v) {
        const uint4 u = __ldcs(reinterpret_cast<const uint4*>(row + at + (v * (int)blockDim.x + (int)threadIdx.x) * 8));
        w[4 * v] = u.x; w[4 * v + 1] = u.y; w[4 * v + 2] = u.z; w[4 * v + 3] = u.w;
      }
      return;
    }
#pragma unroll
    for (int v = 0; v < VECS; ++v) {
      const int i = at + (v * (int)blockDim.x + (int)threadIdx.x) * 8;
      if (i >= 0 && i + 8 <= n) {
        const uint4 u = __ldcs(reinterpret_cast<const uint4*>(row + i));
        w[4 * v] = u.x; w[4 * v + 1] = u.y; w[4 * v + 2] = u.z; w[4 * v + 3] = u.w;
      } else {
        const uint16_t* bits = reinterpret_cast<const uint16_t*>(row);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int k = i + 2 * e;
          w[4 * v + e] = (k >= 0 && k < n ? bits[k] : 0xff80u) | (uint32_t)(k + 1 >= 0 && k + 1 < n ? bits[k + 1] : 0xff80u) << 16;
        }
      }
    }
  }
  __device__ __forceinline__ float operator[](int i) const { return __uint_as_float(i & 1 ? w[i >> 1] & 0xffff0000u : w[i >> 1] << 16); }
  __device__ __forceinline__ float top() const {             // two at a time
    uint32_t m = w[0];
#pragma unroll
    for (int i = 1; i < 4 * VECS; ++i) asm("max.NaN.bf16x2 %0, %0, %1;" : "+r"(m) : "r"(w[i]));
    float lo = __uint_as_float(m << 16);
    asm("max.NaN.f32 %0, %0, %1;" : "+f"(lo) : "f"(__uint_as_float(m & 0xffff0000u)));
    return lo;
  }
};
__device__ __forceinline__ float larger(float x, float y) {  // NaN if one is
  asm("max.NaN.f32 %0, %0, %1;" : "+f"(x) : "f"(y));
  return x;
}
__device__ __forceinline__ float exp2_f(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ float2 add2(float2 x, float2 y) {
  float2 z;
  asm("{\n\t.reg .b64 u, v;\n\tmov.b64 u, {%2, %3};\n\tmov.b64 v, {%4, %5};\n\tadd.rn.f32x2 u, u, v;\n\tmov.b64 {%0, %1}, u;\n\t}" : "=f"(z.x), "=f"(z.y) : "f"(x.x), "f"(x.y), "f"(y.x), "f"(y.y));
  return z;
}
// e^(x + c) and e^(y + c) by powers of two
__device__ __forceinline__ float2 powers2(float x, float y, float c) {
  const float2 d = add2(make_float2(x, y), make_float2(c, c));
  float2 e;
  asm("{\n\t.reg .b64 u, v;\n\tmov.b64 u, {%2, %3};\n\tmov.b64 v, {%4, %4};\n\tmul.rn.f32x2 u, u, v;\n\tmov.b64 {%0, %1}, u;\n\t}"
      : "=f"(e.x), "=f"(e.y) : "f"(d.x), "f"(d.y), "f"(1.44269502162933349609375f));      // log2(e)
  return make_float2(exp2_f(e.x), exp2_f(e.y));
}

// The sum of entries I .. I + N - 1's e^(x + c), in pairs: five roundings at most for 64, where one behind the other would be as many (the rest of the sum is in 64 bits).
// Halves one after the other, so that few of them are in registers
template <int I, int N, typename E> __device__ __forceinline__ float2 powers(const E& x, float c) {
  if constexpr (N == 2) return powers2(x[I], x[I + 1], c);
  else return add2(powers<I, N / 2>(x, c), powers<I + N / 2, N / 2>(x, c));
}
// Of threads that have one of GROUPS values each: those whose value is the count-th largest say so
template <int GROUPS> __device__ __forceinline__ bool is_nth(const uint32_t* all, uint32_t own, int count) {
  int above = 0, reached = 0;
#pragma unroll(GROUPS == 64 ? 16 : 8)
  for (int i = 0; i < GROUPS; i += 4) {
    const uint4 y = *reinterpret_cast<const uint4*>(all + i);
    above += (y.x > own) + (y.y > own) + (y.z > own) + (y.w > own);
    reached += (y.x >= own) + (y.y >= own) + (y.z >= own) + (y.w >= own);
  }
  return above < count && reached >= count;
}

// Entries that are at least `least`, as bits; bit i: entry `of(i)` of the thread
template <int VECS> __device__ __forceinline__ unsigned long long reach(const Entries<float, VECS>& x, float least) {
  unsigned long long hits = 0ull;
#pragma unroll
  for (int i = 0; i < 4 * VECS; ++i) hits |= x[i] >= least ? 1ull << i : 0ull;
  return hits;
}
template <int VECS> __device__ __forceinline__ unsigned long long reach(const Entries<__nv_bfloat16, VECS>& x, float least) {      // two at a time
  const uint32_t bound = (__float_as_uint(least) >> 16) * 0x10001u;
  uint32_t hits[2] = {0u, 0u};
#pragma unroll
  for (int i = 0; i < 4 * VECS; ++i) {
    uint32_t m;
    asm("set.ge.u32.bf16x2 %0, %1, %2;" : "=r"(m) : "r"(x.w[i]), "r"(bound));
    hits[i >> 4] |= m & (0x10001u << (i & 15));
  }
  return hits[0] | (unsigned long long)hits[1] << 32;
}
template <typename act_t> __device__ __forceinline__ int of(int bit) { return sizeof(act_t) == 4 ? bit : 2 * (bit & 15) + (bit >> 4 & 1) + 32 * (bit >> 5); }

template <typename act_t, int ENTRIES>
__global__ void __launch_bounds__(THREADS, ENTRIES == 8 ? 8 : sizeof(act_t) == 2 ? (ENTRIES == 64 ? 4 : 5) : 4) beam_parts_kernel(const __grid_constant__ Select a) {
  __shared__ float tops[THREADS / 32];
  __shared__ double sums[THREADS / 32];
  __shared__ __align__(16) unsigned long long bests[THREADS], list[LIST];
  __shared__ unsigned long long bound;
  __shared__ float least_of;
  __shared__ int found;
  pdl_launch_dependents();                                   // the second launch waits for the end of this one
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, lanes = lanes_of(a.count), groups = THREADS / lanes, unit = blockIdx.y * a.splits + blockIdx.x;
  constexpr int PER = rows::PER<act_t>;
  const act_t* logits = reinterpret_cast<const act_t*>(a.logits) + blockIdx.y * a.ld;
  const int at = rows::border(logits) + blockIdx.x * THREADS * ENTRIES;
  Entries<act_t, ENTRIES / PER> x;
  x.load(logits, at, a.vocab);
  auto key = [&](int i) -> unsigned long long {
    const int v = at + (i / PER * THREADS + (int)threadIdx.x) * PER + i % PER;
    return v >= 0 && v < a.vocab ? (unsigned long long)ordered(ld_act(logits, v)) << 32 | (uint32_t)~v : 0ull;
  };
  const float mine = x.top();
  float group = mine;
  if (lanes == 4) {
    group = larger(group, __shfl_xor_sync(0xffffffffu, group, 1));
    group = larger(group, __shfl_xor_sync(0xffffffffu, group, 2));
  }
  uint32_t* firsts = reinterpret_cast<uint32_t*>(bests);   // the groups' largest as integers
  if (threadIdx.x % lanes == 0) firsts[threadIdx.x / lanes] = ordered(group);
  float top = group;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = larger(top, __shfl_xor_sync(0xffffffffu, top, o));
  if (lane == 0) tops[warp] = top;
  if (threadIdx.x == 0) {
    found = 0;
    bound = 0ull;
  }
  __syncthreads();
  // the count-th largest of the groups' values, by counting how many are larger
  if ((int)threadIdx.x < groups) {
    const uint32_t own = firsts[threadIdx.x];
    if (lanes == 4 ? is_nth<64>(firsts, own, a.count) : is_nth<THREADS>(firsts, own, a.count)) least_of = unordered(own);      // the same from all who say it
  }
  top = larger(larger(larger(tops[0], tops[1]), larger(tops[2], tops[3])), larger(larger(tops[4], tops[5]), larger(tops[6], tops[7])));
  const bool out = !(top > -INFINITY && top < INFINITY);   // no sum; the second launch does not look at the keys of a beam that is out
  const float2 sum = powers<0, ENTRIES>(x, out ? 0.f : -top);
  double all = (double)sum.x + (double)sum.y;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) all += __shfl_xor_sync(0xffffffffu, all, o);
  if (lane == 0) sums[warp] = all;
  __syncthreads();
  if (threadIdx.x == 0) {
    double s = 0.0;
    for (int w = 0; w < THREADS / 32; ++w) s += sums[w];
    a.sums[unit] = out ? 0.0 : s;
    a.tops[unit] = top != top ? INFINITY : top;
  }
  // Entries that reach the bound, found again where they come from: what to do with each is written once, not ENTRIES times
  const float least = least_of;
  if (mine >= least) {
    unsigned long long hits = reach(x, least);
    if (__popcll(hits) + found > LIST) atomicMax(&found, LIST + 1);      // many alike: not one after the other
    for (; hits && found <= LIST; hits &= hits - 1) {
      const unsigned long long k = key(of<act_t>(__ffsll((long long)hits) - 1));
      const int to = k ? atomicAdd(&found, 1) : LIST;
      if (to < LIST) list[to] = k;
    }
  }
  __syncthreads();
  if (found > LIST) {                                      // by keys, which are all different
    unsigned long long best = 0ull;
#pragma unroll 4
    for (int i = 0; i < ENTRIES; ++i) best = max(best, key(i));
    if (lanes == 4) {
      best = max(best, __shfl_xor_sync(0xffffffffu, best, 1));
      best = max(best, __shfl_xor_sync(0xffffffffu, best, 2));
    }
    if (threadIdx.x % lanes == 0) bests[threadIdx.x / lanes] = best;
    __syncthreads();
    if (threadIdx.x == 0) found = 0;
    if ((int)threadIdx.x < groups) {
      const unsigned long long own = bests[threadIdx.x];
      int above = 0;
      for (int i = 0; i < groups; ++i) above += bests[i] > own;
      if (above == a.count - 1 && own) bound = own;        // with fewer groups that have entries than that, all there are
    }
    __syncthreads();
    const unsigned long long from = max(bound, 1ull);
    if (best >= from)
#pragma unroll 4
      for (int i = 0; i < ENTRIES; ++i) {
        const unsigned long long k = key(i);
        if (k >= from) {
          const int to = atomicAdd(&found, 1);
          if (to < LIST) list[to] = k;
        }
      }
    __syncthreads();
  }
  const int n = min(found, LIST);
  unsigned long long* keys = a.keys + (size_t)unit * a.count;
  for (int i = threadIdx.x; i < n; i += THREADS) {
    const unsigned long long own = list[i];
    int rank = 0;
#pragma unroll 8
    for (int j = 0; j < n; ++j) rank += list[j] > own;
    if (rank < a.count) keys[rank] = own;
  }
  for (int i = n + (int)threadIdx.x; i < a.count; i += THREADS) keys[i] = 0ull;
}

// What bounds it: a chain of loads, logarithms in 64 bits, and code that runs once.  One group of 512 entries 5.9 us, 48 of 896 10.3 us (with 256 threads 6.9 and 11.2).
constexpr int HELD = 2048, TIES = 1024;      // entries in shared memory; of those that reach the bound
constexpr int SELECTORS = 512, OCTETS = SELECTORS / 8;      // threads; groups of eight, at least as many as are chosen
static_assert(OCTETS >= MOST_COUNT);

// How far a beam's sum may be off in the first launch: a term 2^(d log2 e), d = x - largest, by 3 |d| 2^-24 of itself (the difference, the product and the constant rounded) and
// 2^-22 for the power of two; weighted with the terms |d| is at most ln 16384 < 9.8 in a part of 16384 entries (an entropy); five roundings of 2^-24 in a thread: less than
// 39 x 2^-24, and the logarithm by as much, which depends on where in 16 bytes the row begins, too.  So values of different beams that are closer than twice that (and two roundings
// of either in 64 bits) have no order yet: those beams' sums are formed again, and the selection is repeated.  What was farther apart stays in order when one of two values is
// put right.
__device__ __forceinline__ double nearly(double value) { return 80.0 / 16777216.0 + fabs(value) * 0x1p-50; }

// 2^62 e^d as a whole number, d <= 0: d = n ln 2 + r with ln 2 in two parts (W. J. Cody and W. Waite), of which the first times n is exact, and the Taylor series of e^r, |r| < 0.35:
// its terms from r^14 / 14! on are below 2^-57
__device__ __forceinline__ unsigned long long whole_exp(double d) {
  d = fmax(d, -50.0);                                        // e^-44 is half of 2^-62
  const double y = fma(d, 1.4426950408889634, 0x1.8p52), n = y - 0x1.8p52, r = fma(n, -0x1.9ef35793c7673p-41, fma(n, -0x1.62e42fefa2000p-1, d));
  constexpr double OVER[14] = {1.0, 1.0, 1.0 / 2, 1.0 / 6, 1.0 / 24, 1.0 / 120, 1.0 / 720, 1.0 / 5040, 1.0 / 40320, 1.0 / 362880, 1.0 / 3628800, 1.0 / 39916800, 1.0 / 479001600, 1.0 / 6227020800.0};
  double p = OVER[13];
#pragma unroll
  for (int k = 12; k >= 0; --k) p = fma(p, r, OVER[k]);
  return __double2ull_rn(p * __hiloint2double((__double2loint(y) + 62 + 1023) << 20, 0));
}
// sum_u exp(x_u - top) of a row by the whole block, in whole numbers: the same for the same logits in whatever order; a term is off by 2^-51 of itself and 2^-63.  A row of 100003
// takes 30 us, one of 32000 10: 48 groups of 8 beams that are all alike 275 us, where the selection takes 36 otherwise (with CUDA's exp, whose branches keep the terms apart, 730)
template <typename act_t> __device__ __forceinline__ void add_up(const act_t* row, int vocab, float top, unsigned long long (&sum)[2]) {
  constexpr int ENTRIES = 16;
  unsigned long long lo = 0ull, hi = 0ull;
#pragma unroll 1
  for (int at = rows::border(row); at < vocab; at += SELECTORS * ENTRIES) {
    float x[ENTRIES];
    rows::load<act_t, ENTRIES / rows::PER<act_t>>(row, at, vocab, -INFINITY, x);
#pragma unroll
    for (int i = 0; i < ENTRIES; ++i) {
      const unsigned long long t = whole_exp((double)x[i] - (double)top);
      lo += t & 0xffffffffull;
      hi += t >> 32;                                         // at most 2^30 for each of 2^30 tokens
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    lo += __shfl_xor_sync(0xffffffffu, lo, o);
    hi += __shfl_xor_sync(0xffffffffu, hi, o);
  }
  if (threadIdx.x % 32 == 0) {
    atomicAdd(&sum[0], lo);
    atomicAdd(&sum[1], hi);
  }
}

__global__ void __launch_bounds__(SELECTORS) beam_select_kernel(const __grid_constant__ Select a) {
  __shared__ double logs[MOST_BEAMS];                        // of the sum of exp(x - largest); NaN: the beam is out
  __shared__ float largest[MOST_BEAMS], scores[MOST_BEAMS];
  __shared__ __align__(16) unsigned long long firsts[OCTETS];
  __shared__ Key list[TIES];
  __shared__ __align__(16) unsigned long long held[HELD];    // and then what reaches the bound, in order
  static_assert(HELD * sizeof(unsigned long long) >= TIES * sizeof(Key));
  __shared__ unsigned long long least_of, doubt, last_place, sum[2];      // beams whose sums are formed again; those with a value near the last that is chosen
  __shared__ int found;
  const int group = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5, per = a.splits * a.count, all = a.beams * per;
  const unsigned long long* keys = a.keys + (size_t)group * all;
  if (threadIdx.x == 0) {
    found = 0;
    doubt = last_place = 0ull;
  }
  pdl_wait();
  if (all <= HELD) {
#pragma unroll 4
    for (int i = threadIdx.x; i < all; i += SELECTORS) held[i] = keys[i];
    keys = held;
  }
  for (int w = warp; w < a.beams; w += SELECTORS / 32) {       // a warp for a beam
    const size_t at = ((size_t)group * a.beams + w) * a.splits;
    const float score = a.scores[(size_t)group * a.beams + w];
    float top = -INFINITY, t = -INFINITY;
    double s = 0.0;
    if (lane < a.splits) {
      t = a.tops[at + lane];
      s = a.sums[at + lane];
    }
    top = t;
    for (int i = lane + 32; i < a.splits; i += 32) top = fmaxf(top, a.tops[at + i]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    double sum = t > -INFINITY ? s * exp((double)t - (double)top) : 0.0;
    for (int i = lane + 32; i < a.splits; i += 32) {
      const float u = a.tops[at + i];
      if (u > -INFINITY) sum += a.sums[at + i] * exp((double)u - (double)top);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    const bool out = !(top > -INFINITY && top < INFINITY && fabsf(score) < INFINITY);
    if (lane == 0) {
      logs[w] = out ? NAN : log(sum);
      largest[w] = top;
      scores[w] = score;
    }
  }
  __syncthreads();
  const float over = 1.f / (float)per;
  auto entry = [&](int i, unsigned long long k) -> Key {     // of a beam's and a part's largest the next
    int w = (int)((float)i * over);                          // i / per, or one off: fewer than 2^24 entries
    w += (w + 1) * per <= i;
    w -= w * per > i;
    const double c = logs[w];
    if (c != c) {
      const int r = i - w * per;
      return r < a.count && r < a.vocab ? Key{ordered(-(double)INFINITY), (uint32_t)w * a.vocab + r, (uint32_t)w} : Key{0ull, 0u, 0u};
    }
    // the logarithm last: beams of equal sums whose scores make up for the difference of their logits are alike
    return k ? Key{ordered((double)scores[w] + ((double)unordered((uint32_t)(k >> 32)) - (double)largest[w]) - c), (uint32_t)w * a.vocab + (uint32_t)~k, (uint32_t)w} : Key{0ull, 0u, 0u};
  };
  // the lowest and the highest of values (as integers) that are close to one; none to -inf
  auto below = [](unsigned long long hi) { return unordered(hi) > -(double)INFINITY ? ordered(unordered(hi) - nearly(unordered(hi))) : ~0ull; };
  auto above = [](unsigned long long hi) { return ordered(unordered(hi) + nearly(unordered(hi))); };
  auto put = [&](const Key& k, int rank) {
    const size_t to = (size_t)group * a.count + rank;
    a.values[to] = (float)unordered(k.hi);
    a.from[to] = (int)(k.lo / (uint32_t)a.vocab);
    a.tokens[to] = (int)(k.lo % (uint32_t)a.vocab);
  };
#pragma unroll 1
  for (int round = 0;; ++round) {
    const bool look = round == 0 && a.beams > 1;             // whether values of different beams are too close
    unsigned long long mine = 0ull, least = 0ull;
#pragma unroll 1
    for (int pass = 0; pass < 2; ++pass) {                   // the largest value of each thread; then what reaches the bound, or nearly does
      if (pass == 0 || mine >= least)
#pragma unroll 1
        for (int i = threadIdx.x; i < all; i += SELECTORS) {
          const Key k = entry(i, keys[i]);
          if (pass == 0) {
            mine = max(mine, k.hi);
          } else if (k.hi >= least) {
            const int to = atomicAdd(&found, 1);
            if (to < TIES) list[to] = k;
          }
        }
      if (pass == 1) break;
      unsigned long long best = mine;
#pragma unroll
      for (int o = 1; o < 8; o <<= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
      if (threadIdx.x % 8 == 0) firsts[threadIdx.x / 8] = best;
      __syncthreads();
      if (threadIdx.x < OCTETS) {
        const unsigned long long own = firsts[threadIdx.x];
        int larger = 0, reached = 0;
#pragma unroll 8
        for (int i = 0; i < OCTETS; i += 2) {
          const ulonglong2 y = *reinterpret_cast<const ulonglong2*>(&firsts[i]);
          larger += (y.x > own) + (y.y > own);
          reached += (y.x >= own) + (y.y >= own);
        }
        if (larger < a.count && reached >= a.count) least_of = own;      // the same from all who say it
      }
      __syncthreads();
      least = least_of;                                      // of a number, or 0
      least = least ? ordered(unordered(least) - nearly(unordered(least))) : 1ull;
    }
    __syncthreads();
    const int n = found;
    if (n <= TIES) {
      for (int i = threadIdx.x; i < n; i += SELECTORS) {
        const Key own = list[i];
        int rank = 0;
#pragma unroll 4
        for (int j = 0; j < n; ++j) rank += before(list[j], own);
        if (rank < a.count) put(own, rank);
        if (look) reinterpret_cast<Key*>(held)[rank] = own;
      }
      if (!look) return;
      __syncthreads();
      const Key* sorted = reinterpret_cast<const Key*>(held);
      for (int r = threadIdx.x; r < n - 1; r += SELECTORS) {      // of a run of close values each has a neighbour of another beam, or one of its own that has
        const Key x = sorted[r], y = sorted[r + 1];
        if (x.beam != y.beam && y.hi >= below(x.hi) && (r + 1 < a.count || y.hi >= below(sorted[a.count - 1].hi))) atomicOr(&doubt, 1ull << x.beam | 1ull << y.beam);
      }
      keys = a.keys + (size_t)group * all;
    } else {
      // more values alike than the list holds: one after the other
      Key last{~0ull, 0u, 0u};
      for (int r = 0; r < a.count; ++r) {
        Key next{0ull, 0u, 0u};
        for (int i = threadIdx.x; i < all; i += SELECTORS) {
          const Key k = entry(i, keys[i]);
          if (k.hi && before(last, k) && (next.hi == 0ull || before(k, next))) next = k;
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
          const Key other{__shfl_xor_sync(0xffffffffu, next.hi, o), __shfl_xor_sync(0xffffffffu, next.lo, o), __shfl_xor_sync(0xffffffffu, next.beam, o)};
          if (other.hi && (next.hi == 0ull || before(other, next))) next = other;
        }
        if (lane == 0) list[warp] = next;
        __syncthreads();
        for (int w = 0; w < SELECTORS / 32; ++w)
          if (list[w].hi && (next.hi == 0ull || before(list[w], next))) next = list[w];
        if (threadIdx.x == 0) {
          put(next, r);
          if (look && r > 0 && next.beam != last.beam && next.hi >= below(last.hi)) doubt |= 1ull << next.beam | 1ull << last.beam;
        }
        last = next;
        __syncthreads();
      }
      if (look) {                                            // those that are not chosen: near the last one that is
        const unsigned long long lo = below(last.hi), hi = above(last.hi);
        unsigned long long beams = 0ull;
        for (int i = threadIdx.x; i < all; i += SELECTORS) {
          const Key k = entry(i, keys[i]);
          if (k.hi >= lo && k.hi <= hi) beams |= 1ull << k.beam;
        }
        if (beams) atomicOr(&last_place, beams);
      }
    }
    if (!look) return;
    __syncthreads();
    const unsigned long long again = doubt | (last_place & (last_place - 1ull) ? last_place : 0ull);
    if (!again) return;
    for (int w = 0; w < a.beams; ++w) {
      if (!(again >> w & 1ull)) continue;
      const size_t row = (size_t)group * a.beams + w;
      if (threadIdx.x == 0) sum[0] = sum[1] = 0ull;
      __syncthreads();
      if (a.bf16) add_up(reinterpret_cast<const __nv_bfloat16*>(a.logits) + row * (size_t)a.ld, a.vocab, largest[w], sum);
      else add_up(reinterpret_cast<const float*>(a.logits) + row * (size_t)a.ld, a.vocab, largest[w], sum);
      __syncthreads();
      if (threadIdx.x == 0) logs[w] = log((double)sum[1] * 0x1p-30 + (double)sum[0] * 0x1p-62);
    }
    if (threadIdx.x == 0) found = 0;
    __syncthreads();
  }
}

// Entries of a thread: 32 (bf16: 64) where the parts fill the GPU, else 8, so that more SMs have one
static int entries_of(long long rows, int vocab, int act_dtype) {
  const int large = act_dtype == B2L_BF16 ? 64 : 32;
  return rows * ((vocab + THREADS * large - 1) / (THREADS * large)) >= 2ll * sm_count() ? large : 8;
}
static int splits_of(long long rows, int vocab, int act_dtype) {
  const int per = THREADS * entries_of(rows, vocab, act_dtype);
  return (vocab + 7 + per - 1) / per;                        // 7: a row that does not begin on a border
}

}  // namespace beam
}  // namespace b2l

using namespace b2l;

extern "C" long long b2l_seq_beam_work(int groups, int beams, int vocab, int count, int act_dtype) {
  if (groups <= 0 || beams <= 0 || vocab <= 0 || vocab >= beam::MOST_VOCAB || count <= 0) return 0;
  const long long rows = (long long)groups * beams, parts = rows * beam::splits_of(rows, vocab, act_dtype);
  return parts * (8ll * count + 8 + 4);
}

extern "C" int b2l_seq_beam_select(const void* logits, long long ld, const float* scores, float* values, int* from, int* tokens, void* work, long long work_bytes, int groups, int beams,
                                   int vocab, int count, int act_dtype, b2l_stream_t stream) {
  using namespace beam;
  const char* who = "b2l_seq_beam_select";
  B2L_CHECK_ARG(groups >= 0 && beams > 0 && vocab > 0 && count > 0 && ld >= vocab, "%s: bad sizes", who);
  B2L_CHECK_ARG(groups == 0 || (logits && scores && values && from && tokens), "%s: null pointer", who);
  B2L_CHECK_SUPPORTED(beams <= MOST_BEAMS && count <= MOST_COUNT && (long long)groups * beams < 65536 && vocab < MOST_VOCAB && (long long)beams * vocab < (1ll << 31),
                      "%s: %d groups of %d beams over %d tokens, %d of them: at most 65535 rows, %d beams, %d of them, fewer than %d tokens", who, groups, beams, vocab, count, MOST_BEAMS,
                      MOST_COUNT, MOST_VOCAB);
  B2L_CHECK_ARG(count <= (long long)beams * vocab, "%s: %d of %lld", who, count, (long long)beams * vocab);
  if (groups == 0) return 0;
  const long long need = b2l_seq_beam_work(groups, beams, vocab, count, act_dtype);
  B2L_CHECK_ARG(work && work_bytes >= need && ((uintptr_t)work & 15) == 0, "%s: a work space of %lld bytes is needed", who, need);
  const int rows = groups * beams, splits = splits_of(rows, vocab, act_dtype);
  B2L_CHECK_SUPPORTED((long long)rows * splits < (1ll << 31) && (long long)beams * splits * count < (1ll << 24), "%s: %d rows over %d tokens, %d of them", who, rows, vocab, count);
  Select a{logits, scores, ld, groups, beams, vocab, count, splits};
  a.keys = (unsigned long long*)work;
  a.sums = (double*)(a.keys + (size_t)rows * splits * count);
  a.tops = (float*)(a.sums + (size_t)rows * splits);
  a.values = values;
  a.from = from;
  a.tokens = tokens;
  a.bf16 = act_dtype == B2L_BF16;
  const cudaStream_t st = (cudaStream_t)stream;
  const bool large = entries_of(rows, vocab, act_dtype) > 8;
  B2L_SEQ_DISPATCH(act_dtype, {
    if (large) beam_parts_kernel<act_t, sizeof(act_t) == 2 ? 64 : 32><<<dim3(splits, rows), THREADS, 0, st>>>(a);
    else beam_parts_kernel<act_t, 8><<<dim3(splits, rows), THREADS, 0, st>>>(a);
  });
  B2L_LAUNCH_CHECK("beam_parts_kernel");
  LaunchCfg launch(dim3((unsigned)groups), dim3(SELECTORS), 0, st, true);
  B2L_CUDA(cudaLaunchKernelEx(&launch.cfg, beam_select_kernel, a));
  B2L_LAUNCH_CHECK("beam_select_kernel");
  return 0;
}
