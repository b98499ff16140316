// Beam search's selection: of a group's beams and the vocabulary the `count` largest of
//
//   value[w, v] = score[w] + x[w, v] - log sum_u exp x[w, u],    ties to the lowest w V + v
//
// Within a beam the order is that of its logits, so one pass over them gives the sum and each part's `count` largest, as keys of 64 bits: the logit as an integer of
// the same order, and what is left to the lowest index.  A block holds its part in registers.  Its groups of threads have a largest key each; the count-th largest of
// these is a bound that at least `count` entries reach, all of them in `count` groups, so the few that do are found without a sort and ranked by counting.  A
// second launch, a block for a group of beams, does the same with the beams' parts, by values in 64 bits (scores and logits of different beams may be
// neighbours: what f32 keeps of a sum of 32000 terms would change their order).
//
// A beam whose score or log-probabilities are no numbers (a score of -inf, a logit that is NaN or +inf, none above -inf) is out: its values are -inf.
//
// What bounds it: the logits read once; few beams: two launches.
#include "seq_rows.cuh"

namespace b2l {
namespace beam {

constexpr int THREADS = 256, MOST_COUNT = 64, MOST_BEAMS = 64, LIST = 2048;

struct Key { unsigned long long hi; uint32_t lo; };          // larger first, then the lowest `lo`
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
  float* tops;                                               // [rows][splits]; +inf: a logit that is no number or +inf
  float* values;
  int *from, *tokens;
};

template <typename act_t, int ENTRIES>
__global__ void __launch_bounds__(THREADS) beam_parts_kernel(const __grid_constant__ Select a) {
  __shared__ float tops[THREADS / 32];
  __shared__ double sums[THREADS / 32];
  __shared__ __align__(16) unsigned long long bests[THREADS];
  __shared__ unsigned long long bound, list[LIST];
  __shared__ int found;
  const int row = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const act_t* logits = reinterpret_cast<const act_t*>(a.logits) + row * a.ld;
  constexpr int PER = rows::PER<act_t>;
  const int at = rows::border(logits) + blockIdx.x * THREADS * ENTRIES;
  float x[ENTRIES];
  rows::load<act_t, ENTRIES / PER>(logits, at, a.vocab, -INFINITY, x);
  auto index = [&](int i) { return at + (i / PER * THREADS + (int)threadIdx.x) * PER + i % PER; };
  auto key = [&](int i) {
    const int v = index(i);
    return v >= 0 && v < a.vocab ? (unsigned long long)ordered(x[i]) << 32 | (uint32_t)~v : 0ull;
  };
  float top = -INFINITY;
#pragma unroll
  for (int i = 0; i < ENTRIES; ++i) {
    if (!(x[i] < INFINITY)) x[i] = INFINITY;
    top = fmaxf(top, x[i]);
  }
  const float mine = top;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  if (lane == 0) tops[warp] = top;
  if (threadIdx.x == 0) {
    found = 0;
    bound = 0ull;
  }
  // this thread's largest entry, the first of equal ones (they ascend)
  unsigned long long best = 0ull;
#pragma unroll
  for (int i = ENTRIES - 1; i >= 0; --i)
    if (x[i] == mine) {
      const unsigned long long k = key(i);
      if (k) best = k;
    }
  const int lanes = lanes_of(a.count), keys = THREADS / lanes;
  if (lanes == 4) {
    for (int o = 1; o < 4; o <<= 1) {
      const unsigned long long other = __shfl_xor_sync(0xffffffffu, best, o);
      best = max(best, other);
    }
  }
  if (threadIdx.x % lanes == 0) bests[threadIdx.x / lanes] = best;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < THREADS / 32; ++w) top = fmaxf(top, tops[w]);
  // in pairs: five roundings at most, where one behind the other would be 32 (the rest of the sum is in 64 bits)
  float sum[ENTRIES / 4];
  if (top > -INFINITY && top < INFINITY) {
#pragma unroll
    for (int i = 0; i < ENTRIES; i += 4) sum[i / 4] = (expf(x[i] - top) + expf(x[i + 1] - top)) + (expf(x[i + 2] - top) + expf(x[i + 3] - top));
#pragma unroll
    for (int n = ENTRIES / 8; n > 0; n /= 2)
#pragma unroll
      for (int i = 0; i < n; ++i) sum[i] += sum[i + n];
  } else {
    sum[0] = 0.f;
  }
  double all = sum[0];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) all += __shfl_xor_sync(0xffffffffu, all, o);
  if (lane == 0) sums[warp] = all;
  // the count-th largest of the groups' keys, by counting how many are larger; with fewer groups that have entries than that, all there are
  if ((int)threadIdx.x < keys) {
    const unsigned long long own = bests[threadIdx.x];
    int rank = 0;
    for (int i = 0; i < keys; i += 2) {
      const ulonglong2 y = *reinterpret_cast<const ulonglong2*>(&bests[i]);
      rank += (y.x > own) + (y.y > own);
    }
    if (rank == a.count - 1 && own) bound = own;
  }
  __syncthreads();
  const unsigned long long least = max(bound, 1ull);
  if (threadIdx.x == 0) {
    double s = 0.0;
    for (int w = 0; w < THREADS / 32; ++w) s += sums[w];
    a.sums[(size_t)row * a.splits + blockIdx.x] = s;
    a.tops[(size_t)row * a.splits + blockIdx.x] = top;
  }
  if (best >= least)
#pragma unroll
    for (int i = 0; i < ENTRIES; ++i) {
      const unsigned long long k = key(i);
      if (k >= least) {
        const int to = atomicAdd(&found, 1);
        if (to < LIST) list[to] = k;
      }
    }
  __syncthreads();
  const int n = min(found, LIST);
  unsigned long long* out = a.keys + ((size_t)row * a.splits + blockIdx.x) * a.count;
  for (int i = threadIdx.x; i < n; i += THREADS) {
    const unsigned long long own = list[i];
    int rank = 0;
    for (int j = 0; j < n; ++j) rank += list[j] > own;
    if (rank < a.count) out[rank] = own;
  }
  for (int i = n + (int)threadIdx.x; i < a.count; i += THREADS) out[i] = 0ull;
}

__global__ void __launch_bounds__(THREADS) beam_select_kernel(const __grid_constant__ Select a) {
  __shared__ double offset[MOST_BEAMS];                      // score less the logarithm of the sum of exp(x - largest); NaN: the beam is out
  __shared__ float largest[MOST_BEAMS];
  __shared__ Key bests[THREADS], list[LIST], bound;
  __shared__ int found;
  const int group = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5, per = a.splits * a.count, all = a.beams * per;
  pdl_wait();
  if (threadIdx.x == 0) {
    found = 0;
    bound = Key{0ull, 0u};
  }
  for (int w = warp; w < a.beams; w += THREADS / 32) {       // a warp for a beam
    const size_t at = ((size_t)group * a.beams + w) * a.splits;
    float top = -INFINITY;
    for (int s = lane; s < a.splits; s += 32) top = fmaxf(top, a.tops[at + s]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    double sum = 0.0;
    for (int s = lane; s < a.splits; s += 32) {
      const float t = a.tops[at + s];
      if (t > -INFINITY) sum += a.sums[at + s] * exp((double)t - (double)top);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    const float score = a.scores[(size_t)group * a.beams + w];
    const bool out = !(top > -INFINITY && top < INFINITY && fabsf(score) < INFINITY);
    if (lane == 0) {
      offset[w] = out ? NAN : (double)score - log(sum);
      largest[w] = top;
    }
  }
  __syncthreads();
  const unsigned long long* keys = a.keys + (size_t)group * all;
  auto entry = [&](int i) -> Key {                           // of a beam's and a part's largest the next
    const int w = i / per, r = i - w * per;
    const double c = offset[w];
    if (c != c) return r < a.count && r < a.vocab ? Key{ordered(-(double)INFINITY), (uint32_t)w * a.vocab + r} : Key{0ull, 0u};
    const unsigned long long k = keys[i];
    return k ? Key{ordered(c + ((double)unordered((uint32_t)(k >> 32)) - (double)largest[w])), (uint32_t)w * a.vocab + (uint32_t)~k} : Key{0ull, 0u};
  };
  auto put = [&](const Key& k, int rank) {
    const size_t to = (size_t)group * a.count + rank;
    a.values[to] = (float)unordered(k.hi);
    a.from[to] = (int)(k.lo / (uint32_t)a.vocab);
    a.tokens[to] = (int)(k.lo % (uint32_t)a.vocab);
  };
  if (a.count * ((all + THREADS - 1) / THREADS) > LIST) {    // more than the list is sure to hold: one after the other
    Key last{~0ull, 0u};
    for (int r = 0; r < a.count; ++r) {
      Key best{0ull, 0u};
      for (int i = threadIdx.x; i < all; i += THREADS) {
        const Key k = entry(i);
        if (k.hi && before(last, k) && (best.hi == 0ull || before(k, best))) best = k;
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        const Key other{__shfl_xor_sync(0xffffffffu, best.hi, o), __shfl_xor_sync(0xffffffffu, best.lo, o)};
        if (other.hi && (best.hi == 0ull || before(other, best))) best = other;
      }
      if (lane == 0) bests[warp] = best;
      __syncthreads();
      for (int w = 0; w < THREADS / 32; ++w)
        if (bests[w].hi && (best.hi == 0ull || before(bests[w], best))) best = bests[w];
      if (threadIdx.x == 0) put(best, r);
      last = best;
      __syncthreads();
    }
    return;
  }
  Key best{0ull, 0u};
  for (int i = threadIdx.x; i < all; i += THREADS) {
    const Key k = entry(i);
    if (k.hi && (best.hi == 0ull || before(k, best))) best = k;
  }
  bests[threadIdx.x] = best;
  __syncthreads();
  if (best.hi) {
    int rank = 0;
    for (int i = 0; i < THREADS; ++i) rank += bests[i].hi && before(bests[i], best);
    if (rank == a.count - 1) bound = best;
  }
  __syncthreads();
  const Key least = bound;                                   // none: fewer threads than that have entries
  if (best.hi && (least.hi == 0ull || !before(least, best)))
    for (int i = threadIdx.x; i < all; i += THREADS) {
      const Key k = entry(i);
      if (k.hi && (least.hi == 0ull || !before(least, k))) {
        const int to = atomicAdd(&found, 1);
        if (to < LIST) list[to] = k;
      }
    }
  __syncthreads();
  const int n = min(found, LIST);
  for (int i = threadIdx.x; i < n; i += THREADS) {
    const Key own = list[i];
    int rank = 0;
    for (int j = 0; j < n; ++j) rank += before(list[j], own);
    if (rank < a.count) put(own, rank);
  }
}

// Entries of a thread: 32 where the parts fill the GPU, else 8, so that more SMs have one
static int entries_of(long long rows, int vocab) { return rows * ((vocab + 8191) / 8192) >= 2ll * sm_count() ? 32 : 8; }
static int splits_of(long long rows, int vocab) {
  const int per = THREADS * entries_of(rows, vocab);
  return (vocab + 7 + per - 1) / per;                        // 7: a row that does not begin on a border
}

}  // namespace beam
}  // namespace b2l

using namespace b2l;

extern "C" long long b2l_seq_beam_work(int groups, int beams, int vocab, int count) {
  if (groups <= 0 || beams <= 0 || vocab <= 0 || count <= 0) return 0;
  const long long rows = (long long)groups * beams, parts = rows * beam::splits_of(rows, vocab);
  return parts * (8ll * count + 8 + 4);
}

extern "C" int b2l_seq_beam_select(const void* logits, long long ld, const float* scores, float* values, int* from, int* tokens, void* work, long long work_bytes, int groups, int beams,
                                   int vocab, int count, int act_dtype, b2l_stream_t stream) {
  using namespace beam;
  const char* who = "b2l_seq_beam_select";
  B2L_CHECK_ARG(groups >= 0 && beams > 0 && vocab > 0 && count > 0 && ld >= vocab, "%s: bad sizes", who);
  B2L_CHECK_ARG(groups == 0 || (logits && scores && values && from && tokens), "%s: null pointer", who);
  B2L_CHECK_SUPPORTED(beams <= MOST_BEAMS && count <= MOST_COUNT && (long long)groups * beams < 65536 && (long long)beams * vocab < (1ll << 31),
                      "%s: %d groups of %d beams over %d tokens, %d of them: at most 65535 rows, %d beams, %d of them", who, groups, beams, vocab, count, MOST_BEAMS, MOST_COUNT);
  B2L_CHECK_ARG(count <= (long long)beams * vocab, "%s: %d of %lld", who, count, (long long)beams * vocab);
  if (groups == 0) return 0;
  const long long need = b2l_seq_beam_work(groups, beams, vocab, count);
  B2L_CHECK_ARG(work && work_bytes >= need && ((uintptr_t)work & 15) == 0, "%s: a work space of %lld bytes is needed", who, need);
  const int rows = groups * beams, splits = splits_of(rows, vocab);
  Select a{logits, scores, ld, groups, beams, vocab, count, splits};
  a.keys = (unsigned long long*)work;
  a.sums = (double*)(a.keys + (size_t)rows * splits * count);
  a.tops = (float*)(a.sums + (size_t)rows * splits);
  a.values = values;
  a.from = from;
  a.tokens = tokens;
  const cudaStream_t st = (cudaStream_t)stream;
  const bool large = entries_of(rows, vocab) == 32;
  B2L_SEQ_DISPATCH(act_dtype, {
    if (large) beam_parts_kernel<act_t, 32><<<dim3(splits, rows), THREADS, 0, st>>>(a);
    else beam_parts_kernel<act_t, 8><<<dim3(splits, rows), THREADS, 0, st>>>(a);
  });
  B2L_LAUNCH_CHECK("beam_parts_kernel");
  LaunchCfg launch(dim3((unsigned)groups), dim3(THREADS), 0, st, true);
  B2L_CUDA(cudaLaunchKernelEx(&launch.cfg, beam_select_kernel, a));
  B2L_LAUNCH_CHECK("beam_select_kernel");
  return 0;
}
