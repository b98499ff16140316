// Trees of drafted tokens: what each token sees, and which of them are accepted.
//
// Token i of a sequence's new ones has a parent among those before it (or none: -1), so its ancestors are found by going up.  Its depth is the number of them.
//   target[r] = argmax_v x[r, v]                    or, drawn, argmax_v x[r, v] / T - log q[r, v], q ~ Exp(1): v with probability softmax(x / T)[v]
//   path: the first new token; then, as long as there is one, the first child whose token is its parent's target
// The second launch joins the parts of the rows and goes down the trees, a block for each sequence.
//
// What bounds acceptance: logits (and noise) read once: 758 rows of 32000 f32 logits with noise 38 us for the targets, 5.2 TB/s, a call 40; one tree of 8 tokens: two launches, 4.4
// and 5.7 us by themselves.  Values are compared in 64 bits, as two logits may be neighbours: a block finds its largest in f32 and computes those that f32 cannot tell from it again.
#include "seq_paged.cuh"
#include "seq_rows.cuh"

namespace b2l {
namespace tree {

// ------------------------------------------------------------------------------------------------ ancestors
struct Build {
  const int *parents, *starts, *lengths;
  uint32_t* masks;
  int *depths, *positions;
  int words, rows, seqs, window, first;
};
__global__ void __launch_bounds__(128) tree_build_kernel(const __grid_constant__ Build a) {
  const int row = blockIdx.x * blockDim.x + threadIdx.x;
  if (row >= a.rows) return;
  int lo = 0, hi = a.seqs;                                   // starts[lo] <= row < starts[hi], if any
  const bool in = row >= a.starts[0] && row < a.starts[a.seqs];
  while (in && hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (a.starts[mid] <= row) lo = mid;
    else hi = mid;
  }
  uint32_t* mask = a.masks + (size_t)row * a.words;
  if (!in) {
    for (int w = 0; w < a.words; ++w) mask[w] = 0u;
    a.depths[row] = 0;
    a.positions[row] = 0;
    return;
  }
  const int start = max(a.starts[lo], 0), n = min(a.starts[lo + 1], a.rows) - start, base = max(a.lengths[lo], 0) - n;
  auto parent = [&](int i) {                                 // before its child, or none
    const int p = a.parents[start + i];
    return p >= 0 && p < i ? p : -1;
  };
  int depth = 0;
  for (int i = parent(row - start); i >= 0; i = parent(i)) ++depth;
  int at = a.words - 1, steps = 0;
  uint32_t bits = 0u;
  for (int i = row - start; i >= 0; i = parent(i), ++steps) {      // falling, so the words are written from the last on
    if (i >= 32 * a.words) continue;
    while (i >> 5 < at) {
      mask[at--] = bits;
      bits = 0u;
    }
    if (a.window == 0 || steps < a.window || base + depth - steps < a.first) bits |= 1u << (i & 31);
  }
  for (; at >= 0; --at, bits = 0u) mask[at] = bits;
  a.depths[row] = depth;
  a.positions[row] = base + depth;
}

// ------------------------------------------------------------------------------------------------ targets
struct Best { double value; int at; };
__device__ __forceinline__ bool better(const Best& x, const Best& y) { return x.value > y.value || (x.value == y.value && x.at < y.at); }
struct Targets {
  const void* logits;
  const float* noise;
  long long ld, ldn;
  float temperature;
  int rows, vocab, splits;
  Best* parts;                                               // [rows][splits]
};
// A warp goes through its part of a row by itself, 512 entries at a time: what is near the largest so far it notes, and with barriers between the steps (a block's
// largest first, then what is near it) 32 trees with noise took 49 us in place of 36.
constexpr int THREADS = 256, ENTRIES = 16, ROUNDS = 2, CHUNK = THREADS * ENTRIES * ROUNDS, LIST = 1024;

template <typename act_t, bool DRAWN>
__global__ void __launch_bounds__(THREADS, 5) tree_targets_kernel(const __grid_constant__ Targets a) {
  __shared__ Best bests[THREADS / 32];
  __shared__ int list[DRAWN ? LIST : 1], found;
  pdl_launch_dependents();                                   // the second launch waits for the end of this one
  const int row = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const act_t* logits = reinterpret_cast<const act_t*>(a.logits) + row * a.ld;
  const float* noise = DRAWN ? a.noise + row * a.ldn : nullptr;
  constexpr int PER = rows::PER<act_t>;
  const int at = rows::border(logits) + blockIdx.x * CHUNK;
  const bool even = DRAWN && ((uintptr_t)(noise + at) & 15) == 0;
  const float over = DRAWN ? 1.f / a.temperature : 1.f;
  constexpr float LN2 = 0.693147182464599609375f, SLACK = 1.9073486328125e-6f;      // 2^-19
  Best best{-INFINITY, INT32_MAX};
  auto exactly = [&](int v) {
    if (v < 0 || v >= a.vocab) return;
    const Best here{(double)ld_act(logits, v) / (double)a.temperature - log((double)noise[v]), v};
    if (here.value > -INFINITY && better(here, best)) best = here;
  };
  if (DRAWN) {
    if (threadIdx.x == 0) found = 0;
    __syncthreads();
  }
  float top = -INFINITY;                                     // of the warp so far
#pragma unroll 1
  for (int round = 0; round < ROUNDS; ++round) {
    const int from = at + round * THREADS * ENTRIES;
    if (from >= a.vocab) break;
    float x[ENTRIES];
    rows::load<act_t, ENTRIES / PER>(logits, from, a.vocab, -INFINITY, x);
    auto index = [&](int i) { return from + (i / PER * THREADS + (int)threadIdx.x) * PER + i % PER; };
    if constexpr (!DRAWN) {
#pragma unroll
      for (int i = 0; i < ENTRIES; ++i)
        if (x[i] > best.value) best = {x[i], index(i)};      // no NaN; a thread's entries ascend
    } else {
      float y[ENTRIES];
      if (even && rows::inside<act_t, ENTRIES / PER>(from, a.vocab)) {
        float4 u[ENTRIES / 4];
#pragma unroll
        for (int i = 0; i < ENTRIES / 4; ++i) u[i] = __ldcs(reinterpret_cast<const float4*>(noise + index(4 * i)));
#pragma unroll
        for (int i = 0; i < ENTRIES / 4; ++i) {
          y[4 * i] = u[i].x; y[4 * i + 1] = u[i].y; y[4 * i + 2] = u[i].z; y[4 * i + 3] = u[i].w;
        }
      } else
#pragma unroll
      for (int i = 0; i < ENTRIES; i += 4) {
        const int v = index(i);
        if (even && v >= 0 && v + 4 <= a.vocab) {
          const float4 u = __ldcs(reinterpret_cast<const float4*>(noise + v));
          y[i] = u.x; y[i + 1] = u.y; y[i + 2] = u.z; y[i + 3] = u.w;
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) y[i + e] = v + e >= 0 && v + e < a.vocab ? __ldcs(noise + v + e) : 1.f;
        }
      }
#pragma unroll
      for (int i = 0; i < ENTRIES; ++i) {                    // x / T - log q, off by less than 2^-21 of its two terms together
        asm("lg2.approx.f32 %0, %1;" : "=f"(y[i]) : "f"(y[i]));
        x[i] = fmaf(y[i], -LN2, x[i] * over);
        top = fmaxf(top, x[i]);                              // NaN: not the largest
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
      if (top <= -1e25f) {
        // Nothing but masks: a logarithm does not reach quotients like these in 64 bits either, so the lowest of the largest logits is the one to look at (of a vocabulary
        // that is hidden but for a few tokens all would be near the largest: 758 rows of 32000 190 us, 69 so)
        float most = -INFINITY;
        int first = -1;
#pragma unroll 1
        for (int i = 0; i < ENTRIES; ++i) {
          const int v = index(i);
          if (v < 0 || v >= a.vocab) continue;
          const float q = noise[v], here = ld_act(logits, v);
          if (!(q > 0.f) || over == INFINITY) exactly(v);
          else if (q < INFINITY && here > most) {
            most = here;
            first = v;
          }
        }
        exactly(first);
        continue;
      }
      // Those near the largest, one or two, again in 64 bits: x / T is no larger than its difference and the logarithm together, and a logarithm at most 104, so the
      // largest is off by 2^-21 (208 + |top|) at most and one near it by 2^-21 (|top| + 2 |log q|)
      const float least = top < INFINITY ? top - SLACK * (64.f + 2.f * fabsf(top)) : INFINITY;
      uint32_t hits = 0u;
#pragma unroll
      for (int i = 0; i < ENTRIES; ++i) hits |= fmaf(fabsf(y[i]), SLACK, x[i]) < least ? 0u : 1u << i;      // NaN too: infinities of f32 that 64 bits may not have
      for (; hits; hits &= hits - 1) {
        const int to = atomicAdd(&found, 1), v = index(__ffs(hits) - 1);
        if (to < LIST) list[to] = v;
        else exactly(v);                                     // many alike
      }
    }
  }
  if constexpr (DRAWN) {
    __syncthreads();
    for (int i = threadIdx.x; i < min(found, LIST); i += THREADS) exactly(list[i]);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const Best other{__shfl_xor_sync(0xffffffffu, best.value, o), __shfl_xor_sync(0xffffffffu, best.at, o)};
    if (better(other, best)) best = other;
  }
  if (lane == 0) bests[warp] = best;
  __syncthreads();
  if (threadIdx.x == 0) {
#pragma unroll
    for (int w = 1; w < THREADS / 32; ++w)
      if (better(bests[w], best)) best = bests[w];
    a.parts[(size_t)row * a.splits + blockIdx.x] = best;
  }
}

// ------------------------------------------------------------------------------------------------ the way down
struct Walk {
  const Best* parts;
  int splits;
  int* targets;                                              // [rows]
  const int *parents, *starts;
  const void* tokens;
  int wide;                                                  // tokens of 64 bits
  int rows, seqs;
  int *kept, *counts, *next;
};
__global__ void __launch_bounds__(128) tree_walk_kernel(const __grid_constant__ Walk a) {
  const int b = blockIdx.x, lane = threadIdx.x & 31;
  const int start = min(max(a.starts[b], 0), a.rows), n = max(min(a.starts[b + 1], a.rows) - start, 0);
  if (b == 0)
    for (int r = threadIdx.x; r < start; r += blockDim.x) a.kept[r] = -1;
  if (b == a.seqs - 1)
    for (int r = start + n + threadIdx.x; r < a.rows; r += blockDim.x) a.kept[r] = -1;
  pdl_wait();
  for (int r = start + threadIdx.x; r < start + n; r += blockDim.x) {
    Best best{-INFINITY, INT32_MAX};
    for (int s = 0; s < a.splits; ++s) {
      const Best other = a.parts[(size_t)r * a.splits + s];
      if (better(other, best)) best = other;
    }
    a.targets[r] = best.at == INT32_MAX ? 0 : best.at;       // no logit above -inf: the first token
  }
  __syncthreads();
  if (threadIdx.x >= 32) return;
  int at = 0, count = 0, target = -1;
  while (at < n) {
    if (lane == 0) a.kept[start + count] = at;
    ++count;
    target = a.targets[start + at];
    int child = n;
    for (int j0 = at + 1; j0 < n && child == n; j0 += 32) {
      const int j = j0 + lane;
      bool fits = false;
      if (j < n && a.parents[start + j] == at)
        fits = a.wide ? reinterpret_cast<const long long*>(a.tokens)[start + j] == target : reinterpret_cast<const int*>(a.tokens)[start + j] == target;
      const uint32_t mine = __ballot_sync(0xffffffffu, fits);
      if (mine) child = j0 + __ffs(mine) - 1;
    }
    at = child;
  }
  for (int i = count + lane; i < n; i += 32) a.kept[start + i] = -1;
  if (lane == 0) {
    a.counts[b] = count;
    a.next[b] = target;
  }
}

}  // namespace tree
}  // namespace b2l

using namespace b2l;

extern "C" int b2l_seq_tree_build(const int* parents, const int* starts, const int* lengths, unsigned* masks, int words, int* depths, int* positions, int rows, int seqs, int window,
                                  int first, b2l_stream_t stream) {
  const char* who = "b2l_seq_tree_build";
  B2L_CHECK_ARG(rows >= 0 && seqs >= 0 && words > 0 && window >= 0 && first >= 0, "%s: bad sizes", who);
  B2L_CHECK_ARG(rows == 0 || seqs == 0 || (parents && starts && lengths && masks && depths && positions), "%s: null pointer", who);
  B2L_CHECK_SUPPORTED(rows < (1 << 30), "%s: %d rows", who, rows);
  if (rows == 0 || seqs == 0) return 0;
  tree::tree_build_kernel<<<(rows + 127) / 128, 128, 0, (cudaStream_t)stream>>>({parents, starts, lengths, masks, depths, positions, words, rows, seqs, window, first});
  B2L_LAUNCH_CHECK("tree_build_kernel");
  return 0;
}

static int accept_splits(int vocab) { return (vocab + 7 + tree::CHUNK - 1) / tree::CHUNK; }      // 7: a row that does not begin on a border

extern "C" long long b2l_seq_tree_accept_work(int rows, int vocab) {
  return rows <= 0 || vocab <= 0 ? 0 : (long long)rows * accept_splits(vocab) * (long long)sizeof(tree::Best) + 4ll * rows;
}

extern "C" int b2l_seq_tree_accept(const void* logits, long long ld, const float* noise, long long ldn, float temperature, const int* parents, const int* starts, const void* tokens,
                                   int tokens64, int* kept, int* counts, int* next, void* work, long long work_bytes, int rows, int seqs, int vocab, int act_dtype,
                                   b2l_stream_t stream) {
  using namespace tree;
  const char* who = "b2l_seq_tree_accept";
  B2L_CHECK_ARG(rows >= 0 && seqs >= 0 && vocab > 0, "%s: bad sizes", who);
  B2L_CHECK_ARG(seqs == 0 || (starts && counts && next), "%s: null pointer", who);
  B2L_CHECK_ARG(rows == 0 || seqs == 0 || (logits && parents && tokens && kept), "%s: null pointer", who);
  B2L_CHECK_ARG(ld >= vocab && (!noise || (ldn >= vocab && temperature > 0.f && temperature < INFINITY)), "%s: rows shorter than the vocabulary, or a temperature that is not positive", who);
  B2L_CHECK_SUPPORTED(rows < 65536 && vocab < (1 << 30), "%s: %d rows over %d tokens", who, rows, vocab);
  if (seqs == 0) return 0;
  const long long need = b2l_seq_tree_accept_work(rows, vocab);
  B2L_CHECK_ARG(need == 0 || (work && work_bytes >= need && ((uintptr_t)work & 15) == 0), "%s: a work space of %lld bytes is needed", who, need);
  const cudaStream_t st = (cudaStream_t)stream;
  const int splits = accept_splits(vocab);
  Best* parts = (Best*)work;
  if (rows > 0) {
    const Targets t{logits, noise, ld, ldn, temperature, rows, vocab, splits, parts};
    B2L_SEQ_DISPATCH(act_dtype, {
      if (noise) tree_targets_kernel<act_t, true><<<dim3(splits, rows), THREADS, 0, st>>>(t);
      else tree_targets_kernel<act_t, false><<<dim3(splits, rows), THREADS, 0, st>>>(t);
    });
    B2L_LAUNCH_CHECK("tree_targets_kernel");
  }
  const Walk w{parts, splits, rows > 0 ? (int*)(parts + (size_t)rows * splits) : nullptr, parents, starts, tokens, tokens64, rows, seqs, kept, counts, next};
  LaunchCfg launch(dim3((unsigned)seqs), dim3(128), 0, st, rows > 0);
  B2L_CUDA(cudaLaunchKernelEx(&launch.cfg, tree_walk_kernel, w));
  B2L_LAUNCH_CHECK("tree_walk_kernel");
  return 0;
}
