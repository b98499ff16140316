// Pages and rows moved within paged pools (layout: seq_paged.cuh), in the pools of all layers at once.
//
//   copy   page src -> page dst of keys, values and scales: what a sequence that is forked needs of the page that it goes on writing
//   keep   row base + kept[i] -> base + i, base the position of a sequence's first new token: the accepted tokens of a tree one behind the other
//
// Both move bytes and compute nothing.  What bounds them: HBM, every byte read once and written once: 48 pages of 32 layers of 8 heads of 128, bf16, 805 MB, in 125 us,
// 6.4 TB/s; a page or two: the launch.  Kept rows lie apart, 128 bytes (and a scale of 4) of a head each: 64 sequences of some five rows in 32 layers of 8 heads of int8, 34 MB,
// 16 us from HBM, 11 where L2 has them (as long with blocks that take several layers).  A sequence's rows in a layer are 144 pieces there, two blocks of 128 threads, each with the
// whole chain of lookups.  One sequence 4.4 us by itself.
#include <algorithm>

#include "seq_paged.cuh"

namespace b2l {
namespace paged {

constexpr int MOST_LAYERS = 64;      // of a launch: their addresses are its parameters
struct Pools { uint8_t* at[MOST_LAYERS][4]; };      // keys, values, their scales (or none)

// bytes of a page in each of a layer's pools
struct PageBytes { int of[4]; };
static PageBytes page_bytes(int page, int kv_heads, int K, int V, int store, int act_dtype) {
  const int es = store != ACT ? 1 : act_dtype == B2L_F32 ? 4 : 2, tokens = page * kv_heads, scale = store != ACT ? 4 : 0;
  return {{tokens * K * es, tokens * V * es, tokens * scale, tokens * scale}};
}

constexpr int PIECE = 16384;         // bytes that a block copies: four loads of 16 bytes a thread, all in flight
__global__ void __launch_bounds__(256) paged_copy_kernel(const __grid_constant__ Pools pools, const int2* __restrict__ pairs, int pages, PageBytes bytes) {
  const int2 pair = pairs[blockIdx.y];
  if (pair.x < 0 || pair.x >= pages || pair.y < 0 || pair.y >= pages || pair.x == pair.y) return;
  int piece = blockIdx.x, t = 0;
  while (t < 3 && piece >= (bytes.of[t] + PIECE - 1) / PIECE) piece -= (bytes.of[t++] + PIECE - 1) / PIECE;
  uint8_t* pool = pools.at[blockIdx.z][t];
  const size_t size = bytes.of[t];
  const uint4* src = reinterpret_cast<const uint4*>(pool + pair.x * size + (size_t)piece * PIECE);
  uint4* dst = reinterpret_cast<uint4*>(pool + pair.y * size + (size_t)piece * PIECE);
  const int n = (min((int)size - piece * PIECE, PIECE)) / 16;
  uint4 w[PIECE / 16 / 256];
#pragma unroll
  for (int i = 0; i < PIECE / 16 / 256; ++i)
    if ((int)threadIdx.x + 256 * i < n) w[i] = __ldcs(src + threadIdx.x + 256 * i);
#pragma unroll
  for (int i = 0; i < PIECE / 16 / 256; ++i)
    if ((int)threadIdx.x + 256 * i < n) __stcs(dst + threadIdx.x + 256 * i, w[i]);
}

// A thread has 16 bytes of a head's rows in one layer (or one of its scales), of all rows of one sequence: kept rows ascend and none lies before its new place, so a
// thread that goes through them in order, eight at a time, has read whatever it overwrites.
constexpr int KEEP_ROWS = 64;        // whose places are looked up at a time
__global__ void __launch_bounds__(128) paged_keep_kernel(const __grid_constant__ Pools pools, Step s, const int* __restrict__ kept, const int* __restrict__ counts, int kv_heads,
                                                         int kc, int vc, int scaled) {
  __shared__ int from[KEEP_ROWS], to[KEEP_ROWS];             // rows of head 0; -1: nothing moves
  int start, n, length;
  const int b = blockIdx.y;
  sequence(s, b, start, n, length);
  const int count = min(counts[b], n), base = length - n;
  const int per = kc + vc + 2 * scaled, item = blockIdx.x * blockDim.x + threadIdx.x, h = item / per, c = item % per;
  const bool on = h < kv_heads;
  // a row's bytes here: its stride, this thread's place in it
  const int t = c < kc ? 0 : c < kc + vc ? 1 : c - kc - vc + 2;
  uint8_t* pool = on ? pools.at[blockIdx.z][t] : nullptr;
  const int stride = t == 0 ? 16 * kc : t == 1 ? 16 * vc : 4, at = t == 0 ? 16 * c : t == 1 ? 16 * (c - kc) : 0;
  const long long head = (long long)h << s.shift;            // rows from head 0 to this one
  for (int i0 = 0; i0 < count; i0 += KEEP_ROWS) {
    __syncthreads();
    if (threadIdx.x < KEEP_ROWS) {
      const int i = i0 + threadIdx.x, k = i < count ? kept[start + i] : -1;
      int f = -1, d = -1;
      if (k >= 0 && k < n && k != i && base + i >= 0 && base + k >= 0) {
        const int fp = page_of(s, b, base + k), dp = page_of(s, b, base + i), mask = (1 << s.shift) - 1;
        if (fp >= 0 && dp >= 0) {
          f = ((fp * kv_heads) << s.shift) + ((base + k) & mask);
          d = ((dp * kv_heads) << s.shift) + ((base + i) & mask);
        }
      }
      from[threadIdx.x] = f;
      to[threadIdx.x] = d;
    }
    __syncthreads();
    if (!on) continue;
    for (int i = 0; i < min(count - i0, KEEP_ROWS); i += 8) {
      if (t < 2) {
        uint4 w[8];
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (from[i + e] >= 0) w[e] = *reinterpret_cast<const uint4*>(pool + (from[i + e] + head) * stride + at);
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (from[i + e] >= 0) *reinterpret_cast<uint4*>(pool + (to[i + e] + head) * stride + at) = w[e];
      } else {
        float w[8];
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (from[i + e] >= 0) w[e] = *reinterpret_cast<const float*>(pool + (from[i + e] + head) * 4);
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (from[i + e] >= 0) *reinterpret_cast<float*>(pool + (to[i + e] + head) * 4) = w[e];
      }
    }
  }
}

// the layers' pools, looked at like one layer's
static int check_pools(const char* who, const void* const* pools, int layers, const int* starts, const int* lengths, const int* table, int ldt, int width, int rows, int seqs, int pages,
                       int page, int kv_heads, int K, int V, int store, int act_dtype) {
  B2L_CHECK_ARG(layers >= 0 && (layers == 0 || pools), "%s: null pointer or a negative number of layers", who);
  for (int i = 0; i < layers; ++i)
    if (int rc = check_pool(who, pools[4 * i], pools[4 * i + 1], (const float*)pools[4 * i + 2], (const float*)pools[4 * i + 3], starts, lengths, table, ldt, width, rows, seqs, pages,
                            page, kv_heads, K, V, store, act_dtype))
      return rc;
  B2L_CHECK_SUPPORTED((long long)pages * kv_heads * page < (1ll << 31) && (long long)page * kv_heads * std::max(K, V) * 4 < (1ll << 31), "%s: pools of %d pages of %d heads", who, pages, kv_heads);
  return 0;
}
template <typename F> static int by_layers(const void* const* pools, int layers, int store, F launch) {
  for (int l0 = 0; l0 < layers; l0 += MOST_LAYERS) {
    const int n = std::min(layers - l0, MOST_LAYERS);
    Pools p{};
    for (int i = 0; i < n; ++i)
      for (int t = 0; t < 4; ++t) p.at[i][t] = t < 2 || store != ACT ? (uint8_t*)const_cast<void*>(pools[4 * (l0 + i) + t]) : nullptr;
    launch(p, n);
    B2L_LAUNCH_CHECK("paged moves");
  }
  return 0;
}

}  // namespace paged
}  // namespace b2l

using namespace b2l;

extern "C" int b2l_seq_paged_copy(const void* const* pools, int layers, const int* pairs, int n, int pages, int page, int kv_heads, int K, int V, int store, int act_dtype,
                                  b2l_stream_t stream) {
  using namespace paged;
  const char* who = "b2l_seq_paged_copy";
  B2L_CHECK_ARG(n >= 0 && (n == 0 || pairs), "%s: null pointer or a negative number of pages", who);
  B2L_CHECK_ARG(((uintptr_t)pairs & 7) == 0, "%s: pairs must be 8-byte aligned", who);
  if (int rc = check_pools(who, pools, layers, nullptr, nullptr, nullptr, 1, 1, 0, 0, pages, page, kv_heads, K, V, store, act_dtype)) return rc;
  B2L_CHECK_SUPPORTED(n < 65536, "%s: %d pages", who, n);
  if (n == 0) return 0;
  const PageBytes bytes = page_bytes(page, kv_heads, K, V, store, act_dtype);
  int pieces = 0;
  for (int t = 0; t < 4; ++t) pieces += (bytes.of[t] + PIECE - 1) / PIECE;
  return by_layers(pools, layers, store, [&](const Pools& p, int count) {
    paged_copy_kernel<<<dim3(pieces, n, count), 256, 0, (cudaStream_t)stream>>>(p, (const int2*)pairs, pages, bytes);
  });
}

extern "C" int b2l_seq_paged_keep(const void* const* pools, int layers, const int* starts, const int* lengths, const int* table, int ldt, int width, const int* kept, const int* counts,
                                  int rows, int seqs, int pages, int page, int kv_heads, int K, int V, int store, int act_dtype, b2l_stream_t stream) {
  using namespace paged;
  const char* who = "b2l_seq_paged_keep";
  B2L_CHECK_ARG(rows == 0 || seqs == 0 || (kept && counts), "%s: null pointer", who);
  if (int rc = check_pools(who, pools, layers, starts, lengths, table, ldt, width, rows, seqs, pages, page, kv_heads, K, V, store, act_dtype)) return rc;
  B2L_CHECK_SUPPORTED(seqs < 65536, "%s: %d sequences", who, seqs);
  if (rows == 0 || seqs == 0) return 0;
  const int es = store != ACT ? 1 : act_dtype == B2L_F32 ? 4 : 2, kc = K * es / 16, vc = V * es / 16, scaled = store != ACT ? 1 : 0;
  const long long items = (long long)kv_heads * (kc + vc + 2 * scaled);
  const Step s = step_of(starts, lengths, table, ldt, width, rows, seqs, pages, page);
  return by_layers(pools, layers, store, [&](const Pools& p, int count) {
    paged_keep_kernel<<<dim3((unsigned)((items + 127) / 128), seqs, count), 128, 0, (cudaStream_t)stream>>>(p, s, kept, counts, kv_heads, kc, vc, scaled);
  });
}
