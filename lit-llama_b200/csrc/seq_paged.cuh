// Paged caches: what the kernels that write, read and attend to them share.
//
// A pool holds one layer's keys and values of many sequences in `pages` pages of `page` tokens: k [pages][kv_heads][page][K], v [pages][kv_heads][page][V],
// so the tokens of one head in one page are consecutive bytes, and 16 of them (a page is a power of two of at least 16) never cross a page.  Elements are of
// the activation type, e4m3 or int8; an 8-bit pool has one f32 scale per token and head, [pages][kv_heads][page].
// A step gives sequence b the rows starts[b] .. starts[b + 1] - 1; with them it is lengths[b] tokens long, and its tokens lie in the pages table[b][..].
// Everything is read on the device and clipped to the sizes that the host knows; a table entry outside the pool is a page that is not there: nothing is
// written to it, it reads as zeros and no row sees its keys.
#pragma once
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "seq_common.cuh"

namespace b2l {
namespace paged {

struct Step {
  const int *starts, *lengths, *table;
  int ldt, width;                   // of the table: entries between rows, entries of a sequence
  int rows, seqs, pages, shift;     // shift: log2 of the page
};

// where sequence b's rows begin, how many it has, and how long it is with them
__device__ __forceinline__ void sequence(const Step& s, int b, int& start, int& n, int& length) {
  start = min(max(s.starts[b], 0), s.rows);
  n = max(min(s.starts[b + 1], s.rows) - start, 0);
  length = (int)min((long long)max(s.lengths[b], 0), (long long)s.width << s.shift);
}
// the page with token j of sequence b, or -1
__device__ __forceinline__ int page_of(const Step& s, int b, int j) {
  const int p = s.table[(size_t)b * s.ldt + (j >> s.shift)];
  return p >= 0 && p < s.pages ? p : -1;
}
// The sequence that has `row`, or -1: a whole warp looks, 32 places at a time (two rounds of loads up to 1024 sequences).
__device__ __forceinline__ int sequence_of(const Step& s, int row, int lane) {
  if (s.seqs <= 0 || row < s.starts[0] || row >= s.starts[s.seqs]) return -1;
  int lo = 0, hi = s.seqs;                                 // starts[lo] <= row < starts[hi]
  while (hi - lo > 1) {
    const int by = (hi - lo + 31) / 32, at = lo + lane * by;
    const int below = __popc(__ballot_sync(0xffffffffu, at < hi && s.starts[min(at, hi)] <= row));      // starts do not fall, so these come first
    lo += max(below - 1, 0) * by;
    hi = min(lo + by, hi);
  }
  return lo;
}

// ---- elements of a pool
constexpr int ACT = B2L_SEQ_STORE_ACT, E4M3 = B2L_SEQ_STORE_E4M3, INT8 = B2L_SEQ_STORE_INT8;
// two e4m3 codes (the low 16 bits of w) as f32: every e4m3 value is one of f16, NaN included
__device__ __forceinline__ float2 e4m3_pair(uint32_t w) {
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w & 0xffffu), __NV_E4M3);
  return __half22float2(__half2(h));
}

// ---- host
inline int check_pool(const char* who, const void* k, const void* v, const void* ks, const void* vs, const int* starts, const int* lengths, const int* table, int ldt, int width,
                      int rows, int seqs, int pages, int page, int kv_heads, int K, int V, int store, int act_dtype) {
  B2L_CHECK_ARG(k && v && (rows == 0 || seqs == 0 || (starts && lengths && table)), "%s: null pointer", who);      // empty tensors have no address
  B2L_CHECK_SUPPORTED(act_dtype == B2L_BF16 || act_dtype == B2L_F32, "%s: act_dtype %d unsupported", who, act_dtype);
  B2L_CHECK_SUPPORTED(store == ACT || store == E4M3 || store == INT8, "%s: store %d unsupported", who, store);
  B2L_CHECK_ARG(store == ACT || (ks && vs), "%s: an 8-bit pool needs its scales", who);
  B2L_CHECK_ARG(rows >= 0 && seqs >= 0 && pages > 0 && kv_heads > 0 && width > 0 && ldt >= width, "%s: bad sizes", who);
  B2L_CHECK_SUPPORTED(page >= 16 && page <= 256 && (page & (page - 1)) == 0, "%s: a page of %d tokens: 16, 32, 64, 128 or 256", who, page);
  B2L_CHECK_SUPPORTED(K >= 16 && K <= 256 && K % 16 == 0 && V >= 16 && V <= 256 && V % 16 == 0, "%s: heads of %d and %d entries: multiples of 16 up to 256", who, K, V);
  B2L_CHECK_ARG((((uintptr_t)k | (uintptr_t)v | (uintptr_t)ks | (uintptr_t)vs) & 15) == 0, "%s: the pool must be 16-byte aligned", who);
  return 0;
}
inline Step step_of(const int* starts, const int* lengths, const int* table, int ldt, int width, int rows, int seqs, int pages, int page) {
  return Step{starts, lengths, table, ldt, width, rows, seqs, pages, __builtin_ctz((unsigned)page)};
}

}  // namespace paged
}  // namespace b2l
