// Rows of logits: a block's part of one in registers, whatever the row's alignment.
#pragma once
#include "seq_common.cuh"

namespace b2l {
namespace rows {

// Entries `at + (v blockDim.x + thread) PER + e` of a row of `n`, v < VECS and e < PER the entries of 16 bytes, as f32; `none` where there is none.  `at` is such that
// the 16 bytes lie on their border (at most PER - 1 entries before the row or a part begins).
template <typename T> constexpr int PER = 16 / (int)sizeof(T);
// whether all of a block's entries are the row's
template <typename T, int VECS> __device__ __forceinline__ bool inside(int at, int n) { return at >= 0 && at + VECS * (int)blockDim.x * PER<T> <= n; }
template <typename T, int VECS> __device__ __forceinline__ void load(const T* row, int at, int n, float none, float (&x)[VECS * PER<T>]) {
  auto entries = [&](int v, uint4 u) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int e = 0; e < PER<T>; ++e) x[v * PER<T> + e] = sizeof(T) == 4 ? __uint_as_float(w[e]) : __uint_as_float(e & 1 ? w[e >> 1] & 0xffff0000u : w[e >> 1] << 16);
  };
  if (inside<T, VECS>(at, n)) {                              // without a branch between them, so that they are under way together
    uint4 u[VECS];
#pragma unroll
    for (int v = 0; v < VECS; ++v) u[v] = __ldcs(reinterpret_cast<const uint4*>(row + at + (v * (int)blockDim.x + (int)threadIdx.x) * PER<T>));
#pragma unroll
    for (int v = 0; v < VECS; ++v) entries(v, u[v]);
    return;
  }
#pragma unroll
  for (int v = 0; v < VECS; ++v) {
    const int i = at + (v * (int)blockDim.x + (int)threadIdx.x) * PER<T>;
    if (i >= 0 && i + PER<T> <= n) {
      entries(v, __ldcs(reinterpret_cast<const uint4*>(row + i)));
    } else {
#pragma unroll
      for (int e = 0; e < PER<T>; ++e) x[v * PER<T> + e] = i + e >= 0 && i + e < n ? ld_act(row, i + e) : none;
    }
  }
}
// entries before the row's first 16-byte border, counted down: 0 or minus a few
template <typename T> __device__ __forceinline__ int border(const T* row) { return -(int)(((uintptr_t)row & 15) / sizeof(T)); }

}  // namespace rows
}  // namespace b2l
