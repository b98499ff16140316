// Attention over a paged pool: which rows and keys a CTA has, how results are stored, and the slow form for infinities.
#pragma once
#include "seq_paged.cuh"

namespace b2l {
namespace paged {

// 2^x, documented to 2^-22 of the result and without subnormals: as a weight that leaves out what is below 2^-126 of the largest
__device__ __forceinline__ float exp2_f(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__host__ __device__ inline int atoms_of(int D, int es) { return (D * es + 127) / 128; }      // 128-byte columns of a row

// Scales of values that go into exponents.  A smaller one (of a row of zeros it is 2^-126, of a place never written 0; others are of values below
// 2^-51) or a larger one (values beyond 10^14) makes the row be computed again: so no weight above 2^-40 of the largest is lost from the sum.
constexpr float SMALLEST_SCALE = 8.673617379884035e-19f, LARGEST_SCALE = 1.099511627776e12f;      // 2^-60, 2^40

// The power of two that brings a row's largest entry to 2^14 (1 for a row of zeros or with an infinity), and what its scores are multiplied with then
__device__ __forceinline__ void lift_of(float top, float scale_log2, float& up, float& down) {
  const int e = (int)(__float_as_uint(top) >> 23) - 127, by = top > 0.f && top < INFINITY ? min(14 - e, 120) : 0;
  up = __uint_as_float((uint32_t)(by + 127) << 23);
  down = scale_log2 * __uint_as_float((uint32_t)(127 - by) << 23);
}

// Codes (bytes) A0, A1 and B0, B1 of w as two f16 pairs.  An int8 code x: 1024 + (x + 128) is an f16 with x + 128 in its low byte
template <int STORE, int A0, int A1, int B0, int B1> __device__ __forceinline__ uint2 codes4(uint32_t w) {
  uint2 y;
  if constexpr (STORE == E4M3) {
    if constexpr (A0 != 0 || A1 != 1 || B0 != 2 || B1 != 3) w = __byte_perm(w, 0u, A0 | A1 << 4 | B0 << 8 | B1 << 12);
    asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}" : "=r"(y.x), "=r"(y.y) : "r"(w));
  } else {
    const uint32_t u = w ^ 0x80808080u, off = 0x64806480u;   // 1152 twice
    y.x = __byte_perm(u, 0x64646464u, A0 | 0x40 | A1 << 8 | 0x4000);
    y.y = __byte_perm(u, 0x64646464u, B0 | 0x40 | B1 << 8 | 0x4000);
    asm("sub.rn.f16x2 %0, %0, %1;" : "+r"(y.x) : "r"(off));
    asm("sub.rn.f16x2 %0, %0, %1;" : "+r"(y.y) : "r"(off));
  }
  return y;
}

// packed rows first .. of sequence b, which has n new tokens from row `start` on and is `length` tokens long with them
struct Place { int b, start, n, length, first; };

// The keys that some row of a tile sees, [0, early) and [lo, end), in units of a power of two
struct Keys {
  int early, lo, end, p_min, p_max, window, first;
  __device__ __forceinline__ int early_units(int shift) const { return min((early + (1 << shift) - 1) >> shift, lo >> shift); }
  __device__ __forceinline__ int units(int shift) const { return end <= 0 ? 0 : early_units(shift) + ((end + (1 << shift) - 1) >> shift) - (lo >> shift); }
  __device__ __forceinline__ int key0(int u, int shift) const {
    const int e = early_units(shift);
    return (u < e ? u : u - e + (lo >> shift)) << shift;
  }
  // whether every row of the tile sees all of keys j .. j + size - 1
  __device__ __forceinline__ bool whole(int j, int size) const { return j + size - 1 <= p_min && (window == 0 || j > p_max - window || j + size <= first); }
};

// partial results of `splits` CTAs per row: maximum and sum [splits][count][2], outputs [splits][count][V]
struct Parts { float *ml, *o; int splits; long long count; };

// What the CTAs of the chunk kernel leave for one another: of each the last row tile if it goes on in the next CTA (sequence, first packed row, head, number of
// CTAs that have a part; none: 0), and two places for partial results of 256 rows (the first row tile's, the last one's) [2 ctas][256][2] and [2 ctas][256][V]
struct Shared { int4* last; float *ml, *o; };

struct Attn {
  Step s;
  const void *q, *k, *v;
  const float *ks, *vs;
  void* out;
  long long ldq, hsq;
  int heads, kv_heads, K, V, window, first;
  int few_max;                                               // sequences of at most so many packed rows are the few-row kernel's, the others the chunk kernel's
  float scale_log2;
  int zeros;                                                 // whether rows of no sequence become zeros (else they stay as they are)
  int f32, store_kind, both;                                 // both: the two kernels share the step, few_max packed rows of every sequence and head in `few`
  Parts few;
  Shared many;

  __device__ __forceinline__ bool sees(int pos, int j) const { return j <= pos && (window == 0 || j > pos - window || j < first); }

  // Tile `slot` of the tiles of R packed rows of all sequences, without the first of each; a whole warp looks
  __device__ __forceinline__ bool place(int slot, int R, int lane, Place& pl) const {
    const int G = heads / kv_heads;
    int base = 0;
    for (int b0 = 0; b0 < s.seqs; b0 += 32) {
      const int b = b0 + lane;
      int start = 0, n = 0, length = 0, tiles = 0;
      if (b < s.seqs) {
        sequence(s, b, start, n, length);
        const long long packed = (long long)n * G;
        tiles = max((int)((packed + R - 1) / R) - 1, 0);
      }
      int upto = tiles;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += x;
      }
      const uint32_t past = __ballot_sync(0xffffffffu, slot < base + upto);
      if (past) {
        const int at = __ffs(past) - 1;
        pl.b = b0 + at;
        pl.start = __shfl_sync(0xffffffffu, start, at);
        pl.n = __shfl_sync(0xffffffffu, n, at);
        pl.length = __shfl_sync(0xffffffffu, length, at);
        pl.first = (slot - base - __shfl_sync(0xffffffffu, upto - tiles, at) + 1) * R;
        return true;
      }
      base += __shfl_sync(0xffffffffu, upto, 31);
    }
    return false;
  }
  __device__ __forceinline__ Keys keys(const Place& pl, int R) const {
    const int G = heads / kv_heads, last = min(pl.first + R, pl.n * G) - 1;
    Keys x;
    x.p_min = pl.length - pl.n + pl.first / G;
    x.p_max = pl.length - pl.n + last / G;
    x.end = x.p_max + 1;
    x.lo = window ? max(x.p_min - window + 1, 0) : 0;
    x.early = min(first, x.lo);
    x.window = window;
    x.first = first;
    return x;
  }

  __device__ __forceinline__ void store(size_t at, const float (&x)[4], float inv) const {      // at: of the first of four outputs
    const float4 y = make_float4(x[0] * inv, x[1] * inv, x[2] * inv, x[3] * inv);
    if (f32) st_act4(reinterpret_cast<float*>(out) + at, y);
    else st_act4(reinterpret_cast<__nv_bfloat16*>(out) + at, y);
  }

  __device__ __forceinline__ float element(const void* p, const float* scales, size_t row, int D, int d) const {
    const size_t at = row * D + d;
    if (store_kind == ACT) return f32 ? reinterpret_cast<const float*>(p)[at] : bf2f(reinterpret_cast<const __nv_bfloat16*>(p)[at]);
    const uint8_t c = reinterpret_cast<const uint8_t*>(p)[at];
    return (store_kind == E4M3 ? e4m3_pair(c).x : (float)(int8_t)c) * scales[row];
  }
};

// Zeros in the outputs of rows r0 .. r1 - 1, n heads from `head` on
static __device__ __noinline__ void clear_rows(const Attn& a, int r0, int r1, int head, int n, int me, int threads) {
  const int es = a.f32 ? 4 : 2, pieces = n * a.V * es / 16;
  for (long long i = me; i < (long long)(r1 - r0) * pieces; i += threads)
    *reinterpret_cast<uint4*>(reinterpret_cast<uint8_t*>(a.out) + ((size_t)(r0 + i / pieces) * a.heads + head) * a.V * es + i % pieces * 16) = make_uint4(0u, 0u, 0u, 0u);
}

// One row and head again by a warp, key after key over what the row sees and nothing else.  The products above multiply a hidden value by a weight of
// zero, and an f32 infinity has parts of NaN: a result that is not finite is computed again here, so it is what the formula says.
static __device__ __noinline__ void mend_row(const Attn& a, int b, int pos, int row, int head, int lane) {
  const int h = head / (a.heads / a.kv_heads);
  float q[8], o[8], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int d = lane + 32 * i;
    const size_t at = (size_t)row * a.ldq + (size_t)head * a.hsq + d;
    q[i] = d < a.K ? (a.f32 ? reinterpret_cast<const float*>(a.q)[at] : bf2f(reinterpret_cast<const __nv_bfloat16*>(a.q)[at])) : 0.f;
    o[i] = 0.f;
  }
  for (int j = 0; j <= pos; ++j) {
    if (!a.sees(pos, j)) {
      j = max(j, pos - a.window);                            // the next key is the window's first
      continue;
    }
    const int page = page_of(a.s, b, j);
    if (page < 0) continue;
    const size_t at = (((size_t)page * a.kv_heads + h) << a.s.shift) + (j & ((1 << a.s.shift) - 1));
    float x = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (lane + 32 * i < a.K) x = fmaf(q[i], a.element(a.k, a.ks, at, a.K, lane + 32 * i), x);
    x = warp_sum(x) * a.scale_log2;
    if (x == -INFINITY) continue;
    const float now = fmaxf(m, x), f = m == now ? 1.f : exp2_f(m - now), w = exp2_f(x - now);
    m = now;
    l = l * f + w;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (lane + 32 * i < a.V) o[i] = o[i] * f + w * a.element(a.v, a.vs, at, a.V, lane + 32 * i);
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int d = lane + 32 * i;
    const size_t at = ((size_t)row * a.heads + head) * a.V + d;
    if (d < a.V) {
      if (a.f32) reinterpret_cast<float*>(a.out)[at] = o[i] * inv;
      else reinterpret_cast<__nv_bfloat16*>(a.out)[at] = f2bf(o[i] * inv);
    }
  }
}
__device__ __forceinline__ bool finite4(const float (&x)[4], float inv) {
  return fabsf(x[0] * inv) < INFINITY && fabsf(x[1] * inv) < INFINITY && fabsf(x[2] * inv) < INFINITY && fabsf(x[3] * inv) < INFINITY;
}

// the tensor-core kernel of longer chunks (seq_paged_tc.cu): heads that it takes, the CTAs for at most so many row tiles and keys, its work space, its launch
bool many_takes(int K, int V, int store);
int many_ctas(long long row_tiles, long long keys, int sms);
long long many_floats(int ctas, int V);
int many_launch(Attn& a, int ctas, float* work, cudaStream_t stream);

}  // namespace paged
}  // namespace b2l
