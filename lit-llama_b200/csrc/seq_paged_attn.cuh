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

// What the new tokens of a step see of one another: token i of a sequence those before it and itself, or (TREE) those whose bits its mask has, [rows][words] words of
// 32; then its position is the sequence's first new token's plus its depth
struct Tree { const uint32_t* masks; const int* depths; int words; };

__device__ __forceinline__ uint32_t low_bits(int n) { return n >= 32 ? 0xffffffffu : n <= 0 ? 0u : (1u << n) - 1u; }      // bits 0 .. n-1 (any n)

template <bool TREE> struct Attn {
  static constexpr bool tree = TREE;
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
  Tree nodes;
  bool joined;                                               // the few-row kernel's parts are joined by a cluster of CTAs

  // position of new token i of a sequence whose n new ones begin at position `base` and row `start`
  __device__ __forceinline__ int position(int start, int base, int n, int i) const {
    if constexpr (TREE) return base + min(max(nodes.depths[start + i], 0), n - 1);
    else return base + i;
  }
  __device__ __forceinline__ bool in_window(int pos, int j) const { return window == 0 || j > pos - window || j < first; }
  // Bits i0 .. i0 + 31 of the mask of a row, of a sequence with n new tokens
  __device__ __forceinline__ uint32_t tree_bits(int row, int n, int i0) const {
    if (i0 >= n || i0 <= -32) return 0u;
    const uint32_t* m = nodes.masks + (size_t)row * nodes.words;
    const int w = i0 >> 5;                                   // -1 where the context ends inside
    const uint32_t lo = w >= 0 && w < nodes.words ? m[w] : 0u, hi = w + 1 < nodes.words ? m[w + 1] : 0u;
    return __funnelshift_r(lo, hi, i0 & 31) & low_bits(n - i0);
  }
  // whether a row at position `pos` sees key j; its sequence's n new tokens begin at `base`
  __device__ __forceinline__ bool sees(int pos, int row, int base, int n, int j) const {
    if constexpr (TREE) return j < base ? in_window(pos, j) : (tree_bits(row, n, j - base) & 1u) != 0u;
    else return j <= pos && in_window(pos, j);
  }
  // the same of keys j .. j + 31, as bits
  __device__ __forceinline__ uint32_t seen32(int pos, int row, int base, int n, int j) const {
    uint32_t x = low_bits((TREE ? base : pos + 1) - j);
    if (window) x &= ~low_bits(pos - window + 1 - j) | low_bits(first - j);
    if constexpr (TREE) x |= tree_bits(row, n, j - base);
    return x;
  }

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
    if constexpr (TREE) {                                    // rows of any depth
      x.p_min = pl.length - pl.n;
      x.p_max = pl.length - 1;
      x.end = pl.length;
    } else {
      x.p_min = pl.length - pl.n + pl.first / G;
      x.p_max = pl.length - pl.n + last / G;
      x.end = x.p_max + 1;
    }
    x.lo = window ? max(x.p_min - window + 1, 0) : 0;
    if constexpr (TREE) --x.p_min;                           // the last key that all of them may see
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

  // eight entries from `at` on, of the activation type (scale: none) or codes
  __device__ __forceinline__ void eight(const void* p, size_t at, const float* scale, float (&x)[8]) const {
    if (scale == nullptr) {
      float4 u, v;
      if (f32) {
        u = ld_act4(reinterpret_cast<const float*>(p) + at);
        v = ld_act4(reinterpret_cast<const float*>(p) + at + 4);
      } else {
        u = ld_act4(reinterpret_cast<const __nv_bfloat16*>(p) + at);
        v = ld_act4(reinterpret_cast<const __nv_bfloat16*>(p) + at + 4);
      }
      x[0] = u.x; x[1] = u.y; x[2] = u.z; x[3] = u.w; x[4] = v.x; x[5] = v.y; x[6] = v.z; x[7] = v.w;
      return;
    }
    const uint2 w = *reinterpret_cast<const uint2*>(reinterpret_cast<const uint8_t*>(p) + at);
    const float s = *scale;
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
      const uint32_t u = (i < 4 ? w.x : w.y) >> 8 * (i & 2);
      const float2 y = store_kind == E4M3 ? e4m3_pair(u) : make_float2((float)(int8_t)u, (float)(int8_t)(u >> 8));
      x[i] = y.x * s;
      x[i + 1] = y.y * s;
    }
  }
};

// Zeros in the outputs of rows r0 .. r1 - 1, n heads from `head` on
template <bool TREE> static __device__ __noinline__ void clear_rows(const Attn<TREE>& a, int r0, int r1, int head, int n, int me, int threads) {
  const int es = a.f32 ? 4 : 2, pieces = n * a.V * es / 16;
  for (long long i = me; i < (long long)(r1 - r0) * pieces; i += threads)
    *reinterpret_cast<uint4*>(reinterpret_cast<uint8_t*>(a.out) + ((size_t)(r0 + i / pieces) * a.heads + head) * a.V * es + i % pieces * 16) = make_uint4(0u, 0u, 0u, 0u);
}

// Rows and heads of one sequence and key/value head, again by a warp, over what each sees and nothing else, in f32.  The products above multiply a hidden value by
// a weight of zero, and an f32 infinity has parts of NaN: a result that is not finite is computed again here, so it is what the formula says.
// 32 keys at a time, of which a lane has one for the scores, and then 8 entries of every value, for MENDED rows together: four, and two in the chunk kernel, which
// with more spills registers in its loops.  All of 512 tokens' rows again, 32 / 8 heads of 128 over 4096 keys of an int8 pool: 11.3 ms (78 with a row at a time, key
// after key); one token's over 16384 keys 9.6 ms (37).  Where all of a row is NaN it stays so, and the rest is left out: 1.7 and 0.4 ms with a NaN among the first.
template <int MENDED> struct Again { int n, pos[MENDED], row[MENDED], head[MENDED]; };
template <int MENDED, bool TREE> __device__ __forceinline__ void mend_few(const Attn<TREE>& a, int b, int h, const Again<MENDED>& x, int base, int n_new, int lane) {
  float m[MENDED], l[MENDED], o[MENDED][8];
  int p_min = x.pos[0], p_max = x.pos[0];
#pragma unroll
  for (int r = 0; r < MENDED; ++r) {
    if (r < x.n) {
      p_min = min(p_min, x.pos[r]);
      p_max = max(p_max, x.pos[r]);
    }
    m[r] = -INFINITY;
    l[r] = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) o[r][e] = 0.f;
  }
  if constexpr (TREE) p_max = base + n_new - 1;
  int from = p_min - a.window + 1;                           // the first window; of a tree's new tokens the masks decide
  if constexpr (TREE) from = min(from, base);
  for (int j0 = 0; j0 <= p_max; j0 += 32) {
    if (a.window && j0 >= a.first && j0 + 31 < from) {       // on to it
      j0 = (from & ~31) - 32;
      continue;
    }
    const int j = j0 + lane;
    bool any = false;
#pragma unroll
    for (int r = 0; r < MENDED; ++r) any |= r < x.n && a.sees(x.pos[r], x.row[r], base, n_new, j);
    const int page = any ? page_of(a.s, b, j) : -1;
    const size_t at = (((size_t)max(page, 0) * a.kv_heads + h) << a.s.shift) + (j & ((1 << a.s.shift) - 1));
    float w[MENDED] = {};
    if (page >= 0)
      for (int d = 0; d < a.K; d += 8) {
        float k[8];
        a.eight(a.k, at * a.K + d, a.store_kind == ACT ? nullptr : a.ks + at, k);
#pragma unroll
        for (int r = 0; r < MENDED; ++r) {
          if (r >= x.n) break;
          float q[8];
          a.eight(a.q, (size_t)x.row[r] * a.ldq + (size_t)x.head[r] * a.hsq + d, nullptr, q);
#pragma unroll
          for (int e = 0; e < 8; ++e) w[r] = fmaf(q[e], k[e], w[r]);
        }
      }
    bool has = false;                                        // whether the key has a weight in some row; a weight of -1: it is not seen
#pragma unroll
    for (int r = 0; r < MENDED; ++r) {
      if (r >= x.n) break;
      const float s = page >= 0 && a.sees(x.pos[r], x.row[r], base, n_new, j) ? w[r] * a.scale_log2 : -INFINITY;
      float now = s;
#pragma unroll
      for (int y = 16; y > 0; y >>= 1) now = fmaxf(now, __shfl_xor_sync(0xffffffffu, now, y));
      now = fmaxf(now, m[r]);
      const float f = m[r] == now ? 1.f : exp2_f(m[r] - now);
      m[r] = now;
      w[r] = s == -INFINITY ? -1.f : exp2_f(s - now);
      has |= s != -INFINITY;
      l[r] = l[r] * f + warp_sum(s == -INFINITY ? 0.f : w[r]);
#pragma unroll
      for (int e = 0; e < 8; ++e) o[r][e] *= f;
    }
    const uint32_t mine = __ballot_sync(0xffffffffu, has);
#pragma unroll 2
    for (int i = 0; i < 32; ++i) {
      if (!(mine >> i & 1u)) continue;
      const size_t of = __shfl_sync(0xffffffffu, (unsigned long long)at, i);
      float v[8] = {};
      if (8 * lane < a.V) a.eight(a.v, of * a.V + 8 * lane, a.store_kind == ACT ? nullptr : a.vs + of, v);
#pragma unroll
      for (int r = 0; r < MENDED; ++r) {
        const float y = __shfl_sync(0xffffffffu, w[r], i);
        if (r < x.n && !(y < 0.f))
#pragma unroll
          for (int e = 0; e < 8; ++e) o[r][e] = fmaf(y, v[e], o[r][e]);
      }
    }
    bool over = true;                                        // all of every row is NaN
#pragma unroll
    for (int r = 0; r < MENDED; ++r) {
      bool nan = true;
#pragma unroll
      for (int e = 0; e < 8; ++e) nan = nan && o[r][e] != o[r][e];
      over = over && (r >= x.n || l[r] != l[r] || 8 * lane >= a.V || nan);
    }
    if (__all_sync(0xffffffffu, over)) break;
  }
#pragma unroll
  for (int r = 0; r < MENDED; ++r) {
    if (r >= x.n || 8 * lane >= a.V) break;
    const float inv = l[r] == 0.f ? 0.f : 1.f / l[r];
    const size_t at = ((size_t)x.row[r] * a.heads + x.head[r]) * a.V + 8 * lane;
    const float lo[4] = {o[r][0], o[r][1], o[r][2], o[r][3]}, hi[4] = {o[r][4], o[r][5], o[r][6], o[r][7]};
    a.store(at, lo, inv);
    a.store(at + 4, hi, inv);
  }
}
// Packed rows at + i of sequence b and key/value head h, for the bits i of `left`; its rows begin at `start`, its new tokens at position `pos`
template <int MENDED, bool TREE> static __device__ __noinline__ void mend_rows(const Attn<TREE>& a, int b, int start, int pos, int h, int at, uint32_t left, int lane) {
  const int G = a.heads / a.kv_heads;
  int n = 0;
  if constexpr (TREE) {
    int first_row, length;
    sequence(a.s, b, first_row, n, length);
  }
  while (left) {
    Again<MENDED> x;
    x.n = min(__popc(left), MENDED);
#pragma unroll
    for (int r = 0; r < MENDED; ++r) {
      const int i = at + (left ? __ffs(left) - 1 : 0);       // (one too many is not looked at)
      left &= left - 1;
      x.pos[r] = a.position(start, pos, n, min(i / G, TREE ? n - 1 : i / G));
      x.row[r] = start + i / G;
      x.head[r] = h * G + i % G;
    }
    mend_few<MENDED>(a, b, h, x, pos, n, lane);
  }
}
__device__ __forceinline__ bool finite4(const float (&x)[4], float inv) {
  return fabsf(x[0] * inv) < INFINITY && fabsf(x[1] * inv) < INFINITY && fabsf(x[2] * inv) < INFINITY && fabsf(x[3] * inv) < INFINITY;
}

// the tensor-core kernel of longer chunks (seq_paged_tc.cu): heads that it takes; the CTAs for at most so many packed rows of `tiles` sequences, and keys; its work space;
// its launch.  pair: row tiles of 128 rows that both halves of a CTA compute
bool many_takes(int K, int V, int store);
bool pair_takes(int K, int V, int store);
int many_ctas(bool pair, long long packed, long long tiles, int kv_heads, long long keys, int sms);
long long many_floats(bool pair, int ctas, int V);
template <bool TREE> int many_launch(const Attn<TREE>& a, bool pair, int ctas, float* work, cudaStream_t stream);

}  // namespace paged
}  // namespace b2l
