// Rows into a paged pool, quantised on the way, and out of it (layout: seq_paged.cuh).
//
// A row of size D of one head is quantised by itself: scale s = max(max |x| (1 / c), 2^-126), code = round(x / s) (to nearest, ties to even), c = 448 for e4m3
// and 127 for int8, so a code is off by at most half a step: 2^-4 of itself (e4m3, normal codes) or s / 2 (int8).  The floor of s keeps x / s finite for
// rows of zeros and subnormals.  A row with an infinity or NaN gets the scale NaN and codes 0: it reads back as NaN, and its codes stay finite where a mask
// hides them.  1 / c is rounded to f32, and the division by s is the correctly rounded one, so the codes are the same wherever the formula is computed in f32.
//
// 16 lanes have a row of keys, the other 16 of the warp the row of values of the same token and head, each lane 8 elements at a time: 16-byte loads of bf16.
// What bounds it: the write of prompts, 10367 tokens of 32 + 32 heads of 128 into int8 in 58 us or 4.4 TB/s, by its instructions (the issue is 72% busy:
// largest entry, quotients and codes); their read, 44056 tokens of 8 + 8 heads in 52 us, 5.3 TB/s, by HBM.  Single tokens: the launch and one chain of loads
// (starts, length, table), 2.2 us for one, 3.2 us for 96.
#include <math_constants.h>

#include "seq_paged.cuh"

namespace b2l {
namespace paged {

struct Rows {
  Step s;
  const void *k_new, *v_new;         // or, for reading, where the rows go
  long long ldk, hsk, ldv, hsv;      // elements between tokens and between heads of them
  void *k, *v;
  float *ks, *vs;
  int kv_heads, K, V;
};

__device__ __forceinline__ void store8(float* p, const float (&x)[8]) {
  *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
  *reinterpret_cast<float4*>(p + 4) = make_float4(x[4], x[5], x[6], x[7]);
}
__device__ __forceinline__ void store8(__nv_bfloat16* p, const float (&x)[8]) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __nv_bfloat162 y = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
    w[i] = *reinterpret_cast<const uint32_t*>(&y);
  }
  *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
}
// Eight entries as they lie: the largest absolute value as f32 bits (an infinity's or more where one is not finite), and the entries
struct Raw8f { float4 a, b; };
__device__ __forceinline__ Raw8f raw8(const float* p) { return {*reinterpret_cast<const float4*>(p), *reinterpret_cast<const float4*>(p + 4)}; }
__device__ __forceinline__ uint4 raw8(const __nv_bfloat16* p) { return *reinterpret_cast<const uint4*>(p); }
__device__ __forceinline__ void clear(Raw8f& w) { w.a = w.b = make_float4(0.f, 0.f, 0.f, 0.f); }
__device__ __forceinline__ void clear(uint4& w) { w = make_uint4(0u, 0u, 0u, 0u); }
__device__ __forceinline__ uint32_t largest8(const Raw8f& w) {
  auto bits = [](float x) { return __float_as_uint(x) & 0x7fffffffu; };
  return max(max(max(bits(w.a.x), bits(w.a.y)), max(bits(w.a.z), bits(w.a.w))), max(max(bits(w.b.x), bits(w.b.y)), max(bits(w.b.z), bits(w.b.w))));
}
__device__ __forceinline__ uint32_t largest8(const uint4& w) {      // two entries at a time
  const uint32_t m = __vmaxu2(__vmaxu2(w.x & 0x7fff7fffu, w.y & 0x7fff7fffu), __vmaxu2(w.z & 0x7fff7fffu, w.w & 0x7fff7fffu));
  return max(m << 16, m & 0xffff0000u);
}
__device__ __forceinline__ void entries8(const Raw8f& w, float (&x)[8]) {
  x[0] = w.a.x; x[1] = w.a.y; x[2] = w.a.z; x[3] = w.a.w; x[4] = w.b.x; x[5] = w.b.y; x[6] = w.b.z; x[7] = w.b.w;
}
__device__ __forceinline__ void entries8(const uint4& w, float (&x)[8]) {
  const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = __uint_as_float(u[i] << 16);
    x[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
  }
}
// x / s correctly rounded, two at a time: the quotient by the correctly rounded reciprocal, corrected by its own remainder (Markstein).  The remainder is exact
// while it is a normal number, so for s above 2^-90 or so; below the division operator (a third of the instructions of a row otherwise)
__device__ __forceinline__ void over2(float& x, float& y, float s, float r) {
  asm("{\n\t.reg .b64 a, q, d, r, s;\n\tmov.b64 a, {%0, %1};\n\tmov.b64 r, {%2, %2};\n\tmov.b64 s, {%3, %3};\n\tmul.rn.f32x2 q, a, r;\n\tfma.rn.f32x2 d, q, s, a;\n\t"
      "fma.rn.f32x2 q, d, r, q;\n\tmov.b64 {%0, %1}, q;\n\t}"
      : "+f"(x), "+f"(y)
      : "f"(r), "f"(-s));
}
template <int STORE> __device__ __forceinline__ uint2 codes8(float (&x)[8], float s, float r) {      // s: not NaN
  if (s > 8.077935669463161e-28f) {                          // 2^-90
#pragma unroll
    for (int i = 0; i < 8; i += 2) over2(x[i], x[i + 1], s, r);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = __fdiv_rn(x[i], s);
  }
  uint32_t w[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    if (STORE == E4M3) {
      const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(x[4 * i], x[4 * i + 1]), __NV_SATFINITE, __NV_E4M3);
      const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(x[4 * i + 2], x[4 * i + 3]), __NV_SATFINITE, __NV_E4M3);
      w[i] = lo | hi << 16;
    } else {                                                 // 1.5 2^23 more: the nearest integer in the low byte; |x / s| is at most 127 (1 + 2^-22)
      uint32_t b[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) b[e] = __float_as_uint(x[4 * i + e] + 12582912.f);
      w[i] = __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
    }
  }
  return make_uint2(w[0], w[1]);
}
template <int STORE> __device__ __forceinline__ void values8(uint2 w, float s, float (&x)[8]) {
#pragma unroll
  for (int i = 0; i < 8; i += 4) {
    const uint32_t u = i ? w.y : w.x;
    if (STORE == E4M3) {
      const float2 f = e4m3_pair(u), g = e4m3_pair(u >> 16);
      x[i] = f.x; x[i + 1] = f.y; x[i + 2] = g.x; x[i + 3] = g.y;
    } else {                                                 // 2^23 + 128 + code, less 2^23 + 128 (a conversion is a fourth as fast)
      const uint32_t v = u ^ 0x80808080u;
      x[i] = __uint_as_float(__byte_perm(v, 0x4b000000u, 0x7650)) - 8388736.f;
      x[i + 1] = __uint_as_float(__byte_perm(v, 0x4b000000u, 0x7651)) - 8388736.f;
      x[i + 2] = __uint_as_float(__byte_perm(v, 0x4b000000u, 0x7652)) - 8388736.f;
      x[i + 3] = __uint_as_float(__byte_perm(v, 0x4b000000u, 0x7653)) - 8388736.f;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) x[i + e] *= s;
  }
}

// NI: 128-entry parts of the longest row; HEADS: of a token that a warp takes: one look for its place, the loads of all in flight together
template <typename act_t, int STORE, int NI, int HEADS>
__global__ void __launch_bounds__(256) paged_write_kernel(const __grid_constant__ Rows a) {
  const int lane = threadIdx.x & 31, l = lane & 15;
  const bool value = lane >= 16;
  const uint32_t groups = (uint32_t)(a.kv_heads + HEADS - 1) / HEADS;
  const uint32_t unit = blockIdx.x * (blockDim.x / 32) + threadIdx.x / 32;
  const int row = (int)(unit / groups), h0 = (int)(unit % groups) * HEADS;
  if (row >= a.s.rows) return;
  const int D = value ? a.V : a.K;
  const long long hs = value ? a.hsv : a.hsk;
  const act_t* src = reinterpret_cast<const act_t*>(value ? a.v_new : a.k_new) + row * (value ? a.ldv : a.ldk) + h0 * hs + 8 * l;
  decltype(raw8(src)) raw[HEADS][NI];
#pragma unroll
  for (int h = 0; h < HEADS; ++h)
#pragma unroll
    for (int i = 0; i < NI; ++i)
      if (h0 + h < a.kv_heads && 8 * (l + 16 * i) < D) raw[h][i] = raw8(src + h * hs + 128 * i);
      else clear(raw[h][i]);
  const int b = sequence_of(a.s, row, lane);
  if (b < 0) return;
  int start, n, length;
  sequence(a.s, b, start, n, length);
  const int p = length - n + row - start;
  const int page = p >= 0 ? page_of(a.s, b, p) : -1;
  if (page < 0) return;
  size_t at = (((size_t)page * a.kv_heads + h0) << a.s.shift) + (p & ((1 << a.s.shift) - 1));
#pragma unroll
  for (int h = 0; h < HEADS; ++h, at += (size_t)1 << a.s.shift) {
    if (h0 + h >= a.kv_heads) break;
    if (STORE == ACT) {
      act_t* dst = reinterpret_cast<act_t*>(value ? a.v : a.k) + at * D + 8 * l;
#pragma unroll
      for (int i = 0; i < NI; ++i)
        if (8 * (l + 16 * i) < D) *reinterpret_cast<decltype(raw8(src))*>(dst + 128 * i) = raw[h][i];
      continue;
    }
    uint32_t top = 0u;
#pragma unroll
    for (int i = 0; i < NI; ++i) top = max(top, largest8(raw[h][i]));
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
    const bool odd = top >= 0x7f800000u;                     // an infinity or NaN
    const float s = odd ? CUDART_NAN_F : fmaxf(__uint_as_float(top) * (STORE == E4M3 ? 1.f / 448.f : 1.f / 127.f), 1.17549435e-38f), r = __frcp_rn(s);
    if (l == 0) (value ? a.vs : a.ks)[at] = s;
    uint8_t* dst = reinterpret_cast<uint8_t*>(value ? a.v : a.k) + at * D + 8 * l;
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      if (8 * (l + 16 * i) >= D) break;
      float x[8];
      entries8(raw[h][i], x);
      *reinterpret_cast<uint2*>(dst + 128 * i) = odd ? make_uint2(0u, 0u) : codes8<STORE>(x, s, r);
    }
  }
}

template <typename act_t, int STORE, int NI, int HEADS>
__global__ void __launch_bounds__(256) paged_read_kernel(const __grid_constant__ Rows a) {
  const int lane = threadIdx.x & 31, l = lane & 15;
  const bool value = lane >= 16;
  const uint32_t groups = (uint32_t)(a.kv_heads + HEADS - 1) / HEADS;
  const uint32_t unit = blockIdx.x * (blockDim.x / 32) + threadIdx.x / 32;
  const int row = (int)(unit / groups), h0 = (int)(unit % groups) * HEADS;
  if (row >= a.s.rows) return;
  const int b = sequence_of(a.s, row, lane);
  int start = 0, n = 0, length = 0;
  if (b >= 0) sequence(a.s, b, start, n, length);
  const int p = b >= 0 ? length - n + row - start : -1;      // a row of no sequence reads as one whose page is not there
  const int page = p >= 0 ? page_of(a.s, b, p) : -1;
  const int D = value ? a.V : a.K;
  const size_t at = (((size_t)max(page, 0) * a.kv_heads + h0) << a.s.shift) + (p & ((1 << a.s.shift) - 1)), to_next = (size_t)1 << a.s.shift;
  const long long hs = value ? a.hsv : a.hsk;
  act_t* dst = reinterpret_cast<act_t*>(const_cast<void*>(value ? a.v_new : a.k_new)) + row * (value ? a.ldv : a.ldk) + h0 * hs + 8 * l;
  if (STORE == ACT) {
    const act_t* src = reinterpret_cast<const act_t*>(value ? a.v : a.k) + at * D + 8 * l;
    decltype(raw8(src)) raw[HEADS][NI];
#pragma unroll
    for (int h = 0; h < HEADS; ++h)
#pragma unroll
      for (int i = 0; i < NI; ++i)
        if (page >= 0 && h0 + h < a.kv_heads && 8 * (l + 16 * i) < D) raw[h][i] = raw8(src + h * to_next * D + 128 * i);
        else clear(raw[h][i]);
#pragma unroll
    for (int h = 0; h < HEADS; ++h)
#pragma unroll
      for (int i = 0; i < NI; ++i)
        if (h0 + h < a.kv_heads && 8 * (l + 16 * i) < D) *reinterpret_cast<decltype(raw8(src))*>(dst + h * hs + 128 * i) = raw[h][i];
    return;
  }
  const uint8_t* src = reinterpret_cast<const uint8_t*>(value ? a.v : a.k) + at * D + 8 * l;
  const float* scale = (value ? a.vs : a.ks) + at;
  uint2 w[HEADS][NI];
  float s[HEADS];
#pragma unroll
  for (int h = 0; h < HEADS; ++h) {
    const bool in = page >= 0 && h0 + h < a.kv_heads;
    s[h] = in ? scale[h * to_next] : 0.f;
#pragma unroll
    for (int i = 0; i < NI; ++i) w[h][i] = in && 8 * (l + 16 * i) < D ? *reinterpret_cast<const uint2*>(src + h * to_next * D + 128 * i) : make_uint2(0u, 0u);
  }
#pragma unroll
  for (int h = 0; h < HEADS; ++h)
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      if (h0 + h >= a.kv_heads || 8 * (l + 16 * i) >= D) continue;
      float x[8];
      values8<STORE>(w[h][i], s[h], x);
      store8(dst + h * hs + 128 * i, x);
    }
}

template <bool WRITE>
static int rows_call(const char* who, const void* k_new, long long ldk, long long hsk, const void* v_new, long long ldv, long long hsv, void* k, void* v, float* ks, float* vs,
                     const int* starts, const int* lengths, const int* table, int ldt, int width, int rows, int seqs, int pages, int page, int kv_heads, int K, int V, int store,
                     int act_dtype, b2l_stream_t stream) {
  B2L_CHECK_ARG(rows == 0 || (k_new && v_new), "%s: null pointer", who);
  if (int rc = check_pool(who, k, v, ks, vs, starts, lengths, table, ldt, width, rows, seqs, pages, page, kv_heads, K, V, store, act_dtype)) return rc;
  const int per = act_dtype == B2L_F32 ? 4 : 8;
  B2L_CHECK_ARG((((uintptr_t)k_new | (uintptr_t)v_new) & 15) == 0 && ldk % per == 0 && hsk % per == 0 && ldv % per == 0 && hsv % per == 0,
                "%s: rows must be 16-byte aligned", who);
  if (rows == 0 || seqs == 0) return 0;
  Rows a{step_of(starts, lengths, table, ldt, width, rows, seqs, pages, page), k_new, v_new, ldk, hsk, ldv, hsv, k, v, ks, vs, kv_heads, K, V};
  // Few rows: two heads to a warp and a warp to a block, so they spread over the SMs (96 tokens of 8 heads into e4m3: 3.2 us, 3.7 with four and eight).  Many:
  // more heads, as a warp's look for its place is a third of its work then: prompts of 32 heads into int8 58 us with eight, 60 with four; read 52 with four, 62 with eight
  constexpr int HEADS = WRITE ? 8 : 4;
  const bool many = (long long)rows * kv_heads >= 64 * 148;
  const int per_warp = many ? HEADS : 2, warps = many ? 8 : 1;
  const long long units = (long long)rows * ((kv_heads + per_warp - 1) / per_warp);
  const long long blocks = (units + warps - 1) / warps;
  B2L_CHECK_SUPPORTED(units < (1ll << 31), "%s: %d rows of %d heads", who, rows, kv_heads);
  const cudaStream_t st = (cudaStream_t)stream;
#define LAUNCH(T, ST, NI, H)                                                                       \
  (WRITE ? paged_write_kernel<T, ST, NI, H><<<(unsigned)blocks, 32 * warps, 0, st>>>(a)            \
         : paged_read_kernel<T, ST, NI, H><<<(unsigned)blocks, 32 * warps, 0, st>>>(a))
#define GO(T, ST) \
  (K <= 128 && V <= 128 ? (many ? LAUNCH(T, ST, 1, HEADS) : LAUNCH(T, ST, 1, 2)) : (many ? LAUNCH(T, ST, 2, HEADS) : LAUNCH(T, ST, 2, 2)))
  B2L_SEQ_DISPATCH(act_dtype, if (store == ACT) GO(act_t, ACT); else if (store == E4M3) GO(act_t, E4M3); else GO(act_t, INT8));
#undef GO
#undef LAUNCH
  B2L_LAUNCH_CHECK("paged rows");
  return 0;
}

}  // namespace paged
}  // namespace b2l

extern "C" int b2l_seq_paged_write(const void* k_new, long long ldk, long long hsk, const void* v_new, long long ldv, long long hsv, void* k, void* v, float* k_scale,
                                   float* v_scale, const int* starts, const int* lengths, const int* table, int ldt, int width, int rows, int seqs, int pages, int page,
                                   int kv_heads, int K, int V, int store, int act_dtype, b2l_stream_t stream) {
  return b2l::paged::rows_call<true>("b2l_seq_paged_write", k_new, ldk, hsk, v_new, ldv, hsv, k, v, k_scale, v_scale, starts, lengths, table, ldt, width, rows, seqs, pages, page,
                                     kv_heads, K, V, store, act_dtype, stream);
}

extern "C" int b2l_seq_paged_read(void* k_out, long long ldk, long long hsk, void* v_out, long long ldv, long long hsv, const void* k, const void* v, const float* k_scale,
                                  const float* v_scale, const int* starts, const int* lengths, const int* table, int ldt, int width, int rows, int seqs, int pages, int page,
                                  int kv_heads, int K, int V, int store, int act_dtype, b2l_stream_t stream) {
  return b2l::paged::rows_call<false>("b2l_seq_paged_read", k_out, ldk, hsk, v_out, ldv, hsv, const_cast<void*>(k), const_cast<void*>(v), const_cast<float*>(k_scale),
                                      const_cast<float*>(v_scale), starts, lengths, table, ldt, width, rows, seqs, pages, page, kv_heads, K, V, store, act_dtype, stream);
}
