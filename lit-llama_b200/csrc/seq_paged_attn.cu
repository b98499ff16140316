// Attention of new tokens over a paged pool, many sequences in one call (layout and step: seq_paged.cuh).
//
//   out[r, h] = sum_j w_j v_j / sum_j w_j,   w_j = 2^(c q . k_j - m),   c = scale log2(e),   j the keys that row r sees
//
// The query heads that read one key/value head are packed with the tokens: packed row i G + g is head g of the group at the sequence's new token i.
// paged_few_kernel takes 16 packed rows (one tile of mma.m16n8k16) against the keys of one head, 16 at a time.  A warp has every W-th such unit of its share
// all to itself: its own ring of copies (cp.async; a unit is 16 consecutive rows of one page), its own running maximum, sum and outputs in registers, no
// barrier in the loop.  The warps' results are joined at the end, and those of several CTAs that share a row's keys by paged_merge_kernel.
//
// Operands are fed to the tensor cores as bf16: an e4m3 or int8 code is one exactly, its scale goes into the score (keys) and the weight (values); a weight is
// two bf16 parts (at most 2^-15 of itself is left out); f32 queries, keys, values and weights are three parts each (f32's 24 bits), of whose nine products the six
// above 2^-24 are taken and added to f32 registers unit by unit, because the tensor core truncates where it adds to its accumulator.
// The order of a head's entries and of a unit's keys is free as long as both operands have the same: a lane reads four consecutive entries of a key and
// has them as its share of a k16 step; 8-bit values are transposed as pairs of neighbouring entries.
//
// What bounds it: one pass over the keys and values that the rows see, at HBM's rate, for the rows of a token; 16 rows of f32 are bound by their six products.
#include <algorithm>

#include "seq_paged_attn.cuh"

namespace b2l {
namespace paged {

// ------------------------------------------------------------------------------------------------ pieces
__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool in) {      // 16 bytes, or zeros
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(in ? 16 : 0) : "memory");
}
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ldsm_x4_t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ uint32_t lds32(uint32_t a) { uint32_t v; asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(a) : "memory"); return v; }
__device__ __forceinline__ uint2 lds64(uint32_t a) { uint2 v; asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a) : "memory"); return v; }
__device__ __forceinline__ uint4 lds128(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ uint32_t pack_hi(float x, float y) { return __byte_perm(__float_as_uint(x), __float_as_uint(y), 0x7632); }      // upper halves, x low
__device__ __forceinline__ float hi_of(float x) { return __uint_as_float(__float_as_uint(x) & 0xffff0000u); }
// Two f32 as PARTS pairs of bf16 that add up to them: truncated but for the last, which is rounded
template <int PARTS> __device__ __forceinline__ void parts2(float x, float y, uint32_t (&p)[PARTS]) {
#pragma unroll
  for (int i = 0; i < PARTS - 1; ++i) {
    p[i] = pack_hi(x, y);
    x -= hi_of(x);
    y -= hi_of(y);
  }
  const __nv_bfloat162 r = __floats2bfloat162_rn(x, y);
  p[PARTS - 1] = *reinterpret_cast<const uint32_t*>(&r);
}
// four e4m3 or int8 codes as bf16 pairs (0, 1) and (2, 3): exact, so the upper half of the f32
template <int STORE> __device__ __forceinline__ uint2 codes4(uint32_t w) {
  if (STORE == E4M3) {
    const float2 a = e4m3_pair(w), b = e4m3_pair(w >> 16);
    return make_uint2(pack_hi(a.x, a.y), pack_hi(b.x, b.y));
  }
  const uint32_t u = w ^ 0x80808080u;                        // 2^23 + 128 + x in the low byte of an f32's mantissa
  const float x0 = __uint_as_float(__byte_perm(u, 0x4b000000u, 0x7650)) - 8388736.f, x1 = __uint_as_float(__byte_perm(u, 0x4b000000u, 0x7651)) - 8388736.f;
  const float x2 = __uint_as_float(__byte_perm(u, 0x4b000000u, 0x7652)) - 8388736.f, x3 = __uint_as_float(__byte_perm(u, 0x4b000000u, 0x7653)) - 8388736.f;
  return make_uint2(pack_hi(x0, x1), pack_hi(x2, x3));
}
// of nine products of three parts (index 0 the largest) the six above 2^-24, the smallest first
__device__ constexpr int PART_A[6] = {2, 1, 0, 1, 0, 0}, PART_B[6] = {0, 1, 2, 0, 1, 0};

// c += sum of the products of a's and b's parts; FRESH: in an accumulator of its own, added to c as f32 additions are rounded
template <int AP, int BP, int N, bool FRESH>
__device__ __forceinline__ void product(float (&c)[4], const uint32_t (&a)[AP][4], const uint32_t* b0, const uint32_t* b1) {
  if (!FRESH) {
#pragma unroll
    for (int x = 0; x < N; ++x) mma16816(c, a[AP - 1 - x], b0[0], b1[0]);
    return;
  }
  float z[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int x = 0; x < N; ++x) mma16816(z, a[BP == 3 ? PART_A[x] : AP - 1 - x], b0[BP == 3 ? PART_B[x] : 0], b1[BP == 3 ? PART_B[x] : 0]);
#pragma unroll
  for (int e = 0; e < 4; ++e) c[e] += z[e];
}

// ------------------------------------------------------------------------------------------------ 16 rows
// One unit of keys (16) and values in a ring stage: rows padded so that the loads below meet no bank twice
template <typename act_t, int STORE> struct Unit {
  static constexpr int ES = STORE == ACT ? (int)sizeof(act_t) : 1;
  // words between rows: = 16 (mod 32) for f32, 8 (mod 16) for bf16, 4 (mod 8) for codes, where a lane reads four entries of one of eight keys
  __host__ __device__ static int k_row(int K) {
    const int w = K * ES / 4;
    return 4 * (ES == 4 ? (w % 32 ? w : w + 16) : ES == 2 ? (w % 16 ? w : w + 8) : (w % 8 ? w : w + 4));
  }
  // 4 (mod 8) for the transposing loads, and for f32 (4 mod 16), where a lane reads one entry of four keys
  __host__ __device__ static int v_row(int V) {
    const int w = V * ES / 4;
    return 4 * (w % 8 ? w : w + 4);
  }
  __host__ __device__ static int bytes(int K, int V) { return 16 * (k_row(K) + v_row(V)) + (STORE == ACT ? 0 : 128); }
};

template <typename act_t, int STORE, int NV>      // NV: the most 16-entry parts of a value
__global__ void __launch_bounds__(128) paged_few_kernel(const __grid_constant__ Attn a, int stages) {
  using U = Unit<act_t, STORE>;
  constexpr bool F32 = sizeof(act_t) == 4;
  constexpr int QP = F32 ? 3 : 1, KP = F32 && STORE == ACT ? 3 : 1, WP = F32 ? 3 : 2, PRODUCTS = KP == 3 ? 6 : QP, V_PRODUCTS = KP == 3 ? 6 : WP;
  extern __shared__ __align__(128) uint8_t smem[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, W = blockDim.x >> 5, g = lane >> 2, t = lane & 3;
  const int h = blockIdx.y, split = blockIdx.z, G = a.heads / a.kv_heads, steps = a.K / 16;
  Place pl;
  if (!a.place(blockIdx.x, 16, 0, a.few_max, lane, pl)) return;
  const Keys ks = a.keys(pl, 16);
  const int all = ks.units(4), per = (all + a.few.splits - 1) / a.few.splits;
  const int u_begin = min(split * per, all), u_end = min(u_begin + per, all);
  __shared__ uint32_t bad;                                   // rows whose result is not finite
  if (threadIdx.x == 0) bad = 0u;
  const uint32_t s0 = (uint32_t)__cvta_generic_to_shared(smem), sq = s0;
  const int kr = U::k_row(a.K), vr = U::v_row(a.V), unit_bytes = U::bytes(a.K, a.V);
  const uint32_t ring = s0 + (uint32_t)(QP * steps * 512) + (uint32_t)(warp * stages * unit_bytes);

  // the queries as the A operand's registers, part by part: entry 16 s + 4 t + e of rows g and g + 8
  for (int i = threadIdx.x; i < steps * 32; i += blockDim.x) {
    const int s = i >> 5, l = i & 31;
    float x[2][4];
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int r = pl.first + (l >> 2) + 8 * half;
      if (r < pl.n * G) {
        const float4 f = ld_act4(reinterpret_cast<const act_t*>(a.q) + (pl.start + r / G) * a.ldq + (h * G + r % G) * a.hsq + 16 * s + 4 * (l & 3));
        x[half][0] = f.x; x[half][1] = f.y; x[half][2] = f.z; x[half][3] = f.w;
      } else {
        x[half][0] = x[half][1] = x[half][2] = x[half][3] = 0.f;
      }
    }
    uint32_t p[4][QP];
    parts2<QP>(x[0][0], x[0][1], p[0]);
    parts2<QP>(x[1][0], x[1][1], p[1]);
    parts2<QP>(x[0][2], x[0][3], p[2]);
    parts2<QP>(x[1][2], x[1][3], p[3]);
#pragma unroll
    for (int q = 0; q < QP; ++q) *reinterpret_cast<uint4*>(smem + (q * steps + s) * 512 + l * 16) = make_uint4(p[0][q], p[1][q], p[2][q], p[3][q]);
  }
  __syncthreads();

  const int count = u_begin + warp < u_end ? (u_end - u_begin - warp + W - 1) / W : 0;      // this warp's units: u_begin + warp + W i
  // page of this warp's unit i: 32 at a time, one per lane
  int pages = -1, pages_at = -1;
  auto key0_of = [&](int i) { return ks.key0(u_begin + warp + W * i, 4); };
  auto page_at = [&](int i) {
    if (i / 32 != pages_at) {
      pages_at = i / 32;
      const int mine = pages_at * 32 + lane;
      pages = mine < count ? page_of(a.s, pl.b, key0_of(mine)) : -1;
    }
    return __shfl_sync(0xffffffffu, pages, i & 31);
  };
  uint32_t skipped = 0;                                      // ring stages whose page is not there
  auto load = [&](int i) {
    const int stage = i % stages;
    const uint32_t dst = ring + stage * unit_bytes;
    const int page = i < count ? page_at(i) : -1;
    if (page >= 0) {
      skipped &= ~(1u << stage);
      const int key0 = key0_of(i), valid = min(16, ks.end - key0);      // rows behind the last key that is seen come as zeros
      const size_t at = (((size_t)page * a.kv_heads + h) << a.s.shift) + (key0 & ((1 << a.s.shift) - 1));
#pragma unroll
      for (int kv = 0; kv < 2; ++kv) {
        const int D = kv ? a.V : a.K, row_chunks = D * U::ES / 16, chunks = 16 * row_chunks, row_bytes = kv ? vr : kr;
        const uint8_t* src = reinterpret_cast<const uint8_t*>(kv ? a.v : a.k) + at * D * U::ES;
        const uint32_t base = dst + (kv ? 16 * kr : 0);
        int r = lane / row_chunks, c = lane - r * row_chunks;
        const int dr = 32 / row_chunks, dc = 32 - dr * row_chunks;
        for (int x = lane; x < chunks; x += 32) {
          cp16(base + r * row_bytes + c * 16, src + (size_t)x * 16, r < valid);
          r += dr;
          c += dc;
          if (c >= row_chunks) { c -= row_chunks; ++r; }
        }
      }
      if (STORE != ACT && lane < 8) cp16(dst + 16 * (kr + vr) + lane * 16, (lane < 4 ? a.ks : a.vs) + at + 4 * (lane & 3), 4 * (lane & 3) < valid);
    } else {
      skipped |= 1u << stage;
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };

  float o[2 * NV][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
  for (int i = 0; i < 2 * NV; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) o[i][e] = 0.f;
  int pos[2];                                                // of rows g and g + 8
#pragma unroll
  for (int r = 0; r < 2; ++r) pos[r] = pl.first + g + 8 * r < pl.n * G ? pl.length - pl.n + (pl.first + g + 8 * r) / G : -1;

  for (int i = 0; i < stages - 1; ++i) load(i);
  for (int i = 0; i < count; ++i) {
    __syncwarp();                                            // every lane has done with the stage that is filled next
    load(i + stages - 1);
    if (stages == 2) asm volatile("cp.async.wait_group 1;" ::: "memory");
    else if (stages == 3) asm volatile("cp.async.wait_group 2;" ::: "memory");
    else if (stages == 4) asm volatile("cp.async.wait_group 3;" ::: "memory");
    else asm volatile("cp.async.wait_group 5;" ::: "memory");
    __syncwarp();
    if (skipped >> (i % stages) & 1u) continue;
    const uint32_t kb = ring + (i % stages) * unit_bytes, vb = kb + 16 * kr, sb = vb + 16 * vr;
    float s[2][4];
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) s[n][e] = 0.f;
#pragma unroll 2
    for (int k = 0; k < steps; ++k) {
      uint32_t q[QP][4];
#pragma unroll
      for (int p = 0; p < QP; ++p) {
        const uint4 u = lds128(sq + (p * steps + k) * 512 + lane * 16);
        q[p][0] = u.x; q[p][1] = u.y; q[p][2] = u.z; q[p][3] = u.w;
      }
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        const uint32_t at = kb + (8 * n + g) * kr + (16 * k + 4 * t) * U::ES;
        uint32_t b0[KP], b1[KP];
        if (STORE != ACT) {
          const uint2 c = codes4<STORE>(lds32(at));
          b0[0] = c.x;
          b1[0] = c.y;
        } else if (F32) {
          const uint4 u = lds128(at);
          parts2<KP>(__uint_as_float(u.x), __uint_as_float(u.y), b0);
          parts2<KP>(__uint_as_float(u.z), __uint_as_float(u.w), b1);
        } else {
          const uint2 u = lds64(at);
          b0[0] = u.x;
          b1[0] = u.y;
        }
#pragma unroll
        for (int x = 0; x < PRODUCTS; ++x) {
          const int qi = KP == 3 ? PART_A[x] : QP - 1 - x, ki = KP == 3 ? PART_B[x] : 0;
          mma16816(s[n], q[qi], b0[ki], b1[ki]);
        }
      }
    }
    // scores in powers of two; lane: keys 8 n + 2 t, + 1 of rows g (entries 0, 1) and g + 8 (2, 3)
    const int key0 = key0_of(i);
    float top[2] = {-INFINITY, -INFINITY}, vs[2][2] = {{1.f, 1.f}, {1.f, 1.f}};
    const bool whole = ks.whole(key0, 16);
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      float c[2] = {a.scale_log2, a.scale_log2};
      if (STORE != ACT) {
        const uint2 x = lds64(sb + (8 * n + 2 * t) * 4), y = lds64(sb + 64 + (8 * n + 2 * t) * 4);
        c[0] *= __uint_as_float(x.x);
        c[1] *= __uint_as_float(x.y);
        vs[n][0] = __uint_as_float(y.x);
        vs[n][1] = __uint_as_float(y.y);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s[n][e] *= c[e & 1];
        if (!whole && !a.sees(pos[e >> 1], key0 + 8 * n + 2 * t + (e & 1))) s[n][e] = -INFINITY;
        top[e >> 1] = fmaxf(top[e >> 1], s[n][e]);
      }
    }
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 1));
      top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 2));
    }
    if (__any_sync(0xffffffffu, top[0] > m[0] || top[1] > m[1])) {
      float f[2];
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const float now = fmaxf(m[r], top[r]);
        f[r] = m[r] == now ? 1.f : exp2_f(m[r] - now);
        m[r] = now;
        l[r] *= f[r];
      }
#pragma unroll
      for (int x = 0; x < 2 * NV; ++x) {
        o[x][0] *= f[0];
        o[x][1] *= f[0];
        o[x][2] *= f[1];
        o[x][3] *= f[1];
      }
    }
    uint32_t w[4][WP];                                       // the weights as the A operand of the second product
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        float x[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float z = s[n][2 * r + e];
          x[e] = z == -INFINITY ? 0.f : exp2_f(z - m[r]);
          l[r] += x[e];
          if (STORE != ACT) x[e] = z == -INFINITY ? 0.f : x[e] * vs[n][e];      // a scale that no row may see can be NaN
        }
        parts2<WP>(x[0], x[1], w[2 * n + r]);
      }
    uint32_t wa[WP][4];
#pragma unroll
    for (int p = 0; p < WP; ++p)
#pragma unroll
      for (int e = 0; e < 4; ++e) wa[p][e] = w[e][p];
    if (STORE != ACT) {
#pragma unroll
      for (int x = 0; x < (NV + 1) / 2; ++x) {
        if (32 * x >= a.V) break;
        const bool two = 32 * x + 16 < a.V;
        uint32_t r4[4];
        ldsm_x4_t(vb + (lane & 15) * vr + 32 * x + (two ? lane & 16 : 0), r4);
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          if (2 * x + y >= NV || (y && !two)) break;
          const uint2 lo = codes4<STORE>(__byte_perm(r4[2 * y], 0u, 0x3120)), hi = codes4<STORE>(__byte_perm(r4[2 * y + 1], 0u, 0x3120));      // (k0 d0, k1 d0, k0 d1, k1 d1)
          product<WP, 1, V_PRODUCTS, F32>(o[2 * (2 * x + y)], wa, &lo.x, &hi.x);
          product<WP, 1, V_PRODUCTS, F32>(o[2 * (2 * x + y) + 1], wa, &lo.y, &hi.y);
        }
      }
    } else if (!F32) {
#pragma unroll
      for (int x = 0; x < NV; ++x) {
        if (16 * x >= a.V) break;
        uint32_t r4[4];
        ldsm_x4_t(vb + (lane & 15) * vr + 32 * x + (lane & 16), r4);
        product<WP, 1, V_PRODUCTS, F32>(o[2 * x], wa, &r4[0], &r4[1]);
        product<WP, 1, V_PRODUCTS, F32>(o[2 * x + 1], wa, &r4[2], &r4[3]);
      }
    } else {
#pragma unroll
      for (int x = 0; x < 2 * NV; ++x) {
        if (8 * x >= a.V) break;
        const uint32_t at = vb + 2 * t * vr + (8 * x + g) * 4;
        uint32_t b0[KP], b1[KP];
        parts2<KP>(__uint_as_float(lds32(at)), __uint_as_float(lds32(at + vr)), b0);
        parts2<KP>(__uint_as_float(lds32(at + 8 * vr)), __uint_as_float(lds32(at + 9 * vr)), b1);
        product<WP, KP, V_PRODUCTS, F32>(o[x], wa, b0, b1);
      }
    }
  }

  // the warps' results: reference maximum, sum and outputs of 16 rows each
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
    l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
  __syncthreads();
  float* sm = reinterpret_cast<float*>(smem);                // [W][16] maxima, [W][16] sums, [W][16][ov] outputs
  const int ov = a.V + 4;
  float* so = sm + 32 * W;
  if (t == 0) {
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      sm[16 * warp + g + 8 * r] = m[r];
      sm[16 * W + 16 * warp + g + 8 * r] = l[r];
    }
  }
#pragma unroll
  for (int x = 0; x < 2 * NV; ++x) {
    if (16 * (x / 2) >= a.V) break;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int d = STORE != ACT ? 16 * (x / 2) + 4 * t + 2 * (e & 1) + (x & 1) : 8 * x + 2 * t + (e & 1);
      so[(16 * warp + g + 8 * (e >> 1)) * ov + d] = o[x][e];
    }
  }
  __syncthreads();
  const int quads = a.V / 4;
  for (int i = threadIdx.x; i < 16 * quads; i += blockDim.x) {
    const int r = i / quads, d = 4 * (i - r * quads), at = pl.first + r;
    if (at >= pl.n * G) break;
    float M = -INFINITY, L = 0.f, x[4] = {0.f, 0.f, 0.f, 0.f};
    for (int w = 0; w < W; ++w) M = fmaxf(M, sm[16 * w + r]);
    for (int w = 0; w < W; ++w) {
      const float mw = sm[16 * w + r];
      if (mw == -INFINITY && sm[16 * W + 16 * w + r] == 0.f) continue;
      const float f = mw == M ? 1.f : exp2_f(mw - M);
      L += f * sm[16 * W + 16 * w + r];
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = fmaf(f, so[(16 * w + r) * ov + d + e], x[e]);
    }
    const int row = pl.start + at / G, head = h * G + at % G;
    if (a.few.splits > 1) {
      const long long to = (long long)split * a.few.count + (a.compact ? (long long)(pl.b * a.kv_heads + h) * 16 + at : (long long)row * a.heads + head);
      if (d == 0) *reinterpret_cast<float2*>(a.few.ml + 2 * to) = make_float2(M, L);
      *reinterpret_cast<float4*>(a.few.o + to * a.V + d) = make_float4(x[0], x[1], x[2], x[3]);
    } else {
      const float inv = L == 0.f ? 0.f : 1.f / L;
      a.store(((size_t)row * a.heads + head) * a.V + d, x, inv);
      if (!finite4(x, inv)) atomicOr(&bad, 1u << r);
    }
  }
  if (a.few.splits == 1) {
    __syncthreads();
    for (uint32_t left = bad; left; left &= left - 1) {
      const int r = __ffs(left) - 1, at = pl.first + r;
      if (r % W == warp) mend_row(a, pl.b, pl.length - pl.n + at / G, pl.start + at / G, h * G + at % G, lane);
    }
  }
}

// ------------------------------------------------------------------------------------------------ joining parts
// A warp per row and head; rows of sequences whose parts were not split are in place already.
__global__ void __launch_bounds__(256) paged_merge_kernel(const __grid_constant__ Attn a) {
  const int lane = threadIdx.x & 31, G = a.heads / a.kv_heads;
  const long long unit = (long long)blockIdx.x * (blockDim.x / 32) + threadIdx.x / 32;
  const int row = (int)(unit / a.heads), head = (int)(unit % a.heads);
  if (row >= a.s.rows) return;
  const int b = sequence_of(a.s, row, lane);
  if (b < 0) return;
  int start, n, length;
  sequence(a.s, b, start, n, length);
  const bool few = (long long)n * G <= a.few_max;
  const Parts& p = few ? a.few : a.many;
  if (p.splits <= 1) return;
  const int h = head / G;
  const long long at = few && a.compact ? (long long)(b * a.kv_heads + h) * 16 + (row - start) * G + head % G : (long long)row * a.heads + head;
  float M = -INFINITY, L = 0.f;
  for (int i = lane; i < p.splits; i += 32) M = fmaxf(M, p.ml[2 * (i * p.count + at)]);
  M = warp_max(M);
  float x[2][4] = {};
  for (int i = 0; i < p.splits; ++i) {
    const float2 ml = *reinterpret_cast<const float2*>(p.ml + 2 * (i * p.count + at));
    if (ml.x == -INFINITY && ml.y == 0.f) continue;          // saw nothing
    const float f = ml.x == M ? 1.f : exp2_f(ml.x - M);
    L += f * ml.y;
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int d = 4 * (lane + 32 * c);
      if (d >= a.V) break;
      const float4 y = *reinterpret_cast<const float4*>(p.o + (i * p.count + at) * a.V + d);
      x[c][0] = fmaf(f, y.x, x[c][0]);
      x[c][1] = fmaf(f, y.y, x[c][1]);
      x[c][2] = fmaf(f, y.z, x[c][2]);
      x[c][3] = fmaf(f, y.w, x[c][3]);
    }
  }
  const float inv = L == 0.f ? 0.f : 1.f / L;
  bool fine = true;
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    const int d = 4 * (lane + 32 * c);
    if (d >= a.V) break;
    a.store(((size_t)row * a.heads + head) * a.V + d, x[c], inv);
    fine = fine && finite4(x[c], inv);
  }
  if (!__all_sync(0xffffffffu, fine)) {
    __syncwarp();
    mend_row(a, b, length - n + row - start, row, head, lane);
  }
}

// ------------------------------------------------------------------------------------------------ host
struct Plan {
  bool few, many;
  int few_max, few_tiles, many_tiles, few_splits, many_splits, compact;
  long long few_count, many_count, floats;
};
constexpr long long MOST_WORK = 1ll << 27;                   // floats of partial results

static Plan plan_of(int rows, int seqs, int width, int page, int heads, int kv_heads, int K, int V, int window, int first, int max_new, int min_new, int max_length, int store,
                    int act_dtype) {
  Plan p{};
  const int G = heads / kv_heads, sms = sm_count();
  const bool tensor = act_dtype == B2L_BF16 && many_takes(K, V, store);
  const long long packed = (long long)rows * G;
  p.few = !tensor || !(min_new > 0 && (long long)min_new * G > 16);
  p.many = tensor && !(max_new > 0 && (long long)max_new * G <= 16);
  p.few_max = !p.many ? INT32_MAX : p.few ? 16 : 0;
  p.compact = p.few && p.many;
  const int most = std::min(seqs, rows);
  p.few_tiles = p.compact ? most : (int)std::min<long long>(packed / 16 + most, INT32_MAX);
  p.many_tiles = (int)std::min<long long>(packed / 128 + most, INT32_MAX);
  long long keys = (long long)width * page;                  // the most keys that a row sees
  if (max_length > 0) keys = std::min<long long>(keys, max_length);
  if (window > 0) keys = std::min<long long>(keys, (long long)window + first + 16);
  p.few_splits = p.many_splits = 1;
  p.few_count = p.compact ? (long long)seqs * kv_heads * 16 : (long long)rows * heads;
  p.many_count = (long long)rows * heads;
  if (p.few) {
    const long long ctas = (long long)kv_heads * std::max(1, p.few_tiles), want = (4ll * sms + ctas - 1) / ctas;
    p.few_splits = (int)std::max<long long>(1, std::min({want, keys / 256, 128ll, MOST_WORK / (p.few_count * (V + 2) + 1)}));
  }
  auto floats = [&](int splits, long long count) { return splits > 1 ? (2 * splits * count + 3) / 4 * 4 + splits * count * V : 0; };
  p.floats = (p.few ? floats(p.few_splits, p.few_count) : 0) + (p.many ? floats(p.many_splits, p.many_count) : 0);
  return p;
}

template <typename act_t, int STORE, int NV> static int few_launch(const Attn& a, int tiles, cudaStream_t stream) {
  using U = Unit<act_t, STORE>;
  const size_t queries = (size_t)(sizeof(act_t) == 4 ? 3 : 1) * (a.K / 16) * 512, unit = U::bytes(a.K, a.V);
  int W = 4, stages = 0;
  for (size_t room : {(size_t)112 * 1024, (size_t)226 * 1024}) {      // two CTAs per SM, or one
    for (W = 4; W >= 1 && stages == 0; W /= 2) {
      if (room > 112 * 1024 || W == 4) {
        const size_t n = room > queries ? (room - queries) / (W * unit) : 0;
        stages = n >= 6 ? 6 : n >= 4 ? 4 : n >= 2 ? (int)n : 0;
        if (stages) break;
      }
    }
    if (stages) break;
  }
  B2L_CHECK_SUPPORTED(stages > 0, "b2l_seq_paged_attention: heads of %d and %d entries do not fit", a.K, a.V);
  const size_t smem = std::max(queries + W * stages * unit, (size_t)W * (32 + 16 * (a.V + 4)) * 4);
  static DynSmemCache cache;
  auto kernel = paged_few_kernel<act_t, STORE, NV>;
  if (int rc = ensure_dyn_smem(kernel, smem, cache)) return rc;
  kernel<<<dim3((unsigned)tiles, (unsigned)a.kv_heads, (unsigned)a.few.splits), 32 * W, smem, stream>>>(a, stages);
  B2L_LAUNCH_CHECK("paged_few_kernel");
  return 0;
}

}  // namespace paged
}  // namespace b2l

using namespace b2l;

extern "C" long long b2l_seq_paged_attention_work(int rows, int seqs, int width, int page, int heads, int kv_heads, int K, int V, int window, int first, int max_new, int min_new,
                                                  int max_length, int store, int act_dtype) {
  if (rows <= 0 || seqs <= 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads != 0) return 0;
  return paged::plan_of(rows, seqs, width, page, heads, kv_heads, K, V, window, first, max_new, min_new, max_length, store, act_dtype).floats;
}

extern "C" int b2l_seq_paged_attention(const void* q, long long ldq, long long hsq, const void* k, const void* v, const float* k_scale, const float* v_scale, const int* starts,
                                       const int* lengths, const int* table, int ldt, int width, void* out, float* work, long long work_floats, int rows, int seqs, int pages,
                                       int page, int heads, int kv_heads, int K, int V, int window, int first, float scale, int max_new, int min_new, int max_length, int store,
                                       int act_dtype, b2l_stream_t stream) {
  using namespace paged;
  const char* who = "b2l_seq_paged_attention";
  B2L_CHECK_ARG(q && out, "%s: null pointer", who);
  if (int rc = check_pool(who, k, v, k_scale, v_scale, starts, lengths, table, ldt, width, rows, seqs, pages, page, kv_heads, K, V, store, act_dtype)) return rc;
  B2L_CHECK_ARG(heads > 0 && heads % kv_heads == 0, "%s: %d heads over %d key/value heads", who, heads, kv_heads);
  B2L_CHECK_ARG(window >= 0 && first >= 0, "%s: a negative window or number of first tokens", who);
  B2L_CHECK_ARG(scale > 0.f && scale < INFINITY, "%s: the scale must be positive and finite", who);
  const int per = act_dtype == B2L_F32 ? 4 : 8;
  B2L_CHECK_ARG((((uintptr_t)q | (uintptr_t)out | (uintptr_t)work) & 15) == 0 && ldq % per == 0 && hsq % per == 0, "%s: rows must be 16-byte aligned", who);
  B2L_CHECK_SUPPORTED((long long)width * page < (1ll << 30) && kv_heads < 65536 && (long long)rows * heads < (1ll << 31), "%s: sizes beyond the grid's", who);
  if (rows == 0 || seqs == 0) return 0;
  const Plan p = plan_of(rows, seqs, width, page, heads, kv_heads, K, V, window, first, max_new, min_new, max_length, store, act_dtype);
  B2L_CHECK_ARG(p.floats == 0 || (work && work_floats >= p.floats), "%s: a work space of %lld floats is needed", who, p.floats);
  Attn a{};
  a.s = step_of(starts, lengths, table, ldt, width, rows, seqs, pages, page);
  a.q = q; a.k = k; a.v = v; a.ks = k_scale; a.vs = v_scale; a.out = out;
  a.ldq = ldq; a.hsq = hsq;
  a.heads = heads; a.kv_heads = kv_heads; a.K = K; a.V = V;
  a.window = window; a.first = window ? first : 0;
  a.few_max = p.few_max;
  a.scale_log2 = scale * 1.44269502162933349609375f;         // log2(e)
  a.f32 = act_dtype == B2L_F32; a.store_kind = store; a.compact = p.compact;
  auto take = [&](Parts& x, int splits, long long count) {
    x.splits = splits;
    x.count = count;
    if (splits <= 1) return;
    x.ml = work;
    x.o = work + (2 * splits * count + 3) / 4 * 4;
    work = x.o + splits * count * V;
  };
  take(a.few, p.few ? p.few_splits : 1, p.few_count);
  take(a.many, p.many ? p.many_splits : 1, p.many_count);
  const cudaStream_t st = (cudaStream_t)stream;
  if (p.few) {
    int rc = 0;
#define GO(ST) (V <= 128 ? few_launch<act_t, ST, 8>(a, p.few_tiles, st) : few_launch<act_t, ST, 16>(a, p.few_tiles, st))
    B2L_SEQ_DISPATCH(act_dtype, rc = store == ACT ? GO(ACT) : store == E4M3 ? GO(E4M3) : GO(INT8));
#undef GO
    if (rc) return rc;
  }
  if (p.many)
    if (int rc = many_launch(a, p.many_tiles, st)) return rc;
  if (a.few.splits > 1 || a.many.splits > 1) {
    const long long units = (long long)rows * heads;
    const int warps = units >= 8 * 148 ? 8 : 1;
    paged_merge_kernel<<<(unsigned)((units + warps - 1) / warps), 32 * warps, 0, st>>>(a);
    B2L_LAUNCH_CHECK("paged_merge_kernel");
  }
  return 0;
}
