// Attention of new tokens over a paged pool, many sequences in one call (layout and step: seq_paged.cuh).
//
//   out[r, h] = sum_j w_j v_j / sum_j w_j,   w_j = 2^(c q . k_j - m),   c = scale log2(e),   j the keys that row r sees
//
// The query heads that read one key/value head are packed with the tokens: packed row i G + g is head g of the group at the sequence's new token i.
// paged_few_kernel takes 8 or 16 packed rows against the keys of one head, 16 (8-bit: 32) at a time, as mma.m16n8k16 with the keys (and then the entries of a value) for
// its 16 rows and the queries for its 8 columns: a token of a group of up to 8 heads fills the product that it needs, where queries as rows left three
// quarters of the scores and their softmax unused (537 instructions for 16 keys of 128 8-bit entries, now 440 with all beside).  A warp has every W-th such unit of its share
// all to itself: its own ring of tiled copies (16 rows of one page by 128 bytes, swizzled), its own running maximum, sum and outputs in registers, no
// barrier in the loop.  The warps' results are joined at the end, and those of several CTAs that share a row's keys by paged_merge_kernel.
//
// Operands of the tensor cores, all products exact and added in f32:
//   bf16 pool       as it lies; a weight is two bf16 parts (at most 2^-15 of itself is left out)
//   8-bit pool      a code is an f16 exactly (two codes an instruction; bf16 took four times as many), and so the queries: a row of them times the power of
//                   two that brings its largest entry to 2^14 (an entry below 2^-28 of that keeps fewer than 8 bits, off by 2^-39 of it).  The scale of a
//                   key goes into its score, the scale of a value into the exponent of its weight, w s = 2^(t + log2 s - m), m the largest t + log2 s so
//                   far (scales between 2^-60 and 2^40; a row that sees others is computed again): in f16 with a factor of 2^14, off by 2^-11 of itself at most (2^-39 of the largest where it is small), and sum_j w_j adds w s / s
//   f32             three parts each (f32's 24 bits); of the nine products of two f32 operands the six above 2^-24.  They are added to f32 registers unit by
//                   unit, because the tensor core truncates where it adds to its accumulator
// With 8-bit codes a lane has four consecutive entries of a key as its share of a k16 step (queries laid out alike), and values are transposed as pairs
// of neighbouring entries, so 16-byte rows of ldmatrix do for both.  Weights turn from keys by rows into the second product's operand by movmatrix.
//
// What bounds it: one pass over the keys and values that the rows see.  One token over 131072 keys of 4 heads of 128, bf16: 55.5 us, 4.8 TB/s.  Tokens of 48
// sequences over up to 8192 keys of 8 heads, e4m3: 123 us, 4.3 TB/s, where the issue of instructions is busy for half of the cycles and their latency is the
// other half (12 warps on an SM, as many as the copies in flight leave room for).  One token over 1031 keys: 12 us, two launches of a chain of loads each.
// 16 rows of f32 are bound by their six products: 461 tokens over a window of 512, 8 / 2 heads of 128, 73 us.
#include <algorithm>
#include <cmath>

#include "seq_paged_attn.cuh"
#include "tc_common.cuh"

namespace b2l {
namespace paged {

// ------------------------------------------------------------------------------------------------ pieces
__device__ __forceinline__ void bulk64(uint32_t dst, const void* src, uint32_t bar) {      // 64 bytes, 16-byte aligned
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], 64, [%2];" ::"r"(dst), "l"(src), "r"(bar) : "memory");
}
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma16816h(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ldsm_x4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm_x4_t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ uint32_t transposed(uint32_t x) {      // of an 8 x 8 matrix of 16-bit entries, two per lane
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
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
// the same in f16, each part rounded
template <int PARTS> __device__ __forceinline__ void halves2(float x, float y, uint32_t (&p)[PARTS]) {
#pragma unroll
  for (int i = 0; i < PARTS; ++i) {
    const __half2 h = __floats2half2_rn(x, y);
    p[i] = *reinterpret_cast<const uint32_t*>(&h);
    if (i + 1 < PARTS) {
      const float2 f = __half22float2(h);
      x -= f.x;
      y -= f.y;
    }
  }
}
template <bool HALF, int PARTS> __device__ __forceinline__ void operand2(float x, float y, uint32_t (&p)[PARTS]) {
  if constexpr (HALF) halves2<PARTS>(x, y, p);
  else parts2<PARTS>(x, y, p);
}
// of nine products of three parts (index 0 the largest) the six above 2^-24, the smallest first
__device__ constexpr int PART_A[6] = {2, 1, 0, 1, 0, 0}, PART_B[6] = {0, 1, 2, 0, 1, 0};

// c += sum of the products of a's and b's parts (one of a, or three of each); FRESH: in an accumulator of its own, added to c as f32 additions are rounded
template <bool HALF, int AP, int BP, int N, bool FRESH>
__device__ __forceinline__ void product(float (&c)[4], const uint32_t (&a)[AP][4], const uint32_t (&b)[BP][2]) {
  float z[4] = {0.f, 0.f, 0.f, 0.f};
  float (&to)[4] = FRESH ? z : c;
#pragma unroll
  for (int x = 0; x < N; ++x) {
    const int i = AP == 3 ? PART_A[x] : 0, j = AP == 3 ? PART_B[x] : BP - 1 - x;
    if constexpr (HALF) mma16816h(to, a[i], b[j][0], b[j][1]);
    else mma16816(to, a[i], b[j][0], b[j][1]);
  }
  if (FRESH)
#pragma unroll
    for (int e = 0; e < 4; ++e) c[e] += z[e];
}

// ------------------------------------------------------------------------------------------------ 16 rows
constexpr int ATOM = 2048;           // 16 rows of 128 bytes, as a swizzled tiled copy leaves them: 16-byte piece c of row r at piece c ^ (r & 7); the next 16 follow

__host__ __device__ constexpr int most_stages(int store) { return store == ACT ? 8 : 4; }

struct FewMaps { CUtensorMap k, v; };

// NV: the most 16-entry parts of a value (and, up to 8, of a key); NR: columns of 8 rows
template <typename act_t, int STORE, int NV, int NR>
__global__ void __launch_bounds__(128, NV <= 8 ? (NR == 1 && STORE != ACT ? 4 : 3) : 2) paged_few_kernel(const __grid_constant__ Attn a, const __grid_constant__ FewMaps maps, int stages) {
  constexpr bool F32 = sizeof(act_t) == 4, HALF = STORE != ACT;
  constexpr int ES = STORE == ACT ? (int)sizeof(act_t) : 1, R = 8 * NR;
  constexpr int QP = F32 ? 3 : 1, KP = F32 && !HALF ? 3 : 1, WP = F32 ? 3 : HALF ? 1 : 2, PRODUCTS = KP == 3 ? 6 : QP, V_PRODUCTS = KP == 3 ? 6 : WP;
  constexpr int PER = ES == 4 ? 1 : ES == 2 ? 1 : 2;         // k16 steps in the two 16-byte pieces that one ldmatrix takes
  constexpr bool HELD = !F32 && NV <= 8;                     // queries in registers
  constexpr int STAGES = most_stages(STORE);
  constexpr int NK = HALF ? 2 : 1, SHIFT = HALF ? 5 : 4;     // 16-key parts of a unit: half as many copies, waits and maxima for codes' half as many bytes
  constexpr float LIFT = HALF ? 14.f : 0.f;                  // weights up to 2^14 in f16
  extern __shared__ __align__(1024) uint8_t smem[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, W = blockDim.x >> 5, g = lane >> 2, t = lane & 3;
  const int h = blockIdx.y, split = blockIdx.z, G = a.heads / a.kv_heads, steps = (a.K / 16 + PER - 1) / PER * PER;
  // The first tile of every sequence, found without looking through the others, and then the rest of those that have more
  Place pl;
  if ((int)blockIdx.x < a.s.seqs) {
    pl.b = blockIdx.x;
    sequence(a.s, pl.b, pl.start, pl.n, pl.length);
    pl.first = 0;
    if (a.zeros && split == 0) {                             // sequences' rows follow one another: the rest lies before the first and behind the last
      if (pl.b == 0 && pl.start > 0) clear_rows(a, 0, pl.start, h * G, G, threadIdx.x, blockDim.x);
      if (pl.b == a.s.seqs - 1 && pl.start + pl.n < a.s.rows) clear_rows(a, pl.start + pl.n, a.s.rows, h * G, G, threadIdx.x, blockDim.x);
    }
    if (pl.n == 0 || (long long)pl.n * G > a.few_max) return;
  } else if (!a.place(blockIdx.x - a.s.seqs, R, lane, pl)) {
    return;
  }
  __shared__ uint32_t bad;                                   // rows whose result is not finite
  __shared__ uint32_t largest[16];                           // entry of a row of queries, as bits
  __shared__ __align__(8) uint64_t bars[4 * STAGES];
  __shared__ __align__(16) float scales[HALF ? 4 * STAGES * 64 : 4];
  const int ka = atoms_of(a.K, ES), va = atoms_of(a.V, ES), unit_bytes = NK * (ka + va) * ATOM;
  const uint32_t s0 = tc::smem_u32(smem);
  const uint32_t ring = s0 + (uint32_t)(warp * stages * unit_bytes), sq = s0 + (uint32_t)(W * stages * unit_bytes);
  const uint32_t bar0 = tc::smem_u32(bars) + warp * STAGES * 8, sc0 = tc::smem_u32(scales) + warp * STAGES * 256;
  uint8_t* queries = smem + W * stages * unit_bytes;
  if (lane == 0) {
    for (int i = 0; i < stages; ++i) tc::mbar_init(bar0 + 8 * i, 1);
    tc::mbar_init_fence();
  }
  __syncwarp();
  uint32_t dead = (s0 & 1023u) ? 1u : 0u, phase = 0;         // swizzled atoms need 1024-byte alignment
  int fill = 0, stage = 0;                                   // stage that is filled next, and read next
  const Keys ks = a.keys(pl, R);
  const int all = ks.units(SHIFT), per = (all + a.few.splits - 1) / a.few.splits;
  const int u_begin = min(split * per, all), u_end = min(u_begin + per, all);
  // Queries on their way while the first pages are looked up: entries d0, + 1 and d1, + 1 of a row, as the B operand has them: row g of a column by entries 2 t, + 1 and
  // 8 + 2 t, + 1 of a k16 step, or (codes) 4 t .. 4 t + 3
  auto place_of = [&](int i, int& k, int& r, int& l) {
    const int x = threadIdx.x + i * blockDim.x;
    k = x / (32 * NR);
    l = x & 31;
    r = 8 * ((x >> 5) % NR) + (l >> 2);
    return k < steps;
  };
  auto query = [&](int k, int r, int l, float (&x)[4]) {
    const int at = pl.first + r, d0 = HALF ? 4 * (l & 3) : 2 * (l & 3), d1 = HALF ? d0 + 2 : d0 + 8;
    x[0] = x[1] = x[2] = x[3] = 0.f;
    if (at < pl.n * G && 16 * k < a.K) {
      const act_t* src = reinterpret_cast<const act_t*>(a.q) + (pl.start + at / G) * a.ldq + (h * G + at % G) * a.hsq + 16 * k;
      x[0] = ld_act(src, d0);
      x[1] = ld_act(src, d0 + 1);
      x[2] = ld_act(src, d1);
      x[3] = ld_act(src, d1 + 1);
    }
  };
  constexpr int AHEAD = 4;                                   // places of a thread that are loaded ahead: all of them for up to 128 entries and 16 rows
  float early[AHEAD][4];
#pragma unroll
  for (int i = 0; i < AHEAD; ++i) {
    int k, r, l;
    if (place_of(i, k, r, l)) query(k, r, l, early[i]);
  }
  if (threadIdx.x == 0) bad = 0u;
  if (threadIdx.x < 16) largest[threadIdx.x] = 0u;

  const int count = u_begin + warp < u_end ? (u_end - u_begin - warp + W - 1) / W : 0;      // this warp's units: u_begin + warp + W i
  auto key0_of = [&](int i) { return ks.key0(u_begin + warp + W * i, SHIFT); };
  // where 16-key parts of this warp's units begin in the pool: 32 at a time, one per lane; of a page that is not there a row beyond the pool, which reads as
  // zeros
  const int beyond = (a.s.pages * a.kv_heads) << a.s.shift;
  const bool wide = NK == 2 && a.s.shift >= 5;               // a unit is in one page: one copy
  const int copies = ka + va;                                // of a page: up to 16, and 8-bit 4
  int row_of = beyond;
  uint32_t gone = 0;                                         // 16-key parts of the ring's stages whose page is not there
  int next = 0;                                              // unit that is loaded next
  auto load = [&]() {
    if (next >= count) return;
    if ((next & (32 / NK - 1)) == 0) {
      const int mine = next + lane / NK, key0 = key0_of(mine) + 16 * (lane % NK);
      const int page = mine < count && key0 < ks.end ? page_of(a.s, pl.b, key0) : -1;
      row_of = page >= 0 ? ((page * a.kv_heads + h) << a.s.shift) + (key0 & ((1 << a.s.shift) - 1)) : beyond;
    }
    const int at = NK * (next & (32 / NK - 1)), r0 = __shfl_sync(0xffffffffu, row_of, at), r1 = NK == 2 ? __shfl_sync(0xffffffffu, row_of, at + 1) : beyond;
    ++next;
    gone = (gone & ~(3u << 2 * fill)) | ((r0 == beyond ? 1u : 0u) | (r1 == beyond ? 2u : 0u)) << 2 * fill;
    if (r0 != beyond || r1 != beyond) {
      const uint32_t dst = ring + fill * unit_bytes, bar = bar0 + 8 * fill;
      if (lane == 0) tc::mbar_expect_tx(bar, unit_bytes + (HALF ? 256 : 0));
      __syncwarp();                                          // the bytes are expected before they come
      // a lane per copy: one lane after the other took some 100 ns for each
      const int half = lane >= copies ? 1 : 0, x = lane - half * copies;
      const int from = wide ? r0 & ~31 : half ? r1 : r0;     // (a unit's second half may lie behind the last key: its page is not looked for)
      if (lane < (NK == 2 && !wide ? 2 : 1) * copies) {
        if (x < ka) tc::tma_load_2d(dst + x * NK * ATOM + half * ATOM, &maps.k, x * (128 / ES), from, bar);
        else tc::tma_load_2d(dst + x * NK * ATOM + half * ATOM, &maps.v, (x - ka) * (128 / ES), from, bar);
      }
      if (HALF && lane >= 28) {                              // the scales; of a page that is not there any
        const int second = lane & 1, at = wide ? from + 16 * second : second ? r1 : r0;
        bulk64(sc0 + 256 * fill + 64 * (lane - 28), (lane & 2 ? a.vs : a.ks) + (at == beyond ? 0 : at), bar);
      }
      __syncwarp();
    }
    if (++fill == stages) fill = 0;
  };
  for (int i = 0; i < stages - 1; ++i) load();

  __syncthreads();
  auto each_place = [&](auto&& take) {                       // take(place, step, row, lane, entries)
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      int k, r, l;
      if (place_of(i, k, r, l)) take(i, k, r, l, early[i]);
    }
    int k, r, l;
    for (int i = AHEAD; place_of(i, k, r, l); ++i) {
      float x[4];
      query(k, r, l, x);
      take(i, k, r, l, x);
    }
  };
  if (HALF) {                                                // the largest entry of every row
    each_place([&](int, int, int r, int l, const float (&x)[4]) {
      float top = fmaxf(fmaxf(fabsf(x[0]), fabsf(x[1])), fmaxf(fabsf(x[2]), fabsf(x[3])));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      if ((l & 3) == 0) atomicMax(&largest[r], __float_as_uint(top));
    });
    __syncthreads();
  }
  each_place([&](int i, int, int r, int, const float (&x)[4]) {
    float up = 1.f, down;
    if (HALF) lift_of(__uint_as_float(largest[r]), a.scale_log2, up, down);
    uint32_t p[2][QP];
    operand2<HALF, QP>(x[0] * up, x[1] * up, p[0]);
    operand2<HALF, QP>(x[2] * up, x[3] * up, p[1]);
#pragma unroll
    for (int q = 0; q < QP; ++q) *reinterpret_cast<uint2*>(queries + q * steps * NR * 256 + (threadIdx.x + i * blockDim.x) * 8) = make_uint2(p[0][q], p[1][q]);
  });
  __syncthreads();
  uint32_t held[HELD ? NV : 1][NR][1][2];
  if (HELD)
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
      for (int r = 0; r < NR; ++r) {
        const uint2 u = k < steps ? lds64(sq + (k * NR + r) * 256 + lane * 8) : make_uint2(0u, 0u);
        held[k][r][0][0] = u.x;
        held[k][r][0][1] = u.y;
      }

  float o[NR][NV][4], m[NR][2], l[NR][2], cr[NR][2];         // rows 8 r + 2 t, + 1; outputs: entries by rows
  int pos[NR][2];
#pragma unroll
  for (int r = 0; r < NR; ++r) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int at = 8 * r + 2 * t + e;
      m[r][e] = -INFINITY;
      l[r][e] = 0.f;
      cr[r][e] = a.scale_log2;
      if (HALF) {
        float up;
        lift_of(__uint_as_float(largest[at]), a.scale_log2, up, cr[r][e]);
      }
      pos[r][e] = pl.first + at < pl.n * G ? pl.length - pl.n + (pl.first + at) / G : -1;
    }
#pragma unroll
    for (int x = 0; x < NV; ++x)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[r][x][e] = 0.f;
  }
  // where this lane's row of an ldmatrix lies: row lane & 15, piece lane / 16 of two; or (bf16 values) row (lane & 7) + 8 (lane / 16), piece lane / 8 % 2
  const uint32_t at_16 = (lane & 15) * 128 + (((lane >> 4) ^ (lane & 7)) << 4), at_8 = ((lane & 7) + (lane >> 4) * 8) * 128 + (((lane >> 3 & 1) ^ (lane & 7)) << 4);

  for (int i = 0; i < count; ++i) {
    __syncwarp();                                            // every lane has done with the stage that is filled next
    load();
    const int st = stage;
    if (++stage == stages) stage = 0;
    const uint32_t lost = gone >> 2 * st & 3u;
    if (lost == 3u) continue;
    tc::mbar_wait_warp(bar0 + 8 * st, phase >> st & 1u, dead);
    phase ^= 1u << st;
    if (dead) break;
    const uint32_t kb = ring + st * unit_bytes, vb = kb + NK * ka * ATOM, sb = sc0 + 256 * st;
    const int key0 = key0_of(i), valid = ks.end - key0;
    if (valid < 16 * NK) {                                   // the last unit: what lies behind the last key that is seen may be anything
      for (int x = lane; x < (16 * NK - valid) * 8 * va; x += 32) {
        const int r = valid + x / (8 * va), c = x % (8 * va);
        asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(vb + (c >> 3) * NK * ATOM + r * 128 + (c & 7) * 16), "r"(0u) : "memory");
      }
      __syncwarp();
    }
    float s[NK][NR][4];
#pragma unroll
    for (int n = 0; n < NK; ++n)
#pragma unroll
      for (int r = 0; r < NR; ++r)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[n][r][e] = 0.f;
    auto score = [&](int n, int k, const uint32_t (&key)[KP][4]) {
#pragma unroll
      for (int r = 0; r < NR; ++r) {
        if constexpr (HELD) {
          product<HALF, KP, QP, PRODUCTS, false>(s[n][r], key, held[k][r]);
        } else {
          uint32_t q[QP][2];
#pragma unroll
          for (int p = 0; p < QP; ++p) {
            const uint2 u = lds64(sq + ((p * steps + k) * NR + r) * 256 + lane * 8);
            q[p][0] = u.x;
            q[p][1] = u.y;
          }
          product<HALF, KP, QP, PRODUCTS, false>(s[n][r], key, q);
        }
      }
    };
    auto key_pieces = [&](int j) {                           // pieces 2 j, 2 j + 1 of the keys: PER steps
#pragma unroll
      for (int n = 0; n < NK; ++n) {
        uint32_t r4[4];
        ldsm_x4(kb + ((j >> 2) * NK + n) * ATOM + (at_16 ^ ((j & 3) << 5)), r4);
#pragma unroll
        for (int x = 0; x < PER; ++x) {
          uint32_t key[KP][4];
          if constexpr (HALF) {
            const uint2 u = codes4<STORE, 0, 1, 2, 3>(r4[2 * x]), v = codes4<STORE, 0, 1, 2, 3>(r4[2 * x + 1]);
            key[0][0] = u.x; key[0][1] = v.x; key[0][2] = u.y; key[0][3] = v.y;
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) key[0][e] = r4[e];
          }
          score(n, PER * j + x, key);
        }
      }
    };
    if constexpr (F32 && !HALF) {
#pragma unroll 2
      for (int k = 0; k < steps; ++k) {
        uint32_t key[KP][4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {                        // rows g, g + 8 by entries 2 t and 8 + 2 t
          const uint32_t c = 4 * (k & 1) + (t >> 1) + (e & 2);
          const uint2 u = lds64(kb + (k >> 1) * ATOM + (g + 8 * (e & 1)) * 128 + ((c ^ g) << 4) + 8 * (t & 1));
          uint32_t p[KP];
          parts2<KP>(__uint_as_float(u.x), __uint_as_float(u.y), p);
#pragma unroll
          for (int x = 0; x < KP; ++x) key[x][e] = p[x];
        }
        score(0, k, key);
      }
    } else if constexpr (HELD) {
#pragma unroll
      for (int j = 0; j < NV / PER; ++j) {
        if (PER * j >= steps) break;
        key_pieces(j);
      }
    } else {
#pragma unroll 2
      for (int j = 0; j < steps / PER; ++j) key_pieces(j);
    }
    // Scores in powers of two; lane: keys 16 n + g (entries 0, 1) and 16 n + g + 8 (2, 3) of rows 2 t and 2 t + 1.  Codes: a lane prepares one key's scales
    float c[NK][2], add[NK][2], over[NK][2], rest[NK][2];    // one over what of the values' scales is in the exponent; what is not
    bool zeros = false;                                      // whether a value counts as zeros
    if constexpr (HALF) {
      const float k1 = __uint_as_float(lds32(sb + lane * 4)), v = __uint_as_float(lds32(sb + 128 + lane * 4));
      const bool zero = v >= 0.f && v <= 1.17549435e-38f;    // 2^-126 (a row of zeros) or 0 (never written): counts as zeros
      const float some = zero ? SMALLEST_SCALE : v;
      float a1, o1, r1;
      if (F32) {                                             // the power of two: exact; the rest of it goes with the weight
        const int exponent = (int)(__float_as_uint(some) >> 23 & 255u);
        a1 = (float)(exponent - 127);
        o1 = __uint_as_float((uint32_t)(254 - exponent) << 23);
        r1 = zero ? 0.f : v * o1;
      } else {                                               // all of it, to 2^-22 (of log2 s where that is larger than 1)
        asm("lg2.approx.f32 %0, %1;" : "=f"(a1) : "f"(some));
        asm("rcp.approx.f32 %0, %1;" : "=f"(o1) : "f"(some));
        r1 = zero ? 0.f : 1.f;
        zeros = __any_sync(0xffffffffu, zero);
      }
      if (!(some >= SMALLEST_SCALE && some <= LARGEST_SCALE)) o1 = NAN;
#pragma unroll
      for (int n = 0; n < NK; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int from = 16 * n + 8 * e + g;
          c[n][e] = __shfl_sync(0xffffffffu, k1, from);
          add[n][e] = __shfl_sync(0xffffffffu, a1, from);
          over[n][e] = __shfl_sync(0xffffffffu, o1, from);
          if (F32) rest[n][e] = __shfl_sync(0xffffffffu, r1, from);
        }
      if (!F32 && zeros)
#pragma unroll
        for (int n = 0; n < NK; ++n)
#pragma unroll
          for (int e = 0; e < 2; ++e) rest[n][e] = __shfl_sync(0xffffffffu, r1, 16 * n + 8 * e + g);
    }
    const bool whole = lost == (NK == 2 ? 0u : 2u) && ks.whole(key0, 16 * NK);
    bool grows = false;
    float top[NR][2];
#pragma unroll
    for (int r = 0; r < NR; ++r) {
#pragma unroll
      for (int n = 0; n < NK; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          s[n][r][e] = HALF ? fmaf(s[n][r][e] * c[n][e >> 1], cr[r][e & 1], add[n][e >> 1]) : s[n][r][e] * a.scale_log2;
          if (!whole && (lost >> n & 1u || !a.sees(pos[r][e & 1], key0 + 16 * n + g + 8 * (e >> 1)))) s[n][r][e] = -INFINITY;
        }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        top[r][e] = fmaxf(s[0][r][e], s[0][r][2 + e]);
        if (NK == 2) top[r][e] = fmaxf(top[r][e], fmaxf(s[NK - 1][r][e], s[NK - 1][r][2 + e]));
        top[r][e] = fmaxf(top[r][e], __shfl_xor_sync(0xffffffffu, top[r][e], 4));
        top[r][e] = fmaxf(top[r][e], __shfl_xor_sync(0xffffffffu, top[r][e], 8));
        top[r][e] = fmaxf(top[r][e], __shfl_xor_sync(0xffffffffu, top[r][e], 16));
        grows |= top[r][e] > m[r][e];
      }
    }
    if (__any_sync(0xffffffffu, grows)) {
#pragma unroll
      for (int r = 0; r < NR; ++r) {
        float f[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float now = fmaxf(m[r][e], top[r][e]);
          f[e] = m[r][e] == now ? 1.f : exp2_f(m[r][e] - now);
          m[r][e] = now;
          l[r][e] *= f[e];
        }
#pragma unroll
        for (int x = 0; x < NV; ++x)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[r][x][e] *= f[e & 1];
      }
    }
    uint32_t wb[NK][NR][WP][2];                              // the weights as the B operand of the second product
#pragma unroll
    for (int n = 0; n < NK; ++n)
#pragma unroll
      for (int r = 0; r < NR; ++r)
#pragma unroll
        for (int k = 0; k < 2; ++k) {                        // key g or g + 8
          float x[2];
          uint32_t w[WP];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float z = s[n][r][2 * k + e];
            x[e] = exp2_f(F32 ? (z - m[r][e]) + LIFT : z - (m[r][e] - LIFT));
            if (z == -INFINITY) x[e] = 0.f;                  // hidden, or of no weight: whatever its scale is, and while the maximum is -inf
            else l[r][e] = HALF ? fmaf(x[e], over[n][k], l[r][e]) : l[r][e] + x[e];
            if (HALF && (F32 || zeros)) x[e] = z == -INFINITY ? 0.f : x[e] * rest[n][k];
          }
          operand2<HALF, WP>(x[0], x[1], w);
#pragma unroll
          for (int p = 0; p < WP; ++p) wb[n][r][p][k] = transposed(w[p]);
        }
    auto value = [&](int n, int x, const uint32_t (&v)[KP][4]) {      // 16 entries of the values
#pragma unroll
      for (int r = 0; r < NR; ++r) product<HALF, KP, WP, V_PRODUCTS, F32>(o[r][x], v, wb[n][r]);
    };
    if constexpr (F32 && !HALF) {
#pragma unroll
      for (int x = 0; x < NV; ++x) {
        if (16 * x >= a.V) break;
        uint32_t v[KP][4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {                        // entries 16 x + g, + 8 of keys 2 t, 2 t + 1 and 8 more
          float y[2];
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const int r = 2 * t + k + 8 * (e >> 1), c = 4 * x + (g >> 2) + 2 * (e & 1);
            y[k] = __uint_as_float(lds32(vb + (c >> 3) * ATOM + r * 128 + (((c & 7) ^ (r & 7)) << 4) + (g & 3) * 4));
          }
          uint32_t p[KP];
          parts2<KP>(y[0], y[1], p);
#pragma unroll
          for (int k = 0; k < KP; ++k) v[k][e] = p[k];
        }
        value(0, x, v);
      }
    } else if constexpr (HALF) {
#pragma unroll
      for (int x = 0; x < (NV + 1) / 2; ++x) {               // 32 entries at a time; the last 16 may be the copy's zeros
        if (32 * x >= a.V) break;
#pragma unroll
        for (int n = 0; n < NK; ++n) {
          uint32_t r4[4];
          ldsm_x4_t(vb + ((x >> 2) * NK + n) * ATOM + (at_16 ^ ((x & 3) << 5)), r4);
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            if (2 * x + y >= NV) break;
            const uint2 lo = codes4<STORE, 0, 2, 1, 3>(r4[2 * y]), hi = codes4<STORE, 0, 2, 1, 3>(r4[2 * y + 1]);      // entries 2 g and 2 g + 1 of two keys
            const uint32_t v[1][4] = {{lo.x, lo.y, hi.x, hi.y}};
            value(n, 2 * x + y, v);
          }
        }
      }
    } else {
#pragma unroll
      for (int x = 0; x < NV; ++x) {
        if (16 * x >= a.V) break;
        uint32_t v[1][4];
        ldsm_x4_t(vb + (x >> 2) * ATOM + (at_8 ^ ((x & 3) << 5)), v[0]);
        value(0, x, v);
      }
    }
  }
  if (dead) {                                                // copies under way end before the CTA does; the rows are computed again from memory
    uint32_t late = 0;
    for (int i = 0; i < stages; ++i) tc::mbar_wait_warp(bar0 + 8 * i, phase >> i & 1u, late);
#pragma unroll
    for (int r = 0; r < NR; ++r) l[r][0] = l[r][1] = NAN;
  }

  // the warps' results: reference maximum, sum and outputs of R rows each
#pragma unroll
  for (int r = 0; r < NR; ++r)
#pragma unroll
    for (int e = 0; e < 2; ++e)
#pragma unroll
      for (int k = 4; k < 32; k <<= 1) l[r][e] += __shfl_xor_sync(0xffffffffu, l[r][e], k);
  __syncthreads();
  float* sm = reinterpret_cast<float*>(smem);                // [W][R] maxima, [W][R] sums, [W][R][ov] outputs
  const int ov = a.V + 4;
  float* so = sm + 2 * R * W;
#pragma unroll
  for (int r = 0; r < NR; ++r) {
    if (g == 0)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        sm[R * warp + 8 * r + 2 * t + e] = m[r][e];
        sm[R * (W + warp) + 8 * r + 2 * t + e] = l[r][e];
      }
#pragma unroll
    for (int x = 0; x < NV; ++x) {
      if (16 * x >= a.V) break;
#pragma unroll
      for (int e = 0; e < 4; ++e) so[(R * warp + 8 * r + 2 * t + (e & 1)) * ov + 16 * x + (HALF ? 2 * g + (e >> 1) : g + 8 * (e >> 1))] = o[r][x][e];
    }
  }
  __syncthreads();
  const int quads = a.V / 4;
  for (int i = threadIdx.x; i < R * quads; i += blockDim.x) {
    const int r = i / quads, d = 4 * (i - r * quads), at = pl.first + r;
    if (at >= pl.n * G) break;
    float M = -INFINITY, L = 0.f, x[4] = {0.f, 0.f, 0.f, 0.f};
    for (int w = 0; w < W; ++w) M = fmaxf(M, sm[R * w + r]);
    for (int w = 0; w < W; ++w) {
      const float mw = sm[R * w + r];
      if (mw == -INFINITY && sm[R * (W + w) + r] == 0.f) continue;
      const float f = mw == M ? 1.f : exp2_f(mw - M);
      L += f * sm[R * (W + w) + r];
      const float4 y = *reinterpret_cast<const float4*>(so + (R * w + r) * ov + d);
      x[0] = fmaf(f, y.x, x[0]);
      x[1] = fmaf(f, y.y, x[1]);
      x[2] = fmaf(f, y.z, x[2]);
      x[3] = fmaf(f, y.w, x[3]);
    }
    const int row = pl.start + at / G, head = h * G + at % G;
    if (a.few.splits > 1) {
      const long long to = (long long)split * a.few.count + (a.both ? (long long)(pl.b * a.kv_heads + h) * a.few_max + at : (long long)row * a.heads + head);
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
    const uint32_t own = (W == 4 ? 0x11111111u : W == 2 ? 0x55555555u : 0xffffffffu) << warp;      // every W-th row
    if (bad & own) mend_rows<4>(a, pl.b, pl.start, pl.length - pl.n, h, pl.first, bad & own, lane);
  }
}

// ------------------------------------------------------------------------------------------------ joining parts
// `per` warps (a power of two) have a row and head, each every per-th part.  Parts are read once, and the loads of a warp's parts do not wait for one another.
constexpr int MERGE_WARPS = 8;
__global__ void __launch_bounds__(32 * MERGE_WARPS) paged_merge_kernel(const __grid_constant__ Attn a, int per) {
  __shared__ float4 sx[MERGE_WARPS][64];
  __shared__ float2 sml[MERGE_WARPS];
  const int lane = threadIdx.x & 31, warp = threadIdx.x / 32;
  const int here = MERGE_WARPS / per, sub = warp / here, own = warp % here;      // part of the unit's warps, unit of the block
  const long long at = (long long)blockIdx.x * here + own;
  int row, head, b = -1;
  if (a.both) {                                              // the packed rows of every sequence and key/value head
    const int G = a.heads / a.kv_heads, r = (int)(at % a.few_max), h = (int)(at / a.few_max % a.kv_heads);
    const long long of = at / a.few_max / a.kv_heads;
    int start = 0, n = 0, length;
    if (of < a.s.seqs) sequence(a.s, (int)of, start, n, length);
    if ((long long)n * G <= a.few_max && r < n * G) b = (int)of;
    row = start + r / G;
    head = h * G + r % G;
  } else {
    row = (int)min(at / a.heads, (long long)a.s.rows);
    head = (int)(at % a.heads);
    if (row < a.s.rows) b = sequence_of(a.s, row, lane);
  }
  const Parts& p = a.few;
  const bool on = b >= 0;
  float M = -INFINITY, L = 0.f;
  float4 x[2] = {};
  pdl_wait();                                                // launched as the last CTAs that compute parts end: they let nothing in earlier
  if (on) {
#pragma unroll 4
    for (int i = sub; i < p.splits; i += per) {
      const float2 ml = *reinterpret_cast<const float2*>(p.ml + 2 * (i * p.count + at));
      const float4* y = reinterpret_cast<const float4*>(p.o + (i * p.count + at) * a.V) + lane;
      float4 z[2];
#pragma unroll
      for (int c = 0; c < 2; ++c) z[c] = 4 * (lane + 32 * c) < a.V ? y[32 * c] : make_float4(0.f, 0.f, 0.f, 0.f);
      if (ml.x == -INFINITY && ml.y == 0.f) continue;        // saw nothing
      const float now = fmaxf(M, ml.x), f = M == now ? 1.f : exp2_f(M - now), w = ml.x == now ? 1.f : exp2_f(ml.x - now);
      M = now;
      L = L * f + w * ml.y;
#pragma unroll
      for (int c = 0; c < 2; ++c) x[c] = make_float4(x[c].x * f + w * z[c].x, x[c].y * f + w * z[c].y, x[c].z * f + w * z[c].z, x[c].w * f + w * z[c].w);
    }
  }
  if (per > 1) {
    if (sub > 0) {
#pragma unroll
      for (int c = 0; c < 2; ++c) sx[warp][lane + 32 * c] = x[c];
      if (lane == 0) sml[warp] = make_float2(M, L);
    }
    __syncthreads();
    if (sub > 0) return;
    for (int w0 = warp + here; w0 < MERGE_WARPS; w0 += here) {
      const float2 ml = sml[w0];
      if (ml.x == -INFINITY && ml.y == 0.f) continue;
      const float now = fmaxf(M, ml.x), f = M == now ? 1.f : exp2_f(M - now), w = ml.x == now ? 1.f : exp2_f(ml.x - now);
      M = now;
      L = L * f + w * ml.y;
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const float4 z = sx[w0][lane + 32 * c];
        x[c] = make_float4(x[c].x * f + w * z.x, x[c].y * f + w * z.y, x[c].z * f + w * z.z, x[c].w * f + w * z.w);
      }
    }
  }
  if (!on) return;
  const float inv = L == 0.f ? 0.f : 1.f / L;
  bool fine = true;
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    const int d = 4 * (lane + 32 * c);
    if (d >= a.V) break;
    const float y[4] = {x[c].x, x[c].y, x[c].z, x[c].w};
    a.store(((size_t)row * a.heads + head) * a.V + d, y, inv);
    fine = fine && finite4(y, inv);
  }
  if (!__all_sync(0xffffffffu, fine)) {
    __syncwarp();
    int start, n, length;
    sequence(a.s, b, start, n, length);
    const int G = a.heads / a.kv_heads;
    mend_rows<4>(a, b, start, length - n, head / G, (row - start) * G + head % G, 1u, lane);
  }
}

// ------------------------------------------------------------------------------------------------ host
struct Plan {
  int few_max, few_rows, few_tiles, few_splits, many_ctas;   // few_tiles: of the few-row kernel, 0 where the chunk kernel takes the step; many_ctas: the other way round
  long long few_count, floats;
};
constexpr long long MOST_WORK = 1ll << 27;                   // floats of partial results

static long long few_floats(int splits, long long count, int V) { return splits > 1 ? (2 * splits * count + 3) / 4 * 4 + splits * count * V : 0; }

// A window, or a number of first tokens, as long as all that a table holds.  (A position below zero less a longer window need not fit 32 bits.)
static bool hides_nothing(int window, int first, int width, int page) { return std::max(window, first) >= (long long)width * page; }

static Plan plan_of(int rows, int seqs, int width, int page, int heads, int kv_heads, int K, int V, int window, int first, int max_new, int max_length, int store, int act_dtype) {
  Plan p{};
  if (hides_nothing(window, first, width, page)) window = first = 0;
  const int G = heads / kv_heads, sms = sm_count(), most = std::min(seqs, rows);
  // packed rows of the longest of the sequences; where the host says nothing, a token each if there are no more rows than sequences
  const long long packed = (long long)rows * G, longest = (long long)(max_new > 0 ? std::min(max_new, rows) : rows <= seqs ? 1 : rows) * G;
  long long keys = (long long)width * page;                  // the most keys that a row sees
  if (max_length > 0) keys = std::min<long long>(keys, max_length);
  if (window > 0) keys = std::min<long long>(keys, (long long)window + first + 16);
  // The chunk kernel takes steps with a sequence of more than 16 packed rows.  Single tokens among them too, at up to 3.5 times the few-row kernel's time from
  // 8-bit pools and 1.3 times from bf16 ones, until what that adds is more than the 12 us of two more launches: a chunk of 512 with 8, 48 or 192 tokens of others
  // over 4096 keys of 8 heads takes 107, 184 or 381 us in both kernels from e4m3, 121, 332 or 1084 in the one; from bf16 with 48 or 192 215 and 573, or 210
  // and 670.  There are at most `singles` of them.  (Heads of 128 in groups of four; other sizes were not measured.)
  long long singles = seqs;
  p.few_max = INT32_MAX;
  if (act_dtype == B2L_BF16 && longest > 16 && many_takes(K, V, store)) {
    p.many_ctas = many_ctas((packed / 256 + most) * kv_heads, keys + (window > 0 ? 256 / G : 0), sms);
    p.floats = many_floats(p.many_ctas, V);
    const long long more = longest / G - 1;                  // rows of the longest beside its first
    singles -= (std::max(rows - seqs, 0) + more - 1) / std::max(more, 1ll);
    const bool both = G <= 16 && singles > 0 && singles * kv_heads * 0.5 * keys * (store == ACT ? 0.015e-3 : 0.119e-3) > 12;
    p.few_max = both ? (G <= 8 ? 8 : 16) : 0;
    if (!both) return p;
    p.few_rows = p.few_max;
    p.few_tiles = seqs;
    p.few_count = (long long)seqs * kv_heads * p.few_max;
  } else {
    // rows of a tile: 8 where a token's heads, or all that the longest of the sequences has, fit
    p.few_rows = (max_new > 0 ? (long long)max_new * G <= 8 : G <= 8 && packed <= 8ll * most) ? 8 : 16;
    p.few_tiles = seqs + (int)std::min<long long>(packed / p.few_rows, INT32_MAX - seqs);
    p.few_count = (long long)rows * heads;
    singles = std::max<long long>(seqs, packed / p.few_rows);
  }
  // An SM has three CTAs at a time (with f32 rows, or heads beyond 128, two or one: then this takes up to three times the parts that fill it, or finds room for parts
  // where there is none; chosen and measured for three).  Few CTAs: as many parts as fill them once, of 128 keys at least (one token over 1031 keys of 32 heads: 15.1 us in 4 parts,
  // 13.0 in 8).  Many: parts of a quarter of that each, of 512 keys at least, so that sequences of different lengths share the SMs evenly (48 over up to 8192
  // keys of an e4m3 pool: 143 us whole, 128 in 4 parts, 140 in 8)
  const long long ctas = (long long)kv_heads * singles, slots = 3ll * sms;
  const bool room = 2 * ctas <= slots;
  const long long want = room ? slots / ctas : (4 * slots + ctas - 1) / ctas;
  p.few_splits = (int)std::max<long long>(1, std::min({want, keys / (room ? 128 : 512), 128ll, MOST_WORK / (p.few_count * (V + 2) + 1)}));
  p.floats += few_floats(p.few_splits, p.few_count, V);
  return p;
}

template <typename act_t, int STORE, int NV, int NR> static int few_launch(const Attn& a, int tiles, cudaStream_t stream) {
  constexpr int ES = STORE == ACT ? (int)sizeof(act_t) : 1, PER = ES == 1 ? 2 : 1;
  const size_t queries = (size_t)(sizeof(act_t) == 4 ? 3 : 1) * ((a.K / 16 + PER - 1) / PER * PER) * NR * 256, unit = (size_t)(atoms_of(a.K, ES) + atoms_of(a.V, ES)) * ATOM * (ES == 1 ? 2 : 1);
  // four warps and as many CTAs on an SM as leave each warp two units in its ring at least; fewer warps where one CTA does not fit
  constexpr size_t SM = 227 * 1024, OTHER = ES == 1 ? 6 * 1024 : 2 * 1024;      // static: barriers, scales; the system's 1 KB
  int W = 4, stages = 0;
  for (int ctas = NV <= 8 ? (NR == 1 && ES == 1 ? 4 : 3) : 2; ctas >= 1 && stages < 2; --ctas)
    for (W = 4; W >= (ctas == 1 ? 1 : 4); W /= 2) {
      const size_t room = SM / ctas - OTHER;
      stages = room > queries ? (int)std::min<size_t>(most_stages(STORE), (room - queries) / (W * unit)) : 0;
      if (stages >= 2) break;
    }
  B2L_CHECK_SUPPORTED(stages >= 2, "b2l_seq_paged_attention: heads of %d and %d entries do not fit", a.K, a.V);
  const size_t smem = std::max(queries + W * stages * unit, (size_t)W * 8 * NR * (a.V + 6) * 4);
  const CUtensorMapDataType type = ES == 1 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : ES == 2 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT32;
  const long long rows = ((long long)a.s.pages * a.kv_heads) << a.s.shift;
  FewMaps maps;
  const int box = ES == 1 && a.s.shift >= 5 ? 32 : 16;
  if (int rc = tc::map_sw128(&maps.k, type, ES, a.k, rows, a.K, a.K, 128 / ES, box)) return rc;
  if (int rc = tc::map_sw128(&maps.v, type, ES, a.v, rows, a.V, a.V, 128 / ES, box)) return rc;
  static DynSmemCache cache;
  auto kernel = paged_few_kernel<act_t, STORE, NV, NR>;
  if (int rc = ensure_dyn_smem(kernel, smem, cache)) return rc;
  kernel<<<dim3((unsigned)tiles, (unsigned)a.kv_heads, (unsigned)a.few.splits), 32 * W, smem, stream>>>(a, maps, stages);
  B2L_LAUNCH_CHECK("paged_few_kernel");
  return 0;
}

}  // namespace paged
}  // namespace b2l

using namespace b2l;

extern "C" long long b2l_seq_paged_attention_work(int rows, int seqs, int width, int page, int heads, int kv_heads, int K, int V, int window, int first, int max_new,
                                                  int max_length, int store, int act_dtype) {
  if (rows <= 0 || seqs <= 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads != 0) return 0;
  return paged::plan_of(rows, seqs, width, page, heads, kv_heads, K, V, window, first, max_new, max_length, store, act_dtype).floats;
}

static int attention(const char* who, bool zeros, const void* q, long long ldq, long long hsq, const void* k, const void* v, const float* k_scale, const float* v_scale,
                     const int* starts, const int* lengths, const int* table, int ldt, int width, void* out, float* work, long long work_floats, int rows, int seqs, int pages,
                     int page, int heads, int kv_heads, int K, int V, int window, int first, float scale, int max_new, int max_length, int store, int act_dtype,
                     b2l_stream_t stream) {
  using namespace paged;
  B2L_CHECK_ARG(rows == 0 || (q && out), "%s: null pointer", who);
  if (int rc = check_pool(who, k, v, k_scale, v_scale, starts, lengths, table, ldt, width, rows, seqs, pages, page, kv_heads, K, V, store, act_dtype)) return rc;
  B2L_CHECK_ARG(heads > 0 && heads % kv_heads == 0, "%s: %d heads over %d key/value heads", who, heads, kv_heads);
  B2L_CHECK_ARG(window >= 0 && first >= 0, "%s: a negative window or number of first tokens", who);
  B2L_CHECK_ARG(scale > 0.f && scale < INFINITY, "%s: the scale must be positive and finite", who);
  const int per = act_dtype == B2L_F32 ? 4 : 8;
  B2L_CHECK_ARG((((uintptr_t)q | (uintptr_t)out | (uintptr_t)work) & 15) == 0 && ldq % per == 0 && hsq % per == 0, "%s: rows must be 16-byte aligned", who);
  B2L_CHECK_SUPPORTED((long long)width * page < (1ll << 30) && kv_heads < 65536 && (long long)rows * heads < (1ll << 31) - 65536 && (long long)pages * kv_heads * page < (1ll << 31),
                      "%s: sizes beyond the grid's or a copy's coordinates", who);
  if (rows == 0 || seqs == 0) return 0;
  if (paged::hides_nothing(window, first, width, page)) window = first = 0;
  const Plan p = plan_of(rows, seqs, width, page, heads, kv_heads, K, V, window, first, max_new, max_length, store, act_dtype);
  B2L_CHECK_ARG(p.floats == 0 || (work && work_floats >= p.floats), "%s: a work space of %lld floats is needed", who, p.floats);
  Attn a{};
  a.s = step_of(starts, lengths, table, ldt, width, rows, seqs, pages, page);
  a.q = q; a.k = k; a.v = v; a.ks = k_scale; a.vs = v_scale; a.out = out;
  a.ldq = ldq; a.hsq = hsq;
  a.heads = heads; a.kv_heads = kv_heads; a.K = K; a.V = V;
  a.window = window; a.first = window ? first : 0;
  a.scale_log2 = scale * 1.44269502162933349609375f;         // log2(e)
  a.f32 = act_dtype == B2L_F32; a.store_kind = store;
  const cudaStream_t st = (cudaStream_t)stream;
  a.few_max = p.few_max;
  a.zeros = zeros;
  a.both = p.few_tiles > 0 && p.many_ctas > 0;
  if (p.many_ctas) {
    const int rc = many_launch(a, p.many_ctas, work, st);
    if (rc || !a.both) return rc;
    a.zeros = 0;                                             // they are there
    work += many_floats(p.many_ctas, V);
  }
  a.few.splits = p.few_splits;
  a.few.count = p.few_count;
  a.few.ml = work;
  a.few.o = work + (2 * p.few_splits * a.few.count + 3) / 4 * 4;
  int rc = 0;
  const bool small = V <= 128 && K <= 128;
#define GO(ST)                                                                                                                              \
  (p.few_rows == 8 ? (small ? few_launch<act_t, ST, 8, 1>(a, p.few_tiles, st) : few_launch<act_t, ST, 16, 1>(a, p.few_tiles, st))            \
                   : (small ? few_launch<act_t, ST, 8, 2>(a, p.few_tiles, st) : few_launch<act_t, ST, 16, 2>(a, p.few_tiles, st)))
  B2L_SEQ_DISPATCH(act_dtype, rc = store == ACT ? GO(ACT) : store == E4M3 ? GO(E4M3) : GO(INT8));
#undef GO
  if (rc || p.few_splits == 1) return rc;
  const int warps = p.few_splits >= 32 ? 8 : p.few_splits >= 16 ? 4 : p.few_splits >= 8 ? 2 : 1, here = MERGE_WARPS / warps;
  LaunchCfg launch(dim3((unsigned)((a.few.count + here - 1) / here)), dim3(32 * MERGE_WARPS), 0, st, true);
  B2L_CUDA(cudaLaunchKernelEx(&launch.cfg, paged_merge_kernel, a, warps));
  B2L_LAUNCH_CHECK("paged_merge_kernel");
  return 0;
}

extern "C" int b2l_seq_paged_attention(const void* q, long long ldq, long long hsq, const void* k, const void* v, const float* k_scale, const float* v_scale, const int* starts,
                                       const int* lengths, const int* table, int ldt, int width, void* out, float* work, long long work_floats, int rows, int seqs, int pages,
                                       int page, int heads, int kv_heads, int K, int V, int window, int first, float scale, int max_new, int max_length, int store,
                                       int act_dtype, b2l_stream_t stream) {
  return attention("b2l_seq_paged_attention", false, q, ldq, hsq, k, v, k_scale, v_scale, starts, lengths, table, ldt, width, out, work, work_floats, rows, seqs, pages, page, heads,
                   kv_heads, K, V, window, first, scale, max_new, max_length, store, act_dtype, stream);
}

extern "C" int b2l_seq_paged_attention_all(const void* q, long long ldq, long long hsq, const void* k, const void* v, const float* k_scale, const float* v_scale, const int* starts,
                                           const int* lengths, const int* table, int ldt, int width, void* out, float* work, long long work_floats, int rows, int seqs, int pages,
                                           int page, int heads, int kv_heads, int K, int V, int window, int first, float scale, int max_new, int max_length, int store,
                                           int act_dtype, b2l_stream_t stream) {
  return attention("b2l_seq_paged_attention_all", true, q, ldq, hsq, k, v, k_scale, v_scale, starts, lengths, table, ldt, width, out, work, work_floats, rows, seqs, pages, page,
                   heads, kv_heads, K, V, window, first, scale, max_new, max_length, store, act_dtype, stream);
}
