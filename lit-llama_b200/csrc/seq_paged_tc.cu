// Attention of chunks over a paged pool on tcgen05: 256 packed rows of one key/value head (seq_paged_attn.cu) against tiles of 128 keys.
//
// Two tiles of 128 rows take turns: while the tensor core multiplies one tile's queries with the keys and the other's weights with the values, four warps
// turn the first one's scores into weights, a thread per row (tensor-memory lane), so no row needs another thread's maximum or sum.
//
//   warp 0        issues the MMAs: for a tile of keys t and each row tile, P(t) V, then Q K^T of t + 1 (one commit tells that the scores are there and
//                 that the output may be touched)
//   warp 1        bf16 pool: tiled copies of pages, 64 columns each, into 128-byte swizzled rows (keys K-major, values MN-major)
//   warps 4..11   softmax of row tile 0 (4..7) and 1 (8..11): scores from tensor memory twice, once for the maximum and once for the weights, which go
//                 back over them in two halves, so the second product begins with the first 64 keys.  A row's reference moves only when it is exceeded
//                 by more than 8 (weights reach 2^8; nothing is rounded by that), so the output in tensor memory is seldom scaled
//   warps 12..15  8-bit pool: codes by 16-byte loads a tile ahead, as f16 (exactly) into the same rows, and the tile's scales
//
// Weights are rounded to one bf16 (by half a step, 2^-8; with 8-bit pools one f16, 2^-11): the first rounding below f32 in the sums, and the price of one
// product instead of two; outputs in bf16 are off by as much themselves.  8-bit pools: queries as f16 times a power of two per row, the scale of a value in
// the exponent of its weight, as the few-row kernel has them.
//
// Tensor memory: scores and weights of the row tiles at columns 0 and 128, outputs at 256 and 384.  Shared memory: the queries of both, two stages of keys
// and values where they fit.  One CTA per SM.
#include <utility>

#include "seq_paged_attn.cuh"
#include "tc_common.cuh"

namespace b2l {
namespace paged {

using namespace tc;

constexpr int KEYS = 128, TILE = 128, ROWS = 2 * TILE, MOST_K = 192, MOST_V = 128;
constexpr int TC_ATOM = 128 * 128;                           // bytes of 64 columns of 128 rows
constexpr int INFOS = 4;

struct alignas(16) Info {                                    // of a tile of keys, for the softmax (read by 16 bytes)
  float ks[KEYS], add[KEYS], over[KEYS];                     // scale of the key, log2 of the value's, one over it (8-bit pools)
  uint32_t there, zero[KEYS / 32];                           // 16 keys each: whether their page is there; keys whose values count as zeros
};
struct Control {
  uint64_t q_full, k_full[2], k_empty[2], v_full[2], v_empty[2], s_full[2], p_half[2][2], o_done[2], info_full[INFOS], tail, gave_up;
  uint32_t tmem;
};
constexpr size_t CONTROL_BYTES = 1024;
template <int STORE> constexpr size_t INFO_BYTES = STORE == ACT ? 1024 : (INFOS * sizeof(Info) + 1023) / 1024 * 1024;
static_assert(sizeof(Control) <= CONTROL_BYTES && sizeof(Info) % 16 == 0);

struct Layout { int ks, vs; size_t smem; };                  // stages of keys and values; none: the sizes do not fit
template <int STORE> static Layout layout(int K, int V) {
  const size_t base = CONTROL_BYTES + INFO_BYTES<STORE>, ka = atoms_of(K, 2), va = atoms_of(V, 2), q = 2 * ka * TC_ATOM, room = 227 * 1024;
  Layout l{0, 0, 0};
  for (const auto& [ks, vs] : {std::pair<int, int>{2, 2}, {2, 1}, {1, 1}})
    if (base + q + (ks * ka + vs * va) * TC_ATOM <= room) {
      l = {ks, vs, base + q + (ks * ka + vs * va) * TC_ATOM};
      break;
    }
  if (l.ks && l.smem < 120 * 1024) l.smem = 120 * 1024;      // one CTA per SM: each takes all of tensor memory
  return l;
}

__device__ __forceinline__ void tmem_ld32(uint32_t a, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, "
      "%28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]),
        "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(a)
      : "memory");
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc, uint32_t lead) {
  asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
               "l"(a), "l"(b), "r"(idesc), "r"(acc), "r"(lead)
               : "memory");
}
// MN-major operand, 128-byte swizzle: rows of 64 consecutive MN entries, one row per k; `lbo` bytes to the next 64 entries
__device__ __forceinline__ uint64_t desc_mn(uint32_t addr, uint32_t lbo) {
  return (uint64_t)((addr & 0x3FFFFu) >> 4) | ((uint64_t)(lbo >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) | ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
__device__ __forceinline__ void st128(uint32_t a, uint4 v) { asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(a), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory"); }
__device__ __forceinline__ float4 ldf4(const float* p) { return *reinterpret_cast<const float4*>(p); }
// bits 0 .. n-1 (any n)
__device__ __forceinline__ uint32_t low_bits(int n) { return n >= 32 ? 0xffffffffu : n <= 0 ? 0u : (1u << n) - 1u; }
// place of the 16-byte piece c of row r in tiles of 128 rows
__device__ __forceinline__ uint32_t piece_at(int r, int c) { return (uint32_t)((c >> 3) * TC_ATOM + r * 128 + (((c & 7) ^ (r & 7)) << 4)); }

template <int STORE>
__global__ void __launch_bounds__(STORE == ACT ? 384 : 512, 1) paged_many_kernel(const __grid_constant__ Attn a, const __grid_constant__ CUtensorMap map_k,
                                                                                  const __grid_constant__ CUtensorMap map_v, int k_stages, int v_stages) {
  constexpr bool HALF = STORE != ACT;
  constexpr float LIFT = HALF ? 6.f : 0.f;                   // weights up to 2^8 times this in f16
  extern __shared__ __align__(1024) uint8_t smem[];
  Control& ct = *reinterpret_cast<Control*>(smem);
  Info* infos = reinterpret_cast<Info*>(smem + CONTROL_BYTES);      // ACT: only `there`, at uint32_t steps
  uint32_t* there_of = reinterpret_cast<uint32_t*>(smem + CONTROL_BYTES);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, G = a.heads / a.kv_heads, h = blockIdx.y, split = blockIdx.z;
  Place pl;
  if (!a.place(gridDim.x - 1 - blockIdx.x, ROWS, a.few_max, INT32_MAX, lane, pl)) return;      // later rows, with more keys, first
  const int rows = min(ROWS, pl.n * G - pl.first), groups = rows > TILE ? 2 : 1;
  const Keys keys = a.keys(pl, ROWS);
  const int all = keys.units(7), per = (all + a.many.splits - 1) / a.many.splits;
  const int t0 = min(split * per, all), n = min(t0 + per, all) - t0;
  const int ka = atoms_of(a.K, 2), va = atoms_of(a.V, 2);
  const uint32_t sq = smem_u32(smem) + CONTROL_BYTES + INFO_BYTES<STORE>, sk = sq + 2 * ka * TC_ATOM, sv = sk + k_stages * ka * TC_ATOM;
  auto bar = [&](const uint64_t& b) { return smem_u32(&b); };
  uint32_t dead = (sq & 1023u) ? 1u : 0u;
  if (tid == 0) {
    mbar_init(bar(ct.q_full), 256);
    for (int i = 0; i < 2; ++i) {
      mbar_init(bar(ct.k_full[i]), HALF ? 128 : 1);
      mbar_init(bar(ct.v_full[i]), HALF ? 128 : 1);
      mbar_init(bar(ct.k_empty[i]), 1);
      mbar_init(bar(ct.v_empty[i]), 1);
      mbar_init(bar(ct.s_full[i]), 1);
      mbar_init(bar(ct.p_half[i][0]), 4);
      mbar_init(bar(ct.p_half[i][1]), 4);
      mbar_init(bar(ct.o_done[i]), 1);
    }
    for (int i = 0; i < INFOS; ++i) mbar_init(bar(ct.info_full[i]), HALF ? 128 : 1);
    mbar_init(bar(ct.tail), 1);
    mbar_init(bar(ct.gave_up), 1);
    mbar_init_fence();
  }
  if (warp == 0) tmem_alloc(smem_u32(&ct.tmem), 512);
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = ct.tmem;
  // 8-bit pool: 512 threads of 128 registers; a tile's codes, loaded a tile ahead, take 80 of the last warpgroup's, and what the first does not need
  // (64 x 128 + 128 x 256 + 184 x 128 <= 128 x 512)
  if (HALF && warp < 4) asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
  if (HALF && warp >= 12) asm volatile("setmaxnreg.inc.sync.aligned.u32 184;");

  if (warp == 0) {
    // ===================== MMA issue =====================
    const uint32_t lead = elect_lane();
    const uint32_t types = HALF ? 0u : (1u << 7) | (1u << 10);      // f16 or bf16, both operands
    const uint32_t id_s = (1u << 4) | types | ((uint32_t)(KEYS >> 3) << 17) | ((uint32_t)(TILE >> 4) << 24);
    const uint32_t id_o = (1u << 4) | types | (1u << 16) | ((uint32_t)(a.V >> 3) << 17) | ((uint32_t)(TILE >> 4) << 24);
    const int steps = a.K / 16;
    auto scores = [&](int g, int st) {
      uint32_t d = tmem + 128 * g;
#pragma unroll 1
      for (int x = 0; 4 * x < steps; ++x) {
        const uint64_t qd = desc_sw128(sq + (g * ka + x) * TC_ATOM), kd = desc_sw128(sk + (st * ka + x) * TC_ATOM);
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (4 * x + k < steps) mma_ss(d, qd + 2 * k, kd + 2 * k, id_s, x + k > 0 ? 1u : 0u, lead);
      }
    };
    auto outputs = [&](int g, int half, int st, bool first) {
      const uint64_t vd = desc_mn(sv + st * va * TC_ATOM + half * (TC_ATOM / 2), TC_ATOM);
#pragma unroll
      for (int k = 0; k < 4; ++k)
        mma_ts(tmem + 256 + 128 * g, tmem + 128 * g + 32 * half + 8 * k, vd + k * (16 * 128 / 16), id_o, first && half == 0 && k == 0 ? 0u : 1u, lead);
    };
    int kst = 0, vst = 0;
    uint32_t kph = 0, vph = 0;
    if (n > 0) {
      mbar_wait(bar(ct.q_full), 0, dead);
      mbar_wait_warp(bar(ct.k_full[0]), 0, dead);
      fence_after();
      for (int g = 0; g < groups && !dead; ++g) {
        scores(g, 0);
        if (lead) commit(bar(ct.s_full[g]));
      }
      if (!dead && lead) commit(bar(ct.k_empty[0]));
      if (++kst == k_stages) { kst = 0; kph ^= 1u; }
    }
    for (int t = 0; t < n && !dead; ++t) {
      const bool more = t + 1 < n;
      mbar_wait_warp(bar(ct.v_full[vst]), vph, dead);
      for (int g = 0; g < groups && !dead; ++g) {
#pragma unroll 1
        for (int half = 0; half < 2 && !dead; ++half) {
          mbar_wait_warp(bar(ct.p_half[g][half]), (uint32_t)t & 1u, dead);
          if (dead) break;
          fence_after();
          outputs(g, half, vst, t == 0);
        }
        if (dead) break;
        if (g == groups - 1 && lead) commit(bar(ct.v_empty[vst]));
        if (more) {
          if (g == 0) mbar_wait_warp(bar(ct.k_full[kst]), kph, dead);
          if (dead) break;
          fence_after();
          scores(g, kst);
          if (lead) {
            commit(bar(ct.s_full[g]));
            if (g == groups - 1) commit(bar(ct.k_empty[kst]));
          }
        } else if (lead) {
          commit(bar(ct.o_done[g]));
        }
        __syncwarp();
      }
      if (++vst == v_stages) { vst = 0; vph ^= 1u; }
      if (++kst == k_stages) { kst = 0; kph ^= 1u; }
    }
    if (dead) {                                              // what was issued ends before tensor memory is given back
      uint32_t late = 0;
      if (lead) commit(bar(ct.gave_up));
      mbar_wait(bar(ct.gave_up), 0, late);
    }
    __syncwarp();
  } else if (warp == 1 && !HALF) {
    // ===================== tiled copies =====================
    const int box = min(1 << a.s.shift, KEYS), boxes = KEYS / box, gone = (a.s.pages * a.kv_heads) << a.s.shift;      // a row beyond the pool: zeros
    int kst = 0, vst = 0;
    uint32_t kph = 1, vph = 1, tail_waits = 0;               // a stage is free at first
    for (int t = 0; t < n; ++t) {
      const int key0 = keys.key0(t0 + t, 7);
      int page = -1;
      if (lane < boxes && key0 + lane * box < keys.end) page = page_of(a.s, pl.b, key0 + lane * box);
      const uint32_t seen = __ballot_sync(0xffffffffu, page >= 0);
      const int row = page >= 0 ? ((page * a.kv_heads + h) << a.s.shift) + ((key0 + lane * box) & ((1 << a.s.shift) - 1)) : gone;
      uint32_t there = 0;                                    // by 16 keys
      for (int i = 0; i < 8; ++i) there |= (seen >> (i * 16 / box) & 1u) << i;
      mbar_wait_warp(bar(ct.k_empty[kst]), kph, dead);
      if (dead) break;
      if (lane == 0) {
        there_of[t % INFOS] = there;
        mbar_arrive(bar(ct.info_full[t % INFOS]));
        mbar_expect_tx(bar(ct.k_full[kst]), ka * TC_ATOM);
      }
      for (int i = 0; i < boxes; ++i) {
        const int r = __shfl_sync(0xffffffffu, row, i);
        if (lane == 0)
          for (int x = 0; x < ka; ++x) tma_load_2d(sk + (kst * ka + x) * TC_ATOM + i * box * 128, &map_k, 64 * x, r, bar(ct.k_full[kst]));
      }
      if (++kst == k_stages) { kst = 0; kph ^= 1u; }
      mbar_wait_warp(bar(ct.v_empty[vst]), vph, dead);
      if (dead) break;
      const int valid = keys.end - key0;
      // behind the last key that is seen the page may hold anything, and a weight of zero does not hide an infinity: zeros there
      const uint32_t to = valid < KEYS ? bar(ct.tail) : bar(ct.v_full[vst]);
      if (lane == 0) mbar_expect_tx(to, va * TC_ATOM);
      for (int i = 0; i < boxes; ++i) {
        const int r = __shfl_sync(0xffffffffu, row, i);
        if (lane == 0)
          for (int x = 0; x < va; ++x) tma_load_2d(sv + (vst * va + x) * TC_ATOM + i * box * 128, &map_v, 64 * x, r, to);
      }
      if (valid < KEYS) {
        mbar_wait_warp(to, tail_waits++ & 1u, dead);
        if (dead) break;
        for (int x = lane; x < (KEYS - valid) * 8 * va; x += 32) st128(sv + vst * va * TC_ATOM + piece_at(valid + x / (8 * va), x % (8 * va)), make_uint4(0, 0, 0, 0));
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(ct.v_full[vst]));
      }
      if (++vst == v_stages) { vst = 0; vph ^= 1u; }
    }
    // every copy has landed before the CTA ends: the MMAs of all tiles come after them, unless a wait ran out
    if (dead) {
      uint32_t late = 0;
      for (int i = 0; i < k_stages; ++i) mbar_wait(bar(ct.k_full[i]), i < kst ? kph ^ 1u : kph, late);
      late = 0;
      for (int i = 0; i < v_stages; ++i) mbar_wait(bar(ct.v_full[i]), i < vst ? vph ^ 1u : vph, late);
    }
    __syncwarp();
  } else if (warp >= 12) {
    // ===================== 8-bit codes to f16 =====================
    if constexpr (HALF) {
      const int me = tid - 384, kc = a.K / 16, vc = a.V / 16;      // 16-byte pieces of a row
      int kst = 0, vst = 0;
      uint32_t kph = 1, vph = 1;
      int pages = -1, key0 = 0;
      auto look = [&](int t) {                               // pages of a tile's 16-key parts, in lanes 0..7
        key0 = keys.key0(t0 + t, 7);
        const int j = key0 + 16 * (lane & 7);
        pages = j < keys.end ? page_of(a.s, pl.b, j) : -1;
      };
      auto row_of = [&](int key) -> long long {              // of the pool, or -1; a whole warp asks
        const int page = __shfl_sync(0xffffffffu, pages, key >> 4);
        const int j = key0 + key;
        return page >= 0 && j < keys.end ? ((long long)(page * a.kv_heads + h) << a.s.shift) + (j & ((1 << a.s.shift) - 1)) : -1;
      };
      const int k_by = 65536 / kc + 1, v_by = 65536 / vc + 1;      // x / pieces = x by >> 16 for x < 128 pieces, pieces <= 12
      auto fetch = [&](const void* pool, int D, int pieces, int by, int i) {
        const int x = i * 128 + me, key = x * by >> 16, c = x - key * pieces;
        const long long row = row_of(key);
        const uint4 w = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint8_t*>(pool) + max(row, 0ll) * D + c * 16);
        return row >= 0 ? w : make_uint4(0u, 0u, 0u, 0u);
      };
      auto put = [&](uint32_t base, int pieces, int by, int i, uint4 w, bool zero) {
        const int x = i * 128 + me, key = x * by >> 16, c = x - key * pieces;
        const uint32_t u[4] = {w.x, w.y, w.z, w.w};
        uint32_t y[8];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint2 f = codes4<STORE, 0, 1, 2, 3>(u[e]);
          y[2 * e] = zero ? 0u : f.x;
          y[2 * e + 1] = zero ? 0u : f.y;
        }
        const int odd = (c >> 2) & 1;                        // neighbours meet different banks
        const uint4 lo = make_uint4(y[0], y[1], y[2], y[3]), hi = make_uint4(y[4], y[5], y[6], y[7]);
        st128(base + piece_at(key, 2 * c + odd), odd ? hi : lo);
        st128(base + piece_at(key, 2 * c + 1 - odd), odd ? lo : hi);
      };
      uint4 kw[MOST_K / 16], vw[MOST_V / 16];
      float ks = 0.f, vs = 0.f;
      auto fetch_keys = [&](int t) {
        look(t);
#pragma unroll
        for (int i = 0; i < MOST_K / 16; ++i)
          if (i < kc) kw[i] = fetch(a.k, a.K, kc, k_by, i);
        const long long row = row_of(me);
        ks = row >= 0 ? a.ks[row] : 0.f;
        vs = row >= 0 ? a.vs[row] : 1.f;
      };
      if (n > 0) fetch_keys(0);
      for (int t = 0; t < n; ++t) {
        Info& info = infos[t % INFOS];
        const bool zero_row = vs <= 1.17549435e-38f && vs >= 0.f;      // 2^-126 (a row of zeros) or 0 (never written): counts as zeros
        const uint32_t there = __ballot_sync(0xffffffffu, pages >= 0) & 0xffu, zeros = __ballot_sync(0xffffffffu, zero_row);
        float add = 0.f, over = 1.f;
        const float some = zero_row ? SMALLEST_SCALE : vs;
        asm("lg2.approx.f32 %0, %1;" : "=f"(add) : "f"(some));
        asm("rcp.approx.f32 %0, %1;" : "=f"(over) : "f"(some));
        if (!(some >= SMALLEST_SCALE && some <= LARGEST_SCALE)) over = NAN;
#pragma unroll
        for (int i = 0; i < MOST_V / 16; ++i)
          if (i < vc) vw[i] = fetch(a.v, a.V, vc, v_by, i);
        mbar_wait_warp(bar(ct.k_empty[kst]), kph, dead);
        if (dead) break;
        info.ks[me] = ks;
        info.add[me] = add;
        info.over[me] = over;
        if (lane == 0) info.zero[warp - 12] = zeros;
        if (me == 0) info.there = there;
        mbar_arrive(bar(ct.info_full[t % INFOS]));
#pragma unroll
        for (int i = 0; i < MOST_K / 16; ++i)
          if (i < kc) put(sk + kst * ka * TC_ATOM, kc, k_by, i, kw[i], false);
        fence_proxy_async();
        mbar_arrive(bar(ct.k_full[kst]));
        if (++kst == k_stages) { kst = 0; kph ^= 1u; }
        if (t + 1 < n) fetch_keys(t + 1);
        mbar_wait_warp(bar(ct.v_empty[vst]), vph, dead);
        if (dead) break;
        mbar_wait_warp(bar(ct.info_full[t % INFOS]), (uint32_t)(t / INFOS) & 1u, dead);      // all four warps' zero rows are known
        if (dead) break;
#pragma unroll
        for (int i = 0; i < MOST_V / 16; ++i)
          if (i < vc) {
            const int key = (i * 128 + me) * v_by >> 16;
            put(sv + vst * va * TC_ATOM, vc, v_by, i, vw[i], info.zero[key >> 5] >> (key & 31) & 1u);
          }
        fence_proxy_async();
        mbar_arrive(bar(ct.v_full[vst]));
        if (++vst == v_stages) { vst = 0; vph ^= 1u; }
      }
    }
  } else if (warp >= 4) {
    // ===================== queries, softmax, outputs =====================
    const int g = (warp - 4) >> 2, r = (warp & 3) * 32 + lane, at = pl.first + TILE * g + r;
    const bool live = TILE * g + r < rows;
    const int token = live ? at / G : 0, head = h * G + (live ? at % G : 0), row = pl.start + token, pos = live ? pl.length - pl.n + token : -1;
    const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16), S = lanes + 128 * g, O = lanes + 256 + 128 * g;
    float cr = a.scale_log2;
    {
      const __nv_bfloat16* src = reinterpret_cast<const __nv_bfloat16*>(a.q) + (size_t)row * a.ldq + (size_t)head * a.hsq;
      float up = 1.f;
      if (HALF) {
        float top = 0.f;
        for (int c = 0; c < a.K / 8 && live; ++c) {
          const float4 x = ld_act4(src + 8 * c), y = ld_act4(src + 8 * c + 4);
          top = fmaxf(fmaxf(fmaxf(fmaxf(top, fabsf(x.x)), fabsf(x.y)), fmaxf(fabsf(x.z), fabsf(x.w))), fmaxf(fmaxf(fabsf(y.x), fabsf(y.y)), fmaxf(fabsf(y.z), fabsf(y.w))));
        }
        lift_of(top, a.scale_log2, up, cr);
      }
      for (int c = 0; c < a.K / 8; ++c) {
        uint4 w = live ? *reinterpret_cast<const uint4*>(src + 8 * c) : make_uint4(0u, 0u, 0u, 0u);
        if (HALF) {
          uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const __half2 f = __floats2half2_rn(__uint_as_float(u[e] << 16) * up, __uint_as_float(u[e] & 0xffff0000u) * up);
            u[e] = *reinterpret_cast<const uint32_t*>(&f);
          }
          w = make_uint4(u[0], u[1], u[2], u[3]);
        }
        st128(sq + g * ka * TC_ATOM + piece_at(r, c), w);
      }
      fence_proxy_async();
      mbar_arrive(bar(ct.q_full));
    }
    float m = -INFINITY, l = 0.f;
    // positions of this group's rows: where all of them see a tile no mask is needed
    const int p_min = pl.length - pl.n + (pl.first + TILE * g) / G, p_max = pl.length - pl.n + (pl.first + min(TILE * (g + 1), rows) - 1) / G;
    if (g < groups) {
      for (int t = 0; t < n; ++t) {
        const int key0 = keys.key0(t0 + t, 7);
        mbar_wait(bar(ct.info_full[t % INFOS]), (uint32_t)(t / INFOS) & 1u, dead);
        mbar_wait_warp(bar(ct.s_full[g]), (uint32_t)t & 1u, dead);
        if (dead) break;
        fence_after();
        const Info& info = infos[t % INFOS];
        const uint32_t there = HALF ? info.there : there_of[t % INFOS];
        const bool whole = there == 0xffu && key0 + KEYS - 1 <= p_min && (a.window == 0 || key0 > p_max - a.window || key0 + KEYS <= a.first);
        // keys that the row sees, as bits of 32
        auto seen = [&](int c) {
          const int j = key0 + 32 * c;
          uint32_t x = low_bits(pos + 1 - j);
          if (a.window) x &= ~low_bits(pos - a.window + 1 - j) | low_bits(a.first - j);
          return x & (((there >> 2 * c & 1u) ? 0xffffu : 0u) | ((there >> (2 * c + 1) & 1u) ? 0xffff0000u : 0u));
        };
        float top = -INFINITY;
#pragma unroll 1
        for (int c = 0; c < 4; ++c) {
          uint32_t u[32];
          tmem_ld32(S + 32 * c, u);
          float x[4] = {top, -INFINITY, -INFINITY, -INFINITY};
          if (HALF) {
#pragma unroll
            for (int i = 0; i < 32; i += 4) {
              const float4 k4 = ldf4(info.ks + 32 * c + i), a4 = ldf4(info.add + 32 * c + i);
              u[i] = __float_as_uint(fmaf(__uint_as_float(u[i]) * k4.x, cr, a4.x));
              u[i + 1] = __float_as_uint(fmaf(__uint_as_float(u[i + 1]) * k4.y, cr, a4.y));
              u[i + 2] = __float_as_uint(fmaf(__uint_as_float(u[i + 2]) * k4.z, cr, a4.z));
              u[i + 3] = __float_as_uint(fmaf(__uint_as_float(u[i + 3]) * k4.w, cr, a4.w));
            }
          }
          if (!whole) {
            const uint32_t mask = seen(c);
#pragma unroll
            for (int i = 0; i < 32; ++i) u[i] = mask >> i & 1u ? u[i] : 0xff800000u;
          }
#pragma unroll
          for (int i = 0; i < 32; ++i) x[i & 3] = fmaxf(x[i & 3], __uint_as_float(u[i]));
          top = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
        }
        if (!HALF) top *= cr;
        const bool grows = top > m + 8.f || (m == -INFINITY && top > m);
        if (__any_sync(0xffffffffu, grows)) {
          const float f = grows ? exp2_f(m - top) : 1.f;     // 0 where nothing was added yet
          if (grows) m = top;
          l *= f;
          if (t > 0) {                                       // these scores came after the product of tile t - 1
#pragma unroll 1
            for (int c = 0; 16 * c < a.V; ++c) {
              uint32_t o[16];
              tmem_ld16(O + 16 * c, o);
#pragma unroll
              for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
              tmem_st16(O + 16 * c, o);
            }
          }
        }
        const float ref = m == -INFINITY ? 0.f : m - LIFT;
        float sum[2] = {0.f, 0.f};
#pragma unroll 1
        for (int c = 0; c < 4; ++c) {
          uint32_t u[32], w[16];
          tmem_ld32(S + 32 * c, u);
          if (!whole) {
            const uint32_t mask = seen(c);
#pragma unroll
            for (int i = 0; i < 32; ++i) u[i] = mask >> i & 1u ? u[i] : 0xff800000u;
          }
          if (HALF) {
#pragma unroll
            for (int i = 0; i < 32; i += 4) {
              const float4 k4 = ldf4(info.ks + 32 * c + i), a4 = ldf4(info.add + 32 * c + i), o4 = ldf4(info.over + 32 * c + i);
              float x[4] = {fmaf(__uint_as_float(u[i]) * k4.x, cr, a4.x), fmaf(__uint_as_float(u[i + 1]) * k4.y, cr, a4.y),
                            fmaf(__uint_as_float(u[i + 2]) * k4.z, cr, a4.z), fmaf(__uint_as_float(u[i + 3]) * k4.w, cr, a4.w)};
              const float ov[4] = {o4.x, o4.y, o4.z, o4.w};
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const bool none = u[i + e] == 0xff800000u;   // hidden: whatever its scales are
                x[e] = none ? 0.f : exp2_f(x[e] - ref);
                sum[e & 1] = fmaf(x[e], none ? 0.f : ov[e], sum[e & 1]);
              }
              const __half2 lo = __floats2half2_rn(x[0], x[1]), hi = __floats2half2_rn(x[2], x[3]);
              w[i / 2] = *reinterpret_cast<const uint32_t*>(&lo);
              w[i / 2 + 1] = *reinterpret_cast<const uint32_t*>(&hi);
            }
          } else {
#pragma unroll
            for (int i = 0; i < 32; i += 2) {
              const float x = exp2_f(fmaf(__uint_as_float(u[i]), cr, -ref)), y = exp2_f(fmaf(__uint_as_float(u[i + 1]), cr, -ref));
              sum[0] += x;
              sum[1] += y;
              const __nv_bfloat162 z = __floats2bfloat162_rn(x, y);
              w[i / 2] = *reinterpret_cast<const uint32_t*>(&z);
            }
          }
          tmem_st16(S + 16 * c, w);
          if (c & 1) {                                       // half of the weights
            tmem_wait_st();
            fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar(ct.p_half[g][c >> 1]));
          }
        }
        l += sum[0] + sum[1];
      }
      if (n > 0) mbar_wait_warp(bar(ct.o_done[g]), 0, dead);
      fence_after();
      if (dead) l = NAN;
      const float inv = a.many.splits > 1 ? 1.f : l == 0.f ? 0.f : 1.f / l;
      bool fine = true;
      const long long to = ((long long)split * a.many.count + (long long)row * a.heads + head);
#pragma unroll 1
      for (int c = 0; 16 * c < a.V; ++c) {
        uint32_t o[16];
        if (n > 0 && !dead) tmem_ld16(O + 16 * c, o);
        float x[4];
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
#pragma unroll
          for (int e = 0; e < 4; ++e) x[e] = dead ? NAN : n > 0 ? __uint_as_float(o[i + e]) : 0.f;
          if (!live) continue;
          if (a.many.splits > 1) *reinterpret_cast<float4*>(a.many.o + to * a.V + 16 * c + i) = make_float4(x[0], x[1], x[2], x[3]);
          else a.store(((size_t)row * a.heads + head) * a.V + 16 * c + i, x, inv);
          fine = fine && finite4(x, inv);
        }
      }
      if (live && a.many.splits > 1) *reinterpret_cast<float2*>(a.many.ml + 2 * to) = make_float2(m, l);
      if (a.many.splits == 1) {
        __syncwarp();
        for (uint32_t left = __ballot_sync(0xffffffffu, live && !(fine && fabsf(l) < INFINITY)); left; left &= left - 1) {
          const int i = __ffs(left) - 1;
          mend_row(a, pl.b, __shfl_sync(0xffffffffu, pos, i), __shfl_sync(0xffffffffu, row, i), __shfl_sync(0xffffffffu, head, i), lane);
        }
      }
    }
  }
  fence_before();
  __syncthreads();
  if (warp == 0) tmem_dealloc(tmem, 512);
}

bool many_takes(int K, int V, int store) {
  if (K > MOST_K || V > MOST_V) return false;
  return (store == ACT ? layout<ACT>(K, V) : layout<INT8>(K, V)).ks > 0;
}

template <int STORE> static int go(const Attn& a, int tiles, cudaStream_t stream) {
  const Layout l = layout<STORE>(a.K, a.V);
  CUtensorMap mk{}, mv{};
  if (STORE == ACT) {
    const long long rows = ((long long)a.s.pages * a.kv_heads) << a.s.shift;
    const int box = 1 << a.s.shift < KEYS ? 1 << a.s.shift : KEYS;
    if (int rc = map_sw128(&mk, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, a.k, rows, a.K, a.K, 64, box)) return rc;
    if (int rc = map_sw128(&mv, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, a.v, rows, a.V, a.V, 64, box)) return rc;
  }
  static DynSmemCache cache;
  if (int rc = ensure_dyn_smem(paged_many_kernel<STORE>, l.smem, cache)) return rc;
  paged_many_kernel<STORE><<<dim3((unsigned)tiles, (unsigned)a.kv_heads, (unsigned)a.many.splits), STORE == ACT ? 384 : 512, l.smem, stream>>>(a, mk, mv, l.ks, l.vs);
  B2L_LAUNCH_CHECK("paged_many_kernel");
  return 0;
}
int many_launch(const Attn& a, int tiles, cudaStream_t stream) {
  return a.store_kind == ACT ? go<ACT>(a, tiles, stream) : a.store_kind == E4M3 ? go<E4M3>(a, tiles, stream) : go<INT8>(a, tiles, stream);
}

}  // namespace paged
}  // namespace b2l
