// Attention of chunks over a paged pool on tcgen05: 256 packed rows of one key/value head (seq_paged_attn.cu) against tiles of 128 keys.
//
// Two tiles of 128 rows take turns: while the tensor core multiplies one tile's queries with the keys and the other's weights with the values, four warps
// turn the first one's scores into weights, a thread per row (tensor-memory lane), so no row needs another thread's maximum or sum.
//
//   warp 0        issues the MMAs: for a tile of keys t and each row tile, P(t) V, then Q K^T of t + 1 (one commit tells that the scores are there and
//                 that the output may be touched).  The other row tile's products fill the time of this one's softmax.  (Two issuing warps fell into step:
//                 both softmaxes at once, then the products, 4300 cycles for a tile; units of 64 keys with two places for their scores took 4160, as an MMA
//                 of N = 64 takes 75 cycles and one of N = 128 103: its rows of A come out of shared memory for half as many keys.)
//   warp 1        tiled copies of pages: bf16, 64 columns each, into 128-byte swizzled rows (keys K-major, values MN-major); codes as they lie, with their
//                 scales, for warps 12..19
//   warps 4..11   softmax of row tile 0 (4..7) and 1 (8..11): a row's scores into registers, its weights back over them in two halves, so the second product
//                 begins with the half that is there.  A row's reference moves only when it is exceeded by more than 8 (weights reach 2^8; nothing is
//                 rounded by that), so the output in tensor memory is seldom scaled.  bf16: of four powers of two the special function unit computes
//                 three and a polynomial the fourth: 2048 tokens over 16384 of 32 / 8 heads take 430 us so, 441 without, 439 with three of eight, 447 with half
//   warps 12..19  8-bit pool: codes times their scale as f16 into the same rows, keys (12..15) and values
//
// Weights are rounded to one bf16 (by half a step, 2^-8; with 8-bit pools one f16, 2^-11): the first rounding below f32 in the sums, and the price of one
// product instead of two; outputs in bf16 are off by as much themselves.
// 8-bit pools: queries as f16 times a power of two per row.  The scale s of a key or value goes into its codes: code times s 2^e rounded to f16 (2^-11), e such
// that the largest s of the CTA's first 128 keys of a row tile comes to 1 .. 2; the scores and the outputs times 2^-e.  (A key's scale times its scores instead, without that
// rounding: every thread needs all of them, 128 KB of reads from shared memory for a tile; 2048 tokens over 16384 keys took 750 us.)  A row that sees a scale
// above 2^7 of that, or one that is not finite, is computed again.  A scale below 2^-12 of that is off by up to 2^-25 (c 2^-25 for its key or value, c the largest
// code), which beside others of the size is nothing.  Where a tile of a row's had one, the row is computed again if it is not nothing: a score's error K 2^15 c 2^-25
// cr may be above 2^-10, or the row's largest output is so small that c 2^-25 is above 2^-12 of it.
//
// Tensor memory: scores and weights of the row tiles at columns 0 and 128, outputs at 256 and 384.  Shared memory: the queries of both, two stages of keys
// and values where they fit (8-bit: of keys, and a tile of codes).  One CTA per SM, which goes through row tiles: the next one's first keys are fetched while the
// outputs of the last are stored.
//
// What bounds it, 2048 tokens over 16384 keys, 32 / 8 heads of 128: bf16 430 us, 1198 TFLOP/s, the tensor core 60% busy; the rest is each row tile's softmax,
// which its next product waits for.  8-bit 645 us (e4m3; int8 690): a row tile waits for its values' codes as well (f16 twice in shared memory do not fit), and queries, keys,
// values and codes keep shared memory's 128 bytes a cycle busy for some 2700 of a tile's 5600 cycles.  (8 warps for keys and values together: 731; with keys a
// tile ahead 787.)
//
// Trees of drafted tokens (TREE) read all of the context for few rows, so what bounds them is the keys on their way: a warp each copies keys and values, three stages of keys
// where they fit, and up to 128 packed rows take row tiles of one half that both halves' warps compute (PAIR, below).  64 tokens each of two sequences of 65536, 32 / 8 heads of
// 128, bf16: 144 us at 1965 MHz, 950 TFLOP/s and 3.7 TB/s (171 with one warp for both, two stages and parts joined one after the other); where they follow one another for more
// than 0.2 s, at the 1450 MHz that 1000 W allow, 173.  37 trees of 32 tokens over 4096 keys: bf16 117 us, 5.3 TB/s (131 in whole row tiles), e4m3 142 us, 2.2 TB/s (206): there
// each tile's values are turned into f16 in 1850 cycles and multiplied in 1100 before the next one's can be, as two stages of f16 values do not fit beside two stages of codes.
//
// Weights meet the values as one bf16 (with codes one f16), as the tensor core takes two operands of one type and a second product for a second part would cost as much as the
// first.  Trees' outputs in bf16 are off by 1.66e-3 of their norm by their own rounding; so they are by 1.67e-3 to 1.77e-3 (few keys and large weights), 5e-4 to 1.6e-3 from what
// f32 weights give.  (Few rows have weights of two bf16 parts, seq_paged_attn.cu: 8e-5.)
#include <algorithm>
#include <utility>

#include "attn_tc.cuh"
#include "seq_paged_attn.cuh"

namespace b2l {
namespace paged {

using namespace tc;
using atc::add2;
using atc::desc_mn;
using atc::fma2;
using atc::mma_ss;

constexpr int KEYS = 128, TILE = 128, MOST_K = 192, MOST_V = 128;
constexpr int TC_ATOM = 128 * 128;                           // bytes of 64 columns of 128 rows
constexpr int INFOS = 4;

// TREE: trees of drafted tokens.  PAIR: a row tile has one half only, 128 rows, and both halves' warps compute it: they take its tiles of keys in turn, each with a
// maximum, a sum and outputs of its own, which are joined at the end.  So one's products and softmax fill the time of the other's as they do in a whole row tile, and the room
// of the second half's queries is free for more stages.  For steps of few rows, whose time is that of the keys on their way.
template <bool TREE_, bool PAIR_> struct Tiles : Attn<TREE_> {
  static constexpr bool TREE = TREE_, PAIR = PAIR_;
  static constexpr int ROWS = PAIR ? TILE : 2 * TILE;
};

struct alignas(16) Info { uint2 k_by[KEYS], v_by[KEYS]; };   // 8-bit pools, of a tile of keys: what a key's and a value's codes are multiplied with
struct alignas(16) Note {                                    // of a tile of keys
  uint32_t there;                                            // 16 keys each: whether their page is there; bits 8 and 9: whether a scale of a key, a value is below 2^-12 of the largest
  float k_up, v_up;                                          // 8-bit pools: powers of two that the scales were multiplied with
};
// PAIR: twice as many as tiles that are prepared at a time, as the one half's next tile may be multiplied while the other still has to look at the one before
template <bool PAIR> constexpr int NOTES = PAIR ? 2 * INFOS : INFOS;
constexpr int MOST_NOTES = NOTES<true>, MOST_STAGES = 3;
// A row tile: 256 (or 128) packed rows of a head, the tiles of its sequence's rows one after the other, then the next head's, then the next sequence's
struct Walk {
  Place pl;
  int h;
  long long at;                                              // cost of all before it
};
struct Control {
  uint64_t q_full, k_full[MOST_STAGES], k_empty[MOST_STAGES], v_full[MOST_STAGES], v_empty[MOST_STAGES], s_full[2], p_half[2][2], o_done[2], info_full[MOST_NOTES], tail, gave_up;
  uint64_t ref_full, rk_full[2], rk_empty[2], rv_full[2], rv_empty[2];   // 8-bit pools: the first tile's largest scales, codes of keys and values
  uint32_t tmem, k_ref[3], v_ref[3];                         // largest scales of the first tile's keys and values, as bits, of a row tile, the next and the one before
  long long x0, x1;                                          // the CTA's part
  Walk at[20];                                               // each warp's row tile
};
struct Scales { float k[KEYS], v[KEYS]; };                   // 8-bit pools: what lies beside a tile's codes
constexpr size_t CONTROL_BYTES = 1024;
template <int STORE> constexpr size_t INFO_BYTES = STORE == ACT ? 1024 : (MOST_NOTES * sizeof(Note) + INFOS * sizeof(Info) + 1023) / 1024 * 1024;
static_assert(sizeof(Control) <= CONTROL_BYTES && sizeof(Info) % 16 == 0 && sizeof(Scales) == 1024);
template <int STORE> constexpr int THREADS = STORE == ACT ? 384 : 640;

// Stages of keys and values, and of 8-bit pools' codes (with both's scales beside the keys'); none: the sizes do not fit.  The first that fits is taken: PAIR with codes in two
// stages before values in two, as a tile of codes comes some 1200 cycles after it is asked for
struct Layout { int ks, vs, raw_ks, raw_vs; size_t smem; };
template <int STORE, bool PAIR, bool TREE = PAIR> static Layout layout(int K, int V) {
  const size_t ka = atoms_of(K, 2), va = atoms_of(V, 2), q = (PAIR ? 1 : 2) * ka * TC_ATOM + (PAIR ? 2048 : 0), room = 227 * 1024;
  constexpr int N = 5;
  const Layout whole[N] = {{2, 2, 1, 1}, {2, 1, 1, 1}, {1, 1, 1, 1}}, pair8[N] = {{2, 2, 2, 2}, {2, 1, 2, 2}, {1, 1, 2, 2}, {2, 1, 1, 1}, {1, 1, 1, 1}}, pair16[N] = {{3, 3, 1, 1}, {3, 2, 1, 1}, {2, 2, 1, 1}, {2, 1, 1, 1}, {1, 1, 1, 1}};
  Layout l{};
  for (int i = 0; i < N && !l.ks; ++i) {
    Layout s = STORE != ACT ? (PAIR ? pair8[i] : whole[i]) : TREE ? pair16[i] : whole[i];
    s.smem = CONTROL_BYTES + INFO_BYTES<STORE> + q + (s.ks * ka + s.vs * va) * TC_ATOM + (STORE == ACT ? 0 : KEYS * (s.raw_ks * K + s.raw_vs * V) + s.raw_ks * sizeof(Scales));
    if (s.ks && s.smem <= room) l = s;
  }
  if (l.ks && l.smem < 120 * 1024) l.smem = 120 * 1024;      // one CTA per SM: each takes all of tensor memory
  return l;
}

// 64 consecutive 32-bit columns of this warp's 32 tensor-memory lanes, on their way: the registers hold them after tmem_wait_ld64, which takes them as operands
// so that nothing uses them before it
__device__ __forceinline__ void tmem_ld64(uint32_t a, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x64.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, "
      "%32, %33, %34, %35, %36, %37, %38, %39, %40, %41, %42, %43, %44, %45, %46, %47, "
      "%48, %49, %50, %51, %52, %53, %54, %55, %56, %57, %58, %59, %60, %61, %62, %63}, [%64];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]),
        "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]),
        "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31]), "=r"(r[32]),
        "=r"(r[33]), "=r"(r[34]), "=r"(r[35]), "=r"(r[36]), "=r"(r[37]), "=r"(r[38]), "=r"(r[39]), "=r"(r[40]), "=r"(r[41]), "=r"(r[42]), "=r"(r[43]),
        "=r"(r[44]), "=r"(r[45]), "=r"(r[46]), "=r"(r[47]), "=r"(r[48]), "=r"(r[49]), "=r"(r[50]), "=r"(r[51]), "=r"(r[52]), "=r"(r[53]), "=r"(r[54]),
        "=r"(r[55]), "=r"(r[56]), "=r"(r[57]), "=r"(r[58]), "=r"(r[59]), "=r"(r[60]), "=r"(r[61]), "=r"(r[62]), "=r"(r[63])
      : "r"(a)
      : "memory");
}
__device__ __forceinline__ void tmem_wait_ld64(uint32_t* r) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int i = 0; i < 64; i += 16)
    asm volatile("" : "+r"(r[i]), "+r"(r[i + 1]), "+r"(r[i + 2]), "+r"(r[i + 3]), "+r"(r[i + 4]), "+r"(r[i + 5]), "+r"(r[i + 6]), "+r"(r[i + 7]), "+r"(r[i + 8]), "+r"(r[i + 9]),
                 "+r"(r[i + 10]), "+r"(r[i + 11]), "+r"(r[i + 12]), "+r"(r[i + 13]), "+r"(r[i + 14]), "+r"(r[i + 15]) : : "memory");
}
// The largest of three, NaN if one is
__device__ __forceinline__ float max3(float x, float y, float z) {
  float m;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(m) : "f"(x), "f"(y), "f"(z));
  return m;
}
__device__ __forceinline__ void mul2(float& a, float& b, float c, float d) {      // a *= c, b *= d
  asm("{\n\t.reg .b64 x, y;\n\tmov.b64 x, {%0, %1};\n\tmov.b64 y, {%2, %3};\n\tmul.rn.f32x2 x, x, y;\n\tmov.b64 {%0, %1}, x;\n\t}" : "+f"(a), "+f"(b) : "f"(c), "f"(d));
}
__device__ __forceinline__ void fma2v(float& a, float& b, float x, float y, float c) {      // a = a x + c, b = b y + c
  asm("{\n\t.reg .b64 u, v, w;\n\tmov.b64 u, {%0, %1};\n\tmov.b64 v, {%2, %3};\n\tmov.b64 w, {%4, %4};\n\tfma.rn.f32x2 u, u, v, w;\n\tmov.b64 {%0, %1}, u;\n\t}"
      : "+f"(a), "+f"(b) : "f"(x), "f"(y), "f"(c));
}
// Two powers of two on the FMA pipe: 2^n times a polynomial in the rest, |rest| <= 1/2 (fitted to the least largest relative error, 2^-13.3, with p(0) = 1; exact
// zero from -127 on down, as n = -127 then takes all of 1's exponent).  No NaN, none above 127.
__device__ __forceinline__ void exp2_poly2(float& x, float& y) {
  constexpr float MAGIC = 12582912.f;                        // 1.5 2^23: adding it rounds to an integer in the low bits
  x = fmaxf(x, -127.f);
  y = fmaxf(y, -127.f);
  float nx = x, ny = y;
  add2(nx, ny, MAGIC, MAGIC);
  float rx = nx, ry = ny;
  add2(rx, ry, -MAGIC, -MAGIC);
  atc::sub2(x, y, rx, ry);
  float px = x, py = y;
  fma2(px, py, 0.055008940398693085f, 0.2422109991312027f, 0.2422109991312027f);
  fma2v(px, py, x, y, 0.6932829022407532f);
  fma2v(px, py, x, y, 1.f);
  x = __uint_as_float(__float_as_uint(px) + (__float_as_uint(nx) << 23));
  y = __uint_as_float(__float_as_uint(py) + (__float_as_uint(ny) << 23));
}
__device__ __forceinline__ uint4 ld128(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ void st128(uint32_t a, uint4 v) { asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(a), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory"); }
// Waits are bounded by time, some ten seconds: others may be computing rows again all the while (32 rows over 16384 keys take 0.1 s).  Counted in tries, one of them
// lasts 40 ns or 4 us: a warp gave up after 0.15 s, and those that waited for it after 17 s.
constexpr long long PATIENCE = 20'000'000'000;               // cycles
__device__ __forceinline__ void wait_for(uint32_t a, uint32_t parity, uint32_t& dead) {
  if (dead) return;
  for (long long begin = 0;;) {
    uint32_t ok;
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(ok) : "r"(a), "r"(parity) : "memory");
    if (ok) return;
    const long long now = clock64();
    if (begin == 0) begin = now;
    if (now - begin > PATIENCE) break;
  }
  dead = 1u;
}
__device__ __forceinline__ void wait_warp(uint32_t a, uint32_t parity, uint32_t& dead) {      // a warp that acts on the outcome together
  wait_for(a, parity, dead);
  dead = __any_sync(0xffffffffu, dead) ? 1u : 0u;
}
// A warp that issues waits and commits by its leading lane alone, without a branch: 32 lanes at a barrier that is complete took 150 cycles, a branch around a
// commit some 100
__device__ __forceinline__ void wait_lead(uint32_t a, uint32_t parity, uint32_t lead, uint32_t& dead) {
  if (dead) return;
  for (long long begin = 0;;) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 q, %3, 0;\n\tsetp.ne.b32 p, 0, 0;\n\t@q mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(a), "r"(parity), "r"(lead)
        : "memory");
    if (__any_sync(0xffffffffu, ok)) return;
    const long long now = clock64();
    if (begin == 0) begin = now;
    if (__any_sync(0xffffffffu, now - begin > PATIENCE)) break;
  }
  dead = 1u;
}
// Three barriers at once, each by a lane of its own; for all lanes
__device__ __forceinline__ void wait_three(uint32_t a, uint32_t parity, int lane, uint32_t& dead) {
  if (dead) return;
  for (long long begin = 0;;) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\tsetp.lt.s32 q, %3, 3;\n\tsetp.eq.b32 p, 0, 0;\n\t@q mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(a), "r"(parity), "r"(lane)
        : "memory");
    if (__all_sync(0xffffffffu, ok)) break;
    const long long now = clock64();
    if (begin == 0) begin = now;
    if (__any_sync(0xffffffffu, now - begin > PATIENCE)) {
      dead = 1u;
      break;
    }
  }
  __syncwarp();
}
__device__ __forceinline__ void commit_by(uint32_t lead, uint32_t mbar) {
  asm volatile("{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(mbar), "r"(lead) : "memory");
}
// two codes (f16) times a factor in two parts, rounded once
__device__ __forceinline__ uint32_t scaled(uint32_t u, uint32_t hi, uint32_t lo) {
  uint32_t y;
  asm("{\n\t.reg .b32 x;\n\tmul.rn.f16x2 x, %1, %3;\n\tfma.rn.f16x2 %0, %1, %2, x;\n\t}" : "=r"(y) : "r"(u), "r"(hi), "r"(lo));
  return y;
}
__device__ __forceinline__ void bulk(uint32_t dst, const void* src, uint32_t bytes, uint32_t mbar) {      // multiples of 16 bytes
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes), "r"(mbar) : "memory");
}
// the power of two that brings a largest scale (as bits; 0: none) to 1 .. 2
__device__ __forceinline__ float value_lift(uint32_t bits) { return bits ? __uint_as_float((254u - (bits >> 23)) << 23) : 1.f; }
// place of the 16-byte piece c of row r in tiles of 128 rows
__device__ __forceinline__ uint32_t piece_at(int r, int c) { return (uint32_t)((c >> 3) * TC_ATOM + r * 128 + (((c & 7) ^ (r & 7)) << 4)); }

// This thread's 16-byte pieces of a tile's codes (rows of D bytes) as f16 into its rows, code times its row's factor (in two parts) rounded once: every `threads`-th
// piece.  HIDE: a factor of 0 hides whatever the codes are
// UNROLL: 2; PAIR 1, with one place in the code for keys and values (37 trees of 32 tokens over 4096 keys, e4m3: 153 us so when it was chosen, 142 with what came later, 173 with 2 and two places, 167 with the loads of
// four pieces together; values in two halves of 64 keys 160, twice as many warps of half the registers 170)
template <int STORE, bool HIDE, int UNROLL> __device__ __forceinline__ void codes_to_f16(uint32_t raw, int D, const uint2* factors, uint32_t base, int me, int threads) {
  const int pieces = D / 16;
  auto one = [&](uint32_t from, uint2 f, uint32_t first, uint32_t second, bool odd) {
    uint4 w = ld128(from);
    if (HIDE && f.x == 0u) w = make_uint4(0u, 0u, 0u, 0u);
    const uint32_t u[4] = {odd ? w.z : w.x, odd ? w.w : w.y, odd ? w.x : w.z, odd ? w.y : w.w};      // neighbours store their halves in turn: they meet different banks
    uint32_t y[8];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint2 p = codes4<STORE, 0, 1, 2, 3>(u[e]);
      y[2 * e] = scaled(p.x, f.x, f.y);
      y[2 * e + 1] = scaled(p.y, f.x, f.y);
    }
    st128(first, make_uint4(y[0], y[1], y[2], y[3]));
    st128(second, make_uint4(y[4], y[5], y[6], y[7]));
  };
  if ((pieces & (pieces - 1)) == 0) {                        // a thread's pieces lie at the same place of every 128th, 64th .. key
    const int by = 31 - __clz(pieces), c = me & (pieces - 1), key = me >> by, step = threads >> by;
    const bool odd = (c >> 2) & 1;
    uint32_t from = raw + 16 * me, first = base + piece_at(key, 2 * c + odd), second = base + piece_at(key, 2 * c + 1 - odd);
#pragma unroll UNROLL
    for (int k = key; k < KEYS; k += step, from += 16 * threads, first += 128 * step, second += 128 * step) one(from, factors[k], first, second, odd);
  } else {
    const int by = 65536 / pieces + 1;                       // x / pieces = x by >> 16 for x < 128 pieces, pieces <= 12
#pragma unroll 1
    for (int x = me; x < KEYS * pieces; x += threads) {
      const int key = x * by >> 16, c = x - key * pieces;
      const bool odd = (c >> 2) & 1;
      one(raw + 16 * x, factors[key], base + piece_at(key, 2 * c + odd), base + piece_at(key, 2 * c + 1 - odd), odd);
    }
  }
  fence_proxy_async();
}

// ---- which CTA computes what: an equal part of the cost of everything, in the order of `Walk`, so a CTA has whole row tiles and begins and ends inside one.
// Every CTA counts the cost itself.  A tile of keys costs 4 (3 where the row tile has one half only), a row tile 16 beside: 6 chunks of up to 512 tokens over
// 6000 keys of an e4m3 pool take 209 us so, 217 with 12 or 8, 224 with 24 (and 250 in row tiles that were all cut into as many parts).  No share is below 16: 64
// tokens over 4096 keys, 41 us, take 55 in shares of 48.
constexpr int EXTRA = 16, LEAST = 2, SMALLEST_SHARE = 16;      // LEAST: tiles of keys that a cut leaves on either side
// PAIR, where a tile costs 2: 8 (a tree of 32 tokens over 4096 keys of 8 heads, e4m3: 31 us so, 36 with 16; EXTRA of 8 takes 162 us for 32 uneven sequences, 157 with 16)
template <bool PAIR> constexpr int LEAST_SHARE = PAIR ? SMALLEST_SHARE / 2 : SMALLEST_SHARE;

struct Cost {
  int all, units, each;                                      // tiles of keys, the same but one at least, cost of each
  __device__ __forceinline__ int total() const { return EXTRA + units * each; }
  __device__ __forceinline__ int cut(long long d) const {      // tiles of keys before a cut at d
    if (d <= 0) return 0;
    if (d >= total()) return units;
    const int y = max((int)d - EXTRA, 0) / each;
    return y < LEAST ? 0 : units - y < LEAST ? units : y;
  }
};
template <class A> __device__ __forceinline__ Cost cost_of(const A& a, const Place& pl) {
  Cost c;
  c.all = a.keys(pl, A::ROWS).units(7);
  c.units = max(c.all, 1);
  c.each = !A::PAIR && pl.n * (a.heads / a.kv_heads) - pl.first > TILE ? 4 : A::PAIR ? 2 : 3;
  return c;
}
// of one head of a sequence, by a whole warp
template <class A> __device__ __forceinline__ long long sequence_cost(const A& a, Place pl, int lane) {
  long long sum = 0;
  for (pl.first = lane * A::ROWS; pl.first < pl.n * (a.heads / a.kv_heads); pl.first += 32 * A::ROWS) sum += cost_of(a, pl).total();
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  return sum;
}
// each sequence lo .. hi - 1 that is this kernel's, until f says true
template <bool TREE, typename F> __device__ __forceinline__ void each_sequence(const Attn<TREE>& a, int lo, int hi, int lane, F f) {
  for (int b0 = lo; b0 < hi; b0 += 32) {
    int start = 0, n = 0, length = 0;
    if (b0 + lane < hi) sequence(a.s, b0 + lane, start, n, length);
    for (uint32_t left = __ballot_sync(0xffffffffu, (long long)n * (a.heads / a.kv_heads) > a.few_max); left; left &= left - 1) {
      const int i = __ffs(left) - 1;
      if (f(Place{b0 + i, __shfl_sync(0xffffffffu, start, i), __shfl_sync(0xffffffffu, n, i), __shfl_sync(0xffffffffu, length, i), 0})) return;
    }
  }
}
// the row tile after this one; pl.n is 0 behind the last
template <class A> __device__ __forceinline__ void advance(const A& a, Walk& w, const Cost& c, int lane) {
  w.at += c.total();
  if (w.pl.n * (a.heads / a.kv_heads) - w.pl.first > A::ROWS) {
    w.pl.first += A::ROWS;
    return;
  }
  w.pl.first = 0;
  if (++w.h < a.kv_heads) return;
  w.h = 0;
  w.pl.n = 0;
  each_sequence(a, w.pl.b + 1, a.s.seqs, lane, [&](const Place& pl) {
    w.pl = pl;
    return true;
  });
}
// Every warp goes through the CTA's row tiles by itself: this one (tiles of keys t0 .. t1 - 1), and what follows it in shared memory, as registers are few
struct Item {
  Place pl;
  int h, t0, t1, n;                                          // n: tiles of keys that its rows see
  bool whole;
};
template <class A> __device__ __forceinline__ bool next(const A& a, Control& ct, int warp, int lane, Item& x) {
  Walk w = ct.at[warp];
  const long long x0 = ct.x0, x1 = ct.x1;
  bool found = false;
  while (!found && w.pl.n > 0 && w.at < x1) {
    const Cost c = cost_of(a, w.pl);
    x.t0 = c.cut(x0 - w.at);
    x.t1 = c.cut(x1 - w.at);
    if ((found = x.t0 < x.t1)) {
      x.pl = w.pl;
      x.h = w.h;
      x.whole = x.t0 == 0 && x.t1 == c.units;
      x.t1 = min(x.t1, c.all);
      x.n = max(x.t1 - x.t0, 0);
    }
    advance(a, w, c, lane);
  }
  __syncwarp();
  if (lane == 0) ct.at[warp] = w;
  __syncwarp();
  return found;
}

// Warps 4 .. 11 among themselves
__device__ __forceinline__ void both_halves() { asm volatile("bar.sync 1, 256;" ::: "memory"); }

template <class A> __device__ __forceinline__ int pl_groups(const Place& pl, int G) { return !A::PAIR && pl.n * G - pl.first > TILE ? 2 : 1; }

template <int STORE, class A>
__global__ void __launch_bounds__(THREADS<STORE>, 1) paged_many_kernel(const __grid_constant__ A a, const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                                                                       int k_stages, int v_stages, int k_codes, int v_codes) {
  constexpr bool HALF = STORE != ACT, TREE = A::TREE, PAIR = A::PAIR;
  constexpr int ROWS = A::ROWS, NOTES = paged::NOTES<PAIR>;
  constexpr int CONVERTERS = PAIR ? 4 : 128;                 // arrivals of those that convert keys, or values
  const int raw_ks = PAIR ? k_codes : 1, raw_vs = PAIR ? v_codes : 1;
  constexpr float LIFT = HALF ? 6.f : 0.f;                   // weights up to 2^14 in f16
  extern __shared__ __align__(1024) uint8_t smem[];
  Control& ct = *reinterpret_cast<Control*>(smem);
  Note* notes_of = reinterpret_cast<Note*>(smem + CONTROL_BYTES);
  Info* infos = reinterpret_cast<Info*>(smem + CONTROL_BYTES + MOST_NOTES * sizeof(Note));      // 8-bit pools
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, G = a.heads / a.kv_heads;
  // this CTA's part, x0 .. x1
  {
    const int warps = blockDim.x / 32, by = (a.s.seqs + warps - 1) / warps, lo = min(warp * by, a.s.seqs), hi = min(lo + by, a.s.seqs);
    long long mine = 0, before = 0, all = 0;
    int r0 = 0, r1 = a.s.rows;                               // rows of no sequence: before r0 and from r1 on; warp 3 has nothing else to do
    if (a.zeros && warp == 3) {
      r0 = min(max(a.s.starts[0], 0), a.s.rows);
      r1 = max(min(a.s.starts[a.s.seqs], a.s.rows), r0);
    }
    each_sequence(a, lo, hi, lane, [&](const Place& pl) {
      mine += sequence_cost(a, pl, lane) * a.kv_heads;
      return false;
    });
    long long* costs = reinterpret_cast<long long*>(smem + CONTROL_BYTES);      // where the tiles' notes come later
    if (lane == 0) costs[warp] = mine;
    __syncthreads();
    for (int i = 0; i < warps; ++i) {
      if (i == warp) before = all;
      all += costs[i];
    }
    if (a.zeros && warp == 3) {                              // every CTA's part of them
      if (r0 > 0) clear_rows(a, 0, r0, 0, a.heads, blockIdx.x * 32 + lane, gridDim.x * 32);
      if (r1 < a.s.rows) clear_rows(a, r1, a.s.rows, 0, a.heads, blockIdx.x * 32 + lane, gridDim.x * 32);
    }
    const long long share = max((all + gridDim.x - 1) / gridDim.x, (long long)LEAST_SHARE<PAIR>);
    const long long x0 = blockIdx.x * share;
    if (x0 >= all) {                                         // nothing is left
      if (tid == 0) a.many.last[blockIdx.x] = make_int4(0, 0, 0, 0);
      return;
    }
    if (tid == 0) {
      ct.x0 = x0;
      ct.x1 = min(x0 + share, all);
    }
    if (before <= x0 && x0 < before + mine)
      each_sequence(a, lo, hi, lane, [&](Place pl) {
        const long long one = sequence_cost(a, pl, lane);
        if (x0 >= before + one * a.kv_heads) {
          before += one * a.kv_heads;
          return false;
        }
        const int h = (int)((x0 - before) / one);
        before += h * one;
        for (int f0 = 0;; f0 += 32 * ROWS) {                 // the row tile of the head's
          pl.first = f0 + lane * ROWS;
          long long upto = pl.first < pl.n * G ? cost_of(a, pl).total() : 0;
#pragma unroll
          for (int o = 1; o < 32; o <<= 1) {
            const long long x = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += x;
          }
          const uint32_t past = __ballot_sync(0xffffffffu, x0 < before + upto);
          if (past) {
            const int k = __ffs(past) - 1, first = __shfl_sync(0xffffffffu, pl.first, k);
            const long long at = __shfl_sync(0xffffffffu, before + upto - cost_of(a, pl).total(), k);
            if (lane < warps) ct.at[lane] = Walk{Place{pl.b, pl.start, pl.n, pl.length, first}, h, at};
            return true;
          }
          before += __shfl_sync(0xffffffffu, upto, 31);
        }
      });
  }
  const int ka = atoms_of(a.K, 2), va = atoms_of(a.V, 2);
  const uint32_t sq = smem_u32(smem) + CONTROL_BYTES + INFO_BYTES<STORE>, sk = sq + (PAIR ? 1 : 2) * ka * TC_ATOM, sv = sk + k_stages * ka * TC_ATOM;
  const uint32_t raw_k = sv + v_stages * va * TC_ATOM, raw_v = raw_k + raw_ks * KEYS * a.K, raw_s = raw_v + raw_vs * KEYS * a.V;      // 8-bit pools: codes, scales
  const Scales* scales_of = reinterpret_cast<const Scales*>(smem + (raw_s - smem_u32(smem)));
  const uint32_t telling = HALF ? raw_s + raw_ks * (uint32_t)sizeof(Scales) : sv + v_stages * va * TC_ATOM;      // PAIR: what the halves tell one another, 2 KB
  auto bar = [&](const uint64_t& b) { return smem_u32(&b); };
  uint32_t dead = (sq & 1023u) ? 1u : 0u;
  if (tid == 0) {
    mbar_init(bar(ct.q_full), 256);
    for (int i = 0; i < 2; ++i) {
      mbar_init(bar(ct.s_full[i]), 1);
      mbar_init(bar(ct.p_half[i][0]), 4);
      mbar_init(bar(ct.p_half[i][1]), 4);
      mbar_init(bar(ct.o_done[i]), 1);
    }
    mbar_init(bar(ct.gave_up), 1);
    for (int i = 0; i < NOTES; ++i) mbar_init(bar(ct.info_full[i]), HALF ? CONVERTERS + 1 : 1);
    mbar_init(bar(ct.tail), 1);
    mbar_init(bar(ct.ref_full), 128);
    for (int i = 0; i < MOST_STAGES; ++i) {
      mbar_init(bar(ct.k_full[i]), HALF ? CONVERTERS : 1);
      mbar_init(bar(ct.v_full[i]), HALF ? CONVERTERS : 1);
      mbar_init(bar(ct.k_empty[i]), 1);
      mbar_init(bar(ct.v_empty[i]), 1);
      if (i >= 2) break;
      mbar_init(bar(ct.rk_full[i]), 1);
      mbar_init(bar(ct.rv_full[i]), 1);
      mbar_init(bar(ct.rk_empty[i]), CONVERTERS);
      mbar_init(bar(ct.rv_empty[i]), CONVERTERS);
    }
    for (int i = 0; i < 3; ++i) ct.k_ref[i] = ct.v_ref[i] = 0u;
    mbar_init_fence();
  }
  if (warp == 0) tmem_alloc(smem_u32(&ct.tmem), 512);
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = ct.tmem;
  Item x;
  if (warp < 4) {
   // 8-bit pool: 48 x 128 + 144 x 256 + 72 x 256 = 96 x 640 registers
   if constexpr (HALF) asm volatile("setmaxnreg.dec.sync.aligned.u32 48;");
   if (warp == 0) {
    // ===================== MMA issue =====================
    const uint32_t lead = elect_lane();
    const uint32_t types = HALF ? 0u : (1u << 7) | (1u << 10);      // f16 or bf16, both operands
    const uint32_t id_s = (1u << 4) | types | ((uint32_t)(KEYS >> 3) << 17) | ((uint32_t)(TILE >> 4) << 24);
    const uint32_t id_o = (1u << 4) | types | (1u << 16) | ((uint32_t)(a.V >> 3) << 17) | ((uint32_t)(TILE >> 4) << 24);
    const int steps = a.K / 16;
    int kst = 0, vst = 0, groups = 0;
    uint32_t kph = 0, vph = 0, item = 0, done[2] = {0, 0};      // row tiles; tiles of keys of each half
    auto scores = [&](int g) {
#pragma unroll 1
      for (int x = 0; 4 * x < steps; ++x) {
        const uint64_t qd = desc_sw128(sq + ((PAIR ? 0 : g) * ka + x) * TC_ATOM), kd = desc_sw128(sk + (kst * ka + x) * TC_ATOM);
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (4 * x + k < steps) mma_ss(tmem + 128 * g, qd + 2 * k, kd + 2 * k, id_s, x + k > 0 ? 1u : 0u, lead);
      }
      commit_by(lead, bar(ct.s_full[g]));
      if (PAIR || g == groups - 1) {
        commit_by(lead, bar(ct.k_empty[kst]));
        if (++kst == k_stages) { kst = 0; kph ^= 1u; }
      }
    };
    while (!dead && next(a, ct, warp, lane, x)) {
     const int n = x.n;
     if (n == 0) continue;                                   // rows that see nothing
     groups = pl_groups<A>(x.pl, G);
     wait_lead(bar(ct.q_full), item++ & 1u, lead, dead);
     if constexpr (PAIR) {
       for (int g = 0; g < min(n, 2) && !dead; ++g) {
         wait_lead(bar(ct.k_full[kst]), kph, lead, dead);
         fence_after();
         if (!dead) scores(g);
       }
#pragma unroll 1
       for (int t = 0; t < n && !dead; ++t) {
         const int g = t & 1;
         wait_lead(bar(ct.v_full[vst]), vph, lead, dead);
#pragma unroll
         for (int half = 1; half >= 0; --half) {
           wait_lead(bar(ct.p_half[g][half]), (done[g] + (t >> 1)) & 1u, lead, dead);
           if (dead) break;
           fence_after();
           const uint64_t vd = desc_mn(sv + vst * va * TC_ATOM + half * (TC_ATOM / 2), TC_ATOM);
#pragma unroll
           for (int k = 0; k < 4; ++k) mma_ts(tmem + 256 + 128 * g, tmem + 128 * g + 64 * half + 8 * k, vd + k * (16 * 128 / 16), id_o, t < 2 && half == 1 && k == 0 ? 0u : 1u, lead);
         }
         if (dead) break;
         commit_by(lead, bar(ct.v_empty[vst]));
         if (t + 2 < n) {
           wait_lead(bar(ct.k_full[kst]), kph, lead, dead);
           if (dead) break;
           fence_after();
           scores(g);
         } else {
           commit_by(lead, bar(ct.o_done[g]));
         }
         if (++vst == v_stages) { vst = 0; vph ^= 1u; }
       }
       done[0] += (n + 1) >> 1;
       done[1] += n >> 1;
       continue;
     }
     wait_lead(bar(ct.k_full[kst]), kph, lead, dead);
     fence_after();
     for (int g = 0; g < groups && !dead; ++g) scores(g);
     for (int t = 0; t < n && !dead; ++t) {
      wait_lead(bar(ct.v_full[vst]), vph, lead, dead);
#pragma unroll 1
      for (int g = 0; g < groups; ++g) {
#pragma unroll
        for (int half = 1; half >= 0; --half) {
          wait_lead(bar(ct.p_half[g][half]), (done[g] + t) & 1u, lead, dead);
          if (dead) break;
          fence_after();
          const uint64_t vd = desc_mn(sv + vst * va * TC_ATOM + half * (TC_ATOM / 2), TC_ATOM);
#pragma unroll
          for (int k = 0; k < 4; ++k) mma_ts(tmem + 256 + 128 * g, tmem + 128 * g + 64 * half + 8 * k, vd + k * (16 * 128 / 16), id_o, t == 0 && half == 1 && k == 0 ? 0u : 1u, lead);
        }
        if (dead) break;
        if (g == groups - 1) commit_by(lead, bar(ct.v_empty[vst]));
        if (t + 1 < n) {
          if (g == 0) wait_lead(bar(ct.k_full[kst]), kph, lead, dead);
          if (dead) break;
          fence_after();
          scores(g);
        } else {
          commit_by(lead, bar(ct.o_done[g]));
        }
      }
      if (++vst == v_stages) { vst = 0; vph ^= 1u; }
     }
     done[0] += n;
     if (groups > 1) done[1] += n;
    }
    if (dead) {                                              // what was issued ends before tensor memory is given back
      uint32_t late = 0;
      commit_by(lead, bar(ct.gave_up));
      wait_for(bar(ct.gave_up), 0, late);
    }
    __syncwarp();
   } else if (warp == 1 || (TREE && warp == 3)) {
    // ===================== tiled copies =====================
    // TREE: keys by warp 1, values by warp 3.  One warp for both asks for the keys of a tile when the place of values before it is free, which is late where nearly all of
    // the time is that of copies: 37 trees of 32 tokens over 4096 keys, bf16, 125 us so, 120 apart
    const bool keys_here = warp == 1, values_here = !TREE || warp == 3;
    const int box = min(1 << a.s.shift, KEYS), boxes = KEYS / box, gone = (a.s.pages * a.kv_heads) << a.s.shift;      // a row beyond the pool: zeros
    int kst = 0, vst = 0;
    uint32_t kph = 1, vph = 1, tail_waits = 0, tile = 0;     // a stage is free at first; 8-bit pools: stages of codes
    while (!dead && next(a, ct, warp, lane, x)) {
     const Keys keys = a.keys(x.pl, ROWS);
     const int h = x.h, sequence = x.pl.b;
     for (int t = x.t0; t < x.t1; ++t, ++tile) {
      const int key0 = keys.key0(t, 7);
      int page = -1;
      if (lane < boxes && key0 + lane * box < keys.end) page = page_of(a.s, sequence, key0 + lane * box);
      const uint32_t seen = __ballot_sync(0xffffffffu, page >= 0);
      const int row = page >= 0 ? ((page * a.kv_heads + h) << a.s.shift) + ((key0 + lane * box) & ((1 << a.s.shift) - 1)) : gone;
      uint32_t there = 0;                                    // by 16 keys
      for (int i = 0; i < 8; ++i) there |= (seen >> (i * 16 / box) & 1u) << i;
      const int b = lane & (boxes - 1), x = lane / boxes, r = __shfl_sync(0xffffffffu, row, b);      // a lane per box, 24 at most
      if (keys_here) {
        const uint32_t k_to = bar(HALF ? ct.rk_full[kst] : ct.k_full[kst]);
        wait_warp(bar(HALF ? ct.rk_empty[kst] : ct.k_empty[kst]), kph, dead);
        if (dead) break;
        if (lane == 0) {
          notes_of[tile % NOTES].there = there;
          mbar_arrive(bar(ct.info_full[tile % NOTES]));
          mbar_expect_tx(k_to, HALF ? KEYS * (a.K + 8) : ka * TC_ATOM);
        }
        __syncwarp();                                        // the bytes are expected before they come
        // one lane after the other took 100 ns for each box, with pages of 16 tokens 3.1 us for a tile
        if (x < (HALF ? 3 : ka)) {
          if (HALF) {
            const int at = r < gone ? r : 0;                 // of a page that is not there: any scales, which nobody takes
            if (x == 0) tma_load_2d(raw_k + kst * KEYS * a.K + b * box * a.K, &map_k, 0, r, k_to);
            else bulk(smem_u32((x == 1 ? scales_of[kst].k : scales_of[kst].v) + b * box), (x == 1 ? a.ks : a.vs) + at, 4 * box, k_to);
          } else {
            tma_load_2d(sk + (kst * ka + x) * TC_ATOM + b * box * 128, &map_k, 64 * x, r, k_to);
          }
        }
        __syncwarp();
        if (++kst == (HALF ? raw_ks : k_stages)) { kst = 0; kph ^= 1u; }
      }
      if (!values_here) continue;
      wait_warp(bar(HALF ? ct.rv_empty[vst] : ct.v_empty[vst]), vph, dead);
      if (dead) break;
      const int valid = keys.end - key0;
      // bf16: behind the last key that is seen the page may hold anything, and a weight of zero does not hide an infinity: zeros there
      const bool cut = !HALF && valid < KEYS;
      const uint32_t v_to = bar(HALF ? ct.rv_full[vst] : cut ? ct.tail : ct.v_full[vst]);
      if (lane == 0) mbar_expect_tx(v_to, HALF ? KEYS * a.V : va * TC_ATOM);
      __syncwarp();
      if (x < (HALF ? 1 : va)) {
        if (HALF) tma_load_2d(raw_v + vst * KEYS * a.V + b * box * a.V, &map_v, 0, r, v_to);
        else tma_load_2d(sv + (vst * va + x) * TC_ATOM + b * box * 128, &map_v, 64 * x, r, v_to);
      }
      __syncwarp();
      if (cut) {
        wait_warp(v_to, tail_waits++ & 1u, dead);
        if (dead) break;
        for (int x = lane; x < (KEYS - valid) * 8 * va; x += 32) st128(sv + vst * va * TC_ATOM + piece_at(valid + x / (8 * va), x % (8 * va)), make_uint4(0, 0, 0, 0));
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(ct.v_full[vst]));
      }
      if (++vst == (HALF ? raw_vs : v_stages)) { vst = 0; vph ^= 1u; }
     }
    }
    // every copy has landed before the CTA ends: what reads them comes after, unless a wait ran out
    if (dead) {
      uint32_t late = 0;
      for (int i = 0; i < (HALF ? raw_ks : k_stages) && keys_here; ++i) wait_for(bar(HALF ? ct.rk_full[i] : ct.k_full[i]), i < kst ? kph ^ 1u : kph, late);
      late = 0;
      for (int i = 0; i < (HALF ? raw_vs : v_stages) && values_here; ++i) wait_for(bar(HALF ? ct.rv_full[i] : ct.v_full[i]), i < vst ? vph ^ 1u : vph, late);
    }
    __syncwarp();
   } else if (warp == 2) {
    // ===================== the row tile that goes on in the next CTAs =====================
    int4 last = make_int4(0, 0, 0, 0);
    Walk w = ct.at[warp];
    const long long x0 = ct.x0, x1 = ct.x1;
    while (w.pl.n > 0 && w.at < x1) {
      const Cost c = cost_of(a, w.pl);
      if (c.cut(x0 - w.at) == 0 && c.cut(x1 - w.at) > 0 && c.cut(x1 - w.at) < c.units) {
        int parts = 1;
        while (c.cut((blockIdx.x + parts) * (x1 - x0) - w.at) < c.units) ++parts;      // x1 - x0 is a whole share: this CTA is not the last one
        last = make_int4(w.pl.b, w.pl.first, w.h, parts);
      }
      advance(a, w, c, lane);
    }
    if (lane == 0) a.many.last[blockIdx.x] = last;
   }
  } else if (warp >= 12) {
    // ===================== 8-bit codes to f16 =====================
    if constexpr (HALF) {
      asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
      const bool keys_too = warp < 16;                       // warps 12 .. 15: the factors of keys and values, and the keys; 16 .. 19: the values
      const int me = tid & 127;
      int st = 0, ref = 0, raw = 0;
      uint32_t ph = 1, tile = 0, item = 0, raw_ph = 0;
      float k_up = 1.f, v_up = 1.f;
      // the factor in two f16, twice each: as precise as 22 bits, or steps of 2^-25 (2^-13 of a factor of 2^-12); NaN where the scale is out of range; 0 for a row of
      // zeros (2^-126) or one never written (0)
      constexpr uint32_t NO = 0x7e007e00u;
      auto factor = [](bool valid, float scale, float up, uint32_t which, uint32_t& low) {
        const float s = scale * up;
        const bool zero = !valid || (scale >= 0.f && scale <= 1.17549435e-38f), good = s >= 0.f && s <= 128.f;
        if (!zero && good && s < 2.44140625e-4f) low |= which;
        const __half hi = __float2half_rn(s), lo = __float2half_rn(s - __half2float(hi));
        return make_uint2(zero ? 0u : good ? __half_as_ushort(hi) * 0x10001u : NO, zero ? 0u : good ? __half_as_ushort(lo) * 0x10001u : NO);
      };
      // PAIR: by a lane of each warp, and waits for three barriers at once (37 trees of 32 tokens over 4096 keys, int8: 154 us so, 157 by all threads and one after the other)
      auto arrive = [&](uint64_t& b) {
        if (!PAIR || lane == 0) mbar_arrive(bar(b));
      };
      while (!dead && next(a, ct, warp, lane, x)) {
       const Keys keys = a.keys(x.pl, ROWS);
       for (int t = x.t0; t < x.t1; ++t, ++tile) {
        Info& info = infos[tile % INFOS];
        Note& note = notes_of[tile % NOTES];
        if (keys_too) {
          wait_warp(bar(ct.rk_full[raw]), raw_ph, dead);
          if (dead) break;
          const float ks = scales_of[raw].k[me], vs = scales_of[raw].v[me];
          // A key that some row sees: behind the last one and before the windows there may be anything, and of a page that is not there the scales are those of
          // another place (`there` was written before the copies were asked for)
          const int j = keys.key0(t, 7) + me;
          const bool valid = j < keys.end && (j >= keys.lo || j < keys.early) && (*reinterpret_cast<volatile uint32_t*>(&note.there) >> (me / 16) & 1u);
          if (t == x.t0) {
            if (valid && ks >= SMALLEST_SCALE && ks <= 1.f / SMALLEST_SCALE) atomicMax(&ct.k_ref[ref], __float_as_uint(ks));
            if (valid && vs >= SMALLEST_SCALE && vs <= 1.f / SMALLEST_SCALE) atomicMax(&ct.v_ref[ref], __float_as_uint(vs));
            mbar_arrive(bar(ct.ref_full));
            wait_warp(bar(ct.ref_full), item++ & 1u, dead);
            if (dead) break;
            k_up = value_lift(*reinterpret_cast<volatile uint32_t*>(&ct.k_ref[ref]));
            v_up = value_lift(*reinterpret_cast<volatile uint32_t*>(&ct.v_ref[ref]));
            if (me == 0) ct.k_ref[ref == 0 ? 2 : ref - 1] = ct.v_ref[ref == 0 ? 2 : ref - 1] = 0u;      // the ones before, which all have read: for the ones after the next
            ref = ref == 2 ? 0 : ref + 1;
          }
          uint32_t low = 0u;
          uint2 k_by = factor(valid, ks, k_up, 256u, low), v_by = factor(valid, vs, v_up, 512u, low);
          if (low) atomicOr(&note.there, low);
          if (v_by.x == NO) {                                // a row that sees this key is computed again: its scores say so
            k_by = v_by;
            v_by = make_uint2(0u, 0u);
          }
          wait_warp(bar(ct.k_empty[st]), ph, dead);
          if (dead) break;
          info.k_by[me] = k_by;
          info.v_by[me] = v_by;
          if (me == 0) {
            note.k_up = k_up;
            note.v_up = v_up;
          }
          if (PAIR) __syncwarp();
          arrive(ct.info_full[tile % NOTES]);
        } else if (!PAIR) {
          wait_warp(bar(ct.rv_full[raw]), raw_ph, dead);
          wait_warp(bar(ct.v_empty[st]), ph, dead);
        }
        // all keys' factors
        const uint32_t info_full = bar(ct.info_full[tile % NOTES]), info_ph = tile / NOTES & 1u;
        if (!PAIR || keys_too) wait_warp(info_full, info_ph, dead);
        else wait_three(lane == 0 ? info_full : lane == 1 ? bar(ct.rv_full[raw]) : bar(ct.v_empty[st]), lane == 0 ? info_ph : lane == 1 ? raw_ph : ph, lane, dead);
        if (dead) break;
        if constexpr (PAIR) {
          codes_to_f16<STORE, true, 1>(keys_too ? raw_k + raw * KEYS * a.K : raw_v + raw * KEYS * a.V, keys_too ? a.K : a.V, keys_too ? info.k_by : info.v_by,
                                       keys_too ? sk + st * ka * TC_ATOM : sv + st * va * TC_ATOM, me, 128);
        } else {
          if (keys_too) codes_to_f16<STORE, false, 2>(raw_k + raw * KEYS * a.K, a.K, info.k_by, sk + st * ka * TC_ATOM, me, 128);
          else codes_to_f16<STORE, true, 2>(raw_v + raw * KEYS * a.V, a.V, info.v_by, sv + st * va * TC_ATOM, me, 128);
        }
        if (PAIR) __syncwarp();
        arrive(keys_too ? ct.k_full[st] : ct.v_full[st]);
        arrive(keys_too ? ct.rk_empty[raw] : ct.rv_empty[raw]);
        if (++raw == (keys_too ? raw_ks : raw_vs)) { raw = 0; raw_ph ^= 1u; }
        if (++st == (keys_too ? k_stages : v_stages)) { st = 0; ph ^= 1u; }
       }
      }
    }
  } else {
    if constexpr (HALF) asm volatile("setmaxnreg.inc.sync.aligned.u32 144;");
    // ===================== queries, softmax, outputs =====================
    const int g = (warp - 4) >> 2, r = (warp & 3) * 32 + lane;
    const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16), S = lanes + 128 * g, O = lanes + 256 + 128 * g;
    uint32_t tile = 0, mine = 0, item = 0, own_items = 0;    // tiles of keys, those of this half; row tiles with keys, those of this half
    while (next(a, ct, warp, lane, x)) {
    const Place pl = x.pl;
    const int n = x.n, t0 = x.t0, rows = min(ROWS, pl.n * G - pl.first), groups = pl_groups<A>(pl, G);
    const int in_tile = (PAIR ? 0 : TILE * g) + r, at = pl.first + in_tile;
    const bool part = !x.whole, live = in_tile < rows;
    const int token = live ? at / G : 0, head = x.h * G + (live ? at % G : 0), row = pl.start + token, base = pl.length - pl.n, pos = live ? a.position(pl.start, base, pl.n, token) : -1;
    const Keys keys = a.keys(pl, ROWS);
    float cr = a.scale_log2;
    const uint32_t told = telling + 4 * r;                   // PAIR: the second half's maxima, sums and notes; factors of the scores
    if (n > 0) {
     if (g < groups) {
      // The warp's 32 rows, neighbouring lanes along a row: with a row per lane the load unit was busy with 32 lines for every instruction, 5400 cycles.  A
      // small loop, as code that runs once is fetched at some 12 cycles an instruction; a row's lane knows where it is
      const int pieces = a.K / 8, by = 65536 / pieces + 1;   // x / pieces = x by >> 16 for x < 32 pieces, pieces <= 24
      const uint32_t own = sq + g * ka * TC_ATOM;
      const unsigned long long from = reinterpret_cast<unsigned long long>(reinterpret_cast<const __nv_bfloat16*>(a.q) + (size_t)row * a.ldq + (size_t)head * a.hsq);
#pragma unroll 2
      for (int x = lane; x < 32 * pieces; x += 32) {
        const int k = x * by >> 16, c = x - k * pieces;
        const unsigned long long src = __shfl_sync(0xffffffffu, from, k);
        atc::cp16(own + piece_at((warp & 3) * 32 + k, c), reinterpret_cast<const void*>(src + 16 * c), TILE * g + (warp & 3) * 32 + k < rows);
      }
      asm volatile("cp.async.wait_all;" ::: "memory");
      if (HALF) {                                            // then a lane has a row: its largest entry, and the row as f16
        __syncwarp();
        uint32_t top2 = 0u;                                  // of two entries' absolute values, as bits: as large as their values are
        for (int c = 0; c < pieces; ++c) {
          const uint4 w = ld128(own + piece_at(r, c));
          top2 = __vmaxu2(__vmaxu2(__vmaxu2(top2, w.x & 0x7fff7fffu), __vmaxu2(w.y & 0x7fff7fffu, w.z & 0x7fff7fffu)), w.w & 0x7fff7fffu);
        }
        float up;
        lift_of(fmaxf(__uint_as_float(top2 << 16), __uint_as_float(top2 & 0xffff0000u)), a.scale_log2, up, cr);
        for (int c = 0; c < pieces; ++c) {
          const uint4 w = ld128(own + piece_at(r, c));
          uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const __half2 f = __floats2half2_rn(__uint_as_float(u[e] << 16) * up, __uint_as_float(u[e] & 0xffff0000u) * up);
            u[e] = *reinterpret_cast<const uint32_t*>(&f);
          }
          st128(own + piece_at(r, c), make_uint4(u[0], u[1], u[2], u[3]));
        }
        if (PAIR) asm volatile("st.shared.f32 [%0+1536], %1;" ::"r"(told), "f"(cr) : "memory");
      }
      fence_proxy_async();
     }
     // A warp whose wait ran out (rows that others compute again, key by key, can take longer) says nothing any more: it no longer keeps pace, and arrivals of
     // its later row tiles would stand for those of a warp that still has to come, whose queries were then multiplied before they are there
     if (!dead) mbar_arrive(bar(ct.q_full));
    }
    float m = -INFINITY, l = 0.f, down = 1.f;
    uint32_t notes = 0;                                      // those of its tiles; bit 31: a score that is NaN or an infinity
    // positions of this group's rows: where all of them see a tile no mask is needed
    const int p_min = TREE ? keys.p_min : pl.length - pl.n + (pl.first + TILE * g) / G, p_max = TREE ? keys.p_max : pl.length - pl.n + (pl.first + min(TILE * (g + 1), rows) - 1) / G;
    int taken = 0;                                           // tiles of keys of this half
    if (PAIR || g < groups) {
      const bool idle = !__any_sync(0xffffffffu, live);
      for (int t = PAIR ? g : 0; t < n; t += PAIR ? 2 : 1, ++taken) {
        const int key0 = keys.key0(t0 + t, 7);
        wait_for(bar(ct.info_full[(tile + t) % NOTES]), (tile + t) / NOTES & 1u, dead);
        wait_warp(bar(ct.s_full[g]), (mine + taken) & 1u, dead);
        if (dead) break;
        if (idle) {                                          // no row: whatever the weights are
          if (lane < 2) mbar_arrive(bar(ct.p_half[g][lane]));
          continue;
        }
        fence_after();
        const Note& note = notes_of[(tile + t) % NOTES];
        const uint32_t there = note.there;
        if (HALF && taken == 0) {
          if (PAIR && g > 0) asm volatile("ld.shared.f32 %0, [%1+1536];" : "=f"(cr) : "r"(told) : "memory");      // there since these scores are
          cr *= 1.f / note.k_up;
          down = 1.f / note.v_up;
        }
        if (HALF) notes |= there;
        const bool whole = (there & 0xffu) == 0xffu && key0 + KEYS - 1 <= p_min && (a.window == 0 || key0 > p_max - a.window || key0 + KEYS <= a.first);
        // keys that the row sees, as bits of 32
        auto seen = [&](int c) {
          const int j = key0 + 32 * c;
          const uint32_t x = live || !TREE ? a.seen32(pos, row, base, pl.n, j) : 0u;
          return x & (((there >> 2 * c & 1u) ? 0xffffu : 0u) | ((there >> (2 * c + 1) & 1u) ? 0xffff0000u : 0u));
        };
        // scores of keys 64 half .. + 63: hidden ones -inf
        auto finish = [&](int half, uint32_t* u) {
          if (!whole) {
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              const uint32_t mask = seen(2 * half + c);
#pragma unroll
              for (int i = 0; i < 32; ++i) u[32 * c + i] = mask >> i & 1u ? u[32 * c + i] : 0xff800000u;
            }
          }
        };
        // the second half's stay in registers from the maximum to the weights, the first is read twice: all 128 in registers took 3% longer
        uint32_t u[KEYS / 2];
        float x4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          tmem_ld64(S + 64 * half, u);
          tmem_wait_ld64(u);
          finish(half, u);
#pragma unroll
          for (int i = 0; i < 64; i += 2) x4[i / 2 & 3] = max3(x4[i / 2 & 3], __uint_as_float(u[i]), __uint_as_float(u[i + 1]));
        }
        const float top = max3(max3(x4[0], x4[1], x4[2]), x4[3], -INFINITY) * cr;
        if (!(top < INFINITY)) notes |= 1u << 31;            // the row is computed again
        const bool grows = top > m + 8.f || (m == -INFINITY && top > m);
        if (__any_sync(0xffffffffu, grows)) {
          const float f = grows ? exp2_f(m - top) : 1.f;     // 0 where nothing was added yet
          if (grows) m = top;
          l *= f;
          if (taken > 0) {                                   // these scores came after the product of this half's tile before
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
#pragma unroll
        for (int half = 1; half >= 0; --half) {              // the second half first, over its own scores
          if (half == 0) {
            tmem_ld64(S, u);
            tmem_wait_ld64(u);
            finish(0, u);
          }
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            uint32_t w[16];
#pragma unroll
            for (int i = 0; i < 32; i += 2) {
              float x = __uint_as_float(u[32 * c + i]), y = __uint_as_float(u[32 * c + i + 1]);
              fma2(x, y, cr, -ref, -ref);
              if (!HALF && i % 8 == 6) {
                exp2_poly2(x, y);
              } else {
                x = exp2_f(x);
                y = exp2_f(y);
              }
              add2(sum[0], sum[1], x, y);
              if (HALF) {
                const __half2 p = __floats2half2_rn(x, y);
                w[i / 2] = *reinterpret_cast<const uint32_t*>(&p);
              } else {
                const __nv_bfloat162 p = __floats2bfloat162_rn(x, y);
                w[i / 2] = *reinterpret_cast<const uint32_t*>(&p);
              }
            }
            tmem_st16(S + 64 * half + 16 * c, w);
          }
          tmem_wait_st();
          fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(bar(ct.p_half[g][half]));
        }
        l += sum[0] + sum[1];
      }
      const int tiles = PAIR ? (n + 1 - g) >> 1 : n;         // (taken, if no wait ran out)
      if (tiles > 0) wait_warp(bar(ct.o_done[g]), own_items & 1u, dead);
      fence_after();
      if (dead || notes >> 31) l = NAN;
      float f0 = 1.f, f1 = 0.f;                              // of the halves' outputs
      if (PAIR && n > 0) {
        if (g > 0) asm volatile("st.shared.f32 [%0], %1;\n\tst.shared.f32 [%0+512], %2;\n\tst.shared.b32 [%0+1024], %3;" ::"r"(told), "f"(m), "f"(l), "r"(notes) : "memory");
        fence_before();
        both_halves();
        fence_after();
        if (g == 0) {
          float m1, l1;
          uint32_t notes1;
          asm volatile("ld.shared.f32 %0, [%3];\n\tld.shared.f32 %1, [%3+512];\n\tld.shared.b32 %2, [%3+1024];" : "=f"(m1), "=f"(l1), "=r"(notes1) : "r"(told) : "memory");
          const float M = fmaxf(m, m1);
          f0 = m == M ? 1.f : exp2_f(m - M);
          f1 = n < 2 ? 0.f : m1 == M ? 1.f : exp2_f(m1 - M);
          l = l * f0 + (n < 2 ? 0.f : l1 * f1);
          m = M;
          notes |= notes1;
        }
        both_halves();                                       // read before what comes next there
      }
      if (!PAIR || g == 0) {
      const float inv = part ? down : l == 0.f ? 0.f : down / l;
      float peak = 0.f;                                      // the row's largest output, NaN if one is
      const int slot = 2 * (int)blockIdx.x + (t0 == 0 ? 1 : 0), place = !live ? -1 : part ? slot * ROWS + in_tile : row * a.heads + head;      // of the row's outputs
      // Outputs through the warp's rows of the queries (every score of this row tile is done), 128 bytes of each row at a time; then eight lanes along a row (a
      // row per lane took 9500 cycles)
      const int per = part ? 32 : 64;                        // columns
#pragma unroll 1
      for (int c0 = 0; c0 < a.V; c0 += per) {
#pragma unroll 1
        for (int c = c0; c < min(c0 + per, a.V); c += 16) {
          uint32_t o[16];
          if (n > 0 && !dead) tmem_ld16(O + c, o);
          float x[16];
          if (PAIR && n > 1 && !dead) {
            uint32_t o1[16];
            tmem_ld16(O + 128 + c, o1);
#pragma unroll
            for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(fmaf(__uint_as_float(o1[i]), f1, __uint_as_float(o[i]) * f0));
          }
#pragma unroll
          for (int i = 0; i < 16; ++i) x[i] = dead ? NAN : n > 0 ? __uint_as_float(o[i]) * inv : 0.f;
#pragma unroll
          for (int i = 0; i < 16; i += 2) peak = max3(peak, fabsf(x[i]), fabsf(x[i + 1]));
          if (part) {
#pragma unroll
            for (int i = 0; i < 16; i += 4)
              st128(sq + g * ka * TC_ATOM + piece_at(r, (c - c0 + i) / 4), make_uint4(__float_as_uint(x[i]), __float_as_uint(x[i + 1]), __float_as_uint(x[i + 2]), __float_as_uint(x[i + 3])));
          } else {
#pragma unroll
            for (int i = 0; i < 16; i += 8) {
              uint32_t w[4];
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const __nv_bfloat162 y = __floats2bfloat162_rn(x[i + 2 * e], x[i + 2 * e + 1]);
                w[e] = *reinterpret_cast<const uint32_t*>(&y);
              }
              st128(sq + g * ka * TC_ATOM + piece_at(r, (c - c0 + i) / 8), make_uint4(w[0], w[1], w[2], w[3]));
            }
          }
        }
        __syncwarp();
        const int c = lane & 7, column = c0 + c * (per / 8); // this lane's 16 bytes
#pragma unroll 2
        for (int k = lane >> 3; k < 32; k += 4) {
          const int there = __shfl_sync(0xffffffffu, place, k);
          if (there >= 0 && column < a.V) {
            const uint4 y = ld128(sq + g * ka * TC_ATOM + piece_at((warp & 3) * 32 + k, c));
            if (part) *reinterpret_cast<uint4*>(a.many.o + (size_t)there * a.V + column) = y;
            else *reinterpret_cast<uint4*>(reinterpret_cast<__nv_bfloat16*>(a.out) + (size_t)there * a.V + column) = y;
          }
        }
        __syncwarp();
      }
      if constexpr (HALF) {
        constexpr float LARGEST = STORE == E4M3 ? 448.f : 127.f;
        if (notes > 255u && l > 0.f && (((notes & 256u) && cr * (float)a.K * LARGEST > 1.f) || ((notes & 512u) && !(peak >= LARGEST * 1.220703125e-4f * down * (part ? l : 1.f))))) l = NAN;
      }
      if (part) *reinterpret_cast<float2*>(a.many.ml + 2 * (slot * ROWS + in_tile)) = make_float2(m, l);
      if (!part) {
        __syncwarp();
        const uint32_t bad = __ballot_sync(0xffffffffu, live && !(peak < INFINITY && fabsf(l) < INFINITY));
        if (bad) mend_rows<2>(a, pl.b, pl.start, pl.length - pl.n, x.h, pl.first + TILE * g + (warp & 3) * 32, bad, lane);
      }
      }
    }
    if (n > 0) {
      // both halves keep to the same row tile: its products are over before the next one's queries are said to be there
      if (g > 0) wait_warp(bar(ct.o_done[0]), item & 1u, dead);
      ++item;
      tile += n;
      const int tiles = PAIR ? (n + 1 - g) >> 1 : g < groups ? n : 0;
      mine += tiles;
      own_items += tiles > 0;
    }
    }
  }
  fence_before();
  __syncthreads();
  if (warp == 0) tmem_dealloc(tmem, 512);
}

// The row tiles that go on from CTA blockIdx.x to others; a warp has JOINED rows, a lane four columns of each.  Parts are read four at a time: one after the other ten of
// a tile took 18.7 us for 16 tiles.
constexpr int JOINED = 2, JOIN_AHEAD = 4;
template <class A> __global__ void __launch_bounds__(256) paged_join_kernel(const __grid_constant__ A a) {
  constexpr int ROWS = A::ROWS;
  const int lane = threadIdx.x & 31, G = a.heads / a.kv_heads, r0 = blockIdx.y * 8 * JOINED + threadIdx.x / 32 * JOINED;
  pdl_wait();                                                // launched as the last CTAs that compute parts end: they let nothing in earlier
  const int4 last = a.many.last[blockIdx.x];
  if (last.w < 2) return;
  int start, n, length;
  sequence(a.s, last.x, start, n, length);
  const int rows = min(ROWS, n * G - last.y);
  if (r0 >= rows) return;
  float M[JOINED], L[JOINED];
  float4 x[JOINED];
#pragma unroll
  for (int k = 0; k < JOINED; ++k) {
    M[k] = -INFINITY;
    L[k] = 0.f;
    x[k] = make_float4(0.f, 0.f, 0.f, 0.f);
  }
  for (int i0 = 0; i0 < last.w; i0 += JOIN_AHEAD) {
    float2 ml[JOIN_AHEAD][JOINED];
    float4 z[JOIN_AHEAD][JOINED];
#pragma unroll
    for (int e = 0; e < JOIN_AHEAD; ++e) {
      const int i = i0 + e, at = (i == 0 ? 2 * (int)blockIdx.x + 1 : 2 * ((int)blockIdx.x + i)) * ROWS + r0;
#pragma unroll
      for (int k = 0; k < JOINED; ++k) {
        ml[e][k] = make_float2(-INFINITY, 0.f);
        z[e][k] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (i < last.w && r0 + k < rows) {
          ml[e][k] = *reinterpret_cast<const float2*>(a.many.ml + 2 * (at + k));
          if (4 * lane < a.V) z[e][k] = *reinterpret_cast<const float4*>(a.many.o + (size_t)(at + k) * a.V + 4 * lane);
        }
      }
    }
#pragma unroll
    for (int e = 0; e < JOIN_AHEAD; ++e)
#pragma unroll
      for (int k = 0; k < JOINED; ++k) {
        if (ml[e][k].x == -INFINITY && ml[e][k].y == 0.f) continue;      // saw nothing
        const float now = fmaxf(M[k], ml[e][k].x), f = M[k] == now ? 1.f : exp2_f(M[k] - now), w = ml[e][k].x == now ? 1.f : exp2_f(ml[e][k].x - now);
        M[k] = now;
        L[k] = L[k] * f + w * ml[e][k].y;
        x[k] = make_float4(x[k].x * f + w * z[e][k].x, x[k].y * f + w * z[e][k].y, x[k].z * f + w * z[e][k].z, x[k].w * f + w * z[e][k].w);
      }
  }
  uint32_t bad = 0u;
#pragma unroll
  for (int k = 0; k < JOINED; ++k) {
    if (r0 + k >= rows) break;
    const int at = last.y + r0 + k, row = start + at / G, head = last.z * G + at % G;
    const float inv = L[k] == 0.f ? 0.f : 1.f / L[k], y[4] = {x[k].x, x[k].y, x[k].z, x[k].w};
    if (4 * lane < a.V) a.store(((size_t)row * a.heads + head) * a.V + 4 * lane, y, inv);
    if (!__all_sync(0xffffffffu, finite4(y, inv) && fabsf(L[k]) < INFINITY)) bad |= 1u << k;
  }
  __syncwarp();
  if (bad) mend_rows<2>(a, last.x, start, length - n, last.z, last.y + r0, bad, lane);
}

int many_ctas(bool pair, long long packed, long long tiles, int kv_heads, long long keys, int sms) {
  const long long row_tiles = (packed / (pair ? TILE : 2 * TILE) + tiles) * kv_heads, cost = row_tiles * (EXTRA + (pair ? 2 : 4) * ((keys + KEYS - 1) / KEYS + 2));
  return (int)std::max<long long>(1, std::min<long long>(sms, cost / (pair ? LEAST_SHARE<true> : LEAST_SHARE<false>)));
}
long long many_floats(bool pair, int ctas, int V) { return 4ll * ctas + 2ll * ctas * (pair ? TILE : 2 * TILE) * (2 + V); }

bool many_takes(int K, int V, int store) {
  if (K > MOST_K || V > MOST_V) return false;
  return (store == ACT ? layout<ACT, false>(K, V) : layout<INT8, false>(K, V)).ks > 0;
}
bool pair_takes(int K, int V, int store) { return (store == ACT ? layout<ACT, true>(K, V) : layout<INT8, true>(K, V)).ks > 0; }

// Rows of `cols` bytes (a multiple of 16, up to 256), whole ones, as they lie
static int map_rows(CUtensorMap* m, const void* base, long long rows, int cols, int box_rows) {
  EncodeFn fn = encoder();
  if (fn == nullptr) {
    set_error("cuTensorMapEncodeTiled is not available from this driver");
    return B2L_E_STATE;
  }
  const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)cols};
  const cuuint32_t box[2] = {(cuuint32_t)cols, (cuuint32_t)box_rows}, estr[2] = {1, 1};
  const CUresult cr = fn(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE,
                         CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (cr != CUDA_SUCCESS) {
    set_error("cuTensorMapEncodeTiled failed (%d) for %lld x %d", (int)cr, rows, cols);
    return B2L_E_ARG;
  }
  return 0;
}

template <int STORE, class A> static int go(const A& a, int ctas, cudaStream_t stream) {
  const Layout l = layout<STORE, A::PAIR, A::TREE>(a.K, a.V);
  CUtensorMap mk, mv;
  const long long rows = ((long long)a.s.pages * a.kv_heads) << a.s.shift;
  const int box = 1 << a.s.shift < KEYS ? 1 << a.s.shift : KEYS;
  if (STORE == ACT) {
    if (int rc = map_sw128(&mk, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, a.k, rows, a.K, a.K, 64, box)) return rc;
    if (int rc = map_sw128(&mv, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, a.v, rows, a.V, a.V, 64, box)) return rc;
  } else {
    if (int rc = map_rows(&mk, a.k, rows, a.K, box)) return rc;
    if (int rc = map_rows(&mv, a.v, rows, a.V, box)) return rc;
  }
  static DynSmemCache cache;
  if (int rc = ensure_dyn_smem(paged_many_kernel<STORE, A>, l.smem, cache)) return rc;
  paged_many_kernel<STORE, A><<<(unsigned)ctas, THREADS<STORE>, l.smem, stream>>>(a, mk, mv, l.ks, l.vs, l.raw_ks, l.raw_vs);
  B2L_LAUNCH_CHECK("paged_many_kernel");
  return 0;
}
template <class A> static int launch(A& a, int ctas, float* work, cudaStream_t stream) {
  a.many.last = reinterpret_cast<int4*>(work);
  a.many.ml = work + 4 * ctas;
  a.many.o = a.many.ml + 4ll * ctas * A::ROWS;
  const int rc = a.store_kind == ACT ? go<ACT>(a, ctas, stream) : a.store_kind == E4M3 ? go<E4M3>(a, ctas, stream) : go<INT8>(a, ctas, stream);
  if (rc || ctas == 1) return rc;
  LaunchCfg cfg(dim3((unsigned)ctas, A::ROWS / (8 * JOINED)), dim3(256), 0, stream, true);
  B2L_CUDA(cudaLaunchKernelEx(&cfg.cfg, paged_join_kernel<A>, a));
  B2L_LAUNCH_CHECK("paged_join_kernel");
  return 0;
}
template <bool TREE> int many_launch(const Attn<TREE>& a, bool pair, int ctas, float* work, cudaStream_t stream) {
  if constexpr (TREE) {
    if (pair) {
      Tiles<true, true> x{a};
      return launch(x, ctas, work, stream);
    }
  }
  Tiles<TREE, false> x{a};
  return launch(x, ctas, work, stream);
}
template int many_launch<false>(const Attn<false>&, bool, int, float*, cudaStream_t);
template int many_launch<true>(const Attn<true>&, bool, int, float*, cudaStream_t);

}  // namespace paged
}  // namespace b2l
