// What the tensor-core attention kernels share: tensor maps, tcgen05 wrappers, the walk over key tiles, the scores.
//
// Operands reach shared memory as tiles of 128 rows by TMA, in blocks of 64 columns (128-byte rows, 128-byte swizzle; head
// dimensions are filled up to 64 or 128 with zeros by the copy itself).  Such a tile serves tcgen05.mma in two ways:
// K-major, where the product runs along d (scores), and MN-major, where it runs along the rows (weights times rows).  The
// weights are the A operand of the second kind and never leave tensor memory: a thread owns one row (TMEM lane) of a score
// tile, reads it, and writes the 16-bit weights back over it.
//
// Heads that share a key head are packed into the rows of one tile where their number is a power of two: packed row r is
// query r / pg of head r % pg.  A key tile then meets pg times as many rows, and the triangle of a causal mask is cut in
// steps pg times as fine.
//
// Every wait on a barrier is bounded; when one gives up, the block records it, stops issuing work, lets its copies land and its
// products end, makes the rows that it cannot finish NaN, frees its tensor memory and returns.
#pragma once

#include <cuda.h>
#include <string.h>

#include <type_traits>

#include "flk_attn.cuh"
#include "flk_ptx.cuh"

namespace flk {
namespace attn {

using tc::elect_one;
using tc::mbar_arrive;
using tc::mbar_expect_tx;
using tc::mbar_init;
using tc::mma_commit;
using tc::smem_u32;
using tc::tc_fence_after;
using tc::tc_fence_before;
using tc::tmem_alloc;
using tc::tmem_dealloc;
using tc::tmem_relinquish;

constexpr uint32_t kBlockBytes = kTile * 128;  // 128 rows x 64 columns of 16 bits

// Set by a kernel whose bounded wait gave up (one word per translation unit).
static __device__ int g_wait_status;

// Whether the barrier has passed the phase, the same answer for all lanes of a warp.  May suspend the warp for a while.
__device__ __forceinline__ bool passed(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "vote.sync.all.pred q, p, 0xffffffff;\n\t"
      "selp.b32 %0, 1, 0, q;\n\t}"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok != 0;
}
// A whole warp waits, and all of its lanes get the same answer: roles elect a lane for their work, which takes all of them.  A
// waiting warp looks again without sleeping: the other roles of the block wait for what it does next.
static __device__ __forceinline__ bool wait_bar(uint32_t bar, uint32_t parity, uint32_t limit_ns) {
  if (passed(bar, parity)) return true;
  const uint32_t t0 = tc::timer_lo_ns();
  for (uint32_t it = 0; it < (1u << 28); ++it) {
    if (passed(bar, parity)) return true;
    if ((it & 15) == 15 && __any_sync(0xffffffffu, tc::timer_lo_ns() - t0 >= limit_ns)) break;
  }
  atomicExch(&g_wait_status, 1);
  return false;
}
// What a block waits for before it ends, whatever limit its other waits have: copies that are still to land in its shared memory,
// products that are still to read that and to write its tensor memory.
constexpr uint32_t kDrainNs = 1000000000u;
static __device__ __forceinline__ bool drain_bar(uint32_t bar, uint32_t parity) { return wait_bar(bar, parity, kDrainNs); }

__device__ __forceinline__ void tma_load(uint32_t dst, const CUtensorMap* map, int x, int c1, int c2, int c3, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cta.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst),
      "l"(map), "r"(x), "r"(c1), "r"(c2), "r"(c3), "r"(bar)
      : "memory");
}

__device__ __forceinline__ void prefetch_map(const CUtensorMap* map) {
  asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory");
}

// Shared-memory matrix descriptors of a 128-byte-swizzled tile (8-row groups of 1024 bytes).  Only the low word changes from one
// product to the next: it is kept in one register and stepped by immediates.
constexpr uint32_t kDescHigh = (1024 >> 4)       // from one group of 8 rows to the next
                               | (1u << 14)      // version
                               | (2u << 29);     // SWIZZLE_128B
__device__ __forceinline__ uint32_t desc_low(uint32_t addr, uint32_t lead_bytes) {
  // MN-major: `lead_bytes` from one block of 64 columns to the next; K-major: unused
  return ((addr >> 4) & 0x3FFF) | (lead_bytes >> 4) << 16;
}

template <typename T>
__host__ __device__ constexpr uint32_t instr_desc(int n, bool b_mn_major) {
  const uint32_t type = sizeof(T) == 2 && std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
  return (1u << 4) | (type << 7) | (type << 10) | ((b_mn_major ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(kTile >> 4) << 24);
}

// A and B from shared memory
__device__ __forceinline__ void mma_ss(uint32_t d_tmem, uint32_t a_low, uint32_t b_low, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\t"
      "setp.ne.b32 p, %5, 0;\n\t"
      "mov.b64 a, {%1, %3};\n\t"
      "mov.b64 b, {%2, %3};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %4, p;\n\t}" ::"r"(d_tmem),
      "r"(a_low), "r"(b_low), "r"(kDescHigh), "r"(idesc), "r"(accumulate)
      : "memory");
}
// A from tensor memory (16-bit values, two per column), B from shared memory
__device__ __forceinline__ void mma_ts(uint32_t d_tmem, uint32_t a_tmem, uint32_t b_low, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 b;\n\t"
      "setp.ne.b32 p, %5, 0;\n\t"
      "mov.b64 b, {%2, %3};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %4, p;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "r"(b_low), "r"(kDescHigh), "r"(idesc), "r"(accumulate)
      : "memory");
}

// scores: D[128 x 128] = A B^T along DP columns
template <typename T, int DP>
__device__ __forceinline__ void issue_scores(uint32_t d_tmem, uint32_t a, uint32_t b) {
  const uint32_t al = desc_low(a, 16), bl = desc_low(b, 16);
#pragma unroll
  for (int ks = 0; ks < DP / 16; ++ks) {
    const uint32_t off = ((ks / 4) * kBlockBytes + (ks % 4) * 32) >> 4;
    mma_ss(d_tmem, al + off, bl + off, instr_desc<T>(kTile, false), ks > 0);
  }
}
// accumulation: D[128 x DP] (+)= W[128 x 128] B, with the weights W in tensor memory and the 128 rows of B.  The 128 columns of
// scores that the weights came from are shared by 128 / OWN threads of a row; each has put its weights, two per column, at the
// start of its own OWN columns.
template <typename T, int DP, int OWN>
__device__ __forceinline__ void issue_weighted(uint32_t d_tmem, uint32_t w_tmem, uint32_t b, bool accumulate) {
  const uint32_t bl = desc_low(b, kBlockBytes);
  constexpr int kPer = OWN / 16;  // products per thread's share
#pragma unroll
  for (int ks = 0; ks < kTile / 16; ++ks)
    mma_ts(d_tmem, w_tmem + ks / kPer * OWN + ks % kPer * 8, bl + ks * (2048 >> 4), instr_desc<T>(DP, true), accumulate || ks > 0);
}

// Tensor memory into registers, N columns of this thread's row.  The load is asynchronous; its wait is part of the same statement, so
// that no register is on its way where the compiler may move or spill it.
__device__ __forceinline__ void tmem_read16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_read32(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
        "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
        "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_read64(uint32_t taddr, uint32_t (&r)[32], uint32_t (&u)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x64.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, "
      "%32, %33, %34, %35, %36, %37, %38, %39, %40, %41, %42, %43, %44, %45, %46, %47, "
      "%48, %49, %50, %51, %52, %53, %54, %55, %56, %57, %58, %59, %60, %61, %62, %63}, [%64];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
        "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
        "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31]),
        "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]), "=r"(u[6]), "=r"(u[7]),
        "=r"(u[8]), "=r"(u[9]), "=r"(u[10]), "=r"(u[11]), "=r"(u[12]), "=r"(u[13]), "=r"(u[14]), "=r"(u[15]),
        "=r"(u[16]), "=r"(u[17]), "=r"(u[18]), "=r"(u[19]), "=r"(u[20]), "=r"(u[21]), "=r"(u[22]), "=r"(u[23]),
        "=r"(u[24]), "=r"(u[25]), "=r"(u[26]), "=r"(u[27]), "=r"(u[28]), "=r"(u[29]), "=r"(u[30]), "=r"(u[31])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_st4(uint32_t taddr, const uint32_t (&r)[4]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x4.b32 [%0], {%1, %2, %3, %4};" ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]) : "memory");
}
__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]),
               "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

template <typename T>
__device__ __forceinline__ uint32_t pack16(float lo, float hi) {
  uint32_t r;
  if constexpr (std::is_same<T, __nv_bfloat16>::value)
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  else
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
// Forward, weights are exp2(s - m + kLift) with a maximum m that may be 8 behind.  fp16 ends at 2^-25 and just below 2^16, so there
// they are lifted to where the largest is 2^15: up to 2^32 times smaller ones count, of which a long row may have many.
template <typename T>
constexpr float kLift = std::is_same<T, __nv_bfloat16>::value ? 0.f : 7.f;

// the pair of fp32 values that a packed pair holds
template <typename T>
__device__ __forceinline__ uint64_t unpack16(uint32_t v) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value) {
    return tc::pack2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
  } else {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&v));
    return tc::pack2(f.x, f.y);
  }
}
__device__ __forceinline__ float rcp_approx(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// The tanh of capped scores.  Where all of a warp's arguments x = scale s lie in [-1/2, 1/2], and scores of up to half the cap do,
// an odd polynomial on the FMA pipe takes the place of an exponential and a reciprocal: tanh(x) = x p(x^2) with p of degree 4
// fitted to tanh(x) / x at Chebyshev nodes (relative error 6e-8 in fp32); up to 1/8 degree 2 does (6e-9).  With both on the MUFU
// unit, the exponential of the weight included, that unit would set the pace: three operations for each score of a tile of
// 128 x 128, 16 per cycle, are three times the 1024 cycles of the two products.  The scale is multiplied into the coefficients once
// per call (Tanh), which saves a multiplication per score.  Where one of the warp's arguments is larger, every score is scaled first
// and takes the polynomial or the MUFU unit by its own size: 1 - 2 / (1 + e^2x) is off by 2e-7 whatever x is, and the cap, which may
// be as large as it likes, multiplies that.
__device__ __forceinline__ uint64_t both(float x) { return tc::pack2(x, x); }
constexpr double kTanh4[5] = {1.0, -0.3333306908607483, 0.133247509598732, -0.05298423767089844, 0.017131345346570015};
constexpr double kTanh2[3] = {0.999999993627153, -0.33332598923104395, 0.1320774045773301};
struct Tanh {
  uint64_t c[5], low[3];   // coefficients, twice each
  float limit, low_limit;  // largest |s| of the polynomials; -1: none
};
// The polynomials whose coefficients times powers of the scale fp32 holds as normal numbers: the last ones are 0.017 scale^9 and
// 0.13 scale^5.  Smaller scales (caps of a million scores) leave what reads `c` with the short polynomial, or with none.
inline Tanh make_tanh(float scale) {
  const float size = scale < 0 ? -scale : scale;
  const bool four = size > 1e-4f && size < 1e3f, two = size > 1e-7f && size < 1e3f;
  auto twice = [](double x) {
    const float v = (float)x;
    uint32_t u;
    memcpy(&u, &v, 4);
    return (uint64_t)u << 32 | u;
  };
  Tanh t;
  double f = scale;
  for (int k = 0; k < 5; ++k, f *= (double)scale * scale) {
    t.c[k] = twice(four ? kTanh4[k] * f : k < 3 ? kTanh2[k] * f : 0.0);
    if (k < 3) t.low[k] = twice(kTanh2[k] * f);
  }
  t.low_limit = two ? 0.125f / size : -1.f;
  t.limit = four ? 0.5f / size : t.low_limit;
  return t;
}
// which way a warp goes: 2, 1 (polynomial of degree 2, 4) or 0
template <int N>
__device__ __forceinline__ int tanh_way(const uint32_t (&s)[N][32], const Tanh& t) {
  float big = 0.f;
#pragma unroll
  for (int p = 0; p < N; ++p)
#pragma unroll
    for (int c = 0; c < 32; c += 2) big = fmaxf(fmaxf(big, fabsf(__uint_as_float(s[p][c]))), fabsf(__uint_as_float(s[p][c + 1])));
  return __all_sync(0xffffffffu, big <= t.low_limit) ? 2 : __all_sync(0xffffffffu, big <= t.limit) ? 1 : 0;
}
template <bool LOW>
__device__ __forceinline__ uint64_t tanh_slope(uint64_t s, const Tanh& t) {  // tanh(scale s) / s
  const uint64_t z = tc::mul2(s, s);
  if (LOW) return tc::fma2(tc::fma2(z, t.low[2], t.low[1]), z, t.low[0]);
  uint64_t y = tc::fma2(z, t.c[4], t.c[3]);
  y = tc::fma2(y, z, t.c[2]);
  y = tc::fma2(y, z, t.c[1]);
  return tc::fma2(y, z, t.c[0]);
}
// tanh(scale s) whatever the two are
__device__ __forceinline__ float tanh_any(float s, float scale) {
  const float x = s * scale, z = x * x;
  const float p = x * fmaf(fmaf(fmaf(fmaf((float)kTanh4[4], z, (float)kTanh4[3]), z, (float)kTanh4[2]), z, (float)kTanh4[1]), z, (float)kTanh4[0]);
  const float m = fmaf(-2.f, rcp_approx(1.f + ex2_approx(x * (2.f * kLog2e))), 1.f);
  return fabsf(x) <= 0.5f ? p : m;
}
template <bool LOW, int N>
__device__ __forceinline__ void by_polynomial(uint32_t (&s)[N][32], const Tanh& t) {
#pragma unroll
  for (int p = 0; p < N; ++p)
#pragma unroll
    for (int c = 0; c < 32; c += 2) {
      const uint64_t x = tc::pack2(__uint_as_float(s[p][c]), __uint_as_float(s[p][c + 1]));
      float y0, y1;
      tc::unpack2(tc::mul2(tanh_slope<LOW>(x, t), x), y0, y1);
      s[p][c] = __float_as_uint(y0);
      s[p][c + 1] = __float_as_uint(y1);
    }
}
// s -> tanh(scale s) in place, N x 32 raw scores of a row
template <int N>
__device__ __forceinline__ void to_tanh(uint32_t (&s)[N][32], const Tanh& t, float scale) {
  const int way = tanh_way(s, t);
  if (way == 2) {
    by_polynomial<true>(s, t);
  } else if (way == 1) {
    by_polynomial<false>(s, t);
  } else {
#pragma unroll
    for (int p = 0; p < N; ++p)
#pragma unroll
      for (int c = 0; c < 32; ++c) s[p][c] = __float_as_uint(tanh_any(__uint_as_float(s[p][c]), scale));
  }
}

// The block's first barrier (id 1): the loading warp, which has set up the mbarriers, goes on to its copies without waiting for
// the others.
template <int THREADS>
__device__ __forceinline__ void start_arrive() { asm volatile("barrier.cta.arrive 1, %0;" ::"n"(THREADS) : "memory"); }
template <int THREADS>
__device__ __forceinline__ void start_wait() { asm volatile("barrier.cta.sync 1, %0;" ::"n"(THREADS) : "memory"); }

// A warp's 32 rows of N 16-byte pieces each, from a row per lane to lanes side by side in a row: `piece(p)` gives the lane's own
// pieces, `put(row, p, v)` takes them.  A store of a row per lane would touch 32 cache lines at a time; this touches 32 / N rows.
// `room`: 32 * N * 16 bytes of shared memory of the warp's own, 16-byte aligned.
template <int N, typename Piece, typename Put>
__device__ __forceinline__ void store_rows32(uint32_t room, Piece piece, Put put) {
  const uint32_t lane = threadIdx.x & 31;
  __syncwarp();
#pragma unroll
  for (uint32_t p = 0; p < N; ++p) {
    const uint4 v = piece(p);
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(room + (lane * N + (p ^ (lane & (N - 1)))) * 16), "r"(v.x), "r"(v.y), "r"(v.z),
                 "r"(v.w)
                 : "memory");
  }
  __syncwarp();
#pragma unroll
  for (uint32_t e = 0; e < N; ++e) {
    const uint32_t at = e * 32 + lane, row = at / N, p = at % N;
    uint4 v;
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(room + (row * N + (p ^ (row & (N - 1)))) * 16) : "memory");
    put((int)row, (int)p, v);
  }
  __syncwarp();
}

// 16 bytes of NaN in any of the types
__device__ __forceinline__ uint4 nan_piece() { return make_uint4(0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu); }

// What the tensor-core kernels need on top of Args.
struct TcArgs {
  Args a;
  int pg, pg_shift;  // heads packed into the rows of a tile (a power of two), its logarithm
  int hp, rows;      // hq / pg, nq * pg
  int blocks;        // row blocks per (sequence, packed head)
  int splits;        // parts of the key axis
  float* part_o;     // [split][b][hp][rows][d] partial results of the parts, fp32
  float* part_lse;   // [split][b][hp][rows], base 2
  Tanh tanh;         // of the cap
  // the order in which the row blocks (backward: the key tiles) of all sequences start: sequence * blocks + block, or null
  const int* order;
  uint32_t wait_ns;      // limit of a wait; 0: the issuing warp gives up before its first product
};

// The tiles of [first, last) that a block has to look at: all of them or, with documents, those whose labels overlap [lo, hi].
// `tab` has the smallest and largest label of every tile and whether one of its rows has none.  Used by whole warps.
struct Tile {
  int at;     // index, -1 behind the last
  int label;  // the one label of all its rows, -1 where there is no such
  bool dirty; // it holds rows that nobody may see
};
struct TileWalk {
  const int4* tab;
  int at, last, lo, hi;
  uint32_t mask[4];  // what is left of 128 tiles from `base` on
  int base;
  __device__ __forceinline__ TileWalk(const int4* table, int first, int end, int l, int h)
      : tab(table), at(first), last(end), lo(l), hi(h), mask{0, 0, 0, 0}, base(first - 128) {}
  __device__ __forceinline__ Tile next() {
    if (tab == nullptr) return Tile{at < last ? at++ : -1, -1, false};
    while ((mask[0] | mask[1] | mask[2] | mask[3]) == 0) {
      base += 128;
      if (base >= last) return Tile{-1, -1, false};
      int4 r[4];
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const int t = base + 32 * w + (int)(threadIdx.x & 31);
        r[w] = t < last ? __ldg(tab + t) : make_int4(1, 0, 0, 0);
      }
#pragma unroll
      for (int w = 0; w < 4; ++w) mask[w] = __ballot_sync(0xffffffffu, r[w].x <= hi && lo <= r[w].y && r[w].x <= r[w].y);
    }
    int w = 0, found = 0;
#pragma unroll
    for (int e = 3; e >= 0; --e)
      if (mask[e] != 0) w = e, found = __ffs(mask[e]) - 1;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (e == w) mask[e] &= mask[e] - 1;
    const int t = base + 32 * w + found;
    const int4 r = __ldg(tab + t);
    return Tile{t, r.z == 0 && r.x == r.y ? r.x : -1, r.z != 0};
  }
};
// how many tiles such a walk visits
__device__ __forceinline__ int count_tiles(const int4* tab, int first, int last, int lo, int hi) {
  if (tab == nullptr) return max(last - first, 0);
  int n = 0;
  for (int t0 = first + (int)(threadIdx.x & 31); t0 < last; t0 += 256) {
    int4 r[8];
#pragma unroll
    for (int w = 0; w < 8; ++w) r[w] = t0 + 32 * w < last ? __ldg(tab + t0 + 32 * w) : make_int4(1, 0, 0, 0);
#pragma unroll
    for (int w = 0; w < 8; ++w) n += r[w].x <= hi && lo <= r[w].y && r[w].x <= r[w].y;
  }
  __syncwarp();
  for (int o = 16; o > 0; o >>= 1) n += __shfl_xor_sync(0xffffffffu, n, o);
  return n;
}
// The loading warp tells the others which tile a step works on through a ring of 16 slots; it is never that many steps ahead
// of them, its copies having fewer stages.
constexpr int kSlots = 16;
__device__ __forceinline__ void put_tile(uint32_t slots, int step, const Tile& t) {
  asm volatile("st.shared.v2.b32 [%0], {%1, %2};" ::"r"(slots + (step % kSlots) * 8), "r"(t.at | (t.dirty ? 1 << 30 : 0)), "r"(t.label) : "memory");
}
__device__ __forceinline__ Tile get_tile(uint32_t slots, int step) {
  int x, y;
  asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(x), "=r"(y) : "r"(slots + (step % kSlots) * 8) : "memory");
  return Tile{x & ~(1 << 30), y, (x >> 30 & 1) != 0};
}

// Writes zeros over the rows of a 128-row operand tile that are not `kept(row)`, so that what they hold meets no product.
// One warp.
template <int DP, typename Kept>
__device__ __forceinline__ void clean_rows(uint32_t tile, Kept kept) {
  for (int r = threadIdx.x & 31; r < kTile; r += 32) {
    if (kept(r)) continue;
#pragma unroll
    for (int b = 0; b < DP / 64; ++b)
#pragma unroll
      for (int c = 0; c < 128; c += 16)
        asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(tile + b * kBlockBytes + r * 128 + c), "r"(0) : "memory");
  }
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  __syncwarp();
}
// The same for keys that nobody may see: row index >= end, or label < 0.
template <int DP>
__device__ __forceinline__ void clean_tile(uint32_t tile, int r0, int end, const int* docs) {
  clean_rows<DP>(tile, [&](int r) { return r0 + r < end && (docs == nullptr || __ldg(docs + r0 + r) >= 0); });
}

// Bit c: column c of 32 lies before `stop`
__device__ __forceinline__ uint32_t columns_before(int stop) { return stop >= 32 ? 0xffffffffu : stop <= 0 ? 0u : (1u << stop) - 1u; }
// Bit c: column c of 32 has the label of this lane's row.  The lanes of a whole warp bring a column's label (`theirs`) and a
// row's (`my`) each; a round for every label that the rows have, one or two where documents follow one another.
__device__ __forceinline__ uint32_t same_label(int theirs, int my) {
  uint32_t bits = 0, todo = 0xffffffffu;
  while (todo != 0) {
    const int label = __shfl_sync(0xffffffffu, my, __ffs(todo) - 1);
    const uint32_t columns = __ballot_sync(0xffffffffu, theirs == label);
    if (my == label) bits = columns;
    todo &= ~__ballot_sync(0xffffffffu, my == label);
  }
  return bits;
}
// -infinity in the columns whose bit is not set
__device__ __forceinline__ void hide_columns(uint32_t (&s)[32], uint32_t seen) {
#pragma unroll
  for (int c = 0; c < 32; ++c)
    asm volatile("{\n\t.reg .pred p;\n\tsetp.eq.u32 p, %1, 0;\n\t@p mov.b32 %0, 0xff800000;\n\t}" : "+r"(s[c]) : "r"(seen & (1u << c)));
}

// smallest and largest label of the queries [i0, i1), and whether one of them has none; a whole warp
struct LabelRange {
  int lo, hi;
  bool bad;
};
__device__ __forceinline__ LabelRange labels_of(const int* docs, int i0, int i1) {
  LabelRange r{INT32_MAX, INT32_MIN, false};
#pragma unroll 4
  for (int i = i0 + (int)(threadIdx.x & 31); i < i1; i += 32) {
    const int id = __ldg(docs + i);
    if (id >= 0) {
      r.lo = min(r.lo, id);
      r.hi = max(r.hi, id);
    } else {
      r.bad = true;
    }
  }
  for (int o = 16; o > 0; o >>= 1) {
    r.lo = min(r.lo, __shfl_xor_sync(0xffffffffu, r.lo, o));
    r.hi = max(r.hi, __shfl_xor_sync(0xffffffffu, r.hi, o));
  }
  r.bad = __any_sync(0xffffffffu, r.bad);
  return r;
}

// ---------------------------------------------------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------------------------------------------------
// Limit of a wait in the calls that follow, in ns (flk_attention_wait_limit).
inline std::atomic<uint32_t> g_wait_limit{1000000000u};
inline uint32_t wait_limit() { return g_wait_limit.load(std::memory_order_relaxed); }

using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                              const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                              CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
inline EncodeFn encode_fn() {
  static EncodeFn fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult r;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &r) != cudaSuccess) p = nullptr;
    return reinterpret_cast<EncodeFn>(p);
  }();
  return fn;
}

// (d, heads, rows, batch), boxes of 64 columns x `heads_box` heads x `rows_box` rows
inline int make_map(CUtensorMap* m, const Tensor4& t, int dtype, int d, int h, int n, int b, int heads_box, int rows_box) {
  EncodeFn fn = encode_fn();
  if (fn == nullptr) return fail(FLK_ERR_CUDA, "cuTensorMapEncodeTiled is not available");
  const cuuint64_t dims[4] = {(cuuint64_t)d, (cuuint64_t)h, (cuuint64_t)n, (cuuint64_t)b};
  // the stride of a dimension of one entry is never used, but has to be valid
  const cuuint64_t one = (cuuint64_t)round_up(d * 2, 16);
  const cuuint64_t strides[3] = {h > 1 ? (cuuint64_t)t.sh * 2 : one, n > 1 ? (cuuint64_t)t.sn * 2 : one, b > 1 ? (cuuint64_t)t.sb * 2 : one};
  const cuuint32_t box[4] = {64, (cuuint32_t)heads_box, (cuuint32_t)rows_box, 1}, unit[4] = {1, 1, 1, 1};
  const CUresult r = fn(m, dtype == FLK_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, t.p, dims, strides, box,
                        unit, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(FLK_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d)", (int)r);
  return FLK_OK;
}

}  // namespace attn
}  // namespace flk
