// PTX wrappers of the tensor-core kernels (mbarriers, bulk copies, TMEM, tcgen05) and packed fp32 arithmetic.
#pragma once

#include "flk_common.cuh"

namespace flk {
namespace tc {

constexpr uint64_t kWaitTimeoutNs = 1000000000ull;  // every device-side wait gives up after 1 s

// ---------------------------------------------------------------------------------------------
// PTX wrappers
// ---------------------------------------------------------------------------------------------
__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }

// One lane of a converged warp.  Issuing tcgen05.mma / commit / bulk copies under this predicate
// (instead of `lane == 0` inside a divergent branch) lets the compiler keep descriptors and
// addresses in uniform registers; a divergent single-lane issue path costs well over a hundred
// cycles per MMA.
__device__ __forceinline__ bool elect_one() {
  uint32_t pred = 0;
  asm volatile(
      "{\n\t.reg .b32 rx;\n\t.reg .pred px;\n\t"
      "elect.sync rx|px, 0xFFFFFFFF;\n\t"
      "selp.b32 %0, 1, 0, px;\n\t}"
      : "=r"(pred));
  return pred != 0;
}

__device__ __forceinline__ void mbar_init(uint32_t bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void mbar_expect_tx(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
// A warp that read a shared-memory buffer with ordinary loads hands it back to a bulk-copy producer, which will
// overwrite it through the async proxy.  Two things must hold before the arrive that releases the buffer: the
// loads have returned -- an arrive does not wait for loads in flight, and nothing else does when their consumers
// were scheduled after it; `dep` must depend on the last of them (the running sums they feed), and the returned
// zero is added to the barrier address, so the arrive cannot issue earlier -- and the generic and the async proxy are
// ordered by a proxy fence.  Without this a vector tile was overwritten under the loads of the previous one
// whenever the producer stood waiting for exactly that buffer (wrong sums in a few rows, varying from run to run).
__device__ __forceinline__ uint32_t smem_reads_done(uint64_t dep) {
  uint32_t lo, hi, zero;
  asm volatile("mov.b64 {%0, %1}, %2;" : "=r"(lo), "=r"(hi) : "l"(dep));
  asm volatile("and.b32 %0, %1, 0;" : "=r"(zero) : "r"(lo ^ hi));
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  return zero;
}
__device__ __forceinline__ bool mbar_try_wait(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.b32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok != 0;
}
// Low 32 bits of the nanosecond timer (wraps every 4.29 s; differences of two readings stay valid below that).
__device__ __forceinline__ uint32_t timer_lo_ns() {
  uint32_t t;
  asm volatile("mov.u32 %0, %%globaltimer_lo;" : "=r"(t));
  return t;
}
// Bounded wait: false when the phase did not complete within about a second (kWaitTimeoutNs), or after 2^26
// probes, whichever comes first.  A waiting warp backs off with a short nanosleep between probes: a warp that
// spins on a barrier competes for issue slots with the epilogue warps of its SM sub-partition (measured: the
// sub-partition hosting the spinning MMA warp ran its epilogue warps almost 2x slower and set the pace of the
// whole CTA).  Inlined and kept to two registers (start time, probe count): the kernels that use it re-partition
// their registers between warp roles (setmaxnreg), which rules out out-of-line calls.
#ifndef FLK_TC_BACKOFF_NS
#define FLK_TC_BACKOFF_NS 20
#endif
__device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t parity) {
  if (mbar_try_wait(bar, parity)) return true;
  const uint32_t t0 = timer_lo_ns();
  for (uint32_t it = 0; it < (1u << 26); ++it) {
    if (FLK_TC_BACKOFF_NS > 0) __nanosleep(FLK_TC_BACKOFF_NS);
    if (mbar_try_wait(bar, parity)) return true;
    if (timer_lo_ns() - t0 > (uint32_t)kWaitTimeoutNs) return false;
  }
  return false;
}
__device__ __forceinline__ void fence_barrier_init() {
  asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
}
__device__ __forceinline__ void bulk_copy_g2s(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
               "l"(src), "r"(bytes), "r"(bar)
               : "memory");
}

// Register re-partitioning between warp roles; both are executed by all four warps of a warpgroup.
template <int N>
__device__ __forceinline__ void reg_release() {  // lower this warpgroup's register count to N
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void reg_claim() {  // raise it to N (waits until the pool holds enough)
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}

__device__ __forceinline__ void tmem_alloc(uint32_t dst_smem, uint32_t ncols) {
  asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(dst_smem), "r"(ncols)
               : "memory");
}
__device__ __forceinline__ void tmem_relinquish() {
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_dealloc(uint32_t taddr, uint32_t ncols) {
  asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(ncols) : "memory");
}
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

__device__ __forceinline__ void mma_f16(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                        uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void mma_commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
// The two wrappers below carry extra operands whose only purpose is to pin the instruction order the
// software pipeline needs (the compiler is otherwise free to move independent arithmetic across
// them): a load is issued BEFORE the evaluation of the piece that is already in registers, and the
// wait for it comes AFTER that evaluation.
//   tmem_ld32(taddr, dst, held): issues the load into `dst`; `held` (the piece about to be
//     evaluated) is tied as read-write, so its evaluation cannot be scheduled above the issue.
//   tmem_ld_wait_on(dst, acc): waits for the load into `dst`; the running sums `acc` are tied as
//     read-write, so every evaluation that feeds them is scheduled above the wait.
#define FLK_R32_OUT(r)                                                                                         \
  "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),  \
      "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),   \
      "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),  \
      "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
#define FLK_R32_INOUT(r)                                                                                       \
  "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]),  \
      "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]),   \
      "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]), "+r"(r[24]),  \
      "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])
#define FLK_TMEM_LD32_TEXT                                                                   \
  "tcgen05.ld.sync.aligned.32x32b.x32.b32 "                                                  \
  "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "                  \
  "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"

__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(FLK_TMEM_LD32_TEXT : FLK_R32_OUT(r) : "r"(taddr) : "memory");
}
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t (&r)[32], uint32_t (&held)[32]) {
  // operands 0-31 = destination, 32 = address, 33.. = the held piece (tied only)
  asm volatile(FLK_TMEM_LD32_TEXT
               : FLK_R32_OUT(r)
               : "r"(taddr), "r"(held[0]), "r"(held[4]), "r"(held[8]), "r"(held[12]), "r"(held[16]), "r"(held[20]),
                 "r"(held[24]), "r"(held[28])
               : "memory");
}
__device__ __forceinline__ void tmem_ld_wait_on(uint32_t (&r)[32], uint64_t (&acc)[2]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" : FLK_R32_INOUT(r), "+l"(acc[0]), "+l"(acc[1]) : : "memory");
}
__device__ __forceinline__ void tmem_ld_wait_on(uint32_t (&r)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" : FLK_R32_INOUT(r) : : "memory");
}
__device__ __forceinline__ void tmem_ld_wait_on(uint32_t (&r)[32], float (&acc)[4]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : FLK_R32_INOUT(r), "+f"(acc[0]), "+f"(acc[1]), "+f"(acc[2]), "+f"(acc[3])
               :
               : "memory");
}
// 16-column variants for the many-column epilogue (its 32 running sums leave room for 16 accumulator columns).
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_ld_wait_on(uint32_t (&r)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                 "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
               :
               : "memory");
}

// ---------------------------------------------------------------------------------------------
// Packed fp32 pairs (sm_100 add/sub/fma.f32x2: two fp32 operations per issued instruction).  The
// epilogue is bound by instruction issue once part of the exponentials leaves the MUFU unit, so
// everything that can be done on two columns at once is.
// ---------------------------------------------------------------------------------------------
__device__ __forceinline__ uint64_t pack2(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ void unpack2(uint64_t v, float& lo, float& hi) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ void ld_shared_f4(uint32_t addr, float& a, float& b, float& c, float& d) {
  asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(a), "=f"(b), "=f"(c), "=f"(d) : "r"(addr) : "memory");
}
__device__ __forceinline__ void st_shared_f4(uint32_t addr, float a, float b, float c, float d) {
  asm volatile("st.shared.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "f"(a), "f"(b), "f"(c), "f"(d) : "memory");
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ uint64_t sub2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("sub.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}

// 2^x on the FMA pipe for a pair of arguments: n = round(x) through the 1.5 * 2^23 trick, degree-5
// minimax polynomial of 2^f on f = x - n in [-1/2, 1/2] (relative error 2.4e-7), exponent patched
// in with integer arithmetic.  x is clamped at -126 so the patched exponent never wraps; arguments
// a hair above zero (rounding, coincident points) are fine.
__device__ __forceinline__ void ex2_fma_pair(float x0, float x1, float& y0, float& y1) {
  const uint64_t magic = pack2(12582912.0f, 12582912.0f);
  const uint64_t x = pack2(fmaxf(x0, -126.0f), fmaxf(x1, -126.0f));
  const uint64_t t = add2(x, magic);
  const uint64_t f = sub2(x, sub2(t, magic));
  uint64_t p = pack2(0.001327647129073739f, 0.001327647129073739f);
  p = fma2(p, f, pack2(0.009675540961325169f, 0.009675540961325169f));
  p = fma2(p, f, pack2(0.05550713092088699f, 0.05550713092088699f));
  p = fma2(p, f, pack2(0.24022120237350464f, 0.24022120237350464f));
  p = fma2(p, f, pack2(0.6931469440460205f, 0.6931469440460205f));
  p = fma2(p, f, pack2(1.0000001192092896f, 1.0000001192092896f));
  float p0, p1, t0, t1;
  unpack2(p, p0, p1);
  unpack2(t, t0, t1);
  y0 = __int_as_float(__float_as_int(p0) + (__float_as_int(t0) << 23));
  y1 = __int_as_float(__float_as_int(p1) + (__float_as_int(t1) << 23));
}

}  // namespace tc
}  // namespace flk
