// Forward attention on tcgen05: out, and the log-sum-exp of every row.
//
// A block has 18 warps: two groups of eight turn scores into weights, one issues the matrix products, one the copies.  A group
// serves one score tile; two threads share a row, each with half of the columns, and tell each other the largest score.  Tensor
// memory holds two score tiles of 128 x 128 and two accumulators of 128 x DP, all 512 columns.  The two groups take turns on the
// tensor cores: while one turns its scores into weights, the products of the other run.  With a group of four warps (a row
// per thread) a step of two tiles took 3470 cycles, of which 1570 were spent waiting for the next scores; the products take 2048.
//   PAIR   two row tiles (256 rows) against the same key tiles, for prompts and training
//   !PAIR  one row tile; the groups take the even and the odd key tiles, and end with a partial result each: few
//          rows over a long key axis (single tokens)
// Weights are exp2(s - m) with a maximum m that follows the running one only when that has grown by more than 8: weights
// stay below 2^8 (fp16: 2^15, see kLift), and the accumulator is rescaled a few times in a row's life instead of once per tile.
// Weights are rounded to the data's 16 bits before they meet V (a relative error of half a step each, which is what the result
// itself is rounded by: rms error of bf16 results 2.3e-3 of their size, of results rounded once 1.7e-3; a second product with what
// is left would be half as much work again).
// The result is divided by the sum of the rounded weights, so that their common error cancels; the log-sum-exp, which the
// backward pass makes exact weights from, has the sum of the weights as they were.  Sums, maximum and accumulators are fp32.
// Where blocks are fewer than SMs, the key axis is cut into parts, whose normalised fp32 results a second kernel joins.
//
// Measured: 2 x 6000 rows, 16 heads of 128 on 8, causal with a prefix: 318 us, 0.95 PFLOP/s of visible pairs; tensor pipe and MUFU
// 50 % busy each.  A step of two tiles takes 3.9 k cycles, 1.5 k of them waiting for scores, whose place in tensor memory the
// weights still hold.  8192 rows of documents, capped: 115 us; 4 x 2048 rows, heads of 64, distance bias: 83 us.
#pragma once

#include "flk_attn_tc.cuh"

namespace flk {
namespace attn {
namespace fwd {

constexpr int kThreads = 640;
// registers: 640 threads are launched with 96 each (61440); four warpgroups of 104 and one of 64 make the same sum
constexpr int kRegsSoftmax = 104, kRegsOther = 64;
static_assert(4 * 128 * kRegsSoftmax + 128 * kRegsOther <= kThreads * 96, "registers");
constexpr int kMmaWarp = 16, kLoadWarp = 17;

template <int DP, bool PAIR>
struct Layout {
  static constexpr uint32_t kTileBytes = DP / 64 * kBlockBytes;
  static constexpr uint32_t kQ = 0;
  static constexpr uint32_t kRing = (PAIR ? 2 : 1) * kTileBytes;
  static constexpr int kStages = (int)((224 * 1024 - kRing) / kTileBytes) < 8 ? (int)((224 * 1024 - kRing) / kTileBytes) : 8;
  static constexpr uint32_t kBars = kRing + kStages * kTileBytes;
  static constexpr uint32_t kBytes = kBars + 512 + 2048 + 512;  // barriers and slots, the halves' maxima, and some room
};
static_assert(Layout<128, true>::kBytes <= 227 * 1024 && Layout<128, false>::kBytes <= 227 * 1024, "shared memory");

// packed head, sequence, part of the key axis, first row of the block
__device__ __forceinline__ int4 get_place(uint32_t at) {
  int4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
  return v;
}

// Scores in base 2 from raw scores (or their tanh) and the distance bias; column 0 lies d0 before the row's position.  Where all
// columns lie on one side of all rows of the warp, the bias is linear: one base per 8 columns and 4 pairs of offsets that all of
// them share.
__device__ __forceinline__ void add_bias(uint32_t (&s)[2][32], float f2, float slope2, float d0) {
  const uint64_t f = both(f2);
  auto put = [&](int p, int c, uint64_t bias) {
    const uint64_t x = tc::pack2(__uint_as_float(s[p][c]), __uint_as_float(s[p][c + 1]));
    float y0, y1;
    tc::unpack2(tc::fma2(x, f, bias), y0, y1);
    s[p][c] = __float_as_uint(y0);
    s[p][c + 1] = __float_as_uint(y1);
  };
  if (__all_sync(0xffffffffu, d0 >= 63.f)) {
    uint64_t off[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) off[j] = tc::pack2(slope2 * (2 * j), slope2 * (2 * j + 1));
#pragma unroll
    for (int p = 0; p < 2; ++p)
#pragma unroll
      for (int c = 0; c < 32; c += 8) {
        const uint64_t at = both(-slope2 * (d0 - (32 * p + c)));
#pragma unroll
        for (int j = 0; j < 4; ++j) put(p, c + 2 * j, tc::add2(at, off[j]));
      }
  } else {
#pragma unroll
    for (int p = 0; p < 2; ++p)
#pragma unroll
      for (int c = 0; c < 32; c += 2) put(p, c, tc::pack2(-slope2 * fabsf(d0 - (32 * p + c)), -slope2 * fabsf(d0 - (32 * p + c + 1))));
  }
}

template <typename T, int DP, bool CAP, bool BIAS, bool PAIR>
__global__ void __launch_bounds__(kThreads, 1)
    kernel(const __grid_constant__ CUtensorMap tq, const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv, const TcArgs t) {
  using L = Layout<DP, PAIR>;
  constexpr int kStages = L::kStages;
  extern __shared__ __align__(1024) uint8_t raw[];
  const Args& a = t.a;
  const uint32_t base = smem_u32(raw), bars = base + L::kBars;
  auto full = [&](int s) { return bars + s * 8; };
  auto empty = [&](int s) { return bars + 64 + s * 8; };
  auto sfull = [&](int w) { return bars + 128 + w * 8; };
  auto pfull = [&](int w) { return bars + 144 + w * 8; };
  auto odone = [&](int w) { return bars + 160 + w * 8; };
  const uint32_t qfull = bars + 176, tmem_at = bars + 184, slots = bars + 192, place = bars + 320, drained = bars + 400, halves = bars + 512;
  auto xbar = [&](int w) { return bars + 384 + w * 8; };
  auto wait = [&](uint32_t bar, uint32_t parity) { return wait_bar(bar, parity, t.wait_ns); };
  const int warp = threadIdx.x >> 5;
  if (threadIdx.x < 3) prefetch_map(threadIdx.x == 0 ? &tq : threadIdx.x == 1 ? &tk : &tv);

  // block -> (row block, part of the key axis, sequence, packed head); those with the most keys start first, which under a
  // causal mask are the late ones
  uint32_t id = blockIdx.x;
  const int hp = (int)(id % (uint32_t)t.hp);
  id /= (uint32_t)t.hp;
  int b, rb;
  const int split = (int)(id % (uint32_t)t.splits);
  id /= (uint32_t)t.splits;
  if (t.order != nullptr) {
    const uint32_t place = (uint32_t)__ldg(t.order + id);
    b = (int)(place / (uint32_t)t.blocks);
    rb = (int)(place % (uint32_t)t.blocks);
  } else {
    b = (int)(id % (uint32_t)a.b);
    rb = t.blocks - 1 - (int)(id / (uint32_t)a.b);
  }
  constexpr int kRows = PAIR ? 256 : 128;
  const int row0 = rb * kRows, hk = (int)((uint32_t)(hp * t.pg) / (uint32_t)a.grp);
  const int i0 = row0 >> t.pg_shift, i1 = min(a.nq, (row0 + kRows) >> t.pg_shift);  // queries of this block
  const Limits lim = limits_of(a, b);
  const int* kd = a.kdocs ? a.kdocs + (int64_t)b * a.nk_pad : nullptr;
  const int* qd = a.qdocs ? a.qdocs + (int64_t)b * a.nq_pad : nullptr;
  const int4* ktab = kd ? a.ktab + (int64_t)b * (a.nk_pad / kTile) : nullptr;
  const int tiles = (lim.row_end(i1 - 1, a.causal) + kTile - 1) / kTile;
  // parts of at most one tile more than others
  const int even = (int)((uint32_t)tiles / (uint32_t)t.splits), odd = tiles - even * t.splits;
  const int first = split * even + min(split, odd), last = first + even + (split < odd ? 1 : 0);
  LabelRange lab{0, 0, false};
  if (kd) lab = labels_of(qd, i0, i1);
  const int steps = count_tiles(ktab, first, last, lab.lo, lab.hi);

  if (warp == kLoadWarp) {
    if (elect_one()) {
      for (int s = 0; s < kStages; ++s) mbar_init(full(s), 1), mbar_init(empty(s), 1);
      for (int w = 0; w < 2; ++w) mbar_init(sfull(w), 1), mbar_init(pfull(w), 8), mbar_init(odone(w), 1), mbar_init(xbar(w), 8);
      mbar_init(qfull, 1), mbar_init(drained, 1);
      asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(place + 16), "r"(lim.len), "r"(lim.start), "r"(lim.prefix), "r"(lim.at) : "memory");
      asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(place), "r"(hp), "r"(b), "r"(split), "r"(row0) : "memory");
      tc::fence_barrier_init();
    }
    __syncwarp();
    start_arrive<kThreads>();
  } else {
    if (warp == kMmaWarp) {
      tmem_alloc(tmem_at, 512);
      tmem_relinquish();
    }
    tc_fence_before();
    start_wait<kThreads>();
    tc_fence_after();
  }
  uint32_t tmem;
  asm volatile("ld.shared.b32 %0, [%1];" : "=r"(tmem) : "r"(tmem_at));
  auto ts = [&](int w) { return tmem + (uint32_t)w * kTile; };                  // scores, then weights
  auto to = [&](int w) { return tmem + 2 * kTile + (uint32_t)w * DP; };  // accumulators

  if (warp >= kMmaWarp) {
    tc::reg_release<kRegsOther>();
    if (warp == kLoadWarp) {
      TileWalk walk(ktab, first, last, lab.lo, lab.hi);
      bool ok = true;
      if (steps > 0 && elect_one()) {
        mbar_expect_tx(qfull, (PAIR ? 2 : 1) * L::kTileBytes);
#pragma unroll
        for (int r = 0; r < (PAIR ? 2 : 1); ++r)
#pragma unroll
          for (int c = 0; c < DP / 64; ++c)
            tma_load(base + r * L::kTileBytes + c * kBlockBytes, &tq, c * 64, hp * t.pg, (row0 + r * kTile) >> t.pg_shift, b, qfull);
      }
      __syncwarp();
      int n = 0;  // copies issued
      for (int step = 0; step < steps && ok; ++step) {
        const Tile e = walk.next();
#pragma unroll
        for (int kv = 0; kv < 2; ++kv) {
          const int s = n % kStages;
          if (n >= kStages) ok = ok && wait(empty(s), (uint32_t)(n / kStages - 1) & 1);
          if (!ok) break;
          if (elect_one()) {
            if (kv == 0) put_tile(slots, step, e);
            mbar_expect_tx(full(s), L::kTileBytes);
#pragma unroll
            for (int c = 0; c < DP / 64; ++c)
              tma_load(base + L::kRing + s * L::kTileBytes + c * kBlockBytes, kv == 0 ? &tk : &tv, c * 64, hk, e.at * kTile, b, full(s));
          }
          __syncwarp();
          ++n;
        }
      }
      // no copy may land after the block has gone
      if (steps > 0) drain_bar(qfull, 0);
      for (int i = n > kStages ? n - kStages : 0; i < n; ++i) drain_bar(full(i % kStages), (uint32_t)(i / kStages) & 1);
    } else if (warp == kMmaWarp) {
      bool ok = steps == 0 || (t.wait_ns != 0 && wait(qfull, 0));
      auto stage = [&](int n) { return base + L::kRing + (uint32_t)(n % kStages) * L::kTileBytes; };
      auto ready = [&](int n) { return wait(full(n % kStages), (uint32_t)(n / kStages) & 1); };
      auto clean = [&](int step) {
        const Tile e = get_tile(slots, step);
        if (e.dirty || (e.at + 1) * kTile > lim.len) clean_tile<DP>(stage(2 * step + 1), e.at * kTile, lim.len, kd);
      };
      // copy 2 i is the key tile, copy 2 i + 1 the value tile of step i
      if (steps > 0) {
        ok = ok && ready(0);
        tc_fence_after();
        if (ok && elect_one()) {
          issue_scores<T, DP>(ts(0), base, stage(0));
          mma_commit(sfull(0));
          if constexpr (PAIR) {
            issue_scores<T, DP>(ts(1), base + L::kTileBytes, stage(0));
            mma_commit(sfull(1));
          }
          mma_commit(empty(0));
        }
        __syncwarp();
      }
      for (int i = 0; i < steps && ok; ++i) {
        const bool more = i + 1 < steps;
        if constexpr (PAIR) {
          ok = ready(2 * i + 1);
          if (ok) clean(i);
          for (int w = 0; w < 2 && ok; ++w) {
            ok = wait(pfull(w), (uint32_t)i & 1);
            if (ok && w == 0 && more) ok = ready(2 * i + 2);
            tc_fence_after();
            if (ok && elect_one()) {
              issue_weighted<T, DP, 64>(to(w), ts(w), stage(2 * i + 1), i > 0);
              if (w == 1) mma_commit(empty((2 * i + 1) % kStages));
              if (more) {
                issue_scores<T, DP>(ts(w), base + w * L::kTileBytes, stage(2 * i + 2));
                mma_commit(sfull(w));
                if (w == 1) mma_commit(empty((2 * i + 2) % kStages));
              }
            }
            __syncwarp();
          }
        } else {
          // step i belongs to warpgroup i & 1: its scores are issued one step ahead of the weighted sum
          const int w = i & 1;
          if (more) {
            ok = ready(2 * i + 2);
            tc_fence_after();
            // the other score tile was consumed by the weighted sum of step i - 1, issued before
            if (ok && elect_one()) {
              issue_scores<T, DP>(ts(w ^ 1), base, stage(2 * i + 2));
              mma_commit(sfull(w ^ 1));
              mma_commit(empty((2 * i + 2) % kStages));
            }
            __syncwarp();
          }
          ok = ok && ready(2 * i + 1);
          if (ok) clean(i);
          ok = ok && wait(pfull(w), (uint32_t)(i >> 1) & 1);
          tc_fence_after();
          if (ok && elect_one()) {
            issue_weighted<T, DP, 64>(to(w), ts(w), stage(2 * i + 1), i > 1);
            mma_commit(empty((2 * i + 1) % kStages));
          }
          __syncwarp();
        }
      }
      if (steps > 0 && ok && elect_one()) {
        mma_commit(odone(0));
        mma_commit(odone(1));
      }
      __syncwarp();
      // no product may run, and no arrival come, after the block has gone
      if (elect_one()) mma_commit(drained);
      __syncwarp();
      drain_bar(drained, 0);
    }
  } else {
    tc::reg_claim<kRegsSoftmax>();
    const int w = warp >> 3, side = (warp >> 2) & 1;       // score tile; half of its columns
    const uint32_t lane_at = (uint32_t)(warp & 3) << 21;  // TMEM lane 32 (warp % 4) in bits 16 and up
    const int r = row0 + (PAIR ? w * kTile : 0) + (int)(threadIdx.x & 127);  // packed row
    const bool live = (r & ~31) < t.rows;                                   // some row of this warp exists
    const uint32_t mine = halves + (w * 256 + side * 128 + (threadIdx.x & 127)) * 4, other = side == 0 ? mine + 512 : mine - 512;
    const int i = r >> t.pg_shift, h = hp * t.pg + (r & (t.pg - 1));
    const float slope2 = BIAS && a.slopes != nullptr ? a.slopes[h] * kLog2e : 0.f;
    // for the tile of this warpgroup: keys before `x` are visible to every row that exists; `y` is the one label of its queries
    const uint32_t rule = place + 32 + 8 * w;
    {
      const int tile_i0 = (row0 + (PAIR ? w * kTile : 0)) >> t.pg_shift;
      int only = -1;
      if (kd) {
        const LabelRange mine = labels_of(qd, min(tile_i0, a.nq), min(a.nq, (tile_i0 + (kTile >> t.pg_shift))));
        if (!mine.bad && mine.lo == mine.hi) only = mine.lo;
      }
      // all eight warps write the same
      asm volatile("st.shared.v2.b32 [%0], {%1, %2};" ::"r"(rule), "r"(lim.row_end(min(tile_i0, a.nq - 1), a.causal)), "r"(only) : "memory");
      __syncwarp();
    }
    const float f2 = CAP ? a.cap2 : a.scale;  // raw score, or its tanh -> base 2; done last where there is no bias
    float m = -INFINITY;       // of the weights, base 2
    float l = 0.f, lr = 0.f;  // sums of the weights, and of the rounded weights
    bool ok = true;
    // what the two threads of a row tell each other: one value per phase of `xbar`, which all warps of the tile pass
    uint32_t phase = 0;
    auto exchange = [&](float v, float& theirs) {
      asm volatile("st.shared.f32 [%0], %1;" ::"r"(mine), "f"(v) : "memory");
      __syncwarp();
      if (elect_one()) mbar_arrive(xbar(w));
      __syncwarp();
      const bool ok = wait(xbar(w), phase & 1);
      ++phase;
      asm volatile("ld.shared.f32 %0, [%1];" : "=f"(theirs) : "r"(other) : "memory");
      return ok;
    };
    for (int step = PAIR ? 0 : w; step < steps; step += PAIR ? 1 : 2) {
      ok = wait(sfull(w), (uint32_t)(PAIR ? step : step >> 1) & 1);
      if (!ok) break;
      if (!live) {  // the weights of rows that do not exist reach nothing
        if (elect_one()) {
          mbar_arrive(xbar(w));
          mbar_arrive(pfull(w));
        }
        ++phase;
        __syncwarp();
        continue;
      }
      tc_fence_after();
      const Tile e = get_tile(slots, step);
      const int k0 = e.at * kTile + 64 * side;
      int all_before, only;
      asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(all_before), "=r"(only) : "r"(rule) : "memory");
      const bool whole = k0 + 64 <= all_before && (a.kdocs == nullptr || (e.label >= 0 && e.label == only));
      uint32_t s[2][32];
      const uint32_t at = ts(w) + lane_at + 64 * side;
      tmem_read64(at, s[0], s[1]);
      if constexpr (CAP) to_tanh(s, t.tanh, a.scale);
      if constexpr (BIAS) {  // (read again instead of held in a register)
        const int r = get_place(place).w + (PAIR ? w * kTile : 0) + (int)(threadIdx.x & 127);
        add_bias(s, f2, slope2, (float)(get_place(place + 16).w + (r >> t.pg_shift) - k0));
      }
      if (!whole) {
        uint32_t seen[2];
        const int4 x = get_place(place + 16);
        const int r = row0 + (PAIR ? w * kTile : 0) + (int)(threadIdx.x & 127);
        const int end = r < t.rows ? Limits{x.x, x.y, x.z}.row_end(r >> t.pg_shift, a.causal) : 0;
#pragma unroll
        for (int p = 0; p < 2; ++p) seen[p] = columns_before(end - k0 - 32 * p);
        if (a.kdocs != nullptr) {
          const int b = get_place(place).y, *labels = a.kdocs + (int64_t)b * a.nk_pad + k0 + (threadIdx.x & 31);
          const int l0 = __ldg(labels), l1 = __ldg(labels + 32), my = r < t.rows ? __ldg(a.qdocs + (int64_t)b * a.nq_pad + (r >> t.pg_shift)) : -2;
          seen[0] &= same_label(l0, my);
          seen[1] &= same_label(l1, my);
        }
#pragma unroll
        for (int p = 0; p < 2; ++p) hide_columns(s[p], seen[p]);
      }
      float top[4];
#pragma unroll
      for (int p = 0; p < 4; ++p) {
        const int c0 = 16 * (p & 1);
        top[p] = fmaxf(__uint_as_float(s[p / 2][c0]), __uint_as_float(s[p / 2][c0 + 1]));
#pragma unroll
        for (int c = 2; c < 16; c += 2) top[p] = fmaxf(fmaxf(top[p], __uint_as_float(s[p / 2][c0 + c])), __uint_as_float(s[p / 2][c0 + c + 1]));
      }
      float mt = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])), theirs;
      ok = exchange(mt, theirs);
      if (!ok) break;
      mt = fmaxf(mt, theirs);
      if constexpr (!BIAS) mt *= f2;
      const bool grow = mt > m + 8.f;
      if (__any_sync(0xffffffffu, grow)) {
        const float mn = grow ? mt : m;
        const float f = m == mn ? 1.f : ex2_approx(m - mn);
        if (step > (PAIR ? 0 : 1)) {
          // s_full of this step says that the weighted sums before it are done
#pragma unroll 1
          for (int c = side * (DP / 2); c < (side + 1) * (DP / 2); c += 16) {
            uint32_t o[16];
            tmem_read16(to(w) + lane_at + c, o);
#pragma unroll
            for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
            tmem_st16(to(w) + lane_at + c, o);
          }
        }
        l *= f;
        lr *= f;
        m = mn;
      }
      const float mb = (m == -INFINITY ? 0.f : m) - kLift<T>;
      const uint64_t f2v = tc::pack2(f2, f2), mv = tc::pack2(-mb, -mb);
      uint64_t sum = 0, rounded = 0;
#pragma unroll
      for (int p = 0; p < 4; ++p) {
        uint32_t o[8];
#pragma unroll
        for (int c = 0; c < 16; c += 2) {
          const int at = 16 * (p & 1) + c;
          const uint64_t v = tc::pack2(__uint_as_float(s[p / 2][at]), __uint_as_float(s[p / 2][at + 1]));
          const uint64_t x = BIAS ? tc::add2(v, mv) : tc::fma2(v, f2v, mv);
          float x0, x1, p0, p1;
          tc::unpack2(x, x0, x1);
          p0 = ex2_approx(x0);
          p1 = ex2_approx(x1);
          sum = tc::add2(sum, tc::pack2(p0, p1));
          o[c / 2] = pack16<T>(p0, p1);
          rounded = tc::add2(rounded, unpack16<T>(o[c / 2]));
        }
        tmem_st8(at + 8 * p, o);
      }
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (elect_one()) mbar_arrive(pfull(w));
      __syncwarp();
      float u0, u1;
      tc::unpack2(sum, u0, u1);
      l += u0 + u1;
      tc::unpack2(rounded, u0, u1);
      lr += u0 + u1;
    }
    // ---- results
    const bool worked = steps > (PAIR ? 0 : w);
    if (worked && ok) {
      // the products being done, all warps of the tile have passed the last step's exchange
      ok = wait(odone(w), 0);
      // both sums, through what was the ring (behind what the stores below use)
      const uint32_t sums = base + L::kRing + 65536;
      static_assert(L::kStages * L::kTileBytes >= 65536 + 512 * 8, "ring");
      asm volatile("st.shared.v2.f32 [%0], {%1, %2};" ::"r"(sums + threadIdx.x * 8), "f"(l), "f"(lr) : "memory");
      __syncwarp();
      if (elect_one()) mbar_arrive(xbar(w));
      __syncwarp();
      ok = ok && wait(xbar(w), phase & 1);
      float x, y;
      asm volatile("ld.shared.v2.f32 {%0, %1}, [%2];" : "=f"(x), "=f"(y) : "r"(sums + (threadIdx.x ^ 128) * 8) : "memory");
      l = side == 0 ? l + x : x + l;  // the same sums on both sides
      lr = side == 0 ? lr + y : y + lr;
    }
    tc_fence_after();
    // nothing seen: all weights were zero (a score that is not a number makes the sums, and so the row, NaN)
    const bool none = l == 0.f;
    if (live && !ok) {  // the joining kernel makes a row of parts NaN by the part's log-sum-exp alone
      const int4 at = get_place(place);
      const int hp = at.x, b = at.y, split = at.z, r = at.w + (PAIR ? w * kTile : 0) + (int)(threadIdx.x & 127);
      const int i = r >> t.pg_shift, h = hp * t.pg + (r & (t.pg - 1));
      if (r < t.rows && (!PAIR || t.splits > 1)) {
        t.part_lse[(((int64_t)(PAIR ? split : 2 * split + w) * a.b + b) * t.hp + hp) * t.rows + r] = NAN;
      } else if (r < t.rows) {
        if (a.lse != nullptr) a.lse[((int64_t)b * a.hq + h) * a.nq + i] = NAN;
        const int64_t row = b * a.o.sb + (int64_t)i * a.o.sn + h * a.o.sh;
        for (int c = 0; c < a.d; c += 8) {
          *reinterpret_cast<uint4*>(reinterpret_cast<T*>(a.o.p) + row + c) = nan_piece();
          if (a.o_lo != nullptr) *reinterpret_cast<uint4*>(reinterpret_cast<T*>(a.o_lo) + row + c) = nan_piece();
        }
      }
    }
    const float inv = none ? 0.f : 1.0f / lr, lse2 = none ? -INFINITY : m - kLift<T> + log2f(l);
    if (live && ok) {
      // read again instead of held in registers through the loop above
      const int4 at = get_place(place);
      const int hp = at.x, b = at.y, split = at.z, r = at.w + (PAIR ? w * kTile : 0) + (int)(threadIdx.x & 127);
      const int i = r >> t.pg_shift, h = hp * t.pg + (r & (t.pg - 1));
      const bool exists = r < t.rows;
      const bool parts = !PAIR || t.splits > 1;
      const int part = PAIR ? split : 2 * split + w;
      const int64_t prow = (((int64_t)part * a.b + b) * t.hp + hp) * t.rows + r;
      if (exists && side == 0) {
        if (parts)
          t.part_lse[prow] = lse2;
        else if (a.lse != nullptr)
          a.lse[((int64_t)b * a.hq + h) * a.nq + i] = lse2 * kLn2;
      }
      // rows of the warp side by side.  The ring is free: this group has waited for all products, and with them for all copies; a
      // group that had no tile has waited for nothing, but then either nobody had one, or there is nothing to write
      const uint32_t room = base + L::kRing + warp * 4096;
      const int r0 = r - (int)(threadIdx.x & 31);
#pragma unroll
      for (int c = side * (DP / 2); c < (side + 1) * (DP / 2) && (worked || !parts); c += 32) {
        uint32_t o[32];
        if (worked) tmem_read32(to(w) + lane_at + c, o);
#pragma unroll
        for (int e = 0; e < 32; ++e) o[e] = none ? 0u : __float_as_uint(__uint_as_float(o[e]) * inv);
        if (parts) {
          // the joining kernel does not read rows that saw nothing
          const int64_t base_row = (((int64_t)part * a.b + b) * t.hp + hp) * t.rows;
          store_rows32<8>(
              room, [&](uint32_t p) { return make_uint4(o[4 * p], o[4 * p + 1], o[4 * p + 2], o[4 * p + 3]); },
              [&](int e, int p, const uint4& v) {
                if (r0 + e < t.rows && c + 4 * p < a.d) *reinterpret_cast<uint4*>(t.part_o + (base_row + r0 + e) * a.d + c + 4 * p) = v;
              });
        } else {
          auto at_row = [&](int e, int p) -> int64_t {  // -1: not to be written
            const int rr = r0 + e;
            if (rr >= t.rows || c + 8 * p >= a.d) return -1;
            return b * a.o.sb + (int64_t)(rr >> t.pg_shift) * a.o.sn + (hp * t.pg + (rr & (t.pg - 1))) * a.o.sh + c + 8 * p;
          };
          auto piece = [&](uint32_t p, bool low) {
            uint32_t v[4];
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              const float y0 = __uint_as_float(o[8 * p + 2 * q]), y1 = __uint_as_float(o[8 * p + 2 * q + 1]);
              v[q] = low ? pack16<T>(y0 - to_f<T>(from_f<T>(y0)), y1 - to_f<T>(from_f<T>(y1))) : pack16<T>(y0, y1);
            }
            return make_uint4(v[0], v[1], v[2], v[3]);
          };
          store_rows32<4>(
              room, [&](uint32_t p) { return piece(p, false); },
              [&](int e, int p, const uint4& v) {
                const int64_t to = at_row(e, p);
                if (to >= 0) *reinterpret_cast<uint4*>(reinterpret_cast<T*>(a.o.p) + to) = v;
              });
          if (a.o_lo != nullptr)
            store_rows32<4>(
                room, [&](uint32_t p) { return piece(p, true); },
                [&](int e, int p, const uint4& v) {
                  const int64_t to = at_row(e, p);
                  if (to >= 0) *reinterpret_cast<uint4*>(reinterpret_cast<T*>(a.o_lo) + to) = v;
                });
        }
      }
    }
    tc_fence_before();
  }
  __syncthreads();
  if (warp == kMmaWarp) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// Joins the parts of the key axis: out = sum_p w_p o_p with w_p = 2^(lse_p - max) / sum.  A warp per row.
template <typename T>
__global__ void __launch_bounds__(256) join_kernel(const TcArgs t, int parts) {
  const Args& a = t.a;
  const int64_t n = (int64_t)a.b * t.hp * t.rows, row = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (row >= n) return;
  const int r = (int)(row % t.rows), hp = (int)(row / t.rows % t.hp), b = (int)(row / t.rows / t.hp);
  const int i = (int)((uint32_t)r / (uint32_t)t.pg), h = hp * t.pg + (r - i * t.pg);
  float top = -INFINITY;
  for (int p = lane; p < parts; p += 32) top = fmaxf(top, t.part_lse[p * n + row]);
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  if (top == -INFINITY) top = 0.f;
  float sum = 0.f;  // 0 where no part saw a key, NaN where a part's is
  for (int p = lane; p < parts; p += 32) sum += exp2f(t.part_lse[p * n + row] - top);
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  const float inv = sum == 0.f ? 0.f : 1.0f / sum;
  if (lane == 0 && a.lse != nullptr)
    a.lse[((int64_t)b * a.hq + h) * a.nq + i] = sum == 0.f ? -INFINITY : (top + log2f(sum)) * kLn2;
  const int c = lane * 4;
  if (c >= a.d) return;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  if (sum != 0.f) {
#pragma unroll 4
    for (int p = 0; p < parts; ++p) {
      const float e = t.part_lse[p * n + row];
      const float w = exp2f(e - top) * inv;
      // a part that saw nothing has written nothing
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
      if (e != -INFINITY) v = *reinterpret_cast<const float4*>(t.part_o + (p * n + row) * a.d + c);
      acc.x = fmaf(w, v.x, acc.x);
      acc.y = fmaf(w, v.y, acc.y);
      acc.z = fmaf(w, v.z, acc.z);
      acc.w = fmaf(w, v.w, acc.w);
    }
  }
  const int64_t at = b * a.o.sb + (int64_t)i * a.o.sn + h * a.o.sh + c;
  if constexpr (std::is_same<T, float>::value) {
    *reinterpret_cast<float4*>(reinterpret_cast<float*>(a.o.p) + at) = acc;
  } else {
    const uint2 v = make_uint2(pack16<T>(acc.x, acc.y), pack16<T>(acc.z, acc.w));
    *reinterpret_cast<uint2*>(reinterpret_cast<T*>(a.o.p) + at) = v;
    if (a.o_lo != nullptr) {
      const uint2 x = make_uint2(pack16<T>(acc.x - to_f<T>(from_f<T>(acc.x)), acc.y - to_f<T>(from_f<T>(acc.y))),
                                 pack16<T>(acc.z - to_f<T>(from_f<T>(acc.z)), acc.w - to_f<T>(from_f<T>(acc.w))));
      *reinterpret_cast<uint2*>(reinterpret_cast<T*>(a.o_lo) + at) = x;
    }
  }
}

struct Plan {
  bool pair;
  int pg, pg_shift, hp, rows, blocks, splits, parts;
};
// Heads packed into a tile's rows: all that share a key head, where that is a power of two.
inline int packed_heads(int hq, int hk) {
  const int grp = hq / hk;
  return (grp & (grp - 1)) == 0 && grp <= 64 ? grp : 1;
}
// Time of `blocks` x `s` blocks on all SMs, in us: blocks take `longest / s` steps at most and `mean / s` on average, a step
// takes `step` us, a block's start and end 4 us.  Blocks of one length run in waves; blocks of different lengths (uneven) fill
// gaps, all but half of the last one.
inline double time_of(int64_t blocks, int64_t s, double longest, double mean, double step, bool uneven) {
  const double one = longest / s * step + 4;
  if (!uneven) return (double)ceil_div(blocks * s, kNumSMs) * one;
  const double shared = (double)blocks * (mean * step + 4.0 * s) / kNumSMs + one / 2;
  return shared > one ? shared : one;
}
// Parts of the key axis: the number with the lowest estimate, joining included (3 us and its traffic at 5 TB/s).
// Steps of 128 keys take about 1.5 us with heads of 128 and 0.9 us with heads of 64.
inline Plan make_plan(int b, int nq, int nk, int hq, int hk, int d, bool causal, bool documents, bool lens) {
  Plan p{};
  p.pg = packed_heads(hq, hk);
  while ((1 << p.pg_shift) < p.pg) ++p.pg_shift;
  p.hp = hq / p.pg;
  p.rows = nq * p.pg;
  p.pair = p.rows > 128;
  p.blocks = (int)ceil_div(p.rows, p.pair ? 256 : 128);
  const int64_t blocks = (int64_t)p.blocks * p.hp * b, tiles = ceil_div(nk, kTile);
  const double step = d <= 64 ? 0.9 : 1.5, joined = (double)b * p.hp * p.rows * d * 8.0 / 5e6;
  double mean = (double)tiles;
  if (causal && nk > 0) mean *= 1.0 - 0.5 * (nq < nk ? (double)nq / nk : 1.0);
  if (documents) mean *= 0.5;
  if (lens) mean *= 0.75;
  const bool uneven = mean < 0.95 * (double)tiles;
  p.splits = 1;
  double best = 1e300;
  const int64_t least = p.pair ? 4 : 2;  // key tiles of a part
  for (int64_t s = 1; s <= 64 && (s == 1 || s * least <= tiles); ++s) {
    const int64_t parts = p.pair ? s : 2 * s;
    const double cost = time_of(blocks, s, (double)tiles, mean, step, uneven) + (parts > 1 ? 3 + parts * joined : 0);
    if (cost < best * 0.98) best = cost, p.splits = (int)s;
  }
  p.parts = p.pair ? p.splits : 2 * p.splits;
  return p;
}
inline int64_t partial_rows(const Plan& p, int b) { return p.parts > 1 ? (int64_t)p.parts * b * p.hp * p.rows : 0; }

template <typename T, int DP, bool CAP, bool BIAS, bool PAIR>
inline int launch_one(const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv, const TcArgs& t, cudaStream_t st) {
  auto* fn = kernel<T, DP, CAP, BIAS, PAIR>;
  constexpr int kBytes = (int)Layout<DP, PAIR>::kBytes;
  static std::atomic<uint64_t> done{0};
  FLK_TRY(allow_shared(reinterpret_cast<const void*>(fn), kBytes, done));
  const int64_t grid = (int64_t)t.blocks * t.splits * t.a.b * t.hp;
  if (grid > INT32_MAX) return fail(FLK_ERR_UNSUPPORTED, "too many row blocks");
  fn<<<(unsigned)grid, kThreads, kBytes, st>>>(tq, tk, tv, t);
  count_launch();
  return FLK_OK;
}
template <typename T, int DP, bool PAIR>
inline int launch_some(const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv, const TcArgs& t, cudaStream_t st) {
  const bool cap = t.a.cap2 != 0.f;
  // without a cap and a bias the maximum is taken of the raw scores, which needs a positive factor
  const bool bias = t.a.slopes != nullptr || (!cap && !(t.a.scale > 0.f));
  if (cap) return bias ? launch_one<T, DP, true, true, PAIR>(tq, tk, tv, t, st) : launch_one<T, DP, true, false, PAIR>(tq, tk, tv, t, st);
  return bias ? launch_one<T, DP, false, true, PAIR>(tq, tk, tv, t, st) : launch_one<T, DP, false, false, PAIR>(tq, tk, tv, t, st);
}

template <typename T>
inline int launch_join(const TcArgs& t, int parts, cudaStream_t st) {
  join_kernel<T><<<(unsigned)ceil_div((int64_t)t.a.b * t.hp * t.rows, 8), 256, 0, st>>>(t, parts);
  count_launch();
  return FLK_OK;
}

template <typename T>
inline int launch(TcArgs t, const Plan& p, cudaStream_t st) {
  const Args& a = t.a;
  t.wait_ns = wait_limit();
  const int dtype = std::is_same<T, __nv_bfloat16>::value ? FLK_BF16 : FLK_F16;
  t.pg = p.pg, t.pg_shift = p.pg_shift, t.hp = p.hp, t.rows = p.rows, t.blocks = p.blocks, t.splits = p.splits;
  t.tanh = make_tanh(a.scale);
  CUtensorMap tq, tk, tv;
  FLK_TRY(make_map(&tq, a.q, dtype, a.d, a.hq, a.nq, a.b, p.pg, kTile / p.pg));
  FLK_TRY(make_map(&tk, a.k, dtype, a.d, a.hk, a.nk, a.b, 1, kTile));
  FLK_TRY(make_map(&tv, a.v, dtype, a.d, a.hk, a.nk, a.b, 1, kTile));
  if (a.d <= 64)
    FLK_TRY((p.pair ? launch_some<T, 64, true>(tq, tk, tv, t, st) : launch_some<T, 64, false>(tq, tk, tv, t, st)));
  else
    FLK_TRY((p.pair ? launch_some<T, 128, true>(tq, tk, tv, t, st) : launch_some<T, 128, false>(tq, tk, tv, t, st)));
  return p.parts > 1 ? launch_join<T>(t, p.parts, st) : FLK_OK;
}

}  // namespace fwd
}  // namespace attn
}  // namespace flk
