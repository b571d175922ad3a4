// Backward attention on tcgen05: two kernels, one for dK and dV, one for dQ.  No atomics: every gradient is summed by one block
// in a fixed order (or by a few, whose fp32 partial results a last kernel adds in order).  Forming the weights twice costs two
// of seven products; adding dQ up over the blocks of all key tiles instead would cost atomics on fp32, and results that depend
// on their order.
//
//   keys kernel     a block owns 128 keys and walks over the query tiles:  S^T = K Q^T, dP^T = V dO^T  (rows are keys),
//                   P = exp2(S - lse), dV += P^T dO, dS = P (dP - delta), dK += dS^T Q.
//                   Tensor memory: S, dP, dV, dK, 128 columns each.  P and dS replace the scores they were made from.
//                   The tensor cores run dV(i), S(i+1) while dS(i) is being made and dK(i), dP(i+1) while P(i+1) is.
//   queries kernel  a block owns 128 packed query rows and walks over the key tiles:  S = Q K^T (two buffers), dP = dO V^T,
//                   dQ += dS K.
// Both have 20 warps: four warpgroups that turn scores into weights (a thread owns one row and a quarter of the columns), a warp that
// issues products, one that issues copies, and in the keys kernel one that gathers what the columns need (lse, delta, ...).
//
// Measured: 8192 rows of 7 documents, 16 heads of 128 on 2, capped, bf16: dK and dV 162 us (and 10 for adding parts), dQ 120; 4 x 2048
// rows, 12 heads of 64, distance bias, bf16: 106 and 75.  A step takes 4.3 k and 3.0 k cycles with heads of 128 (capped), 3.3 k and
// 2.5 k with 64: the chain product - exponentials - product, 16 warps on one tile; a block's start takes 2 to 5 k, its end 3 k.
//
// P and dS are rounded to the data's 16 bits before their second product, as P is in the forward pass (rms error of a bf16 training
// pass 2.4e-3, of its results rounded once 1.7e-3).  In fp16 they would leave its range: weights are held times 2^12, and the dS of
// a row (a key in the one kernel, a query in the other) times a power of two of its own, which follows what the row has met so far
// as a running maximum does: the first terms take it to 2^4, and terms beyond 2^15 take the row's accumulator down with it.  So no
// row, sequence or head costs another one bits, and terms lost to fp16's lower end are 2^-29 of the row's largest.  The exchange of
// a row's largest term costs fp16 4 to 7% of both kernels (4 x 2048 rows, 12 heads of 128, causal, forward and backward: 340 us,
// bf16 319).
//
// The dS of a row add up to zero, so where a row has few keys the terms of dQ and dK cancel, and the rounding of dS would be the
// largest error (up to 1.8 times that of rounding the result, for rows of ten keys).  With up to 256 queries and keys, where a
// call is bound by its launches, what rounding took from dS is kept beside it, in the other half of its columns, and multiplied
// too.  Beyond, where the error stays at 1.5 times (and more in short documents of a long row, which have it as short rows would),
// the fourth and fifth product would cost 5 to 10% (8192 rows of documents 150 + 120 -> 157 + 135 us; 4 x 2048 rows, heads of 64,
// 104 + 74 -> 115 + 84).
#pragma once

#include "flk_attn_fwd.cuh"

namespace flk {
namespace attn {
namespace bwd {

constexpr int kThreads = 640;
constexpr int kMmaWarp = 16, kLoadWarp = 17, kStatWarp = 18;
// registers: 640 threads are launched with 96 each (61440); four warpgroups of 104 and one of 64 make the same sum
constexpr int kRegsWork = 104, kRegsOther = 64;
static_assert(4 * 128 * kRegsWork + 128 * kRegsOther <= kThreads * 96, "registers");

// what the columns (queries) of a tile bring into the keys kernel
enum { kLse = 0, kDelta = 128, kSlope = 256, kPos = 384, kLabel = 512, kStatWords = 640 };
constexpr int kStatSlots = 4;

template <int DP, bool KEYS>
struct Layout {
  static constexpr uint32_t kTileBytes = DP / 64 * kBlockBytes;
  static constexpr uint32_t kOwn = 0;  // K, V (keys kernel) or Q, dO
  static constexpr uint32_t kRing = 2 * kTileBytes;
  static constexpr uint32_t kStats = KEYS ? kStatSlots * kStatWords * 4 : 0;
  static constexpr int kFit = (int)((224 * 1024 - kRing - kStats) / kTileBytes);
  static constexpr int kStages = kFit < 8 ? kFit : 8;
  static constexpr uint32_t kStatAt = kRing + kStages * kTileBytes;
  static constexpr uint32_t kBars = kStatAt + kStats;
  static constexpr uint32_t kTops = kBars + 512 + (KEYS ? kSlots * 16 : 0);  // fp16: 4 x 128 words
  static constexpr uint32_t kBytes = kTops + 2048;
};
static_assert(Layout<128, true>::kBytes <= 227 * 1024 && Layout<128, false>::kBytes <= 227 * 1024, "shared memory");
static_assert(Layout<128, true>::kStages >= 4 && Layout<128, false>::kStages >= 5, "stages");

// Factors of the data's type: weights are exp2(s - lse + kWeightShift)
template <typename T>
struct Scales {
  static constexpr bool kHalf = !std::is_same<T, __nv_bfloat16>::value;
  static constexpr float kShift = kHalf ? 12.f : 0.f;
  static constexpr float kUnshift = kHalf ? 1.f / 4096.f : 1.f;
};

// fp16: the factor of a row's dS, the same in the four threads that share the row.  They tell each other their largest value
// through shared memory: a word per thread, one phase of an mbarrier per step and warp of the row.
struct RowScale {
  float now = 0.f;  // 0: all terms so far were zero
  // Whether terms of up to `top` need another factor; if so, it is set, and `change` is what to multiply the accumulator with.
  __device__ __forceinline__ bool follow(float top, float& change) {
    change = 1.f;
    if (now == 0.f ? top == 0.f : top * now <= 32768.f) return false;
    const int e = (int)(__float_as_uint(top) >> 23) - 127;  // 2^e <= top < 2^(e + 1)
    const float next = __uint_as_float((uint32_t)(127 + min(max(4 - e, -120), 120)) << 23);
    const bool scaled = now != 0.f;
    if (scaled) change = next / now;
    now = next;
    return scaled;
  }
  // of the finished accumulator
  __device__ __forceinline__ float undo(float scale) const { return now == 0.f ? scale : scale / now; }
};
__device__ __forceinline__ void put_top(uint32_t tops, int w, float v) {
  asm volatile("st.shared.f32 [%0], %1;" ::"r"(tops + (w * kTile + (threadIdx.x & 127)) * 4), "f"(v) : "memory");
}
__device__ __forceinline__ float largest_top(uint32_t tops) {
  float v[4];
#pragma unroll
  for (int w = 0; w < 4; ++w) asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v[w]) : "r"(tops + (w * kTile + (threadIdx.x & 127)) * 4) : "memory");
  return fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3]));
}
// A quarter of the rows' accumulators (DP / 4 columns) times `f`.
template <int DP>
__device__ __forceinline__ void rescale_quarter(uint32_t acc, float f) {
#pragma unroll 1
  for (int c = 0; c < DP / 4; c += 16) {
    uint32_t o[16];
    tmem_read16(acc + c, o);
#pragma unroll
    for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
    tmem_st16(acc + c, o);
  }
}

// What dS is made from later, in the place of the scores s0, s1: the weights, times 1 - tanh^2 where s is the tanh of a capped score
template <bool CAP>
__device__ __forceinline__ void weight_slope(uint32_t& s0, uint32_t& s1, float p0, float p1) {
  if constexpr (CAP) {
    const uint64_t v = tc::pack2(__uint_as_float(s0), __uint_as_float(s1));
    tc::unpack2(tc::mul2(tc::pack2(p0, p1), tc::fma2(tc::mul2(v, both(-1.f)), v, both(1.f))), p0, p1);
  }
  s0 = __float_as_uint(p0);
  s1 = __float_as_uint(p1);
}

// what rounding took from a pair of values, rounded itself
template <typename T>
__device__ __forceinline__ uint32_t left_over(float y0, float y1, uint32_t rounded) {
  tc::unpack2(tc::sub2(tc::pack2(y0, y1), unpack16<T>(rounded)), y0, y1);
  return pack16<T>(y0, y1);
}

// A quarter of the accumulator (DP / 4 columns from c0 on) times f: 16-bit values of 32 rows, rows side by side
// (`at(row)`: where row `row` of the warp begins, or null where it is not to be written).
template <typename T, int DP, typename At>
__device__ __forceinline__ void store_quarter(uint32_t acc, int c0, float f, bool zero, int d, uint32_t room, At at) {
  constexpr int kWords = DP / 4;
  uint32_t o[kWords];
  if constexpr (kWords == 16)
    tmem_read16(acc + c0, o);
  else
    tmem_read32(acc + c0, o);
#pragma unroll
  for (int e = 0; e < kWords; ++e) o[e] = zero ? 0u : __float_as_uint(__uint_as_float(o[e]) * f);
  store_rows32<kWords / 8>(
      room,
      [&](uint32_t p) {
        uint32_t v[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) v[q] = pack16<T>(__uint_as_float(o[8 * p + 2 * q]), __uint_as_float(o[8 * p + 2 * q + 1]));
        return make_uint4(v[0], v[1], v[2], v[3]);
      },
      [&](int row, int p, const uint4& v) {
        T* to = at(row);
        if (to != nullptr && c0 + 8 * p < d) *reinterpret_cast<uint4*>(to + c0 + 8 * p) = v;
      });
}
// The same as fp32 partial results.
template <int DP, typename At>
__device__ __forceinline__ void store_partial(uint32_t acc, int c0, float f, bool zero, int d, uint32_t room, At at) {
  constexpr int kWords = DP / 4;
  uint32_t o[kWords];
  if constexpr (kWords == 16)
    tmem_read16(acc + c0, o);
  else
    tmem_read32(acc + c0, o);
#pragma unroll
  for (int e = 0; e < kWords; ++e) o[e] = zero ? 0u : __float_as_uint(__uint_as_float(o[e]) * f);
  store_rows32<kWords / 4>(
      room, [&](uint32_t p) { return make_uint4(o[4 * p], o[4 * p + 1], o[4 * p + 2], o[4 * p + 3]); },
      [&](int row, int p, const uint4& v) {
        float* to = at(row);
        if (to != nullptr && c0 + 4 * p < d) *reinterpret_cast<uint4*>(to + c0 + 4 * p) = v;
      });
}
// A quarter of a row of one value, zero or NaN (`row`: 16-bit values; `part`: fp32 partial results, unless null)
template <typename T, int DP>
__device__ __forceinline__ void store_same(bool nan, int c0, bool exists, int d, T* row, float* part) {
  if (!exists) return;
  const uint4 v = nan ? nan_piece() : make_uint4(0, 0, 0, 0);
  for (int c = c0; c < c0 + DP / 4 && c < d; c += 8) {
    if (part != nullptr)
      *reinterpret_cast<uint4*>(part + c) = *reinterpret_cast<uint4*>(part + c + 4) = v;
    else
      *reinterpret_cast<uint4*>(row + c) = v;
  }
}

// The steps of the keys kernel: query tiles of each packed head in turn, from step `skip` on.
struct StepWalk {
  const int4* tab;
  int first, last, lo, hi, head;
  TileWalk walk;
  __device__ __forceinline__ StepWalk(const int4* table, int f, int l, int a, int b, int per_head, int skip)
      : tab(table), first(f), last(l), lo(a), hi(b), head(per_head > 0 ? skip / per_head : 0), walk(table, f, l, a, b) {
    int rest = per_head > 0 ? skip % per_head : 0;
    if (tab == nullptr)
      walk.at += rest;
    else
      for (; rest > 0; --rest) walk.next();
  }
  __device__ __forceinline__ Tile next() {
    Tile t = walk.next();
    if (t.at < 0) {
      ++head;
      walk = TileWalk(tab, first, last, lo, hi);
      t = walk.next();
    }
    return t;
  }
};

struct Maps {
  CUtensorMap q, dout, k, v;
};

// ---------------------------------------------------------------------------------------------------------------------
// dK, dV
// ---------------------------------------------------------------------------------------------------------------------
template <typename T, int DP, bool CAP, bool BIAS, bool FINE>
__global__ void __launch_bounds__(kThreads, 1) kernel_keys(const __grid_constant__ Maps maps, const TcArgs t) {
  using L = Layout<DP, true>;
  constexpr int kStages = L::kStages;
  extern __shared__ __align__(1024) uint8_t raw[];
  const Args& a = t.a;
  const uint32_t base = smem_u32(raw), bars = base + L::kBars;
  auto full = [&](int s) { return bars + s * 8; };
  auto empty = [&](int s) { return bars + 64 + s * 8; };
  const uint32_t own = bars + 128, sfull = bars + 136, pfull = bars + 144, dpfull = bars + 152, dsfull = bars + 160, done = bars + 168, tmem_at = bars + 176, drained = bars + 184;
  auto statfull = [&](int s) { return bars + 192 + s * 8; };
  auto statempty = [&](int s) { return bars + 224 + s * 8; };
  const uint32_t slots = bars + 256, hollows = bars + 512;  // 128 bits per slot: rows of the tile that see nothing
  auto xbar = [&](int q) { return bars + 384 + q * 8; };
  auto wait = [&](uint32_t bar, uint32_t parity) { return wait_bar(bar, parity, t.wait_ns); };
  const int warp = threadIdx.x >> 5;
  if (threadIdx.x < 4) prefetch_map(threadIdx.x == 0 ? &maps.k : threadIdx.x == 1 ? &maps.v : threadIdx.x == 2 ? &maps.q : &maps.dout);

  uint32_t id = blockIdx.x;
  const int hk = (int)(id % (uint32_t)a.hk);
  id /= (uint32_t)a.hk;
  const int split = (int)(id % (uint32_t)t.splits);
  id /= (uint32_t)t.splits;
  int b, k0;
  if (t.order != nullptr) {
    const uint32_t place = (uint32_t)__ldg(t.order + id), tiles = (uint32_t)a.nk_pad / kTile;
    b = (int)(place / tiles);
    k0 = (int)(place % tiles) * kTile;
  } else {
    b = (int)(id % (uint32_t)a.b);
    k0 = (int)(id / (uint32_t)a.b) * kTile;
  }
  const Limits lim = limits_of(a, b);
  const int* kd = a.kdocs ? a.kdocs + (int64_t)b * a.nk_pad : nullptr;
  const int* qd = a.qdocs ? a.qdocs + (int64_t)b * a.nq_pad : nullptr;
  const int4* qtab = qd ? a.qtab + (int64_t)b * (a.nq_pad / a.q_rows) : nullptr;
  // query tiles that may see one of these keys
  int first = 0, last = (t.rows + kTile - 1) / kTile;
  if (k0 >= lim.len) last = 0;
  if (a.causal && lim.prefix <= k0) {
    const int64_t i = (int64_t)k0 - lim.start;  // the first query that stands at key k0 or behind it
    first = i <= 0 ? 0 : i >= a.nq ? last : (int)((i << t.pg_shift) / kTile);
  }
  LabelRange lab{0, 0, false};
  if (kd) lab = labels_of(kd, k0, k0 + kTile);
  const int heads = a.grp >> t.pg_shift;
  const int per_head = count_tiles(qtab, first, last, lab.lo, lab.hi);
  // parts of at most one step more than others
  const uint32_t total = (uint32_t)(per_head * heads), even = total / (uint32_t)t.splits, more = total % (uint32_t)t.splits;
  const int skip = (int)(split * even + min((uint32_t)split, more)), steps = (int)(even + ((uint32_t)split < more ? 1 : 0));

  if (warp == kLoadWarp) {
    if (elect_one()) {
      for (int s = 0; s < kStages; ++s) mbar_init(full(s), 1), mbar_init(empty(s), 1);
      mbar_init(own, 1), mbar_init(sfull, 1), mbar_init(pfull, 16), mbar_init(dpfull, 1), mbar_init(dsfull, 16), mbar_init(done, 1), mbar_init(drained, 1);
      if constexpr (Scales<T>::kHalf)
        for (int q = 0; q < 4; ++q) mbar_init(xbar(q), 4);
      for (int s = 0; s < kStatSlots; ++s) mbar_init(statfull(s), 1), mbar_init(statempty(s), 16);
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
  const uint32_t ts = tmem, tp = tmem + 128, tdv = tmem + 256, tdk = tmem + 256 + DP;

  if (warp >= kMmaWarp) {
    tc::reg_release<kRegsOther>();
    if (warp == kLoadWarp) {
      bool ok = true;
      if (steps > 0 && elect_one()) {
        mbar_expect_tx(own, 2 * L::kTileBytes);
#pragma unroll
        for (int c = 0; c < DP / 64; ++c) {
          tma_load(base + c * kBlockBytes, &maps.k, c * 64, hk, k0, b, own);
          tma_load(base + L::kTileBytes + c * kBlockBytes, &maps.v, c * 64, hk, k0, b, own);
        }
      }
      __syncwarp();
      StepWalk walk(qtab, first, last, lab.lo, lab.hi, per_head, skip);
      // queries that see nothing may hold anything; their weights are zero, and what those meet must be finite
      const bool hollow = qd != nullptr || lim.row_end(0, a.causal) == 0;
      int n = 0;
      for (int step = 0; step < steps && ok; ++step) {
        Tile e = walk.next();
        const int h = hk * a.grp + walk.head * t.pg;
        uint32_t none[4] = {0, 0, 0, 0};
        if (hollow) {
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const int r = e.at * kTile + (int)(threadIdx.x & 31) + 32 * x;
            const float lse = r < t.rows ? __ldg(a.lse + ((int64_t)b * a.hq + h + (r & (t.pg - 1))) * a.nq + (r >> t.pg_shift)) : 0.f;
            none[x] = __ballot_sync(0xffffffffu, lse == -INFINITY);
          }
          e.dirty = (none[0] | none[1] | none[2] | none[3]) != 0;
        }
#pragma unroll
        for (int qo = 0; qo < 2; ++qo) {
          const int s = n % kStages;
          if (n >= kStages) ok = ok && wait(empty(s), (uint32_t)(n / kStages - 1) & 1);
          if (!ok) break;
          if (elect_one()) {
            if (qo == 0) {
              put_tile(slots, step, e);
              asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(hollows + (step % kSlots) * 16), "r"(none[0]), "r"(none[1]), "r"(none[2]), "r"(none[3])
                           : "memory");
            }
            mbar_expect_tx(full(s), L::kTileBytes);
#pragma unroll
            for (int c = 0; c < DP / 64; ++c)
              tma_load(base + L::kRing + s * L::kTileBytes + c * kBlockBytes, qo == 0 ? &maps.q : &maps.dout, c * 64, h, (e.at * kTile) >> t.pg_shift, b, full(s));
          }
          __syncwarp();
          ++n;
        }
      }
      if (steps > 0) drain_bar(own, 0);
      for (int i = n > kStages ? n - kStages : 0; i < n; ++i) drain_bar(full(i % kStages), (uint32_t)(i / kStages) & 1);
    } else if (warp >= kStatWarp) {
      // two warps take turns; all loads of a step are under way at once
      bool ok = true;
      StepWalk walk(qtab, first, last, lab.lo, lab.hi, per_head, skip);
      for (int step = 0; step < steps && ok; ++step) {
        const Tile e = walk.next();
        if ((step & 1) != warp - kStatWarp) continue;
        const int slot = step % kStatSlots;
        float lse[4], delta[4], slope[4];
        int label[4];
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const int c = (threadIdx.x & 31) + 32 * x, r = e.at * kTile + c, i = r >> t.pg_shift;
          const int h = hk * a.grp + walk.head * t.pg + (r & (t.pg - 1));
          const bool exists = r < t.rows;
          const int64_t row = ((int64_t)b * a.hq + h) * a.nq + i;
          lse[x] = exists ? __ldg(a.lse + row) : -INFINITY;
          delta[x] = exists ? __ldg(a.delta + row) : 0.f;
          label[x] = qd != nullptr && exists ? __ldg(qd + i) : -2;
          if constexpr (BIAS) slope[x] = a.slopes != nullptr ? __ldg(a.slopes + h) : 0.f;
        }
        if (step >= kStatSlots) ok = wait(statempty(slot), (uint32_t)(step / kStatSlots - 1) & 1);
        if (!ok) break;
        const uint32_t at = base + L::kStatAt + slot * kStatWords * 4;
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const int c = (threadIdx.x & 31) + 32 * x, r = e.at * kTile + c, i = r >> t.pg_shift;
          // rows that see nothing: weights exp2(s - inf) = 0, and no delta, which may be NaN there
          const bool none = lse[x] == -INFINITY;
          auto put = [&](int word, uint32_t v) { asm volatile("st.shared.b32 [%0], %1;" ::"r"(at + (word + c) * 4), "r"(v) : "memory"); };
          put(kLse, __float_as_uint(none ? -INFINITY : fmaf(-lse[x], kLog2e, Scales<T>::kShift)));  // added to the score
          put(kDelta, __float_as_uint(none ? 0.f : -delta[x] * Scales<T>::kUnshift));
          if constexpr (BIAS) {
            put(kSlope, __float_as_uint(-slope[x] * kLog2e));
            put(kPos, __float_as_uint((float)(lim.at + i - k0)));
          }
          put(kLabel, (uint32_t)label[x]);
        }
        __syncwarp();
        if (elect_one()) mbar_arrive(statfull(slot));
        __syncwarp();
      }
    } else if (warp == kMmaWarp) {
      bool ok = steps == 0 || (t.wait_ns != 0 && wait(own, 0));
      auto stage = [&](int n) { return base + L::kRing + (uint32_t)(n % kStages) * L::kTileBytes; };
      auto ready = [&](int n) { return wait(full(n % kStages), (uint32_t)(n / kStages) & 1); };
      auto arrived = [&](int n) {
        if (!ready(n)) return false;
        if (get_tile(slots, n / 2).dirty)
          clean_rows<DP>(stage(n), [&](int r) {
            uint32_t none;
            asm volatile("ld.shared.b32 %0, [%1];" : "=r"(none) : "r"(hollows + n / 2 % kSlots * 16 + r / 32 * 4) : "memory");
            return (none >> (r & 31) & 1) == 0;
          });
        return true;
      };
      if (steps > 0 && ok) {
        ok = arrived(0);
        tc_fence_after();
        if (ok && elect_one()) {
          issue_scores<T, DP>(ts, base, stage(0));
          mma_commit(sfull);
        }
        __syncwarp();
        ok = ok && arrived(1);
        tc_fence_after();
        if (ok && elect_one()) {
          issue_scores<T, DP>(tp, base + L::kTileBytes, stage(1));
          mma_commit(dpfull);
        }
        __syncwarp();
      }
      for (int i = 0; i < steps && ok; ++i) {
        const bool more = i + 1 < steps;
        ok = wait(pfull, (uint32_t)i & 1);
        tc_fence_after();
        if (ok && elect_one()) {
          issue_weighted<T, DP, 32>(tdv, ts, stage(2 * i + 1), i > 0);
          mma_commit(empty((2 * i + 1) % kStages));
        }
        __syncwarp();
        if (more) {
          ok = ok && arrived(2 * i + 2);
          tc_fence_after();
          if (ok && elect_one()) {
            issue_scores<T, DP>(ts, base, stage(2 * i + 2));
            mma_commit(sfull);
          }
          __syncwarp();
        }
        ok = ok && wait(dsfull, (uint32_t)i & 1);
        tc_fence_after();
        if (ok && elect_one()) {
          issue_weighted<T, DP, 32>(tdk, tp, stage(2 * i), i > 0);
          if constexpr (FINE) issue_weighted<T, DP, 32>(tdk, tp + 16, stage(2 * i), true);
          mma_commit(empty((2 * i) % kStages));
        }
        __syncwarp();
        if (more) {
          ok = ok && arrived(2 * i + 3);
          tc_fence_after();
          if (ok && elect_one()) {
            issue_scores<T, DP>(tp, base + L::kTileBytes, stage(2 * i + 3));
            mma_commit(dpfull);
          }
          __syncwarp();
        }
      }
      if (steps > 0 && ok && elect_one()) mma_commit(done);
      __syncwarp();
      // no product may run, and no arrival come, after the block has gone
      if (elect_one()) mma_commit(drained);
      __syncwarp();
      drain_bar(drained, 0);
    }
  } else {
    tc::reg_claim<kRegsWork>();
    const int w = warp >> 2;
    const uint32_t lane_at = (uint32_t)(warp & 3) << 21, mine0 = 32 * w;
    const int key = k0 + (int)(threadIdx.x & 127);
    const float mine = (float)(threadIdx.x & 127);  // key - k0
    const int my = kd ? kd[key] : 0;
    int only = -1;
    if (kd && !lab.bad && lab.lo == lab.hi) only = lab.lo;
    const float f = CAP ? a.cap2 : a.scale;  // raw score, or its tanh -> base 2
    RowScale row_scale;
    // four dS from column c on, in the place of the weights
    auto slopes_at = [&](int c, const uint32_t (&d)[32], uint32_t (&s)[32], uint32_t st, float (&y)[4]) {
      float dl[4];
      tc::ld_shared_f4(st + (kDelta + c) * 4, dl[0], dl[1], dl[2], dl[3]);
#pragma unroll
      for (int q = 0; q < 4; q += 2)
        tc::unpack2(tc::mul2(tc::pack2(__uint_as_float(s[c + q]), __uint_as_float(s[c + q + 1])),
                             tc::fma2(tc::pack2(__uint_as_float(d[c + q]), __uint_as_float(d[c + q + 1])), both(Scales<T>::kUnshift), tc::pack2(dl[q], dl[q + 1]))),
                    y[q], y[q + 1]);
    };
    bool ok = true;
    for (int i = 0; i < steps && ok; ++i) {
      const int slot = i % kStatSlots;
      const uint32_t st = base + L::kStatAt + slot * kStatWords * 4 + mine0 * 4;
      ok = wait(statfull(slot), (uint32_t)(i / kStatSlots) & 1);
      ok = ok && wait(sfull, (uint32_t)i & 1);
      if (!ok) break;
      tc_fence_after();
      const Tile e = get_tile(slots, i);
      const bool whole = k0 + kTile <= lim.row_end((e.at * kTile) >> t.pg_shift, a.causal) && (kd == nullptr || (e.label >= 0 && e.label == only));
      uint32_t seen = 0xffffffffu;  // columns (queries) that see this thread's key
      if (!whole) {
        // under a causal mask the queries from one on, and those that exist
        const int row0 = e.at * kTile + (int)mine0;
        const int from = a.causal && key >= lim.prefix ? min(max(key - lim.start, 0), a.nq) << t.pg_shift : 0;
        seen = key < lim.len ? columns_before(t.rows - row0) & ~columns_before(from - row0) : 0;
        if (kd != nullptr) {
          int label;
          asm volatile("ld.shared.b32 %0, [%1];" : "=r"(label) : "r"(st + (kLabel + (threadIdx.x & 31)) * 4) : "memory");
          seen &= same_label(label, my);
        }
      }
      uint32_t s[1][32];
      uint32_t pr[32];
      tmem_read32(ts + lane_at + mine0, s[0]);
      if constexpr (CAP) to_tanh(s, t.tanh, a.scale);
#pragma unroll
      for (int c = 0; c < 32; c += 4) {
        const uint32_t at = st + c * 4;
        float x[4], add[4];
        tc::ld_shared_f4(at + kLse * 4, add[0], add[1], add[2], add[3]);
        if constexpr (BIAS) {
          float sl[4], ps[4];
          tc::ld_shared_f4(at + kSlope * 4, sl[0], sl[1], sl[2], sl[3]);
          tc::ld_shared_f4(at + kPos * 4, ps[0], ps[1], ps[2], ps[3]);
#pragma unroll
          for (int q = 0; q < 4; ++q) add[q] = fmaf(sl[q], fabsf(ps[q] - mine), add[q]);
        }
#pragma unroll
        for (int q = 0; q < 4; q += 2)
          tc::unpack2(tc::fma2(tc::pack2(__uint_as_float(s[0][c + q]), __uint_as_float(s[0][c + q + 1])), both(f), tc::pack2(add[q], add[q + 1])), x[q], x[q + 1]);
#pragma unroll
        for (int q = 0; q < 4; ++q) pr[c + q] = __float_as_uint(ex2_approx(x[q]));
      }
      if (!whole) {
#pragma unroll
        for (int c = 0; c < 32; ++c)
          if ((seen & (1u << c)) == 0) pr[c] = 0;
      }
#pragma unroll
      for (int p = 0; p < 4; ++p) {
        uint32_t o[4];
#pragma unroll
        for (int c = 8 * p; c < 8 * p + 8; c += 2) {
          const float p0 = __uint_as_float(pr[c]), p1 = __uint_as_float(pr[c + 1]);
          weight_slope<CAP>(s[0][c], s[0][c + 1], p0, p1);
          o[c % 8 / 2] = pack16<T>(p0, p1);
        }
        tmem_st4(ts + lane_at + mine0 + 4 * p, o);
      }
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (elect_one()) mbar_arrive(pfull);
      __syncwarp();
      ok = wait(dpfull, (uint32_t)i & 1);
      if (!ok) break;
      tc_fence_after();
      uint32_t d[32];
      tmem_read32(tp + lane_at + mine0, d);
      if constexpr (Scales<T>::kHalf) {
        float top = 0.f;
#pragma unroll
        for (int c = 0; c < 32; c += 4) {
          float y[4];
          slopes_at(c, d, s[0], st, y);
          top = fmaxf(fmaxf(top, fabsf(y[0])), fabsf(y[1]));
          top = fmaxf(fmaxf(top, fabsf(y[2])), fabsf(y[3]));
#pragma unroll
          for (int q = 0; q < 4; ++q) s[0][c + q] = __float_as_uint(y[q]);
        }
        put_top(base + L::kTops, w, top);
        __syncwarp();
        if (elect_one()) mbar_arrive(xbar(warp & 3));
        __syncwarp();
        ok = wait(xbar(warp & 3), (uint32_t)i & 1);
        if (!ok) break;
        float change;
        const bool changes = row_scale.follow(largest_top(base + L::kTops), change);
        // dP of this step is here, and was issued behind dK of the last one: nothing works on the accumulator
        if (__any_sync(0xffffffffu, changes) && i > 0) rescale_quarter<DP>(tdk + lane_at + w * (DP / 4), change);
      }
#pragma unroll
      for (int p = 0; p < 4; ++p) {
        uint32_t o[4], lo[4];
#pragma unroll
        for (int c = 8 * p; c < 8 * p + 8; c += 4) {
          float y[4];
          if constexpr (Scales<T>::kHalf) {
#pragma unroll
            for (int q = 0; q < 4; q += 2)
              tc::unpack2(tc::mul2(tc::pack2(__uint_as_float(s[0][c + q]), __uint_as_float(s[0][c + q + 1])), both(row_scale.now)), y[q], y[q + 1]);
          } else {
            slopes_at(c, d, s[0], st, y);
          }
          o[c % 8 / 2] = pack16<T>(y[0], y[1]);
          o[c % 8 / 2 + 1] = pack16<T>(y[2], y[3]);
          if constexpr (FINE) {
            lo[c % 8 / 2] = left_over<T>(y[0], y[1], o[c % 8 / 2]);
            lo[c % 8 / 2 + 1] = left_over<T>(y[2], y[3], o[c % 8 / 2 + 1]);
          }
        }
        tmem_st4(tp + lane_at + mine0 + 4 * p, o);
        if constexpr (FINE) tmem_st4(tp + lane_at + mine0 + 16 + 4 * p, lo);
      }
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (elect_one()) {
        mbar_arrive(dsfull);
        mbar_arrive(statempty(slot));
      }
      __syncwarp();
    }
    if (steps > 0 && ok) ok = wait(done, 0);
    tc_fence_after();
    {
      const bool exists = key < a.nk;
      const bool zero = key >= lim.len || (kd != nullptr && my < 0);  // keys that nobody sees
      const int c0 = w * (DP / 4);
      T* rk = reinterpret_cast<T*>(a.dk.p) + b * a.dk.sb + (int64_t)key * a.dk.sn + hk * a.dk.sh;
      T* rv = reinterpret_cast<T*>(a.dv.p) + b * a.dv.sb + (int64_t)key * a.dv.sn + hk * a.dv.sh;
      float *pk = nullptr, *pv = nullptr;
      if (t.splits > 1) {
        const int64_t n = (int64_t)a.b * a.nk * a.hk * a.d, at = (((int64_t)b * a.nk + key) * a.hk + hk) * a.d;
        pk = t.part_o + (int64_t)split * 2 * n + at;
        pv = pk + n;
      }
      if (ok && steps > 0) {
        // the ring is free: all products are done, and with them all copies
        const uint32_t room = base + L::kRing + warp * 4096;
        const float undo = Scales<T>::kHalf ? row_scale.undo(a.scale_raw) : a.scale_raw;
        const int lane = threadIdx.x & 31, first = key - lane, rows = a.nk - first;
        if (pk != nullptr) {
          const int64_t step = (int64_t)a.hk * a.d;
          store_partial<DP>(tdk + lane_at, c0, undo, zero, a.d, room, [&](int r) { return r < rows ? pk + (r - lane) * step : nullptr; });
          store_partial<DP>(tdv + lane_at, c0, Scales<T>::kUnshift, zero, a.d, room, [&](int r) { return r < rows ? pv + (r - lane) * step : nullptr; });
        } else {
          store_quarter<T, DP>(tdk + lane_at, c0, undo, zero, a.d, room, [&](int r) { return r < rows ? rk + (r - lane) * a.dk.sn : nullptr; });
          store_quarter<T, DP>(tdv + lane_at, c0, Scales<T>::kUnshift, zero, a.d, room, [&](int r) { return r < rows ? rv + (r - lane) * a.dv.sn : nullptr; });
        }
      } else {
        store_same<T, DP>(!ok, c0, exists, a.d, rk, pk);
        store_same<T, DP>(!ok, c0, exists, a.d, rv, pv);
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

// Adds the partial results of dK and dV: four values per thread.
template <typename T>
__global__ void __launch_bounds__(256) add_parts_kernel(const TcArgs t) {
  const Args& a = t.a;
  const int64_t n = (int64_t)a.b * a.nk * a.hk * a.d, at = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
  if (at >= n) return;
  const int c = (int)(at % a.d);
  const int64_t row = at / a.d;
  const int hk = (int)(row % a.hk), j = (int)(row / a.hk % a.nk), b = (int)(row / a.hk / a.nk);
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int p = 0; p < t.splits; ++p) {
      const float4 v = *reinterpret_cast<const float4*>(t.part_o + ((int64_t)p * 2 + which) * n + at);
      s.x += v.x, s.y += v.y, s.z += v.z, s.w += v.w;
    }
    const Tensor4& o = which == 0 ? a.dk : a.dv;
    T* out = reinterpret_cast<T*>(o.p) + b * o.sb + (int64_t)j * o.sn + hk * o.sh + c;
    *reinterpret_cast<uint2*>(out) = make_uint2(pack16<T>(s.x, s.y), pack16<T>(s.z, s.w));
  }
}

// ---------------------------------------------------------------------------------------------------------------------
// dQ
// ---------------------------------------------------------------------------------------------------------------------
template <typename T, int DP, bool CAP, bool BIAS, bool FINE>
__global__ void __launch_bounds__(kThreads, 1) kernel_queries(const __grid_constant__ Maps maps, const TcArgs t) {
  using L = Layout<DP, false>;
  constexpr int kStages = L::kStages;
  extern __shared__ __align__(1024) uint8_t raw[];
  const Args& a = t.a;
  const uint32_t base = smem_u32(raw), bars = base + L::kBars;
  auto full = [&](int s) { return bars + s * 8; };
  auto empty = [&](int s) { return bars + 64 + s * 8; };
  auto sfull = [&](int s) { return bars + 128 + s * 8; };
  const uint32_t own = bars + 144, dpfull = bars + 152, dsfull = bars + 160, done = bars + 168, tmem_at = bars + 176, drained = bars + 184, slots = bars + 256;
  auto xbar = [&](int q) { return bars + 384 + q * 8; };
  auto wait = [&](uint32_t bar, uint32_t parity) { return wait_bar(bar, parity, t.wait_ns); };
  const int warp = threadIdx.x >> 5;
  if (threadIdx.x < 4) prefetch_map(threadIdx.x == 0 ? &maps.k : threadIdx.x == 1 ? &maps.v : threadIdx.x == 2 ? &maps.q : &maps.dout);

  uint32_t id = blockIdx.x;
  const int hp = (int)(id % (uint32_t)t.hp);
  id /= (uint32_t)t.hp;
  const int b = (int)(id % (uint32_t)a.b);
  const int row0 = (t.blocks - 1 - (int)(id / (uint32_t)a.b)) * kTile, hk = (int)((uint32_t)(hp * t.pg) / (uint32_t)a.grp);
  const int i0 = row0 >> t.pg_shift, i1 = min(a.nq, (row0 + kTile) >> t.pg_shift);
  const Limits lim = limits_of(a, b);
  const int* kd = a.kdocs ? a.kdocs + (int64_t)b * a.nk_pad : nullptr;
  const int* qd = a.qdocs ? a.qdocs + (int64_t)b * a.nq_pad : nullptr;
  const int4* ktab = kd ? a.ktab + (int64_t)b * (a.nk_pad / kTile) : nullptr;
  const int last = (lim.row_end(i1 - 1, a.causal) + kTile - 1) / kTile;
  // what a working thread has to know of its row; asked for first, so that its time is that of the tables below
  const int r = row0 + (int)(threadIdx.x & 127), i = r >> t.pg_shift, h = hp * t.pg + (r & (t.pg - 1));
  const bool exists = warp < kMmaWarp && r < t.rows;
  float lse = -INFINITY, delta = 0.f, slope = 0.f;
  int my = -2;
  if (exists) {
    const int64_t row = ((int64_t)b * a.hq + h) * a.nq + i;
    lse = __ldg(a.lse + row);
    delta = __ldg(a.delta + row);
    if (qd) my = __ldg(qd + i);
    if (BIAS && a.slopes != nullptr) slope = __ldg(a.slopes + h);
  }
  LabelRange lab{0, 0, false};
  if (kd) lab = labels_of(qd, i0, i1);
  const int steps = count_tiles(ktab, 0, last, lab.lo, lab.hi);

  if (warp == kLoadWarp) {
    if (elect_one()) {
      for (int s = 0; s < kStages; ++s) mbar_init(full(s), 1), mbar_init(empty(s), 1);
      mbar_init(own, 1), mbar_init(sfull(0), 1), mbar_init(sfull(1), 1), mbar_init(dpfull, 1), mbar_init(dsfull, 16), mbar_init(done, 1), mbar_init(drained, 1);
      if constexpr (Scales<T>::kHalf)
        for (int q = 0; q < 4; ++q) mbar_init(xbar(q), 4);
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
  auto ts = [&](int i) { return tmem + (uint32_t)(i & 1) * 128; };
  const uint32_t tp = tmem + 256, tdq = tmem + 384;

  if (warp >= kMmaWarp) {
    tc::reg_release<kRegsOther>();
    if (warp == kLoadWarp) {
      bool ok = true;
      if (steps > 0 && elect_one()) {
        mbar_expect_tx(own, 2 * L::kTileBytes);
#pragma unroll
        for (int c = 0; c < DP / 64; ++c) {
          tma_load(base + c * kBlockBytes, &maps.q, c * 64, hp * t.pg, i0, b, own);
          tma_load(base + L::kTileBytes + c * kBlockBytes, &maps.dout, c * 64, hp * t.pg, i0, b, own);
        }
      }
      __syncwarp();
      TileWalk walk(ktab, 0, last, lab.lo, lab.hi);
      int n = 0;
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
              tma_load(base + L::kRing + s * L::kTileBytes + c * kBlockBytes, kv == 0 ? &maps.k : &maps.v, c * 64, hk, e.at * kTile, b, full(s));
          }
          __syncwarp();
          ++n;
        }
      }
      if (steps > 0) drain_bar(own, 0);
      for (int i = n > kStages ? n - kStages : 0; i < n; ++i) drain_bar(full(i % kStages), (uint32_t)(i / kStages) & 1);
    } else if (warp == kMmaWarp) {
      bool ok = steps == 0 || (t.wait_ns != 0 && wait(own, 0));
      auto stage = [&](int n) { return base + L::kRing + (uint32_t)(n % kStages) * L::kTileBytes; };
      auto ready = [&](int n) { return wait(full(n % kStages), (uint32_t)(n / kStages) & 1); };
      // keys that nobody may see: their weights are zero, and what these meet, dP and K, has to be finite
      auto arrived = [&](int n) {
        if (!ready(n)) return false;
        const Tile e = get_tile(slots, n / 2);
        if (e.dirty || (e.at + 1) * kTile > lim.len) clean_tile<DP>(stage(n), e.at * kTile, lim.len, kd);
        return true;
      };
      auto scores = [&](int i) {
        if (!arrived(2 * i)) return false;
        tc_fence_after();
        if (elect_one()) {
          issue_scores<T, DP>(ts(i), base, stage(2 * i));
          mma_commit(sfull(i & 1));
        }
        __syncwarp();
        return true;
      };
      auto products = [&](int i) {
        if (!arrived(2 * i + 1)) return false;
        tc_fence_after();
        if (elect_one()) {
          issue_scores<T, DP>(tp, base + L::kTileBytes, stage(2 * i + 1));
          mma_commit(dpfull);
          mma_commit(empty((2 * i + 1) % kStages));
        }
        __syncwarp();
        return true;
      };
      if (steps > 0) ok = ok && scores(0) && products(0) && (steps == 1 || scores(1));
      for (int i = 0; i < steps && ok; ++i) {
        ok = wait(dsfull, (uint32_t)i & 1);
        tc_fence_after();
        if (i + 1 < steps) ok = ok && products(i + 1);
        if (ok && elect_one()) {
          issue_weighted<T, DP, 32>(tdq, ts(i), stage(2 * i), i > 0);
          if constexpr (FINE) issue_weighted<T, DP, 32>(tdq, ts(i) + 16, stage(2 * i), true);
          mma_commit(empty((2 * i) % kStages));
        }
        __syncwarp();
        if (i + 2 < steps) ok = ok && scores(i + 2);
      }
      if (steps > 0 && ok && elect_one()) mma_commit(done);
      __syncwarp();
      // no product may run, and no arrival come, after the block has gone
      if (elect_one()) mma_commit(drained);
      __syncwarp();
      drain_bar(drained, 0);
    }
  } else {
    tc::reg_claim<kRegsWork>();
    const int w = warp >> 2;
    const uint32_t lane_at = (uint32_t)(warp & 3) << 21, mine0 = 32 * w;
    const int end = exists ? lim.row_end(i, a.causal) : 0;
    const float slope2 = slope * kLog2e;
    const int pos = lim.at + i;
    const int all_before = lim.row_end(i0, a.causal);
    int only = -1;
    if (kd && !lab.bad && lab.lo == lab.hi) only = lab.lo;
    const float f = CAP ? a.cap2 : a.scale;
    RowScale row_scale;
    // a row that sees nothing has no weights, and no delta, which may be NaN there
    const float add = lse == -INFINITY ? -INFINITY : -lse * kLog2e, nd = lse == -INFINITY ? 0.f : -delta;
    bool ok = true;
    for (int step = 0; step < steps && ok; ++step) {
      ok = wait(sfull(step & 1), (uint32_t)(step >> 1) & 1);
      if (!ok) break;
      tc_fence_after();
      const Tile e = get_tile(slots, step);
      const int k0 = e.at * kTile;
      const bool whole = k0 + kTile <= all_before && (kd == nullptr || (e.label >= 0 && e.label == only));
      uint32_t seen = 0xffffffffu;
      if (!whole) {
        seen = columns_before(end - k0 - (int)mine0);
        if (kd != nullptr) seen &= same_label(__ldg(kd + k0 + (int)mine0 + (int)(threadIdx.x & 31)), my);
      }
      uint32_t s[1][32];
      const uint32_t at = ts(step) + lane_at + mine0;
      tmem_read32(at, s[0]);
      const float d0 = (float)(pos - k0 - (int)mine0);
      if constexpr (CAP) to_tanh(s, t.tanh, a.scale);
#pragma unroll
      for (int c = 0; c < 32; c += 2) {
        float x[2];
        tc::unpack2(tc::fma2(tc::pack2(__uint_as_float(s[0][c]), __uint_as_float(s[0][c + 1])), both(f), both(add)), x[0], x[1]);
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          if constexpr (BIAS) x[q] = fmaf(-slope2, fabsf(d0 - (float)(c + q)), x[q]);
          x[q] = ex2_approx(x[q]);
        }
        weight_slope<CAP>(s[0][c], s[0][c + 1], x[0], x[1]);
      }
      if (!whole) {
#pragma unroll
        for (int c = 0; c < 32; ++c)
          if ((seen & (1u << c)) == 0) s[0][c] = 0;
      }
      ok = wait(dpfull, (uint32_t)step & 1);
      if (!ok) break;
      tc_fence_after();
      uint32_t d[32];
      tmem_read32(tp + lane_at + mine0, d);
      auto slopes_at = [&](int c, float (&y)[2]) {  // two dS, in the place of the weights
        tc::unpack2(tc::mul2(tc::pack2(__uint_as_float(s[0][c]), __uint_as_float(s[0][c + 1])),
                             tc::add2(tc::pack2(__uint_as_float(d[c]), __uint_as_float(d[c + 1])), both(nd))),
                    y[0], y[1]);
      };
      if constexpr (Scales<T>::kHalf) {
        float top = 0.f;
#pragma unroll
        for (int c = 0; c < 32; c += 2) {
          float y[2];
          slopes_at(c, y);
          top = fmaxf(fmaxf(top, fabsf(y[0])), fabsf(y[1]));
          s[0][c] = __float_as_uint(y[0]);
          s[0][c + 1] = __float_as_uint(y[1]);
        }
        put_top(base + L::kTops, w, top);
        __syncwarp();
        if (elect_one()) mbar_arrive(xbar(warp & 3));
        __syncwarp();
        ok = wait(xbar(warp & 3), (uint32_t)step & 1);
        if (!ok) break;
        float change;
        const bool changes = row_scale.follow(largest_top(base + L::kTops), change);
        if (__any_sync(0xffffffffu, changes) && step > 0) {
          // dP of this step was issued ahead of dQ of the last one, which gives its keys' place in the ring back when it is done
          const int n = 2 * (step - 1);
          ok = wait(empty(n % kStages), (uint32_t)(n / kStages) & 1);
          if (!ok) break;
          tc_fence_after();
          rescale_quarter<DP>(tdq + lane_at + w * (DP / 4), change);
        }
      }
#pragma unroll
      for (int p = 0; p < 4; ++p) {
        uint32_t o[4], lo[4];
#pragma unroll
        for (int c = 8 * p; c < 8 * p + 8; c += 2) {
          float y[2];
          if constexpr (Scales<T>::kHalf) {
            tc::unpack2(tc::mul2(tc::pack2(__uint_as_float(s[0][c]), __uint_as_float(s[0][c + 1])), both(row_scale.now)), y[0], y[1]);
          } else {
            slopes_at(c, y);
          }
          o[c % 8 / 2] = pack16<T>(y[0], y[1]);
          if constexpr (FINE) lo[c % 8 / 2] = left_over<T>(y[0], y[1], o[c % 8 / 2]);
        }
        tmem_st4(at + 4 * p, o);
        if constexpr (FINE) tmem_st4(at + 16 + 4 * p, lo);
      }
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (elect_one()) mbar_arrive(dsfull);
      __syncwarp();
    }
    if (steps > 0 && ok) ok = wait(done, 0);
    tc_fence_after();
    {
      T* row = reinterpret_cast<T*>(a.dq.p) + b * a.dq.sb + (int64_t)i * a.dq.sn + h * a.dq.sh;
      const int c0 = w * (DP / 4);
      if (ok && steps > 0)
        store_quarter<T, DP>(tdq + lane_at, c0, Scales<T>::kHalf ? row_scale.undo(a.scale_raw) : a.scale_raw, add == -INFINITY, a.d, base + L::kRing + warp * 4096, [&](int e) {
          const int rr = r - (int)(threadIdx.x & 31) + e;
          return rr < t.rows ? reinterpret_cast<T*>(a.dq.p) + b * a.dq.sb + (int64_t)(rr >> t.pg_shift) * a.dq.sn + (hp * t.pg + (rr & (t.pg - 1))) * a.dq.sh
                             : nullptr;
        });
      else
        store_same<T, DP>(!ok, c0, exists, a.d, row, nullptr);
    }
    tc_fence_before();
  }
  __syncthreads();
  if (warp == kMmaWarp) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

struct Plan {
  int pg, pg_shift, hp, rows, q_blocks, splits;
};
inline Plan make_plan(int b, int nq, int nk, int hq, int hk, int d, bool causal, bool documents) {
  Plan p{};
  const int grp = hq / hk;
  p.pg = fwd::packed_heads(hq, hk);
  while ((1 << p.pg_shift) < p.pg) ++p.pg_shift;
  p.hp = hq / p.pg;
  p.rows = nq * p.pg;
  p.q_blocks = (int)ceil_div(p.rows, kTile);
  // parts of a key tile's query tiles: few or uneven key tiles would leave SMs without work.  The lowest estimate, the
  // traffic of the partial results included; a step takes about 1.6 us with heads of 128, 1 us with heads of 64
  const int64_t blocks = ceil_div(nk, kTile) * hk * b, steps = (int64_t)p.q_blocks * (grp / p.pg);
  const double step = d <= 64 ? 1.0 : 1.6, added = (double)b * nk * hk * d * 16.0 / 5e6;
  // The labels are not known here.  Documents are taken to be half a row long, as forward: over 14 shapes (1024 to 16384 rows, 1 to
  // 12 key heads, both masks) of rows with 1 to 100 documents, equal, growing in steps or doubling, the number of parts that
  // follows costs 2% more than the best one on average, and 25% at most; with a quarter 4% and 35%, an eighth 5% and 71%, the
  // whole row 3% and 37% (8192 rows of 30 equal documents, heads of 128: 1 part 101 us, 2 99, 4 123; of one document: 964, 542, 525).
  const double longest = documents ? 0.5 * (double)steps : (double)steps, mean = causal ? 0.5 * longest : longest;
  p.splits = 1;
  double best = 1e300;
  for (int64_t s = 1; s <= 32 && (s == 1 || s * 4 <= steps); ++s) {
    const double cost = fwd::time_of(blocks, s, longest, mean, step, causal || documents) + (s > 1 ? 3 + s * added : 0);
    if (cost < best * 0.98) best = cost, p.splits = (int)s;
  }
  return p;
}
inline int64_t partial_floats(const Plan& p, int64_t b, int64_t nk, int64_t hk, int64_t d) { return p.splits > 1 ? 2 * p.splits * b * nk * hk * d : 0; }

template <typename T, int DP, bool CAP, bool BIAS, bool FINE>
inline int launch_one(const Maps& m, const TcArgs& t, cudaStream_t st) {
  const Args& a = t.a;
  if (a.dk.p != nullptr) {
    auto* fn = kernel_keys<T, DP, CAP, BIAS, FINE>;
    constexpr int kBytes = (int)Layout<DP, true>::kBytes;
    static std::atomic<uint64_t> done{0};
    FLK_TRY(allow_shared(reinterpret_cast<const void*>(fn), kBytes, done));
    const int64_t grid = ceil_div(a.nk, kTile) * t.splits * a.b * a.hk;
    if (grid > INT32_MAX) return fail(FLK_ERR_UNSUPPORTED, "too many key blocks");
    fn<<<(unsigned)grid, kThreads, kBytes, st>>>(m, t);
    count_launch();
    if (t.splits > 1) {
      add_parts_kernel<T><<<(unsigned)ceil_div((int64_t)a.b * a.nk * a.hk * a.d / 4, 256), 256, 0, st>>>(t);
      count_launch();
    }
  }
  if (a.dq.p != nullptr) {
    auto* fn = kernel_queries<T, DP, CAP, BIAS, FINE>;
    constexpr int kBytes = (int)Layout<DP, false>::kBytes;
    static std::atomic<uint64_t> done{0};
    FLK_TRY(allow_shared(reinterpret_cast<const void*>(fn), kBytes, done));
    const int64_t grid = (int64_t)t.blocks * a.b * t.hp;
    if (grid > INT32_MAX) return fail(FLK_ERR_UNSUPPORTED, "too many row blocks");
    fn<<<(unsigned)grid, kThreads, kBytes, st>>>(m, t);
    count_launch();
  }
  return FLK_OK;
}

template <typename T, int DP, bool FINE>
inline int launch_some(const Maps& m, const TcArgs& t, cudaStream_t st) {
  const bool bias = t.a.slopes != nullptr;
  if (t.a.cap2 != 0.f) return bias ? launch_one<T, DP, true, true, FINE>(m, t, st) : launch_one<T, DP, true, false, FINE>(m, t, st);
  return bias ? launch_one<T, DP, false, true, FINE>(m, t, st) : launch_one<T, DP, false, false, FINE>(m, t, st);
}

template <typename T>
inline int launch(TcArgs t, const Plan& p, cudaStream_t st) {
  const Args& a = t.a;
  t.wait_ns = wait_limit();
  const int dtype = std::is_same<T, __nv_bfloat16>::value ? FLK_BF16 : FLK_F16;
  t.pg = p.pg, t.pg_shift = p.pg_shift, t.hp = p.hp, t.rows = p.rows, t.blocks = p.q_blocks, t.splits = p.splits;
  t.tanh = make_tanh(a.scale);
  Maps m;
  FLK_TRY(make_map(&m.q, a.q, dtype, a.d, a.hq, a.nq, a.b, p.pg, kTile / p.pg));
  FLK_TRY(make_map(&m.dout, a.dout, dtype, a.d, a.hq, a.nq, a.b, p.pg, kTile / p.pg));
  FLK_TRY(make_map(&m.k, a.k, dtype, a.d, a.hk, a.nk, a.b, 1, kTile));
  FLK_TRY(make_map(&m.v, a.v, dtype, a.d, a.hk, a.nk, a.b, 1, kTile));
  const bool fine = a.nq <= 256 && a.nk <= 256;
  if (a.d <= 64) return fine ? launch_some<T, 64, true>(m, t, st) : launch_some<T, 64, false>(m, t, st);
  return fine ? launch_some<T, 128, true>(m, t, st) : launch_some<T, 128, false>(m, t, st);
}

}  // namespace bwd
}  // namespace attn
}  // namespace flk
