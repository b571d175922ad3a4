// Attention of fp32 data on the FP32 pipe, forward and backward.
//
// Tiles of 64 queries x 64 keys, worked on by groups of 256 threads; a thread owns a 4 x 4 patch of the scores (rows 4 ty ..
// 4 ty + 3, columns tx + 16 c) and 4 rows x DM / 16 columns of the accumulators.  Operands come by cp.async: in the forward pass one tile
// ahead of the one that is worked on, in the backward pass while the other group works; rows that no query may see arrive as zeros, so what such rows hold (NaN, infinities) reaches nothing.  All sums run in
// fp32, in pairs (packed multiply-adds), in a fixed order.  Bound by the FP32 pipe and by the shared-memory reads that feed it:
// per 4 values of d a thread reads 8 vectors for 64 multiply-adds.
//
// With heads of up to 64 a block has two groups: one takes the even tiles, one the odd, with accumulators of their own that are
// joined at the end.  Eight warps on an SM would leave its pipes idle for most of the dependent steps (2 x 1000 rows, 4 heads of
// 64, not causal, capped scores, 128 blocks: forward 93 -> 77 us, dK and dV 170 -> 147 us, dQ 133 -> 108 us).  Larger heads leave no
// room for a second set of tiles.  A training pass of 2 x 1000 rows and 4 heads of 128 takes 614 us, as long as elementary torch
// operations, whose products are a library's.  dK and dV have a block per 64 keys of a key head, whatever the number of query heads
// that share it: 1000 rows with 8 heads on one take 1270 us (heads of 64) and 2510 (of 128) on 16 blocks, 0.40 and 0.24 of the speed of
// those elementary operations.
#pragma once

#include "flk_attn_fwd.cuh"

namespace flk {
namespace attn {
namespace simt {

constexpr int kT = 64;
constexpr int kThreads = 256;  // of a group
constexpr int kPs = kT + 4;    // row length of the score tiles in shared memory

template <int DM>
struct Smem {
  static constexpr int kLd = DM + 4;
  static constexpr int kRows = kT * kLd;  // floats of one operand tile
  static constexpr int kPair = kT * kPs;  // floats of one score tile
  static constexpr int kGroups = DM == 64 ? 2 : 1;
};

// A barrier of the threads of one group (number `g`), or of the block where it has one group.
template <int GROUPS>
__device__ __forceinline__ void sync_group(int g) {
  if constexpr (GROUPS == 1)
    __syncthreads();
  else
    asm volatile("barrier.cta.sync %0, %1;" ::"r"(g + 1), "n"(kThreads) : "memory");
}

// rows [r0, r0 + 64) of one head on their way into shared memory; rows at or behind `end`, rows without a label, and queries that
// see nothing (a log-sum-exp of -inf) as zeros
template <int DM>
__device__ __forceinline__ void fetch_tile(float* dst, const Tensor4& t, int b, int h, int r0, int end, int d, const int* docs, int tid,
                                           const float* lse = nullptr) {
  const float* src = (const float*)t.p + b * t.sb + h * t.sh;
  const uint32_t to = tc::smem_u32(dst);
#pragma unroll
  for (int e = tid; e < kT * (DM / 4); e += kThreads) {
    const int r = e / (DM / 4), c = (e - r * (DM / 4)) * 4;
    const bool valid = r0 + r < end && c < d && (docs == nullptr || __ldg(docs + r0 + r) >= 0) && (lse == nullptr || __ldg(lse + r0 + r) != -INFINITY);
    // an address inside the tensor even where nothing is read
    const float* s = src + (valid ? (int64_t)(r0 + r) * t.sn + c : 0);
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to + (r * Smem<DM>::kLd + c) * 4), "l"(s), "r"(valid ? 16 : 0) : "memory");
  }
}

// acc[i][j] = sum over d of A[4 ty + i][:] . B[tx + 16 j][:]
template <int DM>
__device__ __forceinline__ void dots(float (&acc)[4][4], const float* A, const float* B, int ty, int tx) {
  constexpr int kLd = Smem<DM>::kLd;
  uint64_t s[4][4] = {};
#pragma unroll 4
  for (int c = 0; c < DM; c += 4) {
    ulonglong2 x[4], y[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = *reinterpret_cast<const ulonglong2*>(A + (4 * ty + i) * kLd + c);
#pragma unroll
    for (int j = 0; j < 4; ++j) y[j] = *reinterpret_cast<const ulonglong2*>(B + (tx + 16 * j) * kLd + c);
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        s[i][j] = tc::fma2(x[i].x, y[j].x, s[i][j]);
        s[i][j] = tc::fma2(x[i].y, y[j].y, s[i][j]);
      }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float u, v;
      tc::unpack2(s[i][j], u, v);
      acc[i][j] = u + v;
    }
}

// acc[i][:] += sum over t of W[t][4 ty + i] * B[t][4 tx + 64 c ..]   (W is stored [t][row])
template <int DM>
__device__ __forceinline__ void outer(uint64_t (&acc)[4][DM / 32], const float* W, const float* B, int ty, int tx) {
  constexpr int kLd = Smem<DM>::kLd;
#pragma unroll 4
  for (int t = 0; t < kT; ++t) {
    const float4 w = *reinterpret_cast<const float4*>(W + t * kPs + 4 * ty);
    const uint64_t ww[4] = {tc::pack2(w.x, w.x), tc::pack2(w.y, w.y), tc::pack2(w.z, w.z), tc::pack2(w.w, w.w)};
#pragma unroll
    for (int c = 0; c < DM / 64; ++c) {
      const ulonglong2 y = *reinterpret_cast<const ulonglong2*>(B + t * kLd + 4 * tx + 64 * c);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        acc[i][2 * c] = tc::fma2(ww[i], y.x, acc[i][2 * c]);
        acc[i][2 * c + 1] = tc::fma2(ww[i], y.y, acc[i][2 * c + 1]);
      }
    }
  }
}

template <int DM>
__device__ __forceinline__ void store_rows(const Tensor4& t, int b, int h, int r0, int n, int d, const uint64_t (&acc)[4][DM / 32], const float (&f)[4],
                                           int ty, int tx) {
  float* dst = (float*)t.p + b * t.sb + h * t.sh;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = r0 + 4 * ty + i;
    if (r >= n) continue;
#pragma unroll
    for (int c = 0; c < DM / 64; ++c) {
      const int col = 4 * tx + 64 * c;
      float x, y, z, w;
      tc::unpack2(acc[i][2 * c], x, y);
      tc::unpack2(acc[i][2 * c + 1], z, w);
      // a row that saw nothing is zero, whatever met its weights of zero
      if (col < d)
        *reinterpret_cast<float4*>(dst + (int64_t)r * t.sn + col) =
            f[i] == 0.f ? make_float4(0.f, 0.f, 0.f, 0.f) : make_float4(x * f[i], y * f[i], z * f[i], w * f[i]);
    }
  }
}

// The thread's 16 raw dots -> scores in base 2 without the distance bias, and, with a cap, the tanh of each in t (else 0).
// tanh is x p(x^2), p of degree 4 (relative error 6e-8, see to_tanh), where the whole warp's arguments lie in [-1/2, 1/2].
__device__ __forceinline__ void scores(const Args& a, float (&s)[4][4], float (&t)[4][4]) {
  if (a.cap2 == 0.f) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        s[i][j] *= a.scale;
        t[i][j] = 0.f;
      }
    return;
  }
  float big = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      t[i][j] = s[i][j] * a.scale;
      big = fmaxf(big, fabsf(t[i][j]));
    }
  if (__all_sync(0xffffffffu, big <= 0.5f)) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float x = t[i][j], z = x * x;
        t[i][j] = x * fmaf(fmaf(fmaf(fmaf(0.017131345346570015f, z, -0.05298423767089844f), z, 0.133247509598732f), z, -0.3333306908607483f), z, 1.0f);
      }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) t[i][j] = tanhf(t[i][j]);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) s[i][j] = a.cap2 * t[i][j];
}
__device__ __forceinline__ float biased(float s, float slope2, int dist) { return fmaf(-slope2, fabsf((float)dist), s); }

// whether the labels of a query tile and a key tile have a common range
__device__ __forceinline__ bool labels_meet(const Args& a, int b, int q0, int k0) {
  if (a.kdocs == nullptr) return true;
  const int4 x = __ldg(a.qtab + (int64_t)b * (a.nq_pad / a.q_rows) + q0 / a.q_rows), y = __ldg(a.ktab + (int64_t)b * (a.nk_pad / kTile) + k0 / kTile);
  return x.y >= y.x && y.y >= x.x;
}

// Joins the two groups' accumulators: acc = acc * mine + the second group's * theirs, through shared memory (kRows floats).
template <int DM>
__device__ __forceinline__ void put_rows(float* room, const uint64_t (&acc)[4][DM / 32], int ty, int tx) {
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int c = 0; c < DM / 64; ++c)
      *reinterpret_cast<ulonglong2*>(room + (4 * ty + i) * Smem<DM>::kLd + 4 * tx + 64 * c) = make_ulonglong2(acc[i][2 * c], acc[i][2 * c + 1]);
}
template <int DM>
__device__ __forceinline__ void add_rows(const float* room, uint64_t (&acc)[4][DM / 32], const float (&mine)[4], const float (&theirs)[4], int ty, int tx) {
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int c = 0; c < DM / 64; ++c) {
      const ulonglong2 v = *reinterpret_cast<const ulonglong2*>(room + (4 * ty + i) * Smem<DM>::kLd + 4 * tx + 64 * c);
      const uint64_t f = tc::pack2(mine[i], mine[i]), g = tc::pack2(theirs[i], theirs[i]);
      acc[i][2 * c] = tc::fma2(acc[i][2 * c], f, tc::mul2(v.x, g));
      acc[i][2 * c + 1] = tc::fma2(acc[i][2 * c + 1], f, tc::mul2(v.y, g));
    }
}

template <int DM>
__global__ void __launch_bounds__(kThreads* Smem<DM>::kGroups) forward_kernel(const TcArgs t) {
  extern __shared__ float sm[];
  const Args& a = t.a;
  constexpr int kRows = Smem<DM>::kRows, kGroups = Smem<DM>::kGroups;
  const int g = threadIdx.x / kThreads, tid = threadIdx.x % kThreads, tx = tid & 15, ty = tid >> 4;
  float *Q = sm, *K = Q + kRows + g * (4 * kRows + Smem<DM>::kPair), *V = K + 2 * kRows, *P = V + 2 * kRows;
  const int q0 = (int)(blockIdx.x / (uint32_t)t.splits) * kT, split = (int)(blockIdx.x % (uint32_t)t.splits), h = blockIdx.y, b = blockIdx.z, hk = h / a.grp;
  const Limits lim = limits_of(a, b);
  const int* qd = a.qdocs ? a.qdocs + (int64_t)b * a.nq_pad : nullptr;
  const int* kd = a.kdocs ? a.kdocs + (int64_t)b * a.nk_pad : nullptr;
  const float slope2 = a.slopes ? a.slopes[h] * kLog2e : 0.f;
  float m[4], l[4];
  uint64_t acc[4][DM / 32] = {};
  int end[4], id[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = q0 + 4 * ty + i;
    end[i] = r < a.nq ? lim.row_end(r, a.causal) : 0;
    id[i] = qd && r < a.nq ? qd[r] : -2;
    m[i] = -INFINITY;
    l[i] = 0.f;
  }
  // the block's keys: its part of those that its rows see, in whole tiles
  const int tiles = (lim.row_end(min(q0 + kT, a.nq) - 1, a.causal) + kT - 1) / kT;
  const int even = (int)((uint32_t)tiles / (uint32_t)t.splits), odd = tiles - even * t.splits;
  const int first = (split * even + min(split, odd)) * kT, last = first + (even + (split < odd ? 1 : 0)) * kT;
  auto next = [&](int k0) {
    while (k0 < last && !labels_meet(a, b, q0, k0)) k0 += kT * kGroups;
    return k0;
  };
  int k0 = next(first + g * kT), buf = 0;
  if (g == 0) fetch_tile<DM>(Q, a.q, b, h, q0, a.nq, a.d, qd, tid);
  if (k0 < last) fetch_tile<DM>(K, a.k, b, hk, k0, lim.len, a.d, kd, tid);
  cp_async_commit();
  if (k0 < last) fetch_tile<DM>(V, a.v, b, hk, k0, lim.len, a.d, kd, tid);
  cp_async_commit();
  cp_async_wait<1>();
  __syncthreads();  // both groups read Q
  while (k0 < last) {
    const int k1 = next(k0 + kT * kGroups);
    if (k1 < last) fetch_tile<DM>(K + (buf ^ 1) * kRows, a.k, b, hk, k1, lim.len, a.d, kd, tid);
    cp_async_commit();
    cp_async_wait<2>();
    sync_group<kGroups>(g);  // K is here; all have done with the weights and values of the tile before
    if (k1 < last) fetch_tile<DM>(V + (buf ^ 1) * kRows, a.v, b, hk, k1, lim.len, a.d, kd, tid);
    cp_async_commit();
    float s[4][4];
    dots<DM>(s, Q, K + buf * kRows, ty, tx);
    float tanh[4][4];
    scores(a, s, tanh);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int pos = lim.at + q0 + 4 * ty + i;
      float top = -INFINITY;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int col = k0 + tx + 16 * j;
        const float v = biased(s[i][j], slope2, pos - col);
        s[i][j] = col < end[i] && (kd == nullptr || kd[col] == id[i]) ? v : -INFINITY;
        top = fmaxf(top, s[i][j]);
      }
      for (int o = 8; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
      const float mn = fmaxf(m[i], top), base = mn == -INFINITY ? 0.f : mn;
      const float f = ex2_approx(m[i] - base);
      m[i] = mn;
      float sum = 0.f;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        s[i][j] = ex2_approx(s[i][j] - base);
        sum += s[i][j];
      }
      for (int o = 8; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      l[i] = fmaf(l[i], f, sum);
      const uint64_t ff = tc::pack2(f, f);
#pragma unroll
      for (int c = 0; c < DM / 32; ++c) acc[i][c] = tc::mul2(acc[i][c], ff);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) *reinterpret_cast<float4*>(P + (tx + 16 * j) * kPs + 4 * ty) = make_float4(s[0][j], s[1][j], s[2][j], s[3][j]);
    cp_async_wait<2>();
    sync_group<kGroups>(g);  // V is here, and the weights
    outer<DM>(acc, P, V + buf * kRows, ty, tx);
    k0 = k1;
    buf ^= 1;
  }
  cp_async_wait<0>();
  if constexpr (kGroups == 2) {
    __syncthreads();
    float *room = sm + kRows, *stats = room + kRows;  // [row][2] behind the rows
    if (g == 1) {
      put_rows<DM>(room, acc, ty, tx);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (tx == 0) stats[2 * (4 * ty + i)] = m[i], stats[2 * (4 * ty + i) + 1] = l[i];
    }
    __syncthreads();
    if (g == 1) return;
    float fm[4], ft[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float mt = stats[2 * (4 * ty + i)], lt = stats[2 * (4 * ty + i) + 1];
      const float mn = fmaxf(m[i], mt), base = mn == -INFINITY ? 0.f : mn;
      fm[i] = ex2_approx(m[i] - base);
      ft[i] = ex2_approx(mt - base);
      // scores that are not numbers leave the maximum at -inf and the sum NaN
      l[i] = (m[i] == -INFINITY ? l[i] : l[i] * fm[i]) + (mt == -INFINITY ? lt : lt * ft[i]);
      m[i] = mn;
    }
    add_rows<DM>(room, acc, fm, ft, ty, tx);
  }
  float f[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = q0 + 4 * ty + i;
    f[i] = l[i] == 0.f ? 0.f : 1.0f / l[i];
    if (tx != 0 || r >= a.nq) continue;
    const float lse2 = l[i] == 0.f ? -INFINITY : m[i] + log2f(l[i]);
    if (t.splits > 1)
      t.part_lse[(((int64_t)split * a.b + b) * a.hq + h) * a.nq + r] = lse2;
    else if (a.lse != nullptr)
      a.lse[((int64_t)b * a.hq + h) * a.nq + r] = lse2 * kLn2;
  }
  // a part's results are rows of [split][b][hq][nq][d]
  const int64_t rows = (int64_t)a.hq * a.nq * a.d;
  const Tensor4 to = t.splits > 1 ? Tensor4{t.part_o + (int64_t)split * a.b * rows, rows, a.d, (int64_t)a.nq * a.d} : a.o;
  store_rows<DM>(to, b, h, q0, a.nq, a.d, acc, f, ty, tx);
}

// Gradients of 64 keys and values: loops over the query heads that share them and over their query tiles.
template <int DM>
__global__ void __launch_bounds__(kThreads* Smem<DM>::kGroups) backward_kv_kernel(const Args a) {
  extern __shared__ float sm[];
  constexpr int kRows = Smem<DM>::kRows, kGroups = Smem<DM>::kGroups;
  const int g = threadIdx.x / kThreads, tid = threadIdx.x % kThreads, tx = tid & 15, ty = tid >> 4;
  float *K = sm, *V = K + kRows, *Q = V + kRows + g * (2 * kRows + 2 * Smem<DM>::kPair), *G = Q + kRows, *P = G + kRows, *W = P + Smem<DM>::kPair;
  const int k0 = blockIdx.x * kT, hk = blockIdx.y, b = blockIdx.z;
  const Limits lim = limits_of(a, b);
  const int* qd = a.qdocs ? a.qdocs + (int64_t)b * a.nq_pad : nullptr;
  const int* kd = a.kdocs ? a.kdocs + (int64_t)b * a.nk_pad : nullptr;
  uint64_t dk[4][DM / 32] = {}, dv[4][DM / 32] = {};
  int id[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) id[i] = kd ? kd[min(k0 + 4 * ty + i, a.nk_pad - 1)] : 0;
  // steps: query tiles of one head after the other
  const int tiles = (a.nq + kT - 1) / kT;
  const int64_t steps = k0 < lim.len ? (int64_t)a.grp * tiles : 0;
  auto next = [&](int64_t s) {
    for (; s < steps; s += kGroups) {
      const int q0 = (int)(s % tiles) * kT;
      if (lim.row_end(min(q0 + kT, a.nq) - 1, a.causal) > k0 && labels_meet(a, b, q0, k0)) break;
    }
    return s;
  };
  const bool hollow = qd != nullptr || lim.row_end(0, a.causal) == 0;  // some query may see nothing
  auto fetch = [&](int64_t s) {
    const int h = hk * a.grp + (int)(s / tiles), q0 = (int)(s % tiles) * kT;
    const float* lse = hollow ? a.lse + ((int64_t)b * a.hq + h) * a.nq : nullptr;
    fetch_tile<DM>(Q, a.q, b, h, q0, a.nq, a.d, nullptr, tid, lse);
    fetch_tile<DM>(G, a.dout, b, h, q0, a.nq, a.d, nullptr, tid, lse);
  };
  int64_t step = next(g);
  if (g == 0) fetch_tile<DM>(K, a.k, b, hk, k0, lim.len, a.d, kd, tid);
  if (g == kGroups - 1) fetch_tile<DM>(V, a.v, b, hk, k0, lim.len, a.d, kd, tid);
  cp_async_commit();
  if (step < steps) fetch(step);
  cp_async_commit();
  cp_async_wait<1>();
  __syncthreads();  // K and V are here
  while (step < steps) {
    const int64_t after = next(step + kGroups);
    const int h = hk * a.grp + (int)(step / tiles), q0 = (int)(step % tiles) * kT;
    const float slope2 = a.slopes ? a.slopes[h] * kLog2e : 0.f;
    const float *lse = a.lse + ((int64_t)b * a.hq + h) * a.nq, *delta = a.delta + ((int64_t)b * a.hq + h) * a.nq;
    float lse2[4], dl[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int r = q0 + tx + 16 * j;
      lse2[j] = r < a.nq ? __ldg(lse + r) * kLog2e : 0.f;
      dl[j] = r < a.nq ? __ldg(delta + r) : 0.f;
    }
    cp_async_wait<0>();
    sync_group<kGroups>(g);
    float s[4][4], dp[4][4];  // rows: keys, columns: queries
    dots<DM>(s, K, Q, ty, tx);
    dots<DM>(dp, V, G, ty, tx);
    float t[4][4];
    scores(a, s, t);
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int key = k0 + 4 * ty + i, r = q0 + tx + 16 * j;
        const float v = biased(s[i][j], slope2, lim.at + r - key);
        const bool see = r < a.nq && key < lim.row_end(r, a.causal) && (kd == nullptr || qd[r] == id[i]);
        s[i][j] = see ? ex2_approx(v - lse2[j]) : 0.f;
        dp[i][j] = see ? s[i][j] * (dp[i][j] - dl[j]) * (1.f - t[i][j] * t[i][j]) : 0.f;
      }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      *reinterpret_cast<float4*>(P + (tx + 16 * j) * kPs + 4 * ty) = make_float4(s[0][j], s[1][j], s[2][j], s[3][j]);
      *reinterpret_cast<float4*>(W + (tx + 16 * j) * kPs + 4 * ty) = make_float4(dp[0][j], dp[1][j], dp[2][j], dp[3][j]);
    }
    sync_group<kGroups>(g);
    outer<DM>(dv, P, G, ty, tx);
    outer<DM>(dk, W, Q, ty, tx);
    sync_group<kGroups>(g);
    if (after < steps) fetch(after);
    cp_async_commit();
    step = after;
  }
  cp_async_wait<0>();
  if constexpr (kGroups == 2) {
    __syncthreads();
    if (g == 1) {
      put_rows<DM>(sm, dk, ty, tx);
      put_rows<DM>(sm + kRows, dv, ty, tx);
    }
    __syncthreads();
    if (g == 1) return;
    const float both[4] = {1.f, 1.f, 1.f, 1.f};
    add_rows<DM>(sm, dk, both, both, ty, tx);
    add_rows<DM>(sm + kRows, dv, both, both, ty, tx);
  }
  const float one[4] = {1.f, 1.f, 1.f, 1.f}, sc[4] = {a.scale_raw, a.scale_raw, a.scale_raw, a.scale_raw};
  store_rows<DM>(a.dk, b, hk, k0, a.nk, a.d, dk, sc, ty, tx);
  store_rows<DM>(a.dv, b, hk, k0, a.nk, a.d, dv, one, ty, tx);
}

// Gradient of 64 queries.
template <int DM>
__global__ void __launch_bounds__(kThreads* Smem<DM>::kGroups) backward_q_kernel(const Args a) {
  extern __shared__ float sm[];
  constexpr int kRows = Smem<DM>::kRows, kGroups = Smem<DM>::kGroups;
  const int g = threadIdx.x / kThreads, tid = threadIdx.x % kThreads, tx = tid & 15, ty = tid >> 4;
  float *Q = sm, *G = Q + kRows, *K = G + kRows + g * (2 * kRows + Smem<DM>::kPair), *V = K + kRows, *W = V + kRows;
  const int q0 = blockIdx.x * kT, h = blockIdx.y, b = blockIdx.z, hk = h / a.grp;
  const Limits lim = limits_of(a, b);
  const int* qd = a.qdocs ? a.qdocs + (int64_t)b * a.nq_pad : nullptr;
  const int* kd = a.kdocs ? a.kdocs + (int64_t)b * a.nk_pad : nullptr;
  const float slope2 = a.slopes ? a.slopes[h] * kLog2e : 0.f;
  uint64_t dq[4][DM / 32] = {};
  float lse2[4], delta[4];
  int end[4], id[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = q0 + 4 * ty + i;
    end[i] = r < a.nq ? lim.row_end(r, a.causal) : 0;
    id[i] = qd && r < a.nq ? qd[r] : -2;
    lse2[i] = r < a.nq ? a.lse[((int64_t)b * a.hq + h) * a.nq + r] * kLog2e : 0.f;
    delta[i] = r < a.nq ? a.delta[((int64_t)b * a.hq + h) * a.nq + r] : 0.f;
  }
  const int last = lim.row_end(min(q0 + kT, a.nq) - 1, a.causal);
  auto next = [&](int k0) {
    while (k0 < last && !labels_meet(a, b, q0, k0)) k0 += kT * kGroups;
    return k0;
  };
  auto fetch = [&](int k0) {
    fetch_tile<DM>(K, a.k, b, hk, k0, lim.len, a.d, kd, tid);
    fetch_tile<DM>(V, a.v, b, hk, k0, lim.len, a.d, kd, tid);
  };
  int k0 = next(g * kT);
  if (g == 0) fetch_tile<DM>(Q, a.q, b, h, q0, a.nq, a.d, qd, tid);
  if (g == kGroups - 1) fetch_tile<DM>(G, a.dout, b, h, q0, a.nq, a.d, qd, tid);
  cp_async_commit();
  if (k0 < last) fetch(k0);
  cp_async_commit();
  cp_async_wait<1>();
  __syncthreads();  // Q and dO are here
  while (k0 < last) {
    const int k1 = next(k0 + kT * kGroups);
    cp_async_wait<0>();
    sync_group<kGroups>(g);
    float s[4][4], dp[4][4];
    dots<DM>(s, Q, K, ty, tx);
    dots<DM>(dp, G, V, ty, tx);
    float t[4][4];
    scores(a, s, t);
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int col = k0 + tx + 16 * j;
        const float v = biased(s[i][j], slope2, lim.at + q0 + 4 * ty + i - col);
        const bool see = col < end[i] && (kd == nullptr || kd[col] == id[i]);
        s[i][j] = see ? ex2_approx(v - lse2[i]) * (dp[i][j] - delta[i]) * (1.f - t[i][j] * t[i][j]) : 0.f;
      }
#pragma unroll
    for (int j = 0; j < 4; ++j) *reinterpret_cast<float4*>(W + (tx + 16 * j) * kPs + 4 * ty) = make_float4(s[0][j], s[1][j], s[2][j], s[3][j]);
    sync_group<kGroups>(g);
    outer<DM>(dq, W, K, ty, tx);
    sync_group<kGroups>(g);
    if (k1 < last) fetch(k1);
    cp_async_commit();
    k0 = k1;
  }
  cp_async_wait<0>();
  if constexpr (kGroups == 2) {
    __syncthreads();
    if (g == 1) put_rows<DM>(sm, dq, ty, tx);
    __syncthreads();
    if (g == 1) return;
    const float both[4] = {1.f, 1.f, 1.f, 1.f};
    add_rows<DM>(sm, dq, both, both, ty, tx);
  }
  const float sc[4] = {a.scale_raw, a.scale_raw, a.scale_raw, a.scale_raw};
  store_rows<DM>(a.dq, b, h, q0, a.nq, a.d, dq, sc, ty, tx);
}

template <int DM>
constexpr size_t forward_smem() { return (Smem<DM>::kRows + Smem<DM>::kGroups * (4 * Smem<DM>::kRows + Smem<DM>::kPair)) * 4; }
template <int DM>
constexpr size_t kv_smem() { return (2 * Smem<DM>::kRows + Smem<DM>::kGroups * (2 * Smem<DM>::kRows + 2 * Smem<DM>::kPair)) * 4; }
template <int DM>
constexpr size_t q_smem() { return (2 * Smem<DM>::kRows + Smem<DM>::kGroups * (2 * Smem<DM>::kRows + Smem<DM>::kPair)) * 4; }
static_assert(forward_smem<64>() <= 227 * 1024 && forward_smem<128>() <= 227 * 1024, "shared memory");
static_assert(kv_smem<64>() <= 227 * 1024 && kv_smem<128>() <= 227 * 1024, "shared memory");

// Parts of the key axis (see fwd::make_plan): a block takes an SM, and about 5 us per tile of 64 keys with heads of 64, 9 with more
// (100 rows over 3000 keys, 4 heads of 64: 206 us in one part, 31 in parts).
inline int splits_of(int b, int nq, int nk, int hq, int d, bool causal, bool documents, bool lens) {
  const int64_t blocks = ceil_div(nq, kT) * hq * b, tiles = ceil_div(nk, kT);
  double mean = (double)tiles;
  if (causal && nk > 0) mean *= 1.0 - 0.5 * (nq < nk ? (double)nq / nk : 1.0);
  if (documents) mean *= 0.5;
  if (lens) mean *= 0.75;
  const double joined = (double)b * hq * nq * d * 8.0 / 5e6;
  int best = 1;
  double least = 1e300;
  for (int64_t s = 1; s <= 64 && (s == 1 || s * 2 <= tiles); ++s) {
    const double cost = fwd::time_of(blocks, s, (double)tiles, mean, d <= 64 ? 5 : 9, mean < 0.95 * (double)tiles) + (s > 1 ? 3 + s * joined : 0);
    if (cost < least * 0.98) least = cost, best = (int)s;
  }
  return best;
}

template <int DM, typename A>
inline int run(void (*fn)(const A), std::atomic<uint64_t>& done, const dim3& grid, size_t smem, const A& a, cudaStream_t st) {
  FLK_TRY(allow_shared(reinterpret_cast<const void*>(fn), (int)smem, done));
  fn<<<grid, kThreads * Smem<DM>::kGroups, smem, st>>>(a);
  count_launch();
  return FLK_OK;
}
template <int DM>
inline int launch_forward(TcArgs t, int splits, cudaStream_t st) {
  static std::atomic<uint64_t> done{0};
  const Args& a = t.a;
  t.pg = 1, t.hp = a.hq, t.rows = a.nq, t.splits = splits;
  FLK_TRY(run<DM>(forward_kernel<DM>, done, dim3((unsigned)(ceil_div(a.nq, kT) * splits), a.hq, a.b), forward_smem<DM>(), t, st));
  return splits > 1 ? fwd::launch_join<float>(t, splits, st) : FLK_OK;
}
template <int DM>
inline int launch_backward(const Args& a, cudaStream_t st) {
  static std::atomic<uint64_t> done_kv{0}, done_q{0};
  if (a.dk.p != nullptr) FLK_TRY(run<DM>(backward_kv_kernel<DM>, done_kv, dim3((unsigned)ceil_div(a.nk, kT), a.hk, a.b), kv_smem<DM>(), a, st));
  if (a.dq.p != nullptr) FLK_TRY(run<DM>(backward_q_kernel<DM>, done_q, dim3((unsigned)ceil_div(a.nq, kT), a.hq, a.b), q_smem<DM>(), a, st));
  return FLK_OK;
}

}  // namespace simt
}  // namespace attn
}  // namespace flk
