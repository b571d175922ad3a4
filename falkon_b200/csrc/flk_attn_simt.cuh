// Attention on the FP32 pipe, forward and backward: fp32 data, and the check of the tensor-core kernels.
//
// Tiles of 64 queries x 64 keys, 256 threads; a thread owns a 4 x 4 patch of the scores (rows 4 ty .. 4 ty + 3, columns
// tx + 16 c) and 4 rows x DM / 16 columns of the accumulators.  Operands are converted to fp32 in shared memory; rows
// that no query may see are written as zeros there, so what such rows hold (NaN, infinities) reaches nothing.  All sums
// run in fp32 in a fixed order.  Bound by the FP32 pipe and by the shared-memory reads that feed it: per 4 values of d a
// thread reads 8 vectors for 64 multiply-adds.
#pragma once

#include "flk_attn.cuh"

namespace flk {
namespace attn {
namespace simt {

constexpr int kT = 64;
constexpr int kThreads = 256;
constexpr int kPs = kT + 4;  // row length of the score tiles in shared memory

template <int DM>
struct Smem {
  static constexpr int kLd = DM + 4;
  static constexpr int kRows = kT * kLd;  // floats of one operand tile
  static constexpr int kPair = kT * kPs;  // floats of one score tile
};

// rows [r0, r0 + 64) of one head into shared memory as fp32; rows at or behind `end`, and rows that the labels rule
// out, as zeros
template <typename T, int DM>
__device__ __forceinline__ void load_tile(float* dst, const T* src, int64_t sn, int r0, int end, int d, const int* docs) {
  constexpr int kLd = Smem<DM>::kLd;
  for (int e = threadIdx.x; e < kT * (DM / 4); e += kThreads) {
    const int r = e / (DM / 4), c = (e - r * (DM / 4)) * 4;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    if (r0 + r < end && c < d && (docs == nullptr || docs[r0 + r] >= 0)) {
      const T* s = src + (int64_t)(r0 + r) * sn + c;
      if constexpr (sizeof(T) == 4) {
        v = *reinterpret_cast<const float4*>(s);
      } else {
        T t[4];
        *reinterpret_cast<uint2*>(t) = *reinterpret_cast<const uint2*>(s);
        v = make_float4(to_f<T>(t[0]), to_f<T>(t[1]), to_f<T>(t[2]), to_f<T>(t[3]));
      }
    }
    *reinterpret_cast<float4*>(dst + r * kLd + c) = v;
  }
}

// acc[i][j] += sum over d of A[4 ty + i][:] . B[tx + 16 j][:]
template <int DM>
__device__ __forceinline__ void dots(float (&acc)[4][4], const float* A, const float* B, int ty, int tx) {
  constexpr int kLd = Smem<DM>::kLd;
#pragma unroll 4
  for (int c = 0; c < DM; c += 4) {
    float4 x[4], y[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = *reinterpret_cast<const float4*>(A + (4 * ty + i) * kLd + c);
#pragma unroll
    for (int j = 0; j < 4; ++j) y[j] = *reinterpret_cast<const float4*>(B + (tx + 16 * j) * kLd + c);
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        acc[i][j] = fmaf(x[i].x, y[j].x, acc[i][j]);
        acc[i][j] = fmaf(x[i].y, y[j].y, acc[i][j]);
        acc[i][j] = fmaf(x[i].z, y[j].z, acc[i][j]);
        acc[i][j] = fmaf(x[i].w, y[j].w, acc[i][j]);
      }
  }
}

// acc[i][:] += sum over t of W[t][4 ty + i] * B[t][4 tx + 64 c ..]   (W is stored [t][row])
template <int DM>
__device__ __forceinline__ void outer(float (&acc)[4][DM / 16], const float* W, const float* B, int ty, int tx) {
  constexpr int kLd = Smem<DM>::kLd;
#pragma unroll 4
  for (int t = 0; t < kT; ++t) {
    const float4 w = *reinterpret_cast<const float4*>(W + t * kPs + 4 * ty);
    const float ww[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int c = 0; c < DM / 64; ++c) {
      const float4 y = *reinterpret_cast<const float4*>(B + t * kLd + 4 * tx + 64 * c);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        acc[i][4 * c + 0] = fmaf(ww[i], y.x, acc[i][4 * c + 0]);
        acc[i][4 * c + 1] = fmaf(ww[i], y.y, acc[i][4 * c + 1]);
        acc[i][4 * c + 2] = fmaf(ww[i], y.z, acc[i][4 * c + 2]);
        acc[i][4 * c + 3] = fmaf(ww[i], y.w, acc[i][4 * c + 3]);
      }
    }
  }
}

template <typename T, int DM>
__device__ __forceinline__ void store_rows(T* dst, int64_t sn, int r0, int n, int d, const float (&acc)[4][DM / 16], const float (&f)[4],
                                           int ty, int tx, T* lo = nullptr) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = r0 + 4 * ty + i;
    if (r >= n) continue;
#pragma unroll
    for (int c = 0; c < DM / 64; ++c)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int col = 4 * tx + 64 * c + e;
        if (col >= d) continue;
        const float y = acc[i][4 * c + e] * f[i];
        dst[(int64_t)r * sn + col] = from_f<T>(y);
        if (lo != nullptr) lo[(int64_t)r * sn + col] = from_f<T>(y - to_f<T>(from_f<T>(y)));
      }
  }
}

// raw dot -> score in base 2; t = tanh of the capped score (0 without a cap)
__device__ __forceinline__ float score(const Args& a, float raw, float slope2, int dist, float& t) {
  float s = raw * a.scale;
  t = 0.f;
  if (a.cap2 != 0.f) {
    t = tanhf(s);
    s = a.cap2 * t;
  }
  return fmaf(-slope2, fabsf((float)dist), s);
}

template <typename T, int DM>
__global__ void __launch_bounds__(kThreads) forward_kernel(const Args a) {
  extern __shared__ float sm[];
  float *Q = sm, *KV = Q + Smem<DM>::kRows, *P = KV + Smem<DM>::kRows;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const int q0 = blockIdx.x * kT, h = blockIdx.y, b = blockIdx.z, hk = h / a.grp;
  const Limits lim = limits_of(a, b);
  const int* qd = a.qdocs ? a.qdocs + (int64_t)b * a.nq_pad : nullptr;
  const int* kd = a.kdocs ? a.kdocs + (int64_t)b * a.nk_pad : nullptr;
  const float slope2 = a.slopes ? a.slopes[h] * kLog2e : 0.f;
  load_tile<T, DM>(Q, (const T*)a.q.p + b * a.q.sb + h * a.q.sh, a.q.sn, q0, a.nq, a.d, qd);
  float m[4], l[4], acc[4][DM / 16];
  int end[4], id[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = q0 + 4 * ty + i;
    end[i] = r < a.nq ? lim.row_end(r, a.causal) : 0;
    id[i] = qd && r < a.nq ? qd[r] : -2;
    m[i] = -INFINITY;
    l[i] = 0.f;
#pragma unroll
    for (int c = 0; c < DM / 16; ++c) acc[i][c] = 0.f;
  }
  const int last = lim.row_end(min(q0 + kT, a.nq) - 1, a.causal);
  for (int k0 = 0; k0 < last; k0 += kT) {
    if (kd != nullptr) {  // no label in common: nothing to see
      const int4 x = a.qtab[(int64_t)b * (a.nq_pad / a.q_rows) + q0 / a.q_rows], y = a.ktab[(int64_t)b * (a.nk_pad / kTile) + k0 / kTile];
      if (x.y < y.x || y.y < x.x) continue;
    }
    __syncthreads();
    load_tile<T, DM>(KV, (const T*)a.k.p + b * a.k.sb + hk * a.k.sh, a.k.sn, k0, lim.len, a.d, kd);
    __syncthreads();
    float s[4][4] = {};
    dots<DM>(s, Q, KV, ty, tx);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int pos = lim.start + q0 + 4 * ty + i;
      float top = -INFINITY;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int col = k0 + tx + 16 * j;
        float t;
        const float v = score(a, s[i][j], slope2, pos - col, t);
        const bool see = col < end[i] && (kd == nullptr || kd[col] == id[i]);
        s[i][j] = see ? v : -INFINITY;
        top = fmaxf(top, s[i][j]);
      }
      for (int o = 8; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
      const float mn = fmaxf(m[i], top), base = mn == -INFINITY ? 0.f : mn;
      const float f = exp2f(m[i] - base);
      m[i] = mn;
      float sum = 0.f;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        s[i][j] = exp2f(s[i][j] - base);
        sum += s[i][j];
      }
      for (int o = 8; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      l[i] = fmaf(l[i], f, sum);
#pragma unroll
      for (int c = 0; c < DM / 16; ++c) acc[i][c] *= f;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) P[(tx + 16 * j) * kPs + 4 * ty + i] = s[i][j];
    __syncthreads();
    load_tile<T, DM>(KV, (const T*)a.v.p + b * a.v.sb + hk * a.v.sh, a.v.sn, k0, lim.len, a.d, kd);
    __syncthreads();
    outer<DM>(acc, P, KV, ty, tx);
  }
  float f[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = q0 + 4 * ty + i;
    f[i] = l[i] == 0.f ? 0.f : 1.0f / l[i];
    if (l[i] == 0.f)
      for (int c = 0; c < DM / 16; ++c) acc[i][c] = 0.f;
    if (tx == 0 && r < a.nq && a.lse != nullptr)
      a.lse[((int64_t)b * a.hq + h) * a.nq + r] = l[i] == 0.f ? -INFINITY : (m[i] + log2f(l[i])) * kLn2;
  }
  store_rows<T, DM>((T*)a.o.p + b * a.o.sb + h * a.o.sh, a.o.sn, q0, a.nq, a.d, acc, f, ty, tx,
                    a.o_lo == nullptr ? nullptr : (T*)a.o_lo + b * a.o.sb + h * a.o.sh);
}

// delta_i = dO_i . O_i, a group of LANES lanes per row of one head (16 bytes of each array per lane), two rows per group at a time,
// and the largest |dO| of the rows that see something (`amax`, as bits, unless null; a maximum does not depend on the order it
// is taken in).  Bound by the bytes of dO, O and what rounding took from O.
template <typename T, int LANES>
__global__ void __launch_bounds__(256) delta_kernel(const Args a, uint32_t* amax) {
  constexpr int kVec = 16 / sizeof(T), kGroups = 256 / LANES;
  const uint32_t n = (uint32_t)a.nq * (uint32_t)a.hq;
  const int b = blockIdx.y, c = (threadIdx.x % LANES) * kVec;
  const T *dout = (const T*)a.dout.p + b * a.dout.sb, *o = (const T*)a.o.p + b * a.o.sb;
  const T* lo = a.o_lo == nullptr ? nullptr : (const T*)a.o_lo + b * a.o.sb;
  float s[2] = {0.f, 0.f}, top[2] = {0.f, 0.f};
  int64_t at[2];
  bool on[2];
  uint4 u[2], w[2], x[2];
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const uint32_t row = (blockIdx.x * 2 + e) * kGroups + threadIdx.x / LANES;  // (i, h), h fastest
    on[e] = row < n;
    const uint32_t i = on[e] ? row / (uint32_t)a.hq : 0, h = on[e] ? row - i * (uint32_t)a.hq : 0;
    at[e] = ((int64_t)b * a.hq + h) * a.nq + i;
    u[e] = w[e] = x[e] = make_uint4(0, 0, 0, 0);
    if (on[e] && c < a.d) {
      const int64_t off = i * a.o.sn + h * a.o.sh + c;
      u[e] = *reinterpret_cast<const uint4*>(dout + i * a.dout.sn + h * a.dout.sh + c);
      w[e] = *reinterpret_cast<const uint4*>(o + off);
      if (lo != nullptr) x[e] = *reinterpret_cast<const uint4*>(lo + off);
    }
  }
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const T *p = reinterpret_cast<const T*>(&u[e]), *q = reinterpret_cast<const T*>(&w[e]), *r = reinterpret_cast<const T*>(&x[e]);
#pragma unroll
    for (int k = 0; k < kVec; ++k) {
      const float g = to_f<T>(p[k]);
      s[e] = fmaf(g, to_f<T>(q[k]), s[e]);
      if (sizeof(T) == 2) s[e] = fmaf(g, to_f<T>(r[k]), s[e]);
      top[e] = fmaxf(top[e], fabsf(g));
    }
    for (int k = LANES / 2; k > 0; k >>= 1) s[e] += __shfl_xor_sync(0xffffffffu, s[e], k);
    if (c == 0 && on[e]) a.delta[at[e]] = s[e];
  }
  if (amax != nullptr) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      if (!on[e] || a.lse[at[e]] == -INFINITY) top[e] = 0.f;
      for (int k = 16; k > 0; k >>= 1) top[e] = fmaxf(top[e], __shfl_xor_sync(0xffffffffu, top[e], k));
    }
    const uint32_t bits = __float_as_uint(fmaxf(top[0], top[1]));
    if ((threadIdx.x & 31) == 0 && bits > *reinterpret_cast<volatile uint32_t*>(amax)) atomicMax(amax, bits);
  }
}
template <typename T>
inline int launch_delta(const Args& a, uint32_t* amax, cudaStream_t st) {
  constexpr int kVec = 16 / sizeof(T);
  const int64_t n = (int64_t)a.nq * a.hq;
  const int lanes = a.d <= 8 * kVec ? 8 : a.d <= 16 * kVec ? 16 : 32;
  const dim3 grid((unsigned)ceil_div(n, 2 * 256 / lanes), a.b);
  if (lanes == 8) delta_kernel<T, 8><<<grid, 256, 0, st>>>(a, amax);
  else if (lanes == 16) delta_kernel<T, 16><<<grid, 256, 0, st>>>(a, amax);
  else delta_kernel<T, 32><<<grid, 256, 0, st>>>(a, amax);
  count_launch();
  return FLK_OK;
}

// Largest |v| of the rows that may be seen, as bits.
template <typename T>
__global__ void __launch_bounds__(256) largest_value_kernel(const Args a, uint32_t* amax) {
  constexpr int kVec = 16 / sizeof(T);
  const int packs = a.d / kVec;
  const int64_t n = (int64_t)a.b * a.nk * a.hk * packs;
  float top = 0.f;
  for (int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x; e < n; e += (int64_t)gridDim.x * 256) {
    const int c = (int)(e % packs) * kVec;
    const int64_t row = e / packs;
    const int h = (int)(row % a.hk), j = (int)(row / a.hk % a.nk), b = (int)(row / a.hk / a.nk);
    if (j >= (a.kv_lens != nullptr ? a.kv_lens[b] : a.nk) || (a.kdocs != nullptr && a.kdocs[(int64_t)b * a.nk_pad + j] < 0)) continue;
    T u[kVec];
    *reinterpret_cast<uint4*>(u) = *reinterpret_cast<const uint4*>((const T*)a.v.p + b * a.v.sb + j * a.v.sn + h * a.v.sh + c);
#pragma unroll
    for (int x = 0; x < kVec; ++x) top = fmaxf(top, fabsf(to_f<T>(u[x])));
  }
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  if ((threadIdx.x & 31) == 0) atomicMax(amax, __float_as_uint(top));
}

// Gradients of 64 keys and values: loops over the query heads that share them and over their query tiles.
template <typename T, int DM>
__global__ void __launch_bounds__(kThreads) backward_kv_kernel(const Args a) {
  extern __shared__ float sm[];
  constexpr int kRows = Smem<DM>::kRows;
  float *K = sm, *V = K + kRows, *QD = V + kRows, *W = QD + kRows;
  float *sl = W + Smem<DM>::kPair, *sd = sl + kT;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const int k0 = blockIdx.x * kT, hk = blockIdx.y, b = blockIdx.z;
  const Limits lim = limits_of(a, b);
  const int* qd = a.qdocs ? a.qdocs + (int64_t)b * a.nq_pad : nullptr;
  const int* kd = a.kdocs ? a.kdocs + (int64_t)b * a.nk_pad : nullptr;
  load_tile<T, DM>(K, (const T*)a.k.p + b * a.k.sb + hk * a.k.sh, a.k.sn, k0, lim.len, a.d, kd);
  load_tile<T, DM>(V, (const T*)a.v.p + b * a.v.sb + hk * a.v.sh, a.v.sn, k0, lim.len, a.d, kd);
  float dk[4][DM / 16] = {}, dv[4][DM / 16] = {};
  int id[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) id[i] = kd ? kd[min(k0 + 4 * ty + i, a.nk_pad - 1)] : 0;
  for (int g = 0; g < a.grp && k0 < lim.len; ++g) {
    const int h = hk * a.grp + g;
    const float slope2 = a.slopes ? a.slopes[h] * kLog2e : 0.f;
    const float *lse = a.lse + ((int64_t)b * a.hq + h) * a.nq, *delta = a.delta + ((int64_t)b * a.hq + h) * a.nq;
    for (int q0 = 0; q0 < a.nq; q0 += kT) {
      if (lim.row_end(min(q0 + kT, a.nq) - 1, a.causal) <= k0) continue;
      if (kd != nullptr) {
        const int4 x = a.qtab[(int64_t)b * (a.nq_pad / a.q_rows) + q0 / a.q_rows], y = a.ktab[(int64_t)b * (a.nk_pad / kTile) + k0 / kTile];
        if (x.y < y.x || y.y < x.x) continue;
      }
      __syncthreads();
      load_tile<T, DM>(QD, (const T*)a.q.p + b * a.q.sb + h * a.q.sh, a.q.sn, q0, a.nq, a.d, qd);
      if (threadIdx.x < kT) {
        const int r = q0 + threadIdx.x;
        sl[threadIdx.x] = r < a.nq ? lse[r] * kLog2e : 0.f;
        sd[threadIdx.x] = r < a.nq ? delta[r] : 0.f;
      }
      __syncthreads();
      float s[4][4] = {}, p[4][4];  // rows: keys, columns: queries
      dots<DM>(s, K, QD, ty, tx);
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int key = k0 + 4 * ty + i, r = q0 + tx + 16 * j;
          float t;
          const float v = score(a, s[i][j], slope2, lim.start + r - key, t);
          const bool see = r < a.nq && key < lim.row_end(r, a.causal) && (kd == nullptr || qd[r] == id[i]);
          p[i][j] = see ? exp2f(v - sl[tx + 16 * j]) : 0.f;
          s[i][j] = 1.f - t * t;
          W[(tx + 16 * j) * kPs + 4 * ty + i] = p[i][j];
        }
      // dK needs Q after dO has been here: Q is loaded again (from L2); one operand tile less keeps the block small
      __syncthreads();
      load_tile<T, DM>(QD, (const T*)a.dout.p + b * a.dout.sb + h * a.dout.sh, a.dout.sn, q0, a.nq, a.d, qd);
      __syncthreads();
      outer<DM>(dv, W, QD, ty, tx);
      float dp[4][4] = {};
      dots<DM>(dp, V, QD, ty, tx);
      __syncthreads();
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          W[(tx + 16 * j) * kPs + 4 * ty + i] = p[i][j] == 0.f ? 0.f : p[i][j] * (dp[i][j] - sd[tx + 16 * j]) * s[i][j];
      load_tile<T, DM>(QD, (const T*)a.q.p + b * a.q.sb + h * a.q.sh, a.q.sn, q0, a.nq, a.d, qd);
      __syncthreads();
      outer<DM>(dk, W, QD, ty, tx);
    }
  }
  const float one[4] = {1.f, 1.f, 1.f, 1.f}, sc[4] = {a.scale_raw, a.scale_raw, a.scale_raw, a.scale_raw};
  store_rows<T, DM>((T*)a.dk.p + b * a.dk.sb + hk * a.dk.sh, a.dk.sn, k0, a.nk, a.d, dk, sc, ty, tx);
  store_rows<T, DM>((T*)a.dv.p + b * a.dv.sb + hk * a.dv.sh, a.dv.sn, k0, a.nk, a.d, dv, one, ty, tx);
}

// Gradient of 64 queries.
template <typename T, int DM>
__global__ void __launch_bounds__(kThreads) backward_q_kernel(const Args a) {
  extern __shared__ float sm[];
  constexpr int kRows = Smem<DM>::kRows;
  float *Q = sm, *G = Q + kRows, *KV = G + kRows, *W = KV + kRows;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const int q0 = blockIdx.x * kT, h = blockIdx.y, b = blockIdx.z, hk = h / a.grp;
  const Limits lim = limits_of(a, b);
  const int* qd = a.qdocs ? a.qdocs + (int64_t)b * a.nq_pad : nullptr;
  const int* kd = a.kdocs ? a.kdocs + (int64_t)b * a.nk_pad : nullptr;
  const float slope2 = a.slopes ? a.slopes[h] * kLog2e : 0.f;
  load_tile<T, DM>(Q, (const T*)a.q.p + b * a.q.sb + h * a.q.sh, a.q.sn, q0, a.nq, a.d, qd);
  load_tile<T, DM>(G, (const T*)a.dout.p + b * a.dout.sb + h * a.dout.sh, a.dout.sn, q0, a.nq, a.d, qd);
  float dq[4][DM / 16] = {}, lse2[4], delta[4];
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
  for (int k0 = 0; k0 < last; k0 += kT) {
    if (kd != nullptr) {
      const int4 x = a.qtab[(int64_t)b * (a.nq_pad / a.q_rows) + q0 / a.q_rows], y = a.ktab[(int64_t)b * (a.nk_pad / kTile) + k0 / kTile];
      if (x.y < y.x || y.y < x.x) continue;
    }
    float s[4][4] = {}, dp[4][4] = {};
    __syncthreads();
    load_tile<T, DM>(KV, (const T*)a.v.p + b * a.v.sb + hk * a.v.sh, a.v.sn, k0, lim.len, a.d, kd);
    __syncthreads();
    dots<DM>(dp, G, KV, ty, tx);
    __syncthreads();
    load_tile<T, DM>(KV, (const T*)a.k.p + b * a.k.sb + hk * a.k.sh, a.k.sn, k0, lim.len, a.d, kd);
    __syncthreads();
    dots<DM>(s, Q, KV, ty, tx);
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int col = k0 + tx + 16 * j;
        float t;
        const float v = score(a, s[i][j], slope2, lim.start + q0 + 4 * ty + i - col, t);
        const bool see = col < end[i] && (kd == nullptr || kd[col] == id[i]);
        const float p = see ? exp2f(v - lse2[i]) : 0.f;
        W[(tx + 16 * j) * kPs + 4 * ty + i] = see ? p * (dp[i][j] - delta[i]) * (1.f - t * t) : 0.f;
      }
    __syncthreads();
    outer<DM>(dq, W, KV, ty, tx);
  }
  const float sc[4] = {a.scale_raw, a.scale_raw, a.scale_raw, a.scale_raw};
  store_rows<T, DM>((T*)a.dq.p + b * a.dq.sb + h * a.dq.sh, a.dq.sn, q0, a.nq, a.d, dq, sc, ty, tx);
}

template <int DM>
constexpr size_t forward_smem() { return (2 * Smem<DM>::kRows + Smem<DM>::kPair) * 4; }
template <int DM>
constexpr size_t backward_smem() { return (3 * Smem<DM>::kRows + Smem<DM>::kPair + 2 * kT) * 4; }

template <typename T, int DM>
inline int launch_forward(const Args& a, cudaStream_t st) {
  FLK_CUDA_TRY(cudaFuncSetAttribute(forward_kernel<T, DM>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)forward_smem<DM>()));
  forward_kernel<T, DM><<<dim3((unsigned)ceil_div(a.nq, kT), a.hq, a.b), kThreads, forward_smem<DM>(), st>>>(a);
  count_launch();
  return FLK_OK;
}
template <typename T, int DM>
inline int launch_backward(const Args& a, cudaStream_t st) {
  FLK_CUDA_TRY(cudaFuncSetAttribute(backward_kv_kernel<T, DM>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)backward_smem<DM>()));
  FLK_CUDA_TRY(cudaFuncSetAttribute(backward_q_kernel<T, DM>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)backward_smem<DM>()));
  if (a.dk.p != nullptr) {
    backward_kv_kernel<T, DM><<<dim3((unsigned)ceil_div(a.nk, kT), a.hk, a.b), kThreads, backward_smem<DM>(), st>>>(a);
    count_launch();
  }
  if (a.dq.p != nullptr) {
    backward_q_kernel<T, DM><<<dim3((unsigned)ceil_div(a.nq, kT), a.hq, a.b), kThreads, backward_smem<DM>(), st>>>(a);
    count_launch();
  }
  return FLK_OK;
}

}  // namespace simt
}  // namespace attn
}  // namespace flk
