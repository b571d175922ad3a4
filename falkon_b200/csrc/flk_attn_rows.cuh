// Row kernels around attention's products: delta of the backward pass, results of rows that see nothing.
#pragma once

#include "flk_attn.cuh"

namespace flk {
namespace attn {

// delta_i = dO_i . O_i, a group of LANES lanes per row of one head (16 bytes of each array per lane), two rows per group at a time.
// Bound by the bytes of dO, O and what rounding took from O.
template <typename T, int LANES>
__global__ void __launch_bounds__(256) delta_kernel(const Args a) {
  constexpr int kVec = 16 / sizeof(T), kGroups = 256 / LANES;
  const uint32_t n = (uint32_t)a.nq * (uint32_t)a.hq;
  const int b = blockIdx.y, c = (threadIdx.x % LANES) * kVec;
  const T *dout = (const T*)a.dout.p + b * a.dout.sb, *o = (const T*)a.o.p + b * a.o.sb;
  const T* lo = a.o_lo == nullptr ? nullptr : (const T*)a.o_lo + b * a.o.sb;
  float s[2] = {0.f, 0.f};
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
    }
    for (int k = LANES / 2; k > 0; k >>= 1) s[e] += __shfl_xor_sync(0xffffffffu, s[e], k);
    if (c == 0 && on[e]) a.delta[at[e]] = s[e];
  }
}
template <typename T>
inline int launch_delta(const Args& a, cudaStream_t st) {
  constexpr int kVec = 16 / sizeof(T);
  const int lanes = a.d <= 8 * kVec ? 8 : a.d <= 16 * kVec ? 16 : 32;
  const dim3 grid((unsigned)ceil_div((int64_t)a.nq * a.hq, 2 * 256 / lanes), a.b);
  if (lanes == 8) delta_kernel<T, 8><<<grid, 256, 0, st>>>(a);
  else if (sizeof(T) == 2 || lanes == 16) delta_kernel<T, 16><<<grid, 256, 0, st>>>(a);
  else if constexpr (sizeof(T) == 4) delta_kernel<T, 32><<<grid, 256, 0, st>>>(a);
  count_launch();
  return FLK_OK;
}

// Zeros in rows of d values (16 bytes per thread), and -inf in their log-sum-exp (unless null): what a call without keys leaves.
template <typename T>
__global__ void __launch_bounds__(256) nothing_kernel(Tensor4 o, int b, int n, int h, int d, float* lse) {
  constexpr int kVec = 16 / sizeof(T);
  const int packs = d / kVec;
  const int64_t total = (int64_t)b * n * h * packs;
  for (int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x; e < total; e += (int64_t)gridDim.x * 256) {
    const int c = (int)(e % packs) * kVec;
    const int64_t row = e / packs;
    const int hh = (int)(row % h), i = (int)(row / h % n), bb = (int)(row / h / n);
    *reinterpret_cast<uint4*>((T*)o.p + bb * o.sb + i * o.sn + hh * o.sh + c) = make_uint4(0, 0, 0, 0);
    if (c == 0 && lse != nullptr) lse[((int64_t)bb * h + hh) * n + i] = -INFINITY;
  }
}
template <typename T>
inline int launch_nothing(const Tensor4& o, int b, int n, int h, int d, float* lse, cudaStream_t st) {
  const int64_t blocks = ceil_div((int64_t)b * n * h * d * (int)sizeof(T) / 16, 256);
  nothing_kernel<T><<<(unsigned)(blocks < 8 * kNumSMs ? blocks : 8 * kNumSMs), 256, 0, st>>>(o, b, n, h, d, lse);
  count_launch();
  return FLK_OK;
}

}  // namespace attn
}  // namespace flk
