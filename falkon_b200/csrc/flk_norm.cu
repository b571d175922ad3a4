// Layer norm of the rows of a matrix, forward and backward, and its C entry points.
//
//   mu = mean(x), var = mean((x - mu)^2), r = 1 / sqrt(var + eps), xh = (x - mu) r
//   forward    y = xh * w + b                        (mu and r are kept for the backward pass, in fp32)
//   backward   g = dy * w,   dx = r (g - mean(g) - xh mean(g xh)),   dw = sum_rows dy xh,   db = sum_rows dy
//
// Both passes are bound by HBM: forward moves 2 row lengths per row, backward 3.  A row is therefore read once, and every
// statistic is taken from registers (the variance from the centred values, so a large mean costs no digits).  Rows whose
// address and length are multiples of 16 bytes, up to 16384 values, go through the ring kernels: the threads that share a row (16
// values each) copy the rows that come next into a ring in shared memory (cp.async, every thread its own pieces, so nothing
// but the copies' own completion is waited for), and up to 4 rows are under way while others are worked on.  That keeps over
// 64 KB per SM in flight without spending registers on it.  Other rows use plain loads, or, above 16384 values, are read more
// than once.  Measured: 16384 rows of 8192, bf16: forward 117 us (4.6 TB/s), backward 147 us (5.5 TB/s); 300000 rows of 128 out
// of a packed projection 32 us (4.8 TB/s).  What is missing to the 6.5 TB/s of a copy are the two dependent sums of a row.
// Rows of other widths are bound by the number of loads, not by their bytes: 100000 rows of 129, bf16, 39 us forward (1.3 TB/s)
// and 142 with the backward pass, 16384 of 5001 241 (1.4 TB/s) and 920; 2000 of 20000, read three times, 141 us.
// The grid is persistent.  dw and db: every thread adds up its columns in registers over all its rows, every block adds up its
// groups in a fixed order and writes one partial row; a second kernel adds the partial rows, also in a fixed order, so results
// do not depend on timing.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "flk_common.cuh"
#include "flk_ptx.cuh"

namespace flk {
namespace norm {

template <typename T>
__device__ __forceinline__ float to_f(T v);
template <>
__device__ __forceinline__ float to_f<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_f<__half>(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float to_f<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_f(float v);
template <>
__device__ __forceinline__ float from_f<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// VEC values that are loaded and stored at once (16 bytes, or a single value where rows are not 16-byte aligned)
template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) Pack {
  T v[VEC];
};

// Rows of a matrix whose row index has two levels (the heads of a packed projection): offset of row r
struct Rows {
  int64_t inner, s_outer, s_inner;
  __device__ __forceinline__ int64_t at(int64_t r) const {
    if (inner == 1) return r * s_outer;
    if (r < (1ll << 31) && inner < (1ll << 31)) {
      const uint32_t o = (uint32_t)r / (uint32_t)inner;
      return (int64_t)o * s_outer + (int64_t)((uint32_t)r - o * (uint32_t)inner) * s_inner;
    }
    const int64_t o = r / inner;
    return o * s_outer + (r - o * inner) * s_inner;
  }
};

struct Args {
  int64_t n;   // rows
  int d;       // row length
  int tpr;     // threads per row (a power of two)
  int wdtype;  // data type of w and b
  float eps, inv_d;
  const void *x, *dy, *w, *b;
  void *y, *dx;
  Rows xr, dyr;  // y and dx are dense
  float *mean, *rstd;
  float* part;  // [blocks][2][d] partial sums of dw, db
};

__device__ __forceinline__ float load_any(const void* p, int dtype, int64_t i) {
  if (dtype == FLK_F32) return reinterpret_cast<const float*>(p)[i];
  if (dtype == FLK_BF16) return __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(p)[i]);
  return __half2float(reinterpret_cast<const __half*>(p)[i]);
}
__device__ __forceinline__ void store_any(void* p, int dtype, int64_t i, float v) {
  if (dtype == FLK_F32) reinterpret_cast<float*>(p)[i] = v;
  else if (dtype == FLK_BF16) reinterpret_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
  else reinterpret_cast<__half*>(p)[i] = __float2half_rn(v);
}

// Sum of one or two values over the tpr threads of a row group; every thread of the group gets the result.  `red`
// is a 2 x 32 x K shared array: calls alternate between its halves (`flip`), so one barrier per call is enough.
template <int K>
__device__ __forceinline__ void group_sum(float (&v)[K], int tpr, float* red, int& flip) {
  if (tpr < 32) {
    for (int o = tpr >> 1; o > 0; o >>= 1) {
#pragma unroll
      for (int k = 0; k < K; ++k) v[k] += __shfl_xor_sync(0xffffffffu, v[k], o);
    }
    return;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
#pragma unroll
    for (int k = 0; k < K; ++k) v[k] += __shfl_xor_sync(0xffffffffu, v[k], o);
  }
  if (tpr == 32) return;
  float* buf = red + flip * (32 * K);
  flip ^= 1;
  const int warp = threadIdx.x >> 5, at = threadIdx.x & 31, warps = tpr >> 5;
  if (at == 0) {
#pragma unroll
    for (int k = 0; k < K; ++k) buf[warp * K + k] = v[k];
  }
  __syncthreads();
  // every warp adds the sums of its group's warps; their number is a power of two, so lanes take them round and round
  const int from = (warp & ~(warps - 1)) + (at & (warps - 1));
#pragma unroll
  for (int k = 0; k < K; ++k) v[k] = buf[from * K + k];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    if (o < warps) {
#pragma unroll
      for (int k = 0; k < K; ++k) v[k] += __shfl_xor_sync(0xffffffffu, v[k], o);
    }
  }
}
// 1 / sqrt(x): the hardware's approximation and one step of Newton's method
__device__ __forceinline__ float inverse_root(float x) {
  const float r = rsqrtf(x), s = r * fmaf(-0.5f * x * r, r, 1.5f);
  return x > 1e-30f && x < 1e30f ? s : r;  // beyond, the step itself would leave fp32
}

template <typename T, int VEC, int V>
__device__ __forceinline__ void load_row(Pack<T, VEC> (&raw)[V], const T* row, int lane, int tpr, int packs) {
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int p = lane + i * tpr;
    if (p < packs) raw[i] = *reinterpret_cast<const Pack<T, VEC>*>(row + (int64_t)p * VEC);
  }
}

// Rows of up to tpr * V * VEC values.
template <typename T, int VEC, int V>
__global__ void __launch_bounds__(1024 / (V * VEC > 16 ? 2 : 1)) forward_kernel(const Args a) {
  __shared__ float red[2 * 32];
  const int lane = threadIdx.x % a.tpr, group = threadIdx.x / a.tpr, groups = blockDim.x / a.tpr;
  const int packs = a.d / VEC;
  const T* x = reinterpret_cast<const T*>(a.x);
  T* y = reinterpret_cast<T*>(a.y);
  const int64_t step = (int64_t)gridDim.x * groups;
  int flip = 0;
  float w[V][VEC], b[V][VEC];
#pragma unroll
  for (int i = 0; i < V; ++i)
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      const int c = (lane + i * a.tpr) * VEC + j;
      w[i][j] = a.w != nullptr && c < a.d ? load_any(a.w, a.wdtype, c) : 1.f;
      b[i][j] = a.b != nullptr && c < a.d ? load_any(a.b, a.wdtype, c) : 0.f;
    }
  Pack<T, VEC> next[V];
  int64_t row = (int64_t)blockIdx.x * groups + group;
  if (row < a.n) load_row<T, VEC, V>(next, x + a.xr.at(row), lane, a.tpr, packs);
  // every group makes the same number of turns, so that the barriers inside the sums match
  for (int64_t r0 = (int64_t)blockIdx.x * groups; r0 < a.n; r0 += step, row += step) {
    const bool on = row < a.n;
    float v[V][VEC];
    float s[1] = {0.f};
#pragma unroll
    for (int i = 0; i < V; ++i)
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        v[i][j] = lane + i * a.tpr < packs && on ? to_f<T>(next[i].v[j]) : 0.f;
        s[0] += v[i][j];
      }
    if (row + step < a.n) load_row<T, VEC, V>(next, x + a.xr.at(row + step), lane, a.tpr, packs);
    group_sum<1>(s, a.tpr, red, flip);
    const float mu = s[0] * a.inv_d;
    s[0] = 0.f;
#pragma unroll
    for (int i = 0; i < V; ++i)
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        v[i][j] = lane + i * a.tpr < packs ? v[i][j] - mu : 0.f;
        s[0] = fmaf(v[i][j], v[i][j], s[0]);
      }
    group_sum<1>(s, a.tpr, red, flip);
    const float r = inverse_root(fmaf(s[0], a.inv_d, a.eps));
    if (on) {
      if (lane == 0 && a.mean != nullptr) {
        a.mean[row] = mu;
        a.rstd[row] = r;
      }
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const int p = lane + i * a.tpr;
        if (p >= packs) continue;
        Pack<T, VEC> out;
#pragma unroll
        for (int j = 0; j < VEC; ++j) out.v[j] = from_f<T>(fmaf(v[i][j] * r, w[i][j], b[i][j]));
        *reinterpret_cast<Pack<T, VEC>*>(y + row * a.d + (int64_t)p * VEC) = out;
      }
    }
  }
}

// One block per row, rows of any length; the row is read three times (from L2 after the first).  A thread adds up d / 1024 values,
// so a first mean may be off by that many roundings (rows of 2^22 values with a mean of 1000: by 0.01).  The second pass adds up
// the centred values too, and what their mean says is left of the first mean comes off them.
template <typename T>
__global__ void __launch_bounds__(1024) forward_long_kernel(const Args a) {
  __shared__ float red[2 * 32 * 2];
  int flip = 0;
  T* y = reinterpret_cast<T*>(a.y);
  for (int64_t row = blockIdx.x; row < a.n; row += gridDim.x) {
    const T* x = reinterpret_cast<const T*>(a.x) + a.xr.at(row);
    float s[2] = {0.f, 0.f};
    for (int c = threadIdx.x; c < a.d; c += blockDim.x) s[0] += to_f<T>(x[c]);
    group_sum<2>(s, blockDim.x, red, flip);
    const float mu = s[0] * a.inv_d;
    s[0] = s[1] = 0.f;
    for (int c = threadIdx.x; c < a.d; c += blockDim.x) {
      const float v = to_f<T>(x[c]) - mu;
      s[0] += v;
      s[1] = fmaf(v, v, s[1]);
    }
    group_sum<2>(s, blockDim.x, red, flip);
    const float left = s[0] * a.inv_d;
    // mean(v^2) - left^2 without a difference of two large numbers: `left` is a rounding error of the mean
    const float r = inverse_root(fmaxf(fmaf(s[1], a.inv_d, -left * left), 0.f) + a.eps);
    if (threadIdx.x == 0 && a.mean != nullptr) {
      a.mean[row] = mu + left;
      a.rstd[row] = r;
    }
    for (int c = threadIdx.x; c < a.d; c += blockDim.x) {
      const float w = a.w != nullptr ? load_any(a.w, a.wdtype, c) : 1.f, b = a.b != nullptr ? load_any(a.b, a.wdtype, c) : 0.f;
      y[row * a.d + c] = from_f<T>(fmaf((to_f<T>(x[c]) - mu - left) * r, w, b));
    }
  }
}

template <typename T, int VEC, int V>
__global__ void __launch_bounds__(V * VEC > 16 ? 256 : (V * VEC > 8 ? 512 : 1024)) backward_kernel(const Args a) {
  extern __shared__ float sums[];  // [groups][d] when a block has several groups, used once at the end
  __shared__ float red[2 * 32 * 2];
  const int lane = threadIdx.x % a.tpr, group = threadIdx.x / a.tpr, groups = blockDim.x / a.tpr;
  const int packs = a.d / VEC;
  const T *x = reinterpret_cast<const T*>(a.x), *dy = reinterpret_cast<const T*>(a.dy);
  T* dx = reinterpret_cast<T*>(a.dx);
  const int64_t step = (int64_t)gridDim.x * groups;
  int flip = 0;
  float w[V][VEC], dw[V][VEC], db[V][VEC];
#pragma unroll
  for (int i = 0; i < V; ++i)
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      const int c = (lane + i * a.tpr) * VEC + j;
      w[i][j] = a.w != nullptr && c < a.d ? load_any(a.w, a.wdtype, c) : 1.f;
      dw[i][j] = db[i][j] = 0.f;
    }
  Pack<T, VEC> nx[V], ng[V];
  float nmu = 0.f, nr = 0.f;
  int64_t row = (int64_t)blockIdx.x * groups + group;
  if (row < a.n) {
    load_row<T, VEC, V>(nx, x + a.xr.at(row), lane, a.tpr, packs);
    load_row<T, VEC, V>(ng, dy + a.dyr.at(row), lane, a.tpr, packs);
    nmu = a.mean[row];
    nr = a.rstd[row];
  }
  for (int64_t r0 = (int64_t)blockIdx.x * groups; r0 < a.n; r0 += step, row += step) {
    const bool on = row < a.n;
    Pack<T, VEC> cx[V], cg[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
      cx[i] = nx[i];
      cg[i] = ng[i];
    }
    const float mu = nmu, r = nr;
    if (row + step < a.n) {
      load_row<T, VEC, V>(nx, x + a.xr.at(row + step), lane, a.tpr, packs);
      load_row<T, VEC, V>(ng, dy + a.dyr.at(row + step), lane, a.tpr, packs);
      nmu = a.mean[row + step];
      nr = a.rstd[row + step];
    }
    float s[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < V; ++i)
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        if (lane + i * a.tpr >= packs || !on) continue;
        const float g0 = to_f<T>(cg[i].v[j]), xh = (to_f<T>(cx[i].v[j]) - mu) * r, g = g0 * w[i][j];
        s[0] += g;
        s[1] = fmaf(g, xh, s[1]);
        dw[i][j] = fmaf(g0, xh, dw[i][j]);
        db[i][j] += g0;
      }
    group_sum<2>(s, a.tpr, red, flip);
    const float m1 = s[0] * a.inv_d, m2 = s[1] * a.inv_d;
    if (on && dx != nullptr) {
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const int p = lane + i * a.tpr;
        if (p >= packs) continue;
        Pack<T, VEC> out;
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const float xh = (to_f<T>(cx[i].v[j]) - mu) * r;
          out.v[j] = from_f<T>((to_f<T>(cg[i].v[j]) * w[i][j] - m1 - xh * m2) * r);
        }
        *reinterpret_cast<Pack<T, VEC>*>(dx + row * a.d + (int64_t)p * VEC) = out;
      }
    }
  }
  if (a.part == nullptr) return;
  float* part = a.part + (int64_t)blockIdx.x * 2 * a.d;
  if (groups == 1) {
#pragma unroll
    for (int i = 0; i < V; ++i)
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const int c = (lane + i * a.tpr) * VEC + j;
        if (c < a.d) {
          part[c] = dw[i][j];
          part[a.d + c] = db[i][j];
        }
      }
    return;
  }
  for (int which = 0; which < 2; ++which) {
    __syncthreads();
#pragma unroll
    for (int i = 0; i < V; ++i)
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const int c = (lane + i * a.tpr) * VEC + j;
        if (c < a.d) sums[group * a.d + c] = which == 0 ? dw[i][j] : db[i][j];
      }
    __syncthreads();
    for (int c = threadIdx.x; c < a.d; c += blockDim.x) {
      float t = 0.f;
      for (int g = 0; g < groups; ++g) t += sums[g * a.d + c];
      part[which * a.d + c] = t;
    }
  }
}

// One block per row, rows of any length.  The partial sums live in the block's row of the workspace.
template <typename T>
__global__ void __launch_bounds__(1024) backward_long_kernel(const Args a) {
  __shared__ float red[2 * 32 * 2];
  int flip = 0;
  T* dx = reinterpret_cast<T*>(a.dx);
  float* part = a.part == nullptr ? nullptr : a.part + (int64_t)blockIdx.x * 2 * a.d;
  for (int64_t row = blockIdx.x; row < a.n; row += gridDim.x) {
    const T* x = reinterpret_cast<const T*>(a.x) + a.xr.at(row);
    const T* dy = reinterpret_cast<const T*>(a.dy) + a.dyr.at(row);
    const float mu = a.mean[row], r = a.rstd[row];
    float s[2] = {0.f, 0.f};
    for (int c = threadIdx.x; c < a.d; c += blockDim.x) {
      const float g0 = to_f<T>(dy[c]), xh = (to_f<T>(x[c]) - mu) * r;
      const float g = g0 * (a.w != nullptr ? load_any(a.w, a.wdtype, c) : 1.f);
      s[0] += g;
      s[1] = fmaf(g, xh, s[1]);
      if (part != nullptr) {
        const bool first = row == blockIdx.x;
        part[c] = fmaf(g0, xh, first ? 0.f : part[c]);
        part[a.d + c] = (first ? 0.f : part[a.d + c]) + g0;
      }
    }
    group_sum<2>(s, blockDim.x, red, flip);
    const float m1 = s[0] * a.inv_d, m2 = s[1] * a.inv_d;
    if (dx != nullptr)
      for (int c = threadIdx.x; c < a.d; c += blockDim.x) {
        const float xh = (to_f<T>(x[c]) - mu) * r;
        const float g = to_f<T>(dy[c]) * (a.w != nullptr ? load_any(a.w, a.wdtype, c) : 1.f);
        dx[row * a.d + c] = from_f<T>((g - m1 - xh * m2) * r);
      }
  }
}

// ---------------------------------------------------------------------------------------------------------------------
// ring kernels
// ---------------------------------------------------------------------------------------------------------------------
// Shared memory: w (and, forward, b) as fp32, in the order the threads read it (16 bytes per thread and step), then the ring.
// Piece p of a row belongs to thread p % tpr of its group.
template <int VEC>
__device__ __forceinline__ void fill_columns(float* dst, const void* src, int dtype, float missing, int d, int tpr) {
  const int packs = d / VEC;
  for (int e = threadIdx.x; e < packs * (VEC / 4); e += blockDim.x) {
    const int p = e / (VEC / 4), q = e % (VEC / 4), lane = p % tpr, i = p / tpr;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int c = p * VEC + 4 * q + k;
      dst[(((i * (VEC / 4)) + q) * tpr + lane) * 4 + k] = src != nullptr ? load_any(src, dtype, c) : missing;
    }
  }
}
// Values are worked on in pairs (packed fp32): these kernels are short of issue slots before they are short of anything else but
// HBM.  16 bytes of T <-> pairs:
template <typename T>
__device__ __forceinline__ void to_pairs(const uint4& raw, uint64_t (&f)[8 / sizeof(T)]) {
  const uint32_t u[4] = {raw.x, raw.y, raw.z, raw.w};
  if constexpr (sizeof(T) == 4) {
    f[0] = tc::pack2(__uint_as_float(u[0]), __uint_as_float(u[1]));
    f[1] = tc::pack2(__uint_as_float(u[2]), __uint_as_float(u[3]));
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if constexpr (sizeof(T) == 2 && std::is_same<T, __nv_bfloat16>::value) {
        f[k] = tc::pack2(__uint_as_float(u[k] << 16), __uint_as_float(u[k] & 0xffff0000u));
      } else {
        const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&u[k]));
        f[k] = tc::pack2(v.x, v.y);
      }
    }
  }
}
template <typename T>
__device__ __forceinline__ uint4 from_pairs(const uint64_t (&f)[8 / sizeof(T)]) {
  uint32_t u[4];
  float x, y;
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      tc::unpack2(f[k], x, y);
      u[2 * k] = __float_as_uint(x), u[2 * k + 1] = __float_as_uint(y);
    }
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      tc::unpack2(f[k], x, y);
      if constexpr (std::is_same<T, __nv_bfloat16>::value)
        asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(u[k]) : "f"(y), "f"(x));
      else
        asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(u[k]) : "f"(y), "f"(x));
    }
  }
  return make_uint4(u[0], u[1], u[2], u[3]);
}
__device__ __forceinline__ uint64_t both(float v) { return tc::pack2(v, v); }
__device__ __forceinline__ float sum2(uint64_t v) {
  float x, y;
  tc::unpack2(v, x, y);
  return x + y;
}
// `src`: the thread's first 16 bytes; the following ones lie `step` bytes apart
template <int NP>
__device__ __forceinline__ void read_columns(uint64_t (&v)[NP], const char* src, int step, int i) {
#pragma unroll
  for (int q = 0; q < NP / 2; ++q) {
    const ulonglong2 x = *reinterpret_cast<const ulonglong2*>(src + (i * (NP / 2) + q) * step);
    v[2 * q] = x.x, v[2 * q + 1] = x.y;
  }
}
template <typename T, int VEC, int V>
__device__ __forceinline__ void copy_row(char* slot, const T* row, int lane, int tpr, int packs) {
#pragma unroll
  for (int i = 0; i < V; ++i)
    if (lane + i * tpr < packs) cp_async16(slot + (i * blockDim.x + threadIdx.x) * 16, row + (int64_t)(lane + i * tpr) * VEC);
}

// ROWS rows share a turn, and with it the two barriers of their sums: two where the ring has room (16384 rows of 8192, bf16: 128.5 us
// with one, 116.6 with two).
template <typename T, int V, int STAGES, int ROWS>
__global__ void __launch_bounds__(1024) forward_ring_kernel(const Args a) {
  constexpr int VEC = 16 / (int)sizeof(T), NP = VEC / 2;
  static_assert(STAGES % ROWS == 0, "a turn takes ROWS slots of the ring");
  extern __shared__ __align__(16) float cols[];
  __shared__ float red[2 * 32 * ROWS];
  const int lane = threadIdx.x % a.tpr, group = threadIdx.x / a.tpr, groups = blockDim.x / a.tpr, packs = a.d / VEC;
  float *w = cols, *b = cols + a.tpr * V * VEC;
  const char *my_w = reinterpret_cast<const char*>(w) + lane * 16, *my_b = reinterpret_cast<const char*>(b) + lane * 16;
  char* ring = reinterpret_cast<char*>(cols + 2 * a.tpr * V * VEC);
  const int stage_bytes = blockDim.x * V * 16;
  const T* x = reinterpret_cast<const T*>(a.x);
  T* y = reinterpret_cast<T*>(a.y);
  const int64_t step = (int64_t)gridDim.x * groups;
  int64_t row = (int64_t)blockIdx.x * groups + group;
#pragma unroll
  for (int s = 0; s < STAGES; ++s) {
    if (row + s * step < a.n) copy_row<T, VEC, V>(ring + s * stage_bytes, x + a.xr.at(row + s * step), lane, a.tpr, packs);
    cp_async_commit();
  }
  fill_columns<VEC>(w, a.w, a.wdtype, 1.f, a.d, a.tpr);
  fill_columns<VEC>(b, a.b, a.wdtype, 0.f, a.d, a.tpr);
  __syncthreads();
  int flip = 0, at = 0;
  // every group makes the same number of turns, so that the barriers inside the sums match
  for (int64_t r0 = (int64_t)blockIdx.x * groups; r0 < a.n; r0 += ROWS * step, row += ROWS * step) {
    cp_async_wait<STAGES - ROWS>();
    uint64_t v[ROWS][V][NP];
    float s[ROWS], mu[ROWS];
#pragma unroll
    for (int e = 0; e < ROWS; ++e) {
      char* slot = ring + (at + e) * stage_bytes;
      uint64_t acc = 0;
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (row + e * step < a.n && lane + i * a.tpr < packs) {
          to_pairs<T>(*reinterpret_cast<const uint4*>(slot + (i * blockDim.x + threadIdx.x) * 16), v[e][i]);
#pragma unroll
          for (int j = 0; j < NP; ++j) acc = tc::add2(acc, v[e][i][j]);
        }
      if (row + (STAGES + e) * step < a.n) copy_row<T, VEC, V>(slot, x + a.xr.at(row + (STAGES + e) * step), lane, a.tpr, packs);
      cp_async_commit();
      s[e] = sum2(acc);
    }
    at = at + ROWS == STAGES ? 0 : at + ROWS;
    group_sum<ROWS>(s, a.tpr, red, flip);
#pragma unroll
    for (int e = 0; e < ROWS; ++e) {
      mu[e] = s[e] * a.inv_d;
      const uint64_t mu2 = both(mu[e]);
      uint64_t acc = 0;
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (row + e * step < a.n && lane + i * a.tpr < packs) {
#pragma unroll
          for (int j = 0; j < NP; ++j) {
            v[e][i][j] = tc::sub2(v[e][i][j], mu2);
            acc = tc::fma2(v[e][i][j], v[e][i][j], acc);
          }
        }
      s[e] = sum2(acc);
    }
    group_sum<ROWS>(s, a.tpr, red, flip);
#pragma unroll
    for (int e = 0; e < ROWS; ++e) {
      const int64_t out = row + e * step;
      if (out >= a.n) continue;
      const float r = inverse_root(fmaf(s[e], a.inv_d, a.eps));
      if (lane == 0 && a.mean != nullptr) {
        a.mean[out] = mu[e];
        a.rstd[out] = r;
      }
      const uint64_t r2 = both(r);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const int p = lane + i * a.tpr;
        if (p < packs) {
          uint64_t ww[NP], bb[NP];
          read_columns<NP>(ww, my_w, a.tpr * 16, i);
          read_columns<NP>(bb, my_b, a.tpr * 16, i);
#pragma unroll
          for (int j = 0; j < NP; ++j) ww[j] = tc::fma2(tc::mul2(v[e][i][j], r2), ww[j], bb[j]);
          *reinterpret_cast<uint4*>(y + out * a.d + (int64_t)p * VEC) = from_pairs<T>(ww);
        }
      }
    }
  }
}

template <typename T, int V, int STAGES, int THREADS>
__global__ void __launch_bounds__(THREADS, 1) backward_ring_kernel(const Args a) {
  constexpr int VEC = 16 / (int)sizeof(T), NP = VEC / 2;
  extern __shared__ __align__(16) float cols[];
  __shared__ float red[2 * 32 * 2];
  const int lane = threadIdx.x % a.tpr, group = threadIdx.x / a.tpr, groups = blockDim.x / a.tpr, packs = a.d / VEC;
  const int stage_bytes = blockDim.x * V * 32 + blockDim.x * 8;
  float* w = cols;
  const char* my_w = reinterpret_cast<const char*>(w) + lane * 16;
  char* ring = reinterpret_cast<char*>(cols + a.tpr * V * VEC);
  const T *x = reinterpret_cast<const T*>(a.x), *dy = reinterpret_cast<const T*>(a.dy);
  T* dx = reinterpret_cast<T*>(a.dx);
  const int64_t step = (int64_t)gridDim.x * groups;
  // the first lane of a group in each warp fetches mean and rstd for it
  const int lead = threadIdx.x & ~((a.tpr < 32 ? a.tpr : 32) - 1);
  auto fetch = [&](char* slot, int64_t r) {
    copy_row<T, VEC, V>(slot, x + a.xr.at(r), lane, a.tpr, packs);
    copy_row<T, VEC, V>(slot + blockDim.x * V * 16, dy + a.dyr.at(r), lane, a.tpr, packs);
    if ((int)threadIdx.x == lead) {
      cp_async_small<4>(slot + blockDim.x * V * 32 + threadIdx.x * 8, a.mean + r);
      cp_async_small<4>(slot + blockDim.x * V * 32 + threadIdx.x * 8 + 4, a.rstd + r);
    }
  };
  int64_t row = (int64_t)blockIdx.x * groups + group;
#pragma unroll
  for (int s = 0; s < STAGES; ++s) {
    if (row + s * step < a.n) fetch(ring + s * stage_bytes, row + s * step);
    cp_async_commit();
  }
  fill_columns<VEC>(w, a.w, a.wdtype, 1.f, a.d, a.tpr);
  __syncthreads();
  uint64_t dw[V][NP], db[V][NP];
#pragma unroll
  for (int i = 0; i < V; ++i)
#pragma unroll
    for (int j = 0; j < NP; ++j) dw[i][j] = db[i][j] = 0;
  int flip = 0, at = 0;
  for (int64_t r0 = (int64_t)blockIdx.x * groups; r0 < a.n; r0 += step, row += step) {
    const bool on = row < a.n;
    char* slot = ring + at * stage_bytes;
    at = at + 1 == STAGES ? 0 : at + 1;
    cp_async_wait<STAGES - 1>();
    __syncwarp();
    const float2 st = *reinterpret_cast<const float2*>(slot + blockDim.x * V * 32 + lead * 8);
    const float r = st.y;
    const uint64_t mu2 = both(st.x), r2 = both(r);
    // what the second half of the work needs again: with 1024 threads, which have 64 registers, the raw pieces
    constexpr bool kRaw = THREADS == 1024;
    uint64_t g[kRaw ? 1 : V][NP], xh[kRaw ? 1 : V][NP], acc[2] = {0, 0};
    uint4 kx[kRaw ? V : 1], kg[kRaw ? V : 1];
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (on && lane + i * a.tpr < packs) {
        const uint4 px = *reinterpret_cast<const uint4*>(slot + (i * blockDim.x + threadIdx.x) * 16);
        const uint4 pg = *reinterpret_cast<const uint4*>(slot + ((V + i) * blockDim.x + threadIdx.x) * 16);
        uint64_t ww[NP], fx[NP], fg[NP];
        read_columns<NP>(ww, my_w, a.tpr * 16, i);
        to_pairs<T>(px, fx);
        to_pairs<T>(pg, fg);
#pragma unroll
        for (int j = 0; j < NP; ++j) {
          fx[j] = tc::mul2(tc::sub2(fx[j], mu2), r2);
          dw[i][j] = tc::fma2(fg[j], fx[j], dw[i][j]);
          db[i][j] = tc::add2(db[i][j], fg[j]);
          fg[j] = tc::mul2(fg[j], ww[j]);
          acc[0] = tc::add2(acc[0], fg[j]);
          acc[1] = tc::fma2(fg[j], fx[j], acc[1]);
          if constexpr (!kRaw) xh[i][j] = fx[j], g[i][j] = fg[j];
        }
        if constexpr (kRaw) kx[i] = px, kg[i] = pg;
      }
    __syncwarp();  // the slot's mean and rstd have been read
    if (row + STAGES * step < a.n) fetch(slot, row + STAGES * step);
    cp_async_commit();
    float s[2] = {sum2(acc[0]), sum2(acc[1])};
    group_sum<2>(s, a.tpr, red, flip);
    if (on && dx != nullptr) {
      const uint64_t m1 = both(-s[0] * a.inv_d), m2 = both(-s[1] * a.inv_d);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const int p = lane + i * a.tpr;
        if (p < packs) {
          uint64_t out[NP];
          if constexpr (kRaw) {
            uint64_t ww[NP], fx[NP], fg[NP];
            read_columns<NP>(ww, my_w, a.tpr * 16, i);
            to_pairs<T>(kx[i], fx);
            to_pairs<T>(kg[i], fg);
#pragma unroll
            for (int j = 0; j < NP; ++j)
              out[j] = tc::mul2(tc::fma2(tc::mul2(tc::sub2(fx[j], mu2), r2), m2, tc::add2(tc::mul2(fg[j], ww[j]), m1)), r2);
          } else {
#pragma unroll
            for (int j = 0; j < NP; ++j) out[j] = tc::mul2(tc::fma2(xh[i][j], m2, tc::add2(g[i][j], m1)), r2);
          }
          *reinterpret_cast<uint4*>(dx + row * a.d + (int64_t)p * VEC) = from_pairs<T>(out);
        }
      }
    }
  }
  if (a.part == nullptr) return;
  cp_async_wait<0>();
  float* part = a.part + (int64_t)blockIdx.x * 2 * a.d;
  float* sums = reinterpret_cast<float*>(ring);  // [groups][d]: no more than threads * V * VEC values, the ring is larger
  for (int which = 0; which < 2; ++which) {
    if (groups > 1) __syncthreads();
    float* to = groups > 1 ? sums + group * a.d : part + which * a.d;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      if (lane + i * a.tpr >= packs) continue;
#pragma unroll
      for (int j = 0; j < NP; j += 2) {
        const uint64_t v0 = which == 0 ? dw[i][j] : db[i][j], v1 = which == 0 ? dw[i][j + 1] : db[i][j + 1];
        *reinterpret_cast<ulonglong2*>(to + (lane + i * a.tpr) * VEC + 2 * j) = make_ulonglong2(v0, v1);
      }
    }
    if (groups == 1) continue;
    __syncthreads();
    for (int c = threadIdx.x; c < a.d; c += blockDim.x) {
      float t = 0.f;
      for (int q = 0; q < groups; ++q) t += sums[q * a.d + c];
      part[which * a.d + c] = t;
    }
  }
}

// dw, db = sums of the blocks' partial rows: 32 columns per block, 8 slices of partial rows added side by side and then
// in order.
__global__ void __launch_bounds__(256) reduce_kernel(const float* part, int64_t blocks, int d, void* dw, void* db, int wdtype) {
  __shared__ float buf[8][33];
  const int c = blockIdx.x * 32 + (threadIdx.x & 31), slice = threadIdx.x >> 5, which = blockIdx.y;
  float s = 0.f;
  if (c < d)
    for (int64_t i = slice; i < blocks; i += 8) s += part[(i * 2 + which) * d + c];
  buf[slice][threadIdx.x & 31] = s;
  __syncthreads();
  if (slice == 0 && c < d) {
    s = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) s += buf[i][threadIdx.x & 31];
    void* out = which == 0 ? dw : db;
    if (out != nullptr) store_any(out, wdtype, c, s);
  }
}

// How a call is laid out: values per load, loads per thread, threads per row and per block, blocks.
struct Plan {
  int vec, v, tpr, threads, stages;
  bool is_long;
  int64_t blocks;
  size_t smem;
};

static Plan make_plan(int esize, int64_t n, int64_t d, bool aligned, bool backward) {
  Plan p{};
  const int full = 16 / esize;
  int64_t resident;
  if (aligned && d % full == 0 && d <= 16384) {
    // ring kernels: 16 values per thread, fewer where a row has no more than 4 pieces
    p.vec = full;
    const int64_t packs = d / full;
    p.v = 16 / full;
    while (p.v > 1 && packs <= p.v * 2) p.v >>= 1;
    p.tpr = 1;
    while ((int64_t)p.tpr * p.v < packs) p.tpr <<= 1;
    p.threads = p.tpr < 256 ? 256 : p.tpr;
    const size_t columns = (size_t)p.tpr * p.v * full * 4 * (backward ? 1 : 2);
    const size_t stage = backward ? (size_t)p.threads * (p.v * 32 + 8) : (size_t)p.threads * p.v * 16;
    p.stages = columns + 4 * stage <= 224 * 1024 ? 4 : columns + 2 * stage <= 224 * 1024 ? 2 : 1;
    // forward, two blocks with two stages each hide each other's barriers
    if (!backward && p.stages == 4 && columns + 4 * stage > 110 * 1024 && columns + 2 * stage <= 110 * 1024) p.stages = 2;
    p.smem = columns + p.stages * stage;
    // blocks per SM: by shared memory, and by registers (about 64 a thread forward, 96 backward)
    resident = (int64_t)(224 * 1024 / (p.smem + 1024));
    const int64_t by_regs = (backward ? 640 : 1024) / p.threads;
    if (resident > by_regs) resident = by_regs;
  } else {
    p.vec = 1;
    p.is_long = true;
    const int choices[3] = {2, 8, 16};
    for (int i = 0; i < 3 && p.is_long; ++i) {
      p.v = choices[i];
      const int limit = backward ? (p.v > 8 ? 512 : 1024) : 1024;
      int tpr = 4;
      while ((int64_t)tpr * p.v < d) tpr <<= 1;
      if (tpr <= limit && (i > 0 || tpr <= 32)) {
        p.tpr = tpr;
        p.is_long = false;
      }
    }
    if (p.is_long) p.tpr = 1024, p.v = 1;
    p.threads = p.tpr < 256 ? 256 : p.tpr;
    p.smem = backward && !p.is_long && p.tpr < p.threads ? (size_t)(p.threads / p.tpr) * d * 4 : 0;
    resident = backward ? (p.v > 8 ? 512 : 1024) / p.threads : 2048 / p.threads;
  }
  if (resident < 1) resident = 1;
  const int64_t need = ceil_div(n, p.threads / p.tpr);
  p.blocks = need < kNumSMs * resident ? need : kNumSMs * resident;
  if (p.blocks < 1) p.blocks = 1;
  return p;
}

static bool is_aligned(const void* p, int64_t s0, int64_t s1, int esize) {
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && s0 * esize % 16 == 0 && s1 * esize % 16 == 0;
}

static int run(void (*fn)(const Args), const Args& a, const Plan& p, cudaStream_t st) {
  if (p.smem > 40 * 1024) FLK_CUDA_TRY(cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)p.smem));
  fn<<<(unsigned)p.blocks, p.threads, p.smem, st>>>(a);
  count_launch();
  return FLK_OK;
}

static int no_kernel(const Plan& p) { return fail(FLK_ERR_UNSUPPORTED, "no kernel for %d loads per thread, %d threads, %d rows ahead", p.v, p.threads, p.stages); }
// The ring kernels that plans ask for: four rows ahead, fewer only where long rows take the most loads per thread.
template <typename T>
static int forward_ring(const Args& a, const Plan& p, cudaStream_t st) {
  constexpr int kMost = sizeof(T) == 4 ? 4 : 2;
  if (p.stages == 4) {
    if (p.v == 1) return run(forward_ring_kernel<T, 1, 4, 2>, a, p, st);
    if (p.v == kMost) return run(forward_ring_kernel<T, kMost, 4, 2>, a, p, st);
    if (p.v == 2) return run(forward_ring_kernel<T, 2, 4, 2>, a, p, st);  // (fp32)
  } else if (p.v == kMost) {
    if constexpr (sizeof(T) == 2) {
      if (p.stages == 2) return run(forward_ring_kernel<T, kMost, 2, 2>, a, p, st);
    } else {
      if (p.stages == 1) return run(forward_ring_kernel<T, kMost, 1, 1>, a, p, st);
    }
  }
  return no_kernel(p);
}
template <typename T>
static int launch_forward(const Args& a, const Plan& p, cudaStream_t st) {
  if (p.is_long) return run(forward_long_kernel<T>, a, p, st);
  if (p.vec == 1) return p.v == 2 ? run(forward_kernel<T, 1, 2>, a, p, st) : p.v == 8 ? run(forward_kernel<T, 1, 8>, a, p, st) : run(forward_kernel<T, 1, 16>, a, p, st);
  return forward_ring<T>(a, p, st);
}

template <typename T>
static int backward_ring(const Args& a, const Plan& p, cudaStream_t st) {
  constexpr int kMost = sizeof(T) == 4 ? 4 : 2;
  if (p.threads <= 512 && p.stages == 4) {
    if (p.v == 1) return run(backward_ring_kernel<T, 1, 4, 512>, a, p, st);
    if (p.v == kMost) return run(backward_ring_kernel<T, kMost, 4, 512>, a, p, st);
    if (p.v == 2) return run(backward_ring_kernel<T, 2, 4, 512>, a, p, st);  // (fp32)
  } else if (p.v == kMost) {
    if constexpr (sizeof(T) == 2) {
      if (p.threads == 1024 && p.stages == 2) return run(backward_ring_kernel<T, kMost, 2, 1024>, a, p, st);
    } else {
      if (p.threads == 512 && p.stages == 2) return run(backward_ring_kernel<T, kMost, 2, 512>, a, p, st);
      if (p.threads == 1024 && p.stages == 1) return run(backward_ring_kernel<T, kMost, 1, 1024>, a, p, st);
    }
  }
  return no_kernel(p);
}
template <typename T>
static int launch_backward(const Args& a, const Plan& p, cudaStream_t st) {
  if (p.is_long) return run(backward_long_kernel<T>, a, p, st);
  if (p.vec == 1) return p.v == 2 ? run(backward_kernel<T, 1, 2>, a, p, st) : p.v == 8 ? run(backward_kernel<T, 1, 8>, a, p, st) : run(backward_kernel<T, 1, 16>, a, p, st);
  return backward_ring<T>(a, p, st);
}

static int esize_of(int dtype) { return dtype == FLK_F32 ? 4 : 2; }

static int check(const flk_layer_norm_args* p) {
  if (p == nullptr) return fail(FLK_ERR_BAD_ARG, "args: null pointer");
  if (p->dtype != FLK_F32 && p->dtype != FLK_BF16 && p->dtype != FLK_F16)
    return fail(FLK_ERR_BAD_ARG, "layer norm takes fp32, bf16 or fp16 data, not dtype %lld", (long long)p->dtype);
  if (p->wdtype != p->dtype && p->wdtype != FLK_F32)
    return fail(FLK_ERR_BAD_ARG, "weight and bias have the data's type or fp32");
  if (p->n < 0 || p->d < 1 || p->d > (1ll << 24) || p->n > (1ll << 40))
    return fail(FLK_ERR_BAD_ARG, "bad sizes n = %lld, d = %lld (1 <= d <= 2^24)", (long long)p->n, (long long)p->d);
  if (p->x_inner < 1) return fail(FLK_ERR_BAD_ARG, "x_inner must be at least 1");
  if (!(p->eps >= 0)) return fail(FLK_ERR_BAD_ARG, "eps must not be negative");
  return FLK_OK;
}

static Plan plan_of(const flk_layer_norm_args* p, bool backward) {
  const int es = esize_of((int)p->dtype);
  bool al = is_aligned(p->x, p->x_outer_stride, p->x_inner_stride, es);
  if (backward)
    al = al && is_aligned(p->dy, p->dy_outer_stride, p->dy_inner_stride, es) && is_aligned(p->dx, 0, 0, es);
  else
    al = al && is_aligned(p->y, 0, 0, es);
  return make_plan(es, p->n, p->d, al, backward);
}

}  // namespace norm
}  // namespace flk

using namespace flk;

extern "C" {

int flk_layer_norm_forward(const flk_layer_norm_args* p, void* stream) {
  FLK_TRY(norm::check(p));
  if (p->n == 0) return FLK_OK;
  if (p->x == nullptr || p->y == nullptr) return fail(FLK_ERR_BAD_ARG, "x / y: null pointer");
  if ((p->mean == nullptr) != (p->rstd == nullptr)) return fail(FLK_ERR_BAD_ARG, "mean and rstd are given together");
  norm::Args a{};
  a.n = p->n, a.d = (int)p->d, a.wdtype = (int)p->wdtype, a.eps = (float)p->eps, a.inv_d = (float)(1.0 / (double)p->d);
  a.x = p->x, a.w = p->weight, a.b = p->bias, a.y = p->y, a.mean = p->mean, a.rstd = p->rstd;
  a.xr = {p->x_inner, p->x_outer_stride, p->x_inner_stride};
  const norm::Plan plan = norm::plan_of(p, false);
  a.tpr = plan.tpr;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (p->dtype == FLK_F32) FLK_TRY(norm::launch_forward<float>(a, plan, st));
  else if (p->dtype == FLK_BF16) FLK_TRY(norm::launch_forward<__nv_bfloat16>(a, plan, st));
  else FLK_TRY(norm::launch_forward<__half>(a, plan, st));
  FLK_CUDA_TRY(cudaGetLastError());
  return FLK_OK;
}

int64_t flk_layer_norm_workspace_bytes(const flk_layer_norm_args* p) {
  const int s = norm::check(p);
  if (s != FLK_OK) return s;
  if (p->dweight == nullptr && p->dbias == nullptr) return 0;
  return norm::plan_of(p, true).blocks * 2 * p->d * 4;
}

int flk_layer_norm_backward(const flk_layer_norm_args* p, void* stream) {
  FLK_TRY(norm::check(p));
  const bool sums = p->dweight != nullptr || p->dbias != nullptr;
  if (p->n == 0 && !sums) return FLK_OK;
  if (p->dy_inner < 1) return fail(FLK_ERR_BAD_ARG, "dy_inner must be at least 1");
  if (p->n > 0 && (p->x == nullptr || p->dy == nullptr || p->mean == nullptr || p->rstd == nullptr))
    return fail(FLK_ERR_BAD_ARG, "x, dy, mean and rstd are needed");
  norm::Args a{};
  a.n = p->n, a.d = (int)p->d, a.wdtype = (int)p->wdtype, a.eps = (float)p->eps, a.inv_d = (float)(1.0 / (double)p->d);
  a.x = p->x, a.dy = p->dy, a.w = p->weight, a.dx = p->dx, a.mean = p->mean, a.rstd = p->rstd;
  a.xr = {p->x_inner, p->x_outer_stride, p->x_inner_stride};
  a.dyr = {p->dy_inner, p->dy_outer_stride, p->dy_inner_stride};
  const norm::Plan plan = norm::plan_of(p, true);
  a.tpr = plan.tpr;
  if (sums) {
    const int64_t need = plan.blocks * 2 * p->d * 4;
    if (p->workspace == nullptr || p->workspace_bytes < need || reinterpret_cast<uintptr_t>(p->workspace) % 16 != 0)
      return fail(FLK_ERR_WORKSPACE, "layer norm needs %lld bytes of 16-byte aligned workspace", (long long)need);
    a.part = reinterpret_cast<float*>(p->workspace);
  }
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (p->n > 0) {
    if (p->dtype == FLK_F32) FLK_TRY(norm::launch_backward<float>(a, plan, st));
    else if (p->dtype == FLK_BF16) FLK_TRY(norm::launch_backward<__nv_bfloat16>(a, plan, st));
    else FLK_TRY(norm::launch_backward<__half>(a, plan, st));
  }
  if (sums) {
    norm::reduce_kernel<<<dim3((unsigned)ceil_div(p->d, 32), 2), 256, 0, st>>>(a.part, p->n > 0 ? plan.blocks : 0, a.d,
                                                                               p->dweight, p->dbias, a.wdtype);
    count_launch();
  }
  FLK_CUDA_TRY(cudaGetLastError());
  return FLK_OK;
}

}  // extern "C"
