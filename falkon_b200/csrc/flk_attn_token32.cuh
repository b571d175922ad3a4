// Attention of a few query rows over a long key axis (single tokens over a cache): forward, fp32 data.
//
// Bound by the bytes of the cache with one row per key head (32 caches of 4000 keys, 8 heads of 64: 89 us, 5.9 TB/s), by
// instructions with four (8 caches of 16384 keys, 16 heads of 128 on 4: 135 us, 4.0 TB/s).  With the prompts' kernel, tiles of 64
// rows for each query head and the whole cache to a block, these took 545 and 2283 us.  Eight lanes share a key, each with DM / 8 of its columns in registers, so a warp reads four
// keys at a time in pieces of 128 bytes; two keys per lane are under way.  The rows that share a key head (RW at a time, 1 to
// 512 / DM, more in further blocks, which find the keys in L2) stay in registers beside their accumulators.  Each eighth of a warp has its own
// maximum, sum and accumulators, which are joined at the end, so nothing waits for another warp in between, and no sum is
// longer than a sixteenth of the block's keys.  Every block writes partial results (fp32, normalised) that the joining kernel
// of the prompts adds up in a fixed order.
#pragma once

#include "flk_attn_fwd.cuh"
#include "flk_attn_simt.cuh"

namespace flk {
namespace attn {
namespace token32 {

constexpr int kWarps = 4, kLanes = 8, kKeys = kWarps * 32 / kLanes;  // keys that a block works on side by side

template <int DM, int RW>
__global__ void __launch_bounds__(kWarps * 32, RW * DM <= 64 ? 5 : RW * DM <= 128 ? 4 : RW * DM <= 256 ? 3 : 2) kernel(const TcArgs t) {
  constexpr int kPairs = DM / 16, kPieces = DM / 32;
  __shared__ int4 row_of[RW];  // end, label, slope (base 2), position
  __shared__ float shared_m[kKeys][RW], shared_l[kKeys][RW];
  __shared__ __align__(16) float buf[kWarps][RW][DM];
  const Args& a = t.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, part = lane % kLanes, mine = warp * 4 + lane / kLanes;
  uint32_t id = blockIdx.x;
  const uint32_t chunks = (uint32_t)(t.rows + RW - 1) / RW;
  const int r0 = (int)(id % chunks) * RW;
  id /= chunks;
  const int hk = (int)(id % (uint32_t)a.hk);
  id /= (uint32_t)a.hk;
  const int b = (int)(id % (uint32_t)a.b), split = (int)(id / (uint32_t)a.b);
  const Limits lim = limits_of(a, b);
  const int* kd = a.kdocs ? a.kdocs + (int64_t)b * a.nk_pad : nullptr;
  // the block's keys: a share of the groups of 16 up to the last key that a row sees
  const int groups = (lim.row_end(a.nq - 1, a.causal) + kKeys - 1) / kKeys;
  const int even = (int)((uint32_t)groups / (uint32_t)t.splits), odd = groups - even * t.splits;
  const int first = split * even + min(split, odd), last = first + even + (split < odd ? 1 : 0);
  if (threadIdx.x < RW) {
    const int r = r0 + threadIdx.x, i = r / a.grp, h = hk * a.grp + r - i * a.grp;
    const bool exists = r < t.rows;
    row_of[threadIdx.x] = make_int4(exists ? lim.row_end(i, a.causal) : 0, a.qdocs != nullptr && exists ? a.qdocs[(int64_t)b * a.nq_pad + i] : -2,
                                    __float_as_int(a.slopes != nullptr && exists ? a.slopes[h] * kLog2e : 0.f), lim.at + i);
  }
  // columns 4 part + 32 c and up of the rows, in pairs
  uint64_t q[RW][kPairs], acc[RW][kPairs] = {};
  float m[RW], l[RW];
#pragma unroll
  for (int w = 0; w < RW; ++w) {
    const int r = r0 + w, i = r / a.grp;
    const float* row = reinterpret_cast<const float*>(a.q.p) + b * a.q.sb + (int64_t)i * a.q.sn + (int64_t)(hk * a.grp + r - i * a.grp) * a.q.sh;
#pragma unroll
    for (int c = 0; c < kPieces; ++c) {
      ulonglong2 x = make_ulonglong2(0, 0);
      if (r < t.rows && 4 * part + 32 * c < a.d) x = *reinterpret_cast<const ulonglong2*>(row + 4 * part + 32 * c);
      q[w][2 * c] = x.x, q[w][2 * c + 1] = x.y;
    }
    m[w] = -INFINITY;
    l[w] = 0.f;
  }
  const float *K = reinterpret_cast<const float*>(a.k.p) + b * a.k.sb + hk * a.k.sh, *V = reinterpret_cast<const float*>(a.v.p) + b * a.v.sb + hk * a.v.sh;
  __syncthreads();
  // the keys of a turn: two groups of 16; keys that nobody may see are read as zeros
  for (int g = first; g < last; g += 2) {
    ulonglong2 k[2][kPieces], v[2][kPieces];
    int label[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int key = (g + u) * kKeys + mine;
      label[u] = kd != nullptr && key < lim.len ? __ldg(kd + key) : 0;
      const bool valid = g + u < last && key < lim.len && label[u] >= 0;
#pragma unroll
      for (int c = 0; c < kPieces; ++c) {
        const bool in_row = valid && 4 * part + 32 * c < a.d;
        k[u][c] = in_row ? __ldg(reinterpret_cast<const ulonglong2*>(K + key * a.k.sn + 4 * part + 32 * c)) : make_ulonglong2(0, 0);
        v[u][c] = in_row ? __ldg(reinterpret_cast<const ulonglong2*>(V + key * a.v.sn + 4 * part + 32 * c)) : make_ulonglong2(0, 0);
      }
    }
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int key = g + u < last ? (g + u) * kKeys + mine : lim.len;  // (that one is never seen)
#pragma unroll
      for (int w = 0; w < RW; ++w) {
        uint64_t dot = 0;
#pragma unroll
        for (int c = 0; c < kPieces; ++c) {
          dot = tc::fma2(q[w][2 * c], k[u][c].x, dot);
          dot = tc::fma2(q[w][2 * c + 1], k[u][c].y, dot);
        }
        float s0, s1;
        tc::unpack2(dot, s0, s1);
        float s = s0 + s1;
#pragma unroll
        for (int o = kLanes / 2; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        const int4 row = row_of[w];
        s *= a.scale;
        if (a.cap2 != 0.f) s = a.cap2 * tanhf(s);
        s = simt::biased(s, __int_as_float(row.z), row.w - key);
        s = key < row.x && (kd == nullptr || label[u] == row.y) ? s : -INFINITY;
        if (__any_sync(0xffffffffu, s > m[w] + 8.f)) {
          const float mn = fmaxf(m[w], s), f = m[w] == mn ? 1.f : ex2_approx(m[w] - mn);
          const uint64_t ff = tc::pack2(f, f);
          m[w] = mn;
          l[w] *= f;
#pragma unroll
          for (int c = 0; c < kPairs; ++c) acc[w][c] = tc::mul2(acc[w][c], ff);
        }
        const float p = ex2_approx(s - (m[w] == -INFINITY ? 0.f : m[w]));
        l[w] += p;
        const uint64_t pp = tc::pack2(p, p);
#pragma unroll
        for (int c = 0; c < kPieces; ++c) {
          acc[w][2 * c] = tc::fma2(pp, v[u][c].x, acc[w][2 * c]);
          acc[w][2 * c + 1] = tc::fma2(pp, v[u][c].y, acc[w][2 * c + 1]);
        }
      }
    }
  }
  // the 16 results of the block, joined in a fixed order
  if (part == 0) {
#pragma unroll
    for (int w = 0; w < RW; ++w) {
      shared_m[mine][w] = m[w];
      shared_l[mine][w] = l[w];
    }
  }
  __syncthreads();
  const int64_t row0 = (((int64_t)split * a.b + b) * a.hk + hk) * t.rows + r0;
#pragma unroll
  for (int w = 0; w < RW; ++w) {
    float top = -INFINITY, sum = 0.f;
    for (int x = 0; x < kKeys; ++x) top = fmaxf(top, shared_m[x][w]);
    // one whose maximum is -inf has a sum of zero, or NaN where a score is
    for (int x = 0; x < kKeys; ++x) sum += shared_l[x][w] * (shared_m[x][w] == -INFINITY ? 1.f : ex2_approx(shared_m[x][w] - top));
    const float f = sum == 0.f ? 0.f : (m[w] == -INFINITY ? 1.f : ex2_approx(m[w] - top)) / sum;
    if (threadIdx.x == 0 && r0 + w < t.rows) t.part_lse[row0 + w] = sum == 0.f ? -INFINITY : top + log2f(sum);
#pragma unroll
    for (int c = 0; c < kPairs; ++c) {
      float x, y;
      tc::unpack2(acc[w][c], x, y);
      x *= f, y *= f;
#pragma unroll
      for (int o = kLanes; o < 32; o <<= 1) {
        x += __shfl_xor_sync(0xffffffffu, x, o);
        y += __shfl_xor_sync(0xffffffffu, y, o);
      }
      if (lane < kLanes) *reinterpret_cast<float2*>(&buf[warp][w][4 * part + 32 * (c / 2) + 2 * (c % 2)]) = make_float2(x, y);
    }
  }
  __syncthreads();
  for (int e = threadIdx.x; e < RW * DM / 4; e += kWarps * 32) {
    const int w = e / (DM / 4), c = e % (DM / 4) * 4;
    if (c >= a.d || r0 + w >= t.rows) continue;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int x = 0; x < kWarps; ++x) {
      const float4 y = *reinterpret_cast<const float4*>(&buf[x][w][c]);
      v.x += y.x, v.y += y.y, v.z += y.z, v.w += y.w;
    }
    *reinterpret_cast<float4*>(t.part_o + (row0 + w) * a.d + c) = v;
  }
}

// Whether this kernel takes a call, and the parts of the key axis: some blocks more than fit the SMs side by side (two each), so
// that ragged lengths even out, but no less than 128 keys to a block.
inline bool takes(int nq, int grp) { return (int64_t)nq * grp <= 16; }
// Rows that a block takes: as few as there are, a power of two, up to what registers hold.
inline int rows_of(int rows, int d) {
  int n = 1;
  while (n < rows && n < (d <= 64 ? 8 : 4)) n <<= 1;
  return n;
}
inline int splits_of(int b, int nq, int nk, int hq, int hk, int d) {
  const int64_t blocks = (int64_t)b * hk * ceil_div(nq * (hq / hk), rows_of(nq * (hq / hk), d)), want = ceil_div((int64_t)8 * kNumSMs, blocks), most = ceil_div(nk, 128);
  return (int)(want < most ? want : most);
}

inline int launch(TcArgs t, int splits, cudaStream_t st) {
  const Args& a = t.a;
  t.pg = a.grp, t.hp = a.hk, t.rows = a.nq * a.grp, t.splits = splits;
  const int rw = rows_of(t.rows, a.d);
  const int64_t grid = ceil_div(t.rows, rw) * splits * a.b * a.hk;
  if (grid > INT32_MAX) return fail(FLK_ERR_UNSUPPORTED, "too many blocks");
  auto* fn = a.d <= 64 ? (rw == 1 ? kernel<64, 1> : rw == 2 ? kernel<64, 2> : rw == 4 ? kernel<64, 4> : kernel<64, 8>)
                       : (rw == 1 ? kernel<128, 1> : rw == 2 ? kernel<128, 2> : kernel<128, 4>);
  fn<<<(unsigned)grid, kWarps * 32, 0, st>>>(t);
  count_launch();
  return fwd::launch_join<float>(t, splits, st);
}

}  // namespace token32
}  // namespace attn
}  // namespace flk
