// Attention of a few query rows over a long key axis (single tokens over a cache): forward, 16-bit data.
//
// Bound by the bytes of the cache.  The rows that share a key head, up to 16, are the 16 rows of mma.sync tiles; a warp walks
// over 16 keys at a time, which it copies itself (cp.async) into a ring of its own in shared memory, so warps never wait for one
// another before the end.  Scores stay in registers and become the A operand of the second product as they are.  Blocks of four
// warps, two or three to an SM, keep about 128 KB per SM under way, whatever the lengths.  The tensor-core work is far from any bound
// here (16 rows of 16 keys are read once and used once), so the tcgen05 pipeline, its tensor memory and its barriers would only
// add latency: one token over ragged caches of up to 5001 keys, 24 x 16 heads of 64, took 96 us with the prompts' kernel and
// takes 54 us with this one, 38 us being the bytes' time.
// Every block writes partial results (fp32, normalised) that the joining kernel of the prompts adds up in a fixed order.
#pragma once

#include "flk_attn_fwd.cuh"

namespace flk {
namespace attn {
namespace token {

constexpr int kWarps = 4, kRows = 16, kKeys = 16;

template <int DP>
struct Layout {
  static constexpr int kRowBytes = DP * 2;
  static constexpr int kHalf = kKeys * kRowBytes;  // K or V of a stage
  static constexpr int kStages = DP == 64 ? 4 : 3;
  static constexpr int kWarpBytes = kStages * 2 * kHalf;
  static constexpr int kBytes = kWarps * kWarpBytes;
};

__device__ __forceinline__ void cp_async16_zfill(uint32_t dst, const void* src, bool valid) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(valid ? 16 : 0) : "memory");
}
__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
// D (16 x 8, fp32) += A (16 x 16) B (16 x 8)
template <typename T>
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

template <typename T, int DP, bool CAP, bool BIAS>
__global__ void __launch_bounds__(kWarps * 32, DP == 64 ? 3 : 2) kernel(const TcArgs t) {
  using L = Layout<DP>;
  extern __shared__ __align__(1024) uint8_t raw[];
  __shared__ float shared_m[kWarps][kRows], shared_l[kWarps][kRows];
  const Args& a = t.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint32_t id = blockIdx.x;
  const int hk = (int)(id % (uint32_t)a.hk);
  id /= (uint32_t)a.hk;
  const int b = (int)(id % (uint32_t)a.b), split = (int)(id / (uint32_t)a.b);
  const Limits lim = limits_of(a, b);
  const int* kd = a.kdocs ? a.kdocs + (int64_t)b * a.nk_pad : nullptr;
  const int* qd = a.qdocs ? a.qdocs + (int64_t)b * a.nq_pad : nullptr;
  // the block's keys: a share of the groups of 16 up to the last key that a row sees
  const int groups = (lim.row_end(a.nq - 1, a.causal) + kKeys - 1) / kKeys;
  const int even = (int)((uint32_t)groups / (uint32_t)t.splits), odd = groups - even * t.splits;
  const int first = split * even + min(split, odd), last = first + even + (split < odd ? 1 : 0);

  // rows lane / 4 and lane / 4 + 8 of the tile; row r is query r / grp of head r % grp
  int end[2], my[2], pos[2];
  float slope2[2];
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int r = lane / 4 + 8 * e;
    const bool exists = r < t.rows;
    const int i = exists ? (int)((uint32_t)r / (uint32_t)a.grp) : 0, h = hk * a.grp + (exists ? r - i * a.grp : 0);
    end[e] = exists ? lim.row_end(i, a.causal) : 0;
    my[e] = qd != nullptr && exists ? qd[i] : -2;
    slope2[e] = BIAS && a.slopes != nullptr ? a.slopes[h] * kLog2e : 0.f;
    pos[e] = lim.at + i;
  }
  // the queries as A operands: columns 2 (lane % 4) and up of rows lane / 4, lane / 4 + 8
  uint32_t q[DP / 16][4];
  {
    const T* base = reinterpret_cast<const T*>(a.q.p) + b * a.q.sb;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int r = lane / 4 + 8 * e;
      const int i = (int)((uint32_t)r / (uint32_t)a.grp);
      const T* row = base + (int64_t)i * a.q.sn + (int64_t)(hk * a.grp + r - i * a.grp) * a.q.sh;
#pragma unroll
      for (int ks = 0; ks < DP / 16; ++ks)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const int c = ks * 16 + half * 8 + 2 * (lane % 4);
          q[ks][e + 2 * half] = r < t.rows && c < a.d ? *reinterpret_cast<const uint32_t*>(row + c) : 0u;
        }
    }
  }
  const uint32_t ring = tc::smem_u32(raw) + warp * L::kWarpBytes;
  const T *K = reinterpret_cast<const T*>(a.k.p) + b * a.k.sb + hk * a.k.sh, *V = reinterpret_cast<const T*>(a.v.p) + b * a.v.sb + hk * a.v.sh;
  // 16 bytes `chunk` of rows r0, r0 + rows per pass, ... ; rows that nobody may see become zeros
  constexpr int kChunks = DP / 8, kPass = 32 / kChunks;
  const int chunk = lane % kChunks, r0 = lane / kChunks;
  const bool in_row = chunk * 8 < a.d;
  auto fetch = [&](int stage, int group) {
    const uint32_t dst = ring + stage * 2 * L::kHalf;
#pragma unroll
    for (int p = 0; p < kKeys / kPass; ++p) {
      const int r = r0 + p * kPass, key = group * kKeys + r;
      const bool valid = in_row && key < lim.len && (kd == nullptr || __ldg(kd + key) >= 0);
      const uint32_t at = dst + r * L::kRowBytes + ((chunk ^ (r & 7)) * 16);
      // an address inside the tensor even where nothing is read
      const int64_t row = valid ? key : 0;
      cp_async16_zfill(at, K + row * a.k.sn + (valid ? chunk * 8 : 0), valid);
      cp_async16_zfill(at + L::kHalf, V + row * a.v.sn + (valid ? chunk * 8 : 0), valid);
    }
  };
  int at = first + warp;  // group that is worked on
#pragma unroll
  for (int s = 0; s < L::kStages; ++s) {
    if (at + s * kWarps < last) fetch(s, at + s * kWarps);
    cp_async_commit();
  }
  float o[DP / 8][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
  for (int n = 0; n < DP / 8; ++n)
#pragma unroll
    for (int e = 0; e < 4; ++e) o[n][e] = 0.f;
  const float f2 = CAP ? a.cap2 : a.scale;
  int stage = 0;
  for (; at < last; at += kWarps) {
    cp_async_wait<L::kStages - 1>();
    __syncwarp();
    const uint32_t kt = ring + stage * 2 * L::kHalf, vt = kt + L::kHalf;
    float s[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};  // keys 0 to 7 and 8 to 15
#pragma unroll
    for (int ks = 0; ks < DP / 16; ++ks) {
      // matrices: keys 0 to 7 and 8 to 15 by columns 16 ks and 16 ks + 8
      uint32_t f[4];
      const int row = (lane & 7) + ((lane >> 4) << 3), c = 2 * ks + ((lane >> 3) & 1);
      ldmatrix4(f, kt + row * L::kRowBytes + ((c ^ (row & 7)) * 16));
      mma<T>(s[0], q[ks], f[0], f[1]);
      mma<T>(s[1], q[ks], f[2], f[3]);
    }
    const int k0 = at * kKeys + 2 * (lane % 4);
    if constexpr (CAP) {
      float big = 0.f;
#pragma unroll
      for (int e = 0; e < 4; ++e) big = fmaxf(big, fmaxf(fabsf(s[0][e]), fabsf(s[1][e])));
      const bool small = __all_sync(0xffffffffu, big <= t.tanh.limit);
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int e = 0; e < 4; e += 2) {
          const uint64_t x = tc::pack2(s[n][e], s[n][e + 1]);
          if (small) {
            tc::unpack2(tc::mul2(tanh_slope<false>(x, t.tanh), x), s[n][e], s[n][e + 1]);
          } else {
            s[n][e] = tanh_any(s[n][e], a.scale);
            s[n][e + 1] = tanh_any(s[n][e + 1], a.scale);
          }
        }
    }
    float top[2] = {-INFINITY, -INFINITY};
    const float d0[2] = {(float)(pos[0] - k0), (float)(pos[1] - k0)};  // exact where it matters, however far the row and the key lie
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int row = e / 2, key = k0 + 8 * n + e % 2;
        float x = s[n][e] * f2;
        if constexpr (BIAS) x = fmaf(-slope2[row], fabsf(d0[row] - (float)(8 * n + e % 2)), x);
        const bool see = key < end[row] && (kd == nullptr || __ldg(kd + key) == my[row]);
        s[n][e] = see ? x : -INFINITY;
        top[row] = fmaxf(top[row], s[n][e]);
      }
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      top[e] = fmaxf(top[e], __shfl_xor_sync(0xffffffffu, top[e], 1));
      top[e] = fmaxf(top[e], __shfl_xor_sync(0xffffffffu, top[e], 2));
    }
    const bool grow = top[0] > m[0] + 8.f || top[1] > m[1] + 8.f;
    if (__any_sync(0xffffffffu, grow)) {
      float f[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float mn = fmaxf(m[e], top[e]);
        f[e] = m[e] == mn ? 1.f : ex2_approx(m[e] - mn);
        m[e] = mn;
        l[e] *= f[e];
      }
#pragma unroll
      for (int n = 0; n < DP / 8; ++n) {
        o[n][0] *= f[0];
        o[n][1] *= f[0];
        o[n][2] *= f[1];
        o[n][3] *= f[1];
      }
    }
    float p[2][4];
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float base = (m[e / 2] == -INFINITY ? 0.f : m[e / 2]) - kLift<T>;
        p[n][e] = ex2_approx(s[n][e] - base);
        l[e / 2] += p[n][e];
      }
    // rounded to the data's type, as the prompts' kernel does: half a step of each weight, as much as the result itself is rounded by
    // (rms error of bf16 results 2.0e-3 to 2.3e-3 of their size; rounding alone 1.6e-3, and with what rounding takes in a second operand
    // that, but 32 long caches then take 566 us instead of 533, 24 ragged ones 65 instead of 62)
    const uint32_t w[4] = {pack16<T>(p[0][0], p[0][1]), pack16<T>(p[0][2], p[0][3]), pack16<T>(p[1][0], p[1][1]), pack16<T>(p[1][2], p[1][3])};
#pragma unroll
    for (int n = 0; n < DP / 16; ++n) {
      // matrices: keys 0 to 7, 8 to 15 by columns 16 n, then by columns 16 n + 8, transposed
      uint32_t f[4];
      const int row = (lane & 7) + (((lane >> 3) & 1) << 3), c = 2 * n + (lane >> 4);
      ldmatrix4_trans(f, vt + row * L::kRowBytes + ((c ^ (row & 7)) * 16));
      mma<T>(o[2 * n], w, f[0], f[1]);
      mma<T>(o[2 * n + 1], w, f[2], f[3]);
    }
    __syncwarp();  // all lanes have read the stage
    if (at + L::kStages * kWarps < last) fetch(stage, at + L::kStages * kWarps);
    cp_async_commit();
    stage = stage + 1 == L::kStages ? 0 : stage + 1;
  }
  cp_async_wait<0>();
  // the warps' results, joined in order
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    l[e] += __shfl_xor_sync(0xffffffffu, l[e], 1);
    l[e] += __shfl_xor_sync(0xffffffffu, l[e], 2);
    if (lane % 4 == 0) {
      shared_m[warp][lane / 4 + 8 * e] = m[e];
      shared_l[warp][lane / 4 + 8 * e] = l[e];
    }
  }
  __syncthreads();
  float* buf = reinterpret_cast<float*>(raw);  // [warp][row][DP + 4]
  constexpr int kLd = DP + 4;
  static_assert(kWarps * kRows * kLd * 4 <= L::kBytes, "shared memory");
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int r = lane / 4 + 8 * e;
    float top = -INFINITY, sum = 0.f;
#pragma unroll
    for (int x = 0; x < kWarps; ++x) top = fmaxf(top, shared_m[x][r]);
#pragma unroll
    // a warp whose maximum is -inf has a sum of zero, or NaN where a score is
    for (int x = 0; x < kWarps; ++x) sum += shared_l[x][r] * (shared_m[x][r] == -INFINITY ? 1.f : ex2_approx(shared_m[x][r] - top));
    const float f = sum == 0.f ? 0.f : (m[e] == -INFINITY ? 1.f : ex2_approx(m[e] - top)) / sum;
#pragma unroll
    for (int n = 0; n < DP / 8; ++n)
      *reinterpret_cast<float2*>(buf + (warp * kRows + r) * kLd + n * 8 + 2 * (lane % 4)) = make_float2(o[n][2 * e] * f, o[n][2 * e + 1] * f);
    if (warp == 0 && lane % 4 == 0 && r < t.rows)
      t.part_lse[(((int64_t)split * a.b + b) * a.hk + hk) * t.rows + r] = sum == 0.f ? -INFINITY : top - kLift<T> + log2f(sum);
  }
  __syncthreads();
  const int64_t row0 = (((int64_t)split * a.b + b) * a.hk + hk) * t.rows;
  for (int e = threadIdx.x; e < t.rows * (DP / 4); e += kWarps * 32) {
    const int r = e / (DP / 4), c = e % (DP / 4) * 4;
    if (c >= a.d) continue;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int x = 0; x < kWarps; ++x) {
      const float4 y = *reinterpret_cast<const float4*>(buf + (x * kRows + r) * kLd + c);
      v.x += y.x, v.y += y.y, v.z += y.z, v.w += y.w;
    }
    *reinterpret_cast<float4*>(t.part_o + (row0 + r) * a.d + c) = v;
  }
}

// Whether this kernel takes a call, and the parts of the key axis: about 12 blocks per SM, so that ragged lengths even out (32
// caches of 16384 to 32768 keys: 515 us with 2 blocks per SM, 479 with 8, 470 with 12), but no less than 128 keys to a block.
inline bool takes(int nq, int grp) { return (int64_t)nq * grp <= kRows; }
inline int splits_of(int b, int nk, int hk) {
  const int64_t blocks = (int64_t)b * hk, want = ceil_div((int64_t)12 * kNumSMs, blocks), most = ceil_div(nk, 128);
  return (int)(want < most ? want : most);
}

template <typename T, int DP, bool CAP, bool BIAS>
inline int launch_one(const TcArgs& t, cudaStream_t st) {
  auto* fn = kernel<T, DP, CAP, BIAS>;
  constexpr int kBytes = Layout<DP>::kBytes;
  static std::atomic<uint64_t> done{0};
  FLK_TRY(allow_shared(reinterpret_cast<const void*>(fn), kBytes, done));
  const int64_t grid = (int64_t)t.splits * t.a.b * t.a.hk;
  if (grid > INT32_MAX) return fail(FLK_ERR_UNSUPPORTED, "too many blocks");
  fn<<<(unsigned)grid, kWarps * 32, kBytes, st>>>(t);
  count_launch();
  return FLK_OK;
}
template <typename T>
inline int launch(TcArgs t, int splits, cudaStream_t st) {
  const Args& a = t.a;
  t.pg = a.grp, t.hp = a.hk, t.rows = a.nq * a.grp, t.splits = splits;
  t.tanh = make_tanh(a.scale);
  const bool cap = a.cap2 != 0.f, bias = a.slopes != nullptr;
  if (a.d <= 64) {
    if (cap) FLK_TRY((bias ? launch_one<T, 64, true, true>(t, st) : launch_one<T, 64, true, false>(t, st)));
    else FLK_TRY((bias ? launch_one<T, 64, false, true>(t, st) : launch_one<T, 64, false, false>(t, st)));
  } else {
    if (cap) FLK_TRY((bias ? launch_one<T, 128, true, true>(t, st) : launch_one<T, 128, true, false>(t, st)));
    else FLK_TRY((bias ? launch_one<T, 128, false, true>(t, st) : launch_one<T, 128, false, false>(t, st)));
  }
  return fwd::launch_join<T>(t, splits, st);
}

}  // namespace token
}  // namespace attn
}  // namespace flk
