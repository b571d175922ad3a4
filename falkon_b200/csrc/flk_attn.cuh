// Shared definitions of the attention kernels: arguments, visibility, scores.
//
//   r_ij = scale q_i . k_j          s_ij = cap tanh(r_ij / cap)  (or r_ij)  -  slope_h |p_i - j|,   p_i = start + i
//   visible(i, j) = j < L  and  (not causal or j <= p_i or j < prefix)  and  (no documents or dq_i == dk_j >= 0)
//   P = softmax of s over the visible j (all zeros where there is none),  O = P V
//
// Everything about causality, the prefix and the length is one bound per row: row i sees j < row_end(i), among those the
// keys of its document.  Scores are kept in base 2 (multiplied by log2 e), so that the exponential is one ex2.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "flk_common.cuh"

namespace flk {
namespace attn {

constexpr int kMaxHeadDim = 128;
constexpr int kTile = 128;  // tile of the document labels' table (and of the tensor-core kernels)

struct Tensor4 {  // (batch, rows, heads, d), unit stride over d, strides in elements
  void* p;
  int64_t sb, sn, sh;
};

struct Args {
  int b, nq, nk, hq, hk, grp, d;
  int causal;
  float scale;          // of the dot product (without cap: times log2 e)
  float cap2;           // cap * log2 e; 0: no cap.  With a cap, `scale` is scale / cap
  float scale_raw;      // scale as given: the factor of dq and dk
  const float* slopes;  // per query head, or null
  const int *prefix, *kv_lens, *q_starts;
  const int *qdocs, *kdocs;  // padded tables of the workspace ([b][nq_pad], [b][nk_pad]; -2 / -1 where nothing is seen), or null
  const int4 *qtab, *ktab;   // of every tile: smallest, largest label, whether a row has none ([b][nq_pad / q_rows], [b][nk_pad / 128])
  int q_rows;                // queries of a tile of qtab
  int nq_pad, nk_pad;
  Tensor4 q, k, v, o, dout, dq, dk, dv;
  void* o_lo;    // what rounding took from `o` (16-bit types; strides of o), or null
  float* lse;    // (b, hq, nq), natural logarithm; -inf for rows that see nothing
  float* delta;  // (b, hq, nq)
};

struct Limits {  // of one sequence; no query sees keys at or behind `len`
  int len, start, prefix;
  int at;  // `start` as distances are counted from it
  __device__ __forceinline__ int row_end(int i, int causal) const {
    if (!causal) return len;
    const int e = max(start + i + 1, prefix);
    return min(max(e, 0), len);
  }
};
__device__ __forceinline__ Limits limits_of(const Args& a, int b) {
  Limits l;
  l.len = a.kv_lens != nullptr ? min(max(a.kv_lens[b], 0), a.nk) : a.nk;
  // positions stay far from the ends of int, whatever the caller's table holds
  l.start = a.q_starts != nullptr ? min(max(a.q_starts[b], -(1 << 29)), 1 << 29) : l.len - a.nq;
  // Where all queries stand behind all keys, or before them, the distance between the two is the same for every pair and changes
  // no weight; fp32 scores would lose their digits to it.  It is left out of the scores, and of the log-sum-exp that is kept.
  l.at = min(max(l.start, -a.nq), max(l.len, 1) - 1);
  l.prefix = a.prefix != nullptr ? a.prefix[b] : 0;
  // under a causal mask what lies behind the last query (the rest of a cache, say) may hold anything too
  l.len = l.row_end(a.nq - 1, a.causal);
  return l;
}

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

constexpr float kLn2 = 0.6931471805599453f;

}  // namespace attn
}  // namespace flk
