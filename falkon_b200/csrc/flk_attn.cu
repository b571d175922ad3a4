// extern "C" entry points of attention: argument checks, workspace, choice of kernel.
#include "flk_attn.cuh"
#include "flk_attn_bwd.cuh"
#include "flk_attn_fwd.cuh"
#include "flk_attn_rows.cuh"
#include "flk_attn_simt.cuh"
#include "flk_attn_token.cuh"
#include "flk_attn_token32.cuh"

namespace flk {
namespace attn {

int forward_bf16(const TcArgs& t, const fwd::Plan& p, cudaStream_t st);
int forward_f16(const TcArgs& t, const fwd::Plan& p, cudaStream_t st);
int forward_status_bf16(cudaStream_t st, int* out);
int forward_status_f16(cudaStream_t st, int* out);
int token_bf16(const TcArgs& t, int splits, cudaStream_t st);
int token_f16(const TcArgs& t, int splits, cudaStream_t st);
int backward_bf16(const TcArgs& t, const bwd::Plan& p, cudaStream_t st);
int backward_f16(const TcArgs& t, const bwd::Plan& p, cudaStream_t st);
int backward_status_bf16(cudaStream_t st, int* out);
int backward_status_f16(cudaStream_t st, int* out);

// The tables of documents: labels padded to whole tiles, `none` (-1 for keys, -2 for queries) where nothing may be seen, and,
// for every tile of `per` rows (a power of two from 2 to 128), the smallest and largest label and whether a row has none (a tile
// of none: a range that meets no other).  One warp per 128 rows, four rows per lane.
struct DocTable {
  const int* docs;
  int64_t sb;
  const int* lens;
  int n, n_pad, none, per;
  int* out;
  int4* tab;
};
struct DocTables {
  DocTable of[2];  // queries, keys
};
__global__ void __launch_bounds__(128) documents_kernel(const DocTables both) {
  const DocTable& a = both.of[blockIdx.z];
  const int b = blockIdx.y, r0 = (blockIdx.x * 4 + (threadIdx.x >> 5)) * kTile, lane = threadIdx.x & 31;
  if (r0 >= a.n_pad) return;
  const int len = a.lens != nullptr ? min(max(a.lens[b], 0), a.n) : a.n;
  int id[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int i = r0 + 4 * lane + e;
    id[e] = i < len ? a.docs[b * a.sb + i] : -1;
  }
  int lo[2], hi[2], bad[2];
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int x = id[2 * e], y = id[2 * e + 1];
    lo[e] = min(x >= 0 ? x : INT32_MAX, y >= 0 ? y : INT32_MAX);
    hi[e] = max(x >= 0 ? x : INT32_MIN, y >= 0 ? y : INT32_MIN);
    bad[e] = x < 0 || y < 0;
  }
  int4* tab = a.tab + (int64_t)b * (a.n_pad / a.per);
  *reinterpret_cast<int4*>(a.out + (int64_t)b * a.n_pad + r0 + 4 * lane) =
      make_int4(id[0] >= 0 ? id[0] : a.none, id[1] >= 0 ? id[1] : a.none, id[2] >= 0 ? id[2] : a.none, id[3] >= 0 ? id[3] : a.none);
  if (a.per == 2) {
    tab[r0 / 2 + 2 * lane] = make_int4(lo[0], hi[0], bad[0], 0);
    tab[r0 / 2 + 2 * lane + 1] = make_int4(lo[1], hi[1], bad[1], 0);
    return;
  }
  lo[0] = min(lo[0], lo[1]);
  hi[0] = max(hi[0], hi[1]);
  bad[0] |= bad[1];
  for (int o = a.per / 8; o > 0; o >>= 1) {
    lo[0] = min(lo[0], __shfl_xor_sync(0xffffffffu, lo[0], o));
    hi[0] = max(hi[0], __shfl_xor_sync(0xffffffffu, hi[0], o));
    bad[0] |= __shfl_xor_sync(0xffffffffu, bad[0], o);
  }
  if (4 * lane % a.per == 0) tab[(r0 + 4 * lane) / a.per] = make_int4(lo[0], hi[0], bad[0], 0);
}

// The order in which blocks start, those with the most tiles to visit first: with documents of several lengths a block that
// starts late and works long would be what a kernel ends with (8192 rows of 7 documents: forward 128 -> 117 us, dK and dV 188 ->
// 175 us; the blocks of dQ, many and short, gain nothing: 121, and 123 us in order).  One block: the other side's label ranges go to
// shared memory, a few threads per entry count those that its range meets, and rank the counts.
constexpr int kMostOrdered = 1024, kMostRanges = 2048;
struct OrderList {
  bool keys;        // of key tiles, else of row blocks of `per` tiles
  int blocks, per;  // blocks of a sequence
  int* out;
};
__global__ void __launch_bounds__(1024) order_kernel(const Args a, const OrderList o) {
  __shared__ int2 range[kMostRanges];
  __shared__ __align__(16) int work[kMostOrdered];
  const int n = a.b * o.blocks, q_tiles = a.nq_pad / a.q_rows, k_tiles = a.nk_pad / kTile;
  const int others = o.keys ? q_tiles : k_tiles;
  const int4 *own_tab = o.keys ? a.ktab : a.qtab, *tab = o.keys ? a.qtab : a.ktab;
  for (int e = threadIdx.x; e < a.b * others; e += 1024) {
    const int4 r = __ldg(tab + e);
    range[e] = make_int2(r.x, r.y);
  }
  int per = 32;  // threads per entry, a power of two
  while (per > 1 && per * n > 1024) per >>= 1;
  const int e = threadIdx.x / per, lane = threadIdx.x % per;
  const bool on = e < n;
  const int b = on ? e / o.blocks : 0, at = on ? e % o.blocks : 0;
  int4 own = make_int4(0, 0, 0, 0);
  int first = 0, last = 0;
  if (on) {
    const Limits lim = limits_of(a, b);
    if (o.keys) {
      own = __ldg(own_tab + (int64_t)b * k_tiles + at);
      if (a.causal && lim.prefix <= at * kTile) first = min(max(at * kTile - lim.start, 0), a.nq) / a.q_rows;
      last = at * kTile < lim.len ? q_tiles : 0;
    } else {
      own = __ldg(own_tab + (int64_t)b * q_tiles + at * o.per);
      if (o.per == 2 && at * 2 + 1 < q_tiles) {
        const int4 more = __ldg(own_tab + (int64_t)b * q_tiles + at * 2 + 1);
        own.x = min(own.x, more.x);
        own.y = max(own.y, more.y);
      }
      last = (lim.row_end(min(a.nq, (at + 1) * o.per * a.q_rows) - 1, a.causal) + kTile - 1) / kTile;
    }
  }
  __syncthreads();
  int count = 0;
#pragma unroll 4
  for (int x = first + lane; x < last; x += per) {
    const int2 r = range[b * others + x];
    count += r.x <= own.y && own.x <= r.y;
  }
  for (int x = per / 2; x > 0; x >>= 1) count += __shfl_xor_sync(0xffffffffu, count, x);
  const int key = on ? count * kMostOrdered + (kMostOrdered - 1 - e) : -1;  // no two alike
  if (lane == 0) work[e] = key;
  __syncthreads();
  int rank = 0;
#pragma unroll 4
  for (int x = 4 * lane; x < n; x += 4 * per) {
    const int4 w = *reinterpret_cast<const int4*>(work + x);
    rank += (w.x > key) + (w.y > key) + (w.z > key) + (w.w > key);
  }
  for (int x = per / 2; x > 0; x >>= 1) rank += __shfl_xor_sync(0xffffffffu, rank, x);
  if (on && lane == 0) o.out[rank] = e;
}

static int esize_of(int64_t dtype) { return dtype == FLK_F32 ? 4 : 2; }

static int check_sizes(const flk_attention_args* p) {
  if (p == nullptr) return fail(FLK_ERR_BAD_ARG, "args: null pointer");
  if (p->dtype != FLK_F32 && p->dtype != FLK_BF16 && p->dtype != FLK_F16)
    return fail(FLK_ERR_BAD_ARG, "attention takes fp32, bf16 or fp16 data, not dtype %lld", (long long)p->dtype);
  if (p->flags != 0) return fail(FLK_ERR_BAD_ARG, "flags: none are defined, 0 is expected");
  if (p->batch < 0 || p->nq < 0 || p->nk < 0 || p->hq < 1 || p->hk < 1 || p->d < 1)
    return fail(FLK_ERR_BAD_ARG, "negative or empty sizes");
  if (p->batch > 65535 || p->hq > 65535 || p->nq > (1 << 29) || p->nk > (1 << 29))
    return fail(FLK_ERR_UNSUPPORTED, "at most 65535 sequences and heads, and 2^29 rows");
  // (a last tile's rows are counted up to its end)
  if (p->nq * p->hq > INT32_MAX - 1023 || p->nk * p->hk > INT32_MAX - 1023)
    return fail(FLK_ERR_UNSUPPORTED, "at most 2^31 - 1024 rows of all heads of a sequence");
  if (p->hq % p->hk != 0)
    return fail(FLK_ERR_BAD_ARG, "%lld query heads cannot share %lld key heads", (long long)p->hq, (long long)p->hk);
  const int unit = p->dtype == FLK_F32 ? 4 : 8;
  if (p->d > kMaxHeadDim || p->d % unit != 0)
    return fail(FLK_ERR_UNSUPPORTED, "head dimension %lld: a multiple of %d up to %d", (long long)p->d, unit, kMaxHeadDim);
  if (!(p->softcap >= 0) || p->softcap > 1e30 || !(p->scale > -1e30 && p->scale < 1e30))
    return fail(FLK_ERR_BAD_ARG, "scale must be finite, softcap finite and not negative");
  // the tanh's argument, scale / softcap, and the cap itself are held in fp32
  if (p->softcap > 0 && (p->softcap < 1e-30 || (p->scale < 0 ? -p->scale : p->scale) > p->softcap * 1e30))
    return fail(FLK_ERR_UNSUPPORTED, "softcap %g is too small for scale %g", p->softcap, p->scale);
  if ((p->q_documents == nullptr) != (p->k_documents == nullptr))
    return fail(FLK_ERR_BAD_ARG, "q_documents and k_documents are given together");
  if (p->prefix_lens != nullptr && p->causal == 0) return fail(FLK_ERR_BAD_ARG, "prefix_lens needs causal");
  return FLK_OK;
}

static int check_tensor(const char* name, const flk_tensor4& t, int64_t b, int64_t n, int64_t h, int es) {
  if (b == 0 || n == 0) return FLK_OK;
  if (t.data == nullptr) return fail(FLK_ERR_BAD_ARG, "%s: null pointer", name);
  if (reinterpret_cast<uintptr_t>(t.data) % 16 != 0 || (b > 1 && t.stride_b * es % 16 != 0) || (n > 1 && t.stride_n * es % 16 != 0) ||
      (h > 1 && t.stride_h * es % 16 != 0))
    return fail(FLK_ERR_LAYOUT, "%s: address and strides must be multiples of 16 bytes", name);
  return FLK_OK;
}

// The tensor-core kernels take 16-bit data; without keys there is nothing for them to do.
static bool on_tensor_cores(const flk_attention_args* p) {
  return p->dtype != FLK_F32 && p->nk > 0;
}
static fwd::Plan forward_plan(const flk_attention_args* p) {
  return fwd::make_plan((int)p->batch, (int)p->nq, (int)p->nk, (int)p->hq, (int)p->hk, (int)p->d, p->causal != 0, p->q_documents != nullptr,
                        p->kv_lens != nullptr);
}

// A few rows over many keys (their bytes are the bound) go to the kernel for single tokens.
static bool by_token(const flk_attention_args* p) { return on_tensor_cores(p) && token::takes((int)p->nq, (int)(p->hq / p->hk)); }
static int token_splits(const flk_attention_args* p) { return token::splits_of((int)p->batch, (int)p->nk, (int)p->hk); }
// The same for fp32.
static bool by_token32(const flk_attention_args* p) { return p->dtype == FLK_F32 && token32::takes((int)p->nq, (int)(p->hq / p->hk)); }
static int simt_splits(const flk_attention_args* p) {
  return by_token32(p) ? token32::splits_of((int)p->batch, (int)p->nq, (int)p->nk, (int)p->hq, (int)p->hk, (int)p->d)
                       : simt::splits_of((int)p->batch, (int)p->nq, (int)p->nk, (int)p->hq, (int)p->d, p->causal != 0, p->q_documents != nullptr,
                                         p->kv_lens != nullptr);
}
static bwd::Plan backward_plan(const flk_attention_args* p) {
  return bwd::make_plan((int)p->batch, (int)p->nq, (int)p->nk, (int)p->hq, (int)p->hk, (int)p->d, p->causal != 0, p->q_documents != nullptr);
}
// Queries of a tile of the documents' table: those of a tile of 128 packed rows.
static int query_rows(const flk_attention_args* p) { return on_tensor_cores(p) ? kTile / fwd::packed_heads((int)p->hq, (int)p->hk) : kTile; }

static int64_t pad_rows(int64_t n) { return round_up(n, kTile); }
// Entries of the list of blocks in order; 0: they start in the order of their numbers, because all start at once, or are too
// many for the list.
static int64_t ordered(const flk_attention_args* p, bool backward) {
  if (p->q_documents == nullptr || !on_tensor_cores(p) || (!backward && by_token(p))) return 0;
  const int64_t k_tiles = p->batch * ceil_div(p->nk, kTile), q_tiles = p->batch * pad_rows(p->nq) / query_rows(p);
  const fwd::Plan f = forward_plan(p);
  const int64_t entries = backward ? k_tiles : p->batch * f.blocks, ranges = backward ? q_tiles : k_tiles;
  const int64_t blocks = entries * (backward ? p->hk * backward_plan(p).splits : (int64_t)f.hp * f.splits);
  return entries <= kMostOrdered && ranges <= kMostRanges && blocks > kNumSMs ? entries : 0;
}

struct Workspace {
  int64_t qdocs, kdocs, qtab, ktab, order, delta, part_o, part_lse, total;
};
static Workspace plan_workspace(const flk_attention_args* p, bool backward) {
  Workspace w{};
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    const int64_t here = at;
    at += round_up(bytes, 256);
    return here;
  };
  if (p->q_documents != nullptr) {
    w.qdocs = take(p->batch * pad_rows(p->nq) * 4);
    w.kdocs = take(p->batch * pad_rows(p->nk) * 4);
    w.qtab = take(p->batch * pad_rows(p->nq) / query_rows(p) * 16);
    w.ktab = take(p->batch * pad_rows(p->nk) / kTile * 16);
    w.order = take(ordered(p, backward) * 4);
  }
  if (backward) {
    w.delta = take(p->batch * p->hq * p->nq * 4);
    if (on_tensor_cores(p)) w.part_o = take(bwd::partial_floats(backward_plan(p), p->batch, p->nk, p->hk, p->d) * 4);
  }
  if (!backward && p->batch > 0 && p->nq > 0 && p->nk > 0) {
    int64_t rows;
    if (by_token(p) || p->dtype == FLK_F32) {
      const int64_t parts = by_token(p) ? token_splits(p) : simt_splits(p);
      rows = parts > 1 || by_token(p) || by_token32(p) ? parts * p->batch * p->hq * p->nq : 0;
    } else {
      rows = fwd::partial_rows(forward_plan(p), (int)p->batch);
    }
    w.part_o = take(rows * p->d * 4);
    w.part_lse = take(rows * 4);
  }
  w.total = at;
  return w;
}

static Tensor4 tensor_of(const flk_tensor4& t) { return Tensor4{t.data, t.stride_b, t.stride_n, t.stride_h}; }

// Device arguments, and the tables of documents in the workspace.
static int make_args(const flk_attention_args* p, bool backward, Args& a, cudaStream_t st) {
  const Workspace w = plan_workspace(p, backward);
  if (w.total > 0 && (p->workspace == nullptr || p->workspace_bytes < w.total || reinterpret_cast<uintptr_t>(p->workspace) % 256 != 0))
    return fail(FLK_ERR_WORKSPACE, "attention needs %lld bytes of 256-byte aligned workspace", (long long)w.total);
  char* ws = reinterpret_cast<char*>(p->workspace);
  a = Args{};
  a.b = (int)p->batch, a.nq = (int)p->nq, a.nk = (int)p->nk, a.hq = (int)p->hq, a.hk = (int)p->hk;
  a.grp = (int)(p->hq / p->hk), a.d = (int)p->d, a.causal = p->causal != 0;
  a.scale_raw = (float)p->scale;
  a.scale = (float)(p->softcap > 0 ? p->scale / p->softcap : p->scale * 1.4426950408889634);
  a.cap2 = (float)(p->softcap * 1.4426950408889634);
  a.slopes = p->slopes, a.prefix = p->prefix_lens, a.kv_lens = p->kv_lens, a.q_starts = p->q_starts;
  a.q_rows = query_rows(p), a.nq_pad = (int)pad_rows(p->nq), a.nk_pad = (int)pad_rows(p->nk);
  a.q = tensor_of(p->q), a.k = tensor_of(p->k), a.v = tensor_of(p->v), a.o = tensor_of(p->out);
  a.lse = p->lse, a.o_lo = p->dtype == FLK_F32 ? nullptr : p->out_lo;
  if (backward) {
    a.dout = tensor_of(p->dout), a.dq = tensor_of(p->dq), a.dk = tensor_of(p->dk), a.dv = tensor_of(p->dv);
    a.delta = reinterpret_cast<float*>(ws + w.delta);
  }
  if (p->q_documents != nullptr) {
    int *qd = reinterpret_cast<int*>(ws + w.qdocs), *kd = reinterpret_cast<int*>(ws + w.kdocs);
    int4 *qt = reinterpret_cast<int4*>(ws + w.qtab), *kt = reinterpret_cast<int4*>(ws + w.ktab);
    a.qdocs = qd, a.kdocs = kd, a.qtab = qt, a.ktab = kt;
    DocTables tables;
    tables.of[0] = {p->q_documents, p->q_documents_stride, nullptr, a.nq, a.nq_pad, -2, a.q_rows, qd, qt};
    tables.of[1] = {p->k_documents, p->k_documents_stride, p->kv_lens, a.nk, a.nk_pad, -1, kTile, kd, kt};
    const int most = a.nq_pad > a.nk_pad ? a.nq_pad : a.nk_pad;
    if (most > 0) {
      documents_kernel<<<dim3((unsigned)ceil_div(most / kTile, 4), a.b, 2), 128, 0, st>>>(tables);
      count_launch();
    }
  }
  return FLK_OK;
}

static int launch_order(const flk_attention_args* p, bool backward, int* list, TcArgs& t, cudaStream_t st) {
  if (ordered(p, backward) == 0) return FLK_OK;
  const fwd::Plan f = forward_plan(p);
  t.order = list;
  order_kernel<<<1, 1024, 0, st>>>(t.a, OrderList{backward, backward ? (int)ceil_div(p->nk, kTile) : f.blocks, f.pair ? 2 : 1, list});
  count_launch();
  return FLK_OK;
}

// Zeros for a tensor (and -inf for `lse`, unless null): calls without keys, gradients without queries.
static int write_nothing(int64_t dtype, const Tensor4& o, int b, int n, int h, int d, float* lse, cudaStream_t st) {
  if (dtype == FLK_F32) return launch_nothing<float>(o, b, n, h, d, lse, st);
  return launch_nothing<__half>(o, b, n, h, d, lse, st);  // zeros are the same in both 16-bit types
}

}  // namespace attn
}  // namespace flk

using namespace flk;

extern "C" {

int64_t flk_attention_workspace_bytes(const flk_attention_args* p, int backward) {
  const int s = attn::check_sizes(p);
  if (s != FLK_OK) return s;
  return attn::plan_workspace(p, backward != 0).total;
}

int flk_attention_forward(const flk_attention_args* p, void* stream) {
  FLK_TRY(attn::check_sizes(p));
  const int es = attn::esize_of(p->dtype);
  FLK_TRY(attn::check_tensor("q", p->q, p->batch, p->nq, p->hq, es));
  FLK_TRY(attn::check_tensor("k", p->k, p->batch, p->nk, p->hk, es));
  FLK_TRY(attn::check_tensor("v", p->v, p->batch, p->nk, p->hk, es));
  FLK_TRY(attn::check_tensor("out", p->out, p->batch, p->nq, p->hq, es));
  if (reinterpret_cast<uintptr_t>(p->out_lo) % 16 != 0) return fail(FLK_ERR_LAYOUT, "out_lo: not 16-byte aligned");
  if (p->batch == 0 || p->nq == 0) return FLK_OK;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  attn::Args a;
  FLK_TRY(attn::make_args(p, false, a, st));
  if (a.nk == 0) {
    FLK_TRY(attn::write_nothing(p->dtype, a.o, a.b, a.nq, a.hq, a.d, a.lse, st));
    if (a.o_lo != nullptr) FLK_TRY(attn::write_nothing(p->dtype, attn::Tensor4{a.o_lo, a.o.sb, a.o.sn, a.o.sh}, a.b, a.nq, a.hq, a.d, nullptr, st));
  } else {
    attn::TcArgs t{};
    t.a = a;
    const attn::Workspace w = attn::plan_workspace(p, false);
    char* ws = reinterpret_cast<char*>(p->workspace);
    t.part_o = reinterpret_cast<float*>(ws + w.part_o), t.part_lse = reinterpret_cast<float*>(ws + w.part_lse);
    FLK_TRY(attn::launch_order(p, false, reinterpret_cast<int*>(ws + w.order), t, st));
    if (attn::by_token32(p)) {
      FLK_TRY(attn::token32::launch(t, attn::simt_splits(p), st));
    } else if (p->dtype == FLK_F32) {
      FLK_TRY(a.d <= 64 ? attn::simt::launch_forward<64>(t, attn::simt_splits(p), st) : attn::simt::launch_forward<128>(t, attn::simt_splits(p), st));
    } else if (attn::by_token(p)) {
      FLK_TRY(p->dtype == FLK_BF16 ? attn::token_bf16(t, attn::token_splits(p), st) : attn::token_f16(t, attn::token_splits(p), st));
    } else {
      const attn::fwd::Plan plan = attn::forward_plan(p);
      FLK_TRY(p->dtype == FLK_BF16 ? attn::forward_bf16(t, plan, st) : attn::forward_f16(t, plan, st));
    }
  }
  FLK_CUDA_TRY(cudaGetLastError());
  return FLK_OK;
}

int flk_attention_status(void* stream, int* out) {
  if (out == nullptr) return fail(FLK_ERR_BAD_ARG, "status_out: null pointer");
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  int x[4] = {0, 0, 0, 0};
  FLK_TRY(attn::forward_status_bf16(st, &x[0]));
  FLK_TRY(attn::forward_status_f16(st, &x[1]));
  FLK_TRY(attn::backward_status_bf16(st, &x[2]));
  FLK_TRY(attn::backward_status_f16(st, &x[3]));
  *out = x[0] | x[1] | x[2] | x[3];
  return FLK_OK;
}

int flk_attention_wait_limit(int64_t ns) {
  if (ns < 0 || ns > 2000000000) return fail(FLK_ERR_BAD_ARG, "wait limit %lld: 0 to 2e9 ns", (long long)ns);
  attn::g_wait_limit.store((uint32_t)ns, std::memory_order_relaxed);
  return FLK_OK;
}

int flk_attention_backward(const flk_attention_args* p, void* stream) {
  FLK_TRY(attn::check_sizes(p));
  const int es = attn::esize_of(p->dtype);
  FLK_TRY(attn::check_tensor("q", p->q, p->batch, p->nq, p->hq, es));
  FLK_TRY(attn::check_tensor("k", p->k, p->batch, p->nk, p->hk, es));
  FLK_TRY(attn::check_tensor("v", p->v, p->batch, p->nk, p->hk, es));
  FLK_TRY(attn::check_tensor("out", p->out, p->batch, p->nq, p->hq, es));
  if (reinterpret_cast<uintptr_t>(p->out_lo) % 16 != 0) return fail(FLK_ERR_LAYOUT, "out_lo: not 16-byte aligned");
  FLK_TRY(attn::check_tensor("dout", p->dout, p->batch, p->nq, p->hq, es));
  if ((p->dk.data == nullptr) != (p->dv.data == nullptr) && p->nk > 0)
    return fail(FLK_ERR_BAD_ARG, "dk and dv are given together");
  if (p->dq.data != nullptr) FLK_TRY(attn::check_tensor("dq", p->dq, p->batch, p->nq, p->hq, es));
  if (p->dk.data != nullptr) {
    FLK_TRY(attn::check_tensor("dk", p->dk, p->batch, p->nk, p->hk, es));
    FLK_TRY(attn::check_tensor("dv", p->dv, p->batch, p->nk, p->hk, es));
  }
  if (p->batch == 0) return FLK_OK;
  if (p->nq > 0 && p->lse == nullptr) return fail(FLK_ERR_BAD_ARG, "lse: null pointer");
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  attn::Args a;
  FLK_TRY(attn::make_args(p, true, a, st));
  if (a.nq == 0 || a.nk == 0) {
    if (a.nq > 0 && a.dq.p != nullptr) FLK_TRY(attn::write_nothing(p->dtype, a.dq, a.b, a.nq, a.hq, a.d, nullptr, st));
    if (a.nk > 0 && a.dk.p != nullptr) {
      FLK_TRY(attn::write_nothing(p->dtype, a.dk, a.b, a.nk, a.hk, a.d, nullptr, st));
      FLK_TRY(attn::write_nothing(p->dtype, a.dv, a.b, a.nk, a.hk, a.d, nullptr, st));
    }
  } else if (attn::on_tensor_cores(p)) {
    attn::TcArgs t{};
    t.a = a;
    const attn::Workspace w = attn::plan_workspace(p, true);
    char* ws = reinterpret_cast<char*>(p->workspace);
    t.part_o = reinterpret_cast<float*>(ws + w.part_o);
    FLK_TRY(attn::launch_order(p, true, reinterpret_cast<int*>(ws + w.order), t, st));
    const attn::bwd::Plan plan = attn::backward_plan(p);
    if (p->dtype == FLK_BF16) {
      FLK_TRY(attn::launch_delta<__nv_bfloat16>(a, st));
      FLK_TRY(attn::backward_bf16(t, plan, st));
    } else {
      FLK_TRY(attn::launch_delta<__half>(a, st));
      FLK_TRY(attn::backward_f16(t, plan, st));
    }
  } else {
    FLK_TRY(attn::launch_delta<float>(a, st));
    FLK_TRY(a.d <= 64 ? attn::simt::launch_backward<64>(a, st) : attn::simt::launch_backward<128>(a, st));
  }
  FLK_CUDA_TRY(cudaGetLastError());
  return FLK_OK;
}

}  // extern "C"
