// Forward attention kernels of bf16 data.
#include "flk_attn_fwd.cuh"
#include "flk_attn_status.cuh"

namespace flk {
namespace attn {

int forward_bf16(const TcArgs& t, const fwd::Plan& p, cudaStream_t st) { return fwd::launch<__nv_bfloat16>(t, p, st); }
int forward_status_bf16(cudaStream_t st, int* out) { return read_wait_status(st, out); }

}  // namespace attn
}  // namespace flk
