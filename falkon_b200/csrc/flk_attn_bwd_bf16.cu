// Backward attention kernels of bf16 data.
#include "flk_attn_bwd.cuh"
#include "flk_attn_status.cuh"

namespace flk {
namespace attn {

int backward_bf16(const TcArgs& t, const bwd::Plan& p, cudaStream_t st) { return bwd::launch<__nv_bfloat16>(t, p, st); }
int backward_status_bf16(cudaStream_t st, int* out) { return read_wait_status(st, out); }

}  // namespace attn
}  // namespace flk
