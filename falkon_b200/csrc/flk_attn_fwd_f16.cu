// Forward attention kernels of f16 data.
#include "flk_attn_fwd.cuh"
#include "flk_attn_status.cuh"

namespace flk {
namespace attn {

int forward_f16(const TcArgs& t, const fwd::Plan& p, cudaStream_t st) { return fwd::launch<__half>(t, p, st); }
int forward_status_f16(cudaStream_t st, int* out) { return read_wait_status(st, out); }

}  // namespace attn
}  // namespace flk
