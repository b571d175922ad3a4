// Kernels for single tokens of bf16 data.
#include "flk_attn_token.cuh"

namespace flk {
namespace attn {

int token_bf16(const TcArgs& t, int splits, cudaStream_t st) { return token::launch<__nv_bfloat16>(t, splits, st); }

}  // namespace attn
}  // namespace flk
