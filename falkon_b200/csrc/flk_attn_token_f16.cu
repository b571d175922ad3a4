// Kernels for single tokens of f16 data.
#include "flk_attn_token.cuh"

namespace flk {
namespace attn {

int token_f16(const TcArgs& t, int splits, cudaStream_t st) { return token::launch<__half>(t, splits, st); }

}  // namespace attn
}  // namespace flk
