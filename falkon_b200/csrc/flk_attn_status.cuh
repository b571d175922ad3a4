// What the kernels of a translation unit have to say about waits that gave up.
#pragma once

#include <mutex>

#include "flk_attn_tc.cuh"

namespace flk {
namespace attn {

// The status word of this translation unit's kernels, which goes back to 0; waits for the stream.  One query at a time: the word is
// taken to a place that the next one would overwrite.
inline std::mutex g_status_lock;
static __device__ int g_wait_taken;
static __global__ void take_status_kernel() { g_wait_taken = atomicExch(&g_wait_status, 0); }
static int read_wait_status(cudaStream_t st, int* out) {
  const std::lock_guard<std::mutex> alone(g_status_lock);
  take_status_kernel<<<1, 1, 0, st>>>();
  count_launch();
  FLK_CUDA_TRY(cudaGetLastError());
  FLK_CUDA_TRY(cudaMemcpyFromSymbolAsync(out, g_wait_taken, sizeof(int), 0, cudaMemcpyDeviceToHost, st));
  FLK_CUDA_TRY(cudaStreamSynchronize(st));
  return FLK_OK;
}

}  // namespace attn
}  // namespace flk
