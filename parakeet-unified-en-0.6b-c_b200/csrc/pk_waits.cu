// pk_waits.cu -- the bounded device waits that ran out, counted by each translation
// unit of kernels in a word of its own (pk_common.cuh), summed for the host.
//
// One launch reads (and clears) all of the words and one copy brings the sum back:
// a drop-in call on one row of 1024 ends with this check and takes 44 us; with a
// synchronous copy per word to read it and one to clear it 69 us where three units
// had such waits, 94 with five.
#include <mutex>

#include "pk_common.cuh"

namespace {

constexpr int UNITS = 5;
struct Words {
  unsigned *at[UNITS];
};
__device__ unsigned g_sum;

__global__ void sum_waits_kernel(Words w, int reset) {
  unsigned v = 0;
  if (threadIdx.x < UNITS)
    v = reset ? atomicExch(w.at[threadIdx.x], 0u) : *(volatile unsigned *)w.at[threadIdx.x];
  v = __reduce_add_sync(PK_FULL_MASK, v);
  if (threadIdx.x == 0) g_sum = v;
}

std::mutex g_sum_lock;   // one call's launch and copy at a time: g_sum is shared

}  // namespace

// On the current device; waits for the legacy default stream, as the copy does.
extern "C" int pk_wait_timeouts(unsigned *count, int reset) {
  Words w;
  if (pk_softmax_wait_word(&w.at[0]) || pk_conv_wait_word(&w.at[1]) || pk_tc_wait_word(&w.at[2]) ||
      pk_q8_wait_word(&w.at[3]) || pk_rms_wait_word(&w.at[4]))
    return PKCU_ERR_CUDA;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(1);
  cfg.blockDim = dim3(32);
  std::lock_guard<std::mutex> lock(g_sum_lock);
  // (the launch's own status: an error that another call left behind is not this one's)
  if (cudaLaunchKernelEx(&cfg, sum_waits_kernel, w, reset) != cudaSuccess ||
      cudaMemcpyFromSymbol(count, g_sum, sizeof *count) != cudaSuccess)
    return PKCU_ERR_CUDA;
  return PKCU_OK;
}
