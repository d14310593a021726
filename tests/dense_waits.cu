// The two waits of the dense kernels by themselves.  Test helper: compiled with the kernels' source.
#include "../vllm_plugin_b200/csrc/mmoe_dense.cu"

namespace mmoe {
bool chained() { return false; }
ChainScope::ChainScope(bool on) : saved_(on) {}
ChainScope::~ChainScope() {}

namespace {
// Warp 0 idles for `before_ns`, then waits for a barrier, at which warp 1 arrives `after_ns` later still, or (negative) never.  out[0]: 1 when the wait
// gave up, 2 when it ended with the barrier.  Every loop ends by the clock.
__global__ void __launch_bounds__(64) dense_wait_kernel(bool whole_warp, int64_t before_ns, int64_t after_ns, int64_t limit_ns, int32_t* status, int32_t* out) {
  __shared__ uint64_t bar;
  __shared__ int32_t abort_flag;
  if (threadIdx.x == 0) {
    mbar_init(smem_u32(&bar), 1);
    abort_flag = 0;
  }
  __syncthreads();
  const uint64_t t0 = global_timer(), until = t0 + static_cast<uint64_t>(before_ns + (threadIdx.x >= 32 ? max(after_ns, (int64_t)0) : 0));
  DenseWaiter waiter{{&abort_flag, status, 0, kStatusDense, 10 + whole_warp}, limit_ns};
  while (global_timer() < until) __nanosleep(1000);
  __syncwarp();
  if (threadIdx.x >= 32) {
    if (threadIdx.x == 32 && after_ns >= 0) mbar_arrive(smem_u32(&bar));
    return;
  }
  const bool ended = whole_warp ? waiter.wait_uniform(smem_u32(&bar), 0) : waiter.wait_warp(smem_u32(&bar), 0, 0);
  if (threadIdx.x == 0) out[0] = ended ? 2 : 1;
}
}  // namespace
}  // namespace mmoe

extern "C" int run_dense_wait(int whole_warp, int64_t before_ns, int64_t after_ns, int64_t limit_ns, void* status, void* out, void* stream) {
  return static_cast<int>(mmoe::launch_plain(mmoe::dense_wait_kernel, dim3(1), dim3(64), 0, static_cast<cudaStream_t>(stream), whole_warp != 0, before_ns,
                                             after_ns, limit_ns, static_cast<int32_t*>(status), static_cast<int32_t*>(out)));
}
