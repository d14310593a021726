// The two waits that the 8-bit pair kernel has beside those of the other kernels, by themselves.  Test helper: compiled with the kernel's source.
#include "../vllm_plugin_b200/csrc/mmoe_fp8.cu"

namespace mmoe {
bool chained() { return false; }
ChainScope::ChainScope(bool on) : saved_(on) {}
ChainScope::~ChainScope() {}
EncodeFn dense_encoder() { return nullptr; }
int dense_sms() { return 0; }
bool grouped_few_rows(const GroupedProduct&, int) { return false; }
cudaError_t launch_grouped_few(const GroupedProduct&, int, cudaStream_t) { return cudaErrorNotSupported; }

namespace {
// Warp 0 idles for `before_ns`, then waits for a barrier, at which warp 1 arrives `after_ns` later still, or (negative) never; `given_up`: another role has
// given up before.  out[0]: 1 when the wait gave up, 2 when it ended with the barrier; out[1]: the flag that tells the other roles.  The loops of this
// kernel end by the clock.
__global__ void __launch_bounds__(64) fp8_wait_kernel(bool polls, bool given_up, int64_t before_ns, int64_t after_ns, const __grid_constant__ Fp8Params p, int32_t* out) {
  __shared__ uint64_t bar;
  __shared__ Fp8Control ctl;
  if (threadIdx.x == 0) {
    mbar_init(smem_u32(&bar), 1);
    ctl.abort_flag = given_up ? 1 : 0;
  }
  __syncthreads();
  const uint64_t t0 = global_timer(), until = t0 + static_cast<uint64_t>(before_ns + (threadIdx.x >= 32 ? max(after_ns, (int64_t)0) : 0));
  while (global_timer() < until) __nanosleep(1000);
  __syncwarp();
  if (threadIdx.x >= 32) {
    if (threadIdx.x == 32 && after_ns >= 0) mbar_arrive(smem_u32(&bar));
    return;
  }
  DenseWaiter waiter{{&ctl.abort_flag, p.status, 0, kStatusGrouped + 1, 7}, p.timeout_ns};
  const bool ended = polls ? poll(waiter, smem_u32(&bar), 0) : probe_then_wait(p, &ctl, smem_u32(&bar), 0);
  const uint32_t lanes = __ballot_sync(0xffffffffu, ended);
  if (threadIdx.x == 0) out[0] = lanes == 0xffffffffu ? 2 : lanes == 0 ? 1 : 3, out[1] = ctl.abort_flag;
}
}  // namespace
}  // namespace mmoe

extern "C" int run_fp8_wait(int polls, int given_up, int64_t before_ns, int64_t after_ns, int64_t limit_ns, void* status, void* out, void* stream) {
  mmoe::Fp8Params p = {};
  p.status = static_cast<int32_t*>(status), p.timeout_ns = limit_ns;
  return static_cast<int>(mmoe::launch_plain(mmoe::fp8_wait_kernel, dim3(1), dim3(64), 0, static_cast<cudaStream_t>(stream), polls != 0, given_up != 0, before_ns,
                                             after_ns, p, static_cast<int32_t*>(out)));
}
