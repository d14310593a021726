// What the kernels of the dense and of the grouped products share: bounded waits, operand descriptors, products of a pair and of one CTA, copies within a
// cluster, and on the host the instruction descriptor.
#pragma once

#include "mmoe_dense.cuh"
#include "mmoe_tc.cuh"

namespace mmoe {

// kernels in the status words: products on pairs, of few tokens; grouped products on pairs (16 and 8 bits), of few rows
constexpr int kStatusDense = 31, kStatusGrouped = 33;

#ifdef __CUDACC__
// Waits with a limit each, which counts from a wait's 64th probe on: a launch may take as long as its size asks for.  (The layer's limit is one for a
// whole launch, which its buffers bound.)  What waits for a whole tile or for all of a CTA's K says how many stages that are: kStageNs, many times what
// one takes, is added for each.
constexpr int64_t kStageNs = 10000;
struct DenseWaiter {
  Waiter wait;               // its deadline is that of the wait under way
  int64_t limit_ns;
  __device__ __forceinline__ bool late(uint32_t spin, int stages) {
    if (spin != 63u) return wait.abandoned();
    wait.deadline = global_timer() + static_cast<uint64_t>(limit_ns + stages * kStageNs);
    return *wait.abort_flag != 0;
  }
  // both by the whole warp; true when the phase has completed, false when the call is being abandoned (see Waiter for why two)
  __device__ __forceinline__ bool wait_uniform(uint32_t bar, uint32_t parity) {
    for (uint32_t spin = 0;; ++spin) {
      if (__any_sync(0xffffffffu, mbar_try_wait(bar, parity))) return true;
      if ((spin & 63u) == 63u && __any_sync(0xffffffffu, late(spin, 0))) return false;
    }
  }
  __device__ __forceinline__ bool wait_warp(uint32_t bar, uint32_t parity, int stages) {
    if (__all_sync(0xffffffffu, mbar_test_wait(bar, parity))) return true;
    bool ok = true;
    if ((threadIdx.x & 31) == 0)
      for (uint32_t spin = 0;; ++spin) {
        if (mbar_try_wait(bar, parity)) break;
        if ((spin & 63u) == 63u && late(spin, stages)) { ok = false; break; }
      }
    return __shfl_sync(0xffffffffu, ok ? 1 : 0, 0) != 0;
  }
};

// descriptor without its address: 128-byte swizzle; K-major: eight-row groups 1024 bytes apart.  MN-major: groups of eight k's 1024 bytes
// apart, blocks of 64 rows `block` bytes apart.
__device__ __forceinline__ uint64_t operand_desc(bool mn_major, uint32_t block) {
  return desc_hi_sw128() | (mn_major ? static_cast<uint64_t>(block >> 4) << 16 : 0ull);
}

__device__ __forceinline__ void prefetch_bulk(const void* p, uint32_t bytes) {
  asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(p), "r"(bytes) : "memory");
}

template <bool kInt8>
__device__ __forceinline__ void pair_product(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  if (kInt8)
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}"
                 ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
  else
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}"
                 ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}

template <bool kInt8>
__device__ __forceinline__ void single_product(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  if (kInt8)
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}"
                 ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
  else
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
                 ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}

// shared memory of this CTA to that of another one of the cluster, counted on a barrier there
__device__ __forceinline__ void cluster_send(uint32_t dst, uint32_t src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.shared::cta.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
               ::"r"(dst), "r"(src), "r"(bytes), "r"(bar) : "memory");
}

__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }

#endif

// host, per device: the encoder of tensor maps, and the number of SMs (0: prepare_dense() has not run there) of the current one, whose context
// it binds to the calling thread
constexpr int kMaxDevices = 64;
using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                              const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeFn dense_encoder();
int dense_sms();

// Instruction descriptor: [4,6) sums (1 FP32, 2 32-bit integers), [7,10) and [10,13) operands (16 bits: 0 FP16, 1 BF16; 8 bits: 1 signed),
// [15], [16] MN-major operands, [17,23) N >> 3, [24,29) M >> 4.
inline uint32_t product_idesc(int type, bool a_mn, bool b_mn, int rows, int cols) {
  const uint32_t format = type == kDenseFp16 ? 0 : 1;
  return ((type == kDenseInt8 ? 2u : 1u) << 4) | (format << 7) | (format << 10) | ((a_mn ? 1u : 0u) << 15) | ((b_mn ? 1u : 0u) << 16) |
         (static_cast<uint32_t>(cols >> 3) << 17) | (static_cast<uint32_t>(rows >> 4) << 24);
}

}  // namespace mmoe
