// What the kernels of the experts' products share, in 16 and in 8 bits.
#pragma once

#include "mmoe_dense_device.cuh"
#include "mmoe_grouped.cuh"

namespace mmoe {

constexpr int kGroupRows = 128;                       // rows of operand A per CTA

// Where each expert's rows and tiles start
struct GroupPlan {
  int32_t start[kMaxExperts + 1];
  int32_t tile[kMaxExperts + 1];
};

#ifdef __CUDACC__
// By all threads of a CTA: an expert has `each` tiles for every `step` rows that it has begun.  Returns their number.  Every CTA reads `ends` for
// itself, by ordinary loads: the launch in front may have written them.
__device__ __forceinline__ int make_plan(GroupPlan* plan, const int32_t* ends, int experts, int rows, int step, int each, int32_t* status) {
  for (int e = threadIdx.x; e < experts; e += blockDim.x) plan->start[e + 1] = ends != nullptr ? ends[e] : rows;
  if (threadIdx.x == 0) plan->start[0] = 0;
  __syncthreads();
  bool bad = threadIdx.x == 0 && plan->start[experts] > rows;
  for (int e = threadIdx.x; e < experts; e += blockDim.x) bad |= plan->start[e + 1] < plan->start[e];
  if (__syncthreads_or(bad)) {                 // nobody's rows then
    for (int e = threadIdx.x; e <= experts; e += blockDim.x) plan->start[e] = 0;
    if (threadIdx.x == 0 && blockIdx.x == 0) report_bad_index(status);
    __syncthreads();
  }
  if (threadIdx.x < 32) {
    int sum = 0;
    for (int e0 = 0; e0 < experts; e0 += 32) {
      const int e = e0 + threadIdx.x;
      int tiles = e < experts ? (plan->start[e + 1] - plan->start[e] + step - 1) / step * each : 0;
      const int own = tiles;
#pragma unroll
      for (int d = 1; d < 32; d *= 2) {
        const int v = __shfl_up_sync(0xffffffffu, tiles, d);
        if (threadIdx.x >= d) tiles += v;
      }
      if (e < experts) plan->tile[e] = sum + tiles - own;
      sum += __shfl_sync(0xffffffffu, tiles, 31);
    }
    if (threadIdx.x == 0) plan->tile[experts] = sum;
  }
  __syncthreads();
  return plan->tile[experts];
}

// whose the t-th tile is
__device__ __forceinline__ int expert_of(const GroupPlan& plan, int experts, int t) {
  int low = 0, high = experts;                 // tile[low] <= t < tile[high]
  while (high - low > 1) {
    const int mid = (low + high) / 2;
    if (plan.tile[mid] <= t) low = mid;
    else high = mid;
  }
  return low;
}

// Four bytes into shared memory, or zeros
__device__ __forceinline__ void copy_word(uint32_t dst, const float* src, bool there) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(there ? 4 : 0) : "memory");
}

// Zeros from p on, by all threads of the grid
__device__ __forceinline__ void clear_bytes(char* p, int64_t bytes) {
  const int64_t thread = (int64_t)blockIdx.x * blockDim.x + threadIdx.x, threads = (int64_t)gridDim.x * blockDim.x;
  const int64_t head = min(bytes, (int64_t)((16 - (reinterpret_cast<uintptr_t>(p) & 15)) & 15)), body = (bytes - head) / 16;
  for (int64_t i = thread; i < head; i += threads) p[i] = 0;
  for (int64_t i = thread; i < body; i += threads) reinterpret_cast<uint4*>(p + head)[i] = make_uint4(0, 0, 0, 0);
  for (int64_t i = head + body * 16 + thread; i < bytes; i += threads) p[i] = 0;
}

__device__ __forceinline__ void pair_load_4d(uint32_t dst, const CUtensorMap* map, int c0, int c1, int c2, int c3, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];"
      ::"r"(dst), "l"(map), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(bar)
      : "memory");
}
__device__ __forceinline__ void pair_load_5d(uint32_t dst, const CUtensorMap* map, int c0, int c1, int c2, int c3, int c4, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.5d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5, %6}], [%7];"
      ::"r"(dst), "l"(map), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(c4), "r"(bar)
      : "memory");
}

#endif

inline bool encode_map(CUtensorMap* map, int type, const void* base, int rank, const uint64_t (&dims)[5], const uint64_t (&strides)[4], const uint32_t (&box)[5]) {
  const cuuint32_t one[5] = {1, 1, 1, 1, 1};
  const CUtensorMapDataType t = type == kGroupedE4m3 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : type == kDenseBf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  cuuint64_t d[5], st[4];
  cuuint32_t b[5];
  std::copy(dims, dims + 5, d), std::copy(strides, strides + 4, st), std::copy(box, box + 5, b);
  return dense_encoder()(map, t, rank, const_cast<void*>(base), d, st, b, one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                         CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace mmoe
