// Products of a layer's experts over rows that are grouped by expert, in 16 bits (FP32 sums) with what their gradients need, and in 8-bit floating
// point with a scale for each 128 values of a row and each block of 128 x 128 weights; the latter for one weight and all rows too.
#pragma once

#include "mmoe_dense.cuh"

namespace mmoe {

enum { kGroupedE4m3 = 4 };                        // beside DenseType, as an operand type
enum { kGroupedWeights = 3 };                     // beside DenseEpilogueKind: the gradient of the experts' weights
constexpr int kMaxExperts = 1024;                 // a CTA keeps where each expert's rows and tiles start
constexpr int kScaleBlock = 128;

// Rows of expert e: [ends[e - 1], ends[e]), from 0 on for the first; ends == nullptr: all rows are expert 0's.
//   kLinear, kGated, kGatedGrad   out[t, n] = sum_k x[t, k] w[e][n, k] and what follows it, see DenseEpilogueKind.  w_k_rows: w[e] is stored
//                                 as [k, n].  kGated: w[e] holds n gate rows and then n up rows
//   kGroupedWeights               out[e][n, k] = sum over e's rows t of left[t, n] x[t, k], zero without rows
struct GroupedProduct {
  int32_t type, kind;
  const int32_t* ends;
  int32_t experts, rows;
  int32_t n, k;
  const void* w;
  bool w_k_rows;
  const void* left;          // kGroupedWeights: [rows, n] ...
  int64_t left_ld;           // ... with so many elements between rows
  const void* x;
  int64_t x_ld;
  const float* x_scales;     // E4M3: [rows, ceil(k / 128)]
  const float* w_scales;     // [experts][ceil(n / 128) (kGated: twice that, the gate's first)][ceil(k / 128)]
  DenseEpilogue epi;
  bool zero_behind;          // rows of `out` behind the last expert's are set to zero
  int32_t* status;
  int32_t timeout_ms;
};

cudaError_t prepare_grouped();          // behind prepare_dense()
cudaError_t prepare_fp8();
cudaError_t prepare_grouped_few();
cudaError_t launch_grouped(const GroupedProduct& p, cudaStream_t s);      // 16 bits
cudaError_t launch_fp8(const GroupedProduct& p, cudaStream_t s);          // E4M3; rows behind the last expert's are set to zero
bool grouped_few_rows(const GroupedProduct& p, int sms);       // it goes to launch_grouped_few
cudaError_t launch_grouped_few(const GroupedProduct& p, int sms, cudaStream_t s);
cudaError_t launch_quantize_fp8(const void* x, int type, int64_t ld, uint8_t* q, float* scales, int m, int k, cudaStream_t s);

}  // namespace mmoe
