// Products of the dense feed-forward operators: D[m, n] = sum_k A[m, k] B[n, k] in 16 bits (FP32 sums) or in 8-bit integers (exact
// 32-bit sums), with the arithmetic that follows a product done on its sums before they leave the SM.
#pragma once

#include <cuda_fp16.h>

#include "mmoe_common.cuh"

namespace mmoe {

enum DenseType { kDenseBf16 = 0, kDenseFp16 = 1, kDenseInt8 = 2, kDenseFp32 = 3 };

// What becomes of the sums.
//   kLinear     out[m, n] = s [* row_scale[m] * col_scale[n]] [+ bias[n]]
//   kGated      B holds `inter` gate rows and then `inter` up rows; out[m, i] = silu(min(g, c)) * clip(u, -c, c), and, for a backward
//               pass, preact[m, i] = g, preact[m, inter + i] = u
//   kGatedGrad  the sums are the gradient of kGated's output: out[m, i] = that of g, out[m, inter + i] = that of u
enum DenseEpilogueKind { kLinear = 0, kGated = 1, kGatedGrad = 2 };

struct DenseEpilogue {
  void* out;
  int64_t ld_out;
  int32_t out_type;
  int32_t inter;             // kGated, kGatedGrad
  const float* row_scale;    // 8-bit integers: one per row of A ...
  const float* col_scale;    // ... and of B
  const float* bias;
  float* preact;             // float [m, 2 inter]; written by kGated unless null, read by kGatedGrad
  float clamp;               // +inf: none
};

// An operand [rows, k]: row-major with `ld` elements between rows, or (k_rows) stored as its transpose, `ld` elements between the k's.
struct DenseOperand {
  const void* p;
  int64_t ld;
  bool k_rows;
};

struct DenseProduct {
  DenseOperand a, b;
  int32_t m, n, k;           // n: columns of the output; kGated multiplies 2 n rows of B
  int32_t type;              // of both operands
  int32_t kind;
  DenseEpilogue epi;
  int32_t* status;           // int32 [8], see kStatusTimeout
  int32_t timeout_ms;        // of each wait; <= 0: the default
};

cudaError_t prepare_dense();   // once per device, outside stream capture

// One product, or two 16-bit ones that need nothing of each other, at most the first of them kGatedGrad and the others kLinear, in one launch.
constexpr int kMaxParts = 2;
cudaError_t launch_dense(const DenseProduct* p, int parts, cudaStream_t s);
bool dense_few_tokens(const DenseProduct& p);      // it goes by itself
cudaError_t launch_quantize_int8(const void* x, int type, int64_t ld, int8_t* q, float* scales, int m, int k, cudaStream_t s);

#ifdef __CUDACC__
// NaN stays NaN
__device__ __forceinline__ float clip_above(float v, float c) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(v), "f"(c));
  return r;
}
__device__ __forceinline__ float clip_both(float v, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(clip_above(v, c)), "f"(-c));
  return r;
}
// 1 / (1 + exp(-v)) for results of 16 bits: the exponent's rounding is worth 2^-24 |v| of the value, the approximations 2^-21.  0 where the
// exponential or its reciprocal leaves the normal numbers (v below -87).
__device__ __forceinline__ float sigmoid_of(float v) {
  float e, r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(v * -1.4426950408889634f));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.f + e));
  return r;
}

// silu(min(g, c)) * clip(u, -c, c)
__device__ __forceinline__ float gated_value(float g, float u, float c) {
  const float gc = clip_above(g, c);
  return gc * sigmoid_of(gc) * clip_both(u, c);
}

// The same where the result stays FP32 and this is all that is rounded: within 2^-20 of the value over the whole range (and, where exp(g) is no normal
// number, 2^-148 of g u).  Only there: in 16 bits the difference is far below the result's rounding.  exp(-a) = 2^t 2^r, t = -a log2(e) as it is
// rounded and r what that leaves out: the product's rounding, which one fma gives exactly, and that of the constant; 2^r = 1 + r ln 2 for an r
// this small.  The exponential of -|g| does not overflow, and past 128 it is 0.  With expf and a division instead: 3840 tokens 64.2 us, 64 tokens 9.9.
__device__ __forceinline__ float gated_value_fp32(float g, float u, float c) {
  constexpr float kLog2e = 1.44269502f, kLog2eRest = 1.92596299e-8f, kLn2 = 0.693147181f;
  const float gc = clip_above(g, c), a = fminf(fabsf(gc), 128.f), t = -a * kLog2e, r = fmaf(-a, kLog2eRest, fmaf(-a, kLog2e, -t));
  float e, inverse;
  asm("ex2.approx.f32 %0, %1;" : "=f"(e) : "f"(t));
  e = fmaf(e, r * kLn2, e);
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inverse) : "f"(1.f + e));
  return gc * ((gc < 0.f ? e : 1.f) * inverse) * clip_both(u, c);
}

// Its derivatives, times the gradient dh of its value.  A clipped input has none; one on the border has.
__device__ __forceinline__ void gated_grad(float dh, float g, float u, float c, float& dg, float& du) {
  const float gc = clip_above(g, c), s = sigmoid_of(gc), silu = gc * s;
  dg = g > c ? 0.f : dh * clip_both(u, c) * (s + silu * (1.f - s));
  du = fabsf(u) > c ? 0.f : dh * silu;
}

template <typename T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ float from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// Eight neighbouring values of one row, of which the first `valid` exist.  16-byte stores where all do and the place allows it.
template <typename T>
__device__ __forceinline__ void store8(T* dst, const float (&v)[8], int valid) {
  constexpr int kBytes = 8 * sizeof(T);
  if (valid >= 8 && (reinterpret_cast<uintptr_t>(dst) & 15u) == 0) {
    __align__(16) T t[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) t[j] = from_float<T>(v[j]);
#pragma unroll
    for (int j = 0; j < kBytes / 16; ++j) reinterpret_cast<uint4*>(dst)[j] = reinterpret_cast<const uint4*>(t)[j];
    return;
  }
#pragma unroll
  for (int j = 0; j < 8; ++j)
    if (j < valid) dst[j] = from_float<T>(v[j]);
}

// What follows a product, for eight neighbouring columns: made once for the columns, then called for the rows.  `n` ends the columns.
template <int kKind, bool kScaled>
struct DenseFinish {
  const DenseEpilogue& e;
  const int col, valid;
  float cs[8], second[8];              // scales of the columns; kGated: those of the up columns, kLinear: bias
  // by ordinary loads: what is read here may have been written by the launch in front, beside which this one has started
  __device__ __forceinline__ void load8(const float* src, float (&v)[8]) const {
    if (valid >= 8 && (reinterpret_cast<uintptr_t>(src) & 15u) == 0) {
      const float4 lo = reinterpret_cast<const float4*>(src)[0], hi = reinterpret_cast<const float4*>(src)[1];
      v[0] = lo.x, v[1] = lo.y, v[2] = lo.z, v[3] = lo.w, v[4] = hi.x, v[5] = hi.y, v[6] = hi.z, v[7] = hi.w;
      return;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = j < valid ? src[j] : 0.f;
  }
  __device__ __forceinline__ DenseFinish(const DenseEpilogue& epi, int n, int column) : e(epi), col(column), valid(n - column) {
    if (!kScaled) return;
    load8(e.col_scale + col, cs);
    if (kKind == kGated) load8(e.col_scale + e.inter + col, second);
    else if (e.bias != nullptr) load8(e.bias + col, second);
  }
  __device__ __forceinline__ void put(int64_t at, const float (&v)[8]) const {
    if (e.out_type == kDenseBf16) store8(static_cast<__nv_bfloat16*>(e.out) + at, v, valid);
    else if (e.out_type == kDenseFp16) store8(static_cast<__half*>(e.out) + at, v, valid);
    else store8(static_cast<float*>(e.out) + at, v, valid);
  }
  // kGatedGrad: g and u of a row, to be fetched well ahead of row()
  __device__ __forceinline__ void fetch(int row, float (&g)[8], float (&u)[8]) const {
    const float* keep = e.preact + (int64_t)row * 2 * e.inter + col;
    load8(keep, g);
    load8(keep + e.inter, u);
  }
  // `a`: the sums (kGated: the gate's, `b` the up row's; kGatedGrad: `b` and `u` as fetched), `rs` the scale of the row
  __device__ __forceinline__ void row(int row, float rs, float (&a)[8], float (&b)[8], float (&u)[8]) const {
    if (valid <= 0) return;
    const int64_t at = row * e.ld_out + col;
    if (kKind == kLinear) {
      if (kScaled) {
#pragma unroll
        for (int j = 0; j < 8; ++j) a[j] = a[j] * rs * cs[j];
        if (e.bias != nullptr) {
#pragma unroll
          for (int j = 0; j < 8; ++j) a[j] += second[j];
        }
      }
      put(at, a);
    } else if (kKind == kGated) {
      if (kScaled) {
#pragma unroll
        for (int j = 0; j < 8; ++j) a[j] = a[j] * rs * cs[j], b[j] = b[j] * rs * second[j];
      } else if (e.preact != nullptr) {
        float* keep = e.preact + (int64_t)row * 2 * e.inter + col;
        store8(keep, a, valid);
        store8(keep + e.inter, b, valid);
      }
      if (kScaled && e.out_type == kDenseFp32) {
#pragma unroll
        for (int j = 0; j < 8; ++j) a[j] = gated_value_fp32(a[j], b[j], e.clamp);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) a[j] = gated_value(a[j], b[j], e.clamp);
      }
      put(at, a);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) gated_grad(a[j], b[j], u[j], e.clamp, b[j], u[j]);
      put(at, b);
      put(at + e.inter, u);
    }
  }
};
#endif

}  // namespace mmoe
