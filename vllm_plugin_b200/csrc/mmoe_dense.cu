// Products of the dense feed-forward operators for sm_100a (see mmoe_dense.cuh).
#include "mmoe_dense.cuh"

namespace mmoe {

namespace {

// A block per 64 x 64 sums, 2 x 8 of them a thread, operands through shared memory 16 k's at a time.
constexpr int kTile = 64, kDepth = 16;

template <typename T> struct Sum { using type = float; };
template <> struct Sum<int8_t> { using type = int; };
template <typename T> __device__ __forceinline__ typename Sum<T>::type widen(T v) { return static_cast<float>(v); }
template <> __device__ __forceinline__ int widen<int8_t>(int8_t v) { return v; }

template <typename T, int kKind>
__global__ void __launch_bounds__(256) dense_kernel(const DenseProduct p) {
  using S = typename Sum<T>::type;
  constexpr int kParts = kKind == kGated ? 2 : 1;
  __shared__ S sa[kDepth][kTile + 1], sb[kParts][kDepth][kTile + 1];
  const int m0 = blockIdx.y * kTile, n0 = blockIdx.x * kTile, t = threadIdx.x;
  S acc[kParts][2][8] = {};
  const auto at = [&](const DenseOperand& o, int64_t row, int64_t k) {
    return widen(static_cast<const T*>(o.p)[o.k_rows ? k * o.ld + row : row * o.ld + k]);
  };
  for (int k0 = 0; k0 < p.k; k0 += kDepth) {
    for (int i = t; i < kTile * kDepth; i += 256) {
      const int r = i / kDepth, k = i % kDepth;
      const bool in = k0 + k < p.k;
      sa[k][r] = in && m0 + r < p.m ? at(p.a, m0 + r, k0 + k) : S(0);
      for (int c = 0; c < kParts; ++c) sb[c][k][r] = in && n0 + r < p.n ? at(p.b, n0 + r + (int64_t)c * p.n, k0 + k) : S(0);
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kDepth; ++k)
#pragma unroll
      for (int c = 0; c < kParts; ++c)
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int j = 0; j < 8; ++j) acc[c][i][j] += sa[k][(t >> 3) * 2 + i] * sb[c][k][(t & 7) * 8 + j];
    __syncthreads();
  }
  for (int i = 0; i < 2; ++i) {
    const int row = m0 + (t >> 3) * 2 + i;
    if (row >= p.m) break;
    float a[8], b[8];
    for (int j = 0; j < 8; ++j) {
      a[j] = static_cast<float>(acc[0][i][j]);
      b[j] = static_cast<float>(acc[kParts - 1][i][j]);
    }
    dense_finish8<kKind>(p.epi, p.n, row, n0 + (t & 7) * 8, a, b);
  }
}

template <typename T>
cudaError_t launch_typed(const DenseProduct& p, cudaStream_t s) {
  const dim3 grid((p.n + kTile - 1) / kTile, (p.m + kTile - 1) / kTile);
  if (p.kind == kGated) return launch_plain(dense_kernel<T, kGated>, grid, dim3(256), 0, s, p);
  if (p.kind == kGatedGrad) return launch_plain(dense_kernel<T, kGatedGrad>, grid, dim3(256), 0, s, p);
  return launch_plain(dense_kernel<T, kLinear>, grid, dim3(256), 0, s, p);
}

// ---------------------------------------------------------------------------------------------------------------------
// Per-token quantiser: s = max|x| / 127, q = x / s rounded to the nearest whole number, ties to even.
// A block per token; the row stays in registers between the two passes as far as it fits.
// ---------------------------------------------------------------------------------------------------------------------
constexpr int kQuantThreads = 256, kQuantHeld = 4;      // vectors of eight values that a thread keeps

// Exact: t = x / s is known to about an ulp, so rint(t) is the nearest whole number or, next to a border, its neighbour; the remainder
// x - q s is exact in one fma (x has at most 11 bits and is above s / 2 in magnitude where it matters) and tells which.
__device__ __forceinline__ int quantize_one(float x, float s, float inv) {
  float q = rintf(inv > 0.f ? x * inv : __fdiv_rn(x, s));
  const float r = fmaf(-q, s, x), twice = r + r;
  if (fabsf(twice) >= s) {
    const bool odd = (static_cast<int>(q) & 1) != 0;
    if (fabsf(twice) > s || odd) q += copysignf(1.f, r);
  }
  return static_cast<int>(q);
}

template <typename T, bool kVec>
__global__ void __launch_bounds__(kQuantThreads) quantize_int8_kernel(const T* __restrict__ x, int64_t ld, int8_t* __restrict__ q,
                                                                      float* __restrict__ scales, int k) {
  constexpr int kWide = kVec ? 8 : 1;
  struct alignas(sizeof(T) * kWide) Vec { T v[kWide]; };
  struct alignas(kWide) Out { int8_t v[kWide]; };
  const int64_t row = blockIdx.x;
  const Vec* in = reinterpret_cast<const Vec*>(x + row * ld);
  Out* out = reinterpret_cast<Out*>(q + row * k);
  const int n = k / kWide, step = blockDim.x;
  Vec held[kQuantHeld];
  // magnitudes as bits: NaN is above infinity there, so neither is lost
  uint32_t top = 0;
  const auto look = [&](const Vec& v) {
#pragma unroll
    for (int j = 0; j < kWide; ++j) top = max(top, __float_as_uint(fabsf(static_cast<float>(v.v[j]))));
  };
#pragma unroll
  for (int i = 0; i < kQuantHeld; ++i) {
    const int at = threadIdx.x + i * step;
    if (at < n) look(held[i] = in[at]);
  }
  for (int at = threadIdx.x + kQuantHeld * step; at < n; at += step) look(in[at]);
  __shared__ uint32_t tops[kQuantThreads / 32];
  top = __reduce_max_sync(0xffffffffu, top);
  if ((threadIdx.x & 31) == 0) tops[threadIdx.x >> 5] = top;
  __syncthreads();
  for (int w = 0; w < (step >> 5); ++w) top = max(top, tops[w]);
  const float amax = __uint_as_float(top);
  const bool finite = top < 0x7f800000u;
  const float s = !finite ? __uint_as_float(0x7fffffffu) : (top == 0 ? 1.f : __fdiv_rn(amax, 127.f));
  const float inv = s >= 0x1p-100f ? __fdiv_rn(1.f, s) : 0.f;       // of a tiny scale the reciprocal overflows
  const auto put = [&](const Vec& v, int at) {
    Out o;
#pragma unroll
    for (int j = 0; j < kWide; ++j) o.v[j] = finite ? static_cast<int8_t>(quantize_one(static_cast<float>(v.v[j]), s, inv)) : 0;
    out[at] = o;
  };
#pragma unroll
  for (int i = 0; i < kQuantHeld; ++i) {
    const int at = threadIdx.x + i * step;
    if (at < n) put(held[i], at);
  }
  for (int at = threadIdx.x + kQuantHeld * step; at < n; at += step) put(in[at], at);
  if (threadIdx.x == 0) scales[row] = s;
}

template <typename T>
cudaError_t launch_quantize(const void* x, int64_t ld, int8_t* q, float* scales, int m, int k, cudaStream_t s) {
  const T* in = static_cast<const T*>(x);
  const bool vec = k % 8 == 0 && ld % 8 == 0 && reinterpret_cast<uintptr_t>(x) % 16 == 0 && reinterpret_cast<uintptr_t>(q) % 8 == 0;
  // as few threads as keep the same number of vectors each
  const int n = vec ? k / 8 : k, each = (n + kQuantThreads - 1) / kQuantThreads, threads = ((n + each - 1) / each + 31) & ~31;
  return vec ? launch_plain(quantize_int8_kernel<T, true>, dim3(m), dim3(threads), 0, s, in, ld, q, scales, k)
             : launch_plain(quantize_int8_kernel<T, false>, dim3(m), dim3(threads), 0, s, in, ld, q, scales, k);
}

}  // namespace

cudaError_t prepare_dense() { return cudaSuccess; }

cudaError_t launch_dense(const DenseProduct& p, cudaStream_t s) {
  if (p.m <= 0 || p.n <= 0) return cudaSuccess;
  if (p.type == kDenseInt8) return launch_typed<int8_t>(p, s);
  return p.type == kDenseBf16 ? launch_typed<__nv_bfloat16>(p, s) : launch_typed<__half>(p, s);
}

cudaError_t launch_quantize_int8(const void* x, int type, int64_t ld, int8_t* q, float* scales, int m, int k, cudaStream_t s) {
  if (m <= 0) return cudaSuccess;
  return type == kDenseBf16 ? launch_quantize<__nv_bfloat16>(x, ld, q, scales, m, k, s) : launch_quantize<__half>(x, ld, q, scales, m, k, s);
}

}  // namespace mmoe
