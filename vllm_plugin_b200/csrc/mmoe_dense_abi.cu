// extern "C" entry points of the dense feed-forward operators (declared in include/mmoe.h): argument checks and the products of a call.
// Nothing here allocates device memory; only mmoe_dense_read_status synchronises.
#include <string.h>

#include "mmoe_dense_abi.h"
#include "mmoe_grouped.cuh"

namespace {

int check_feed_forward(const MmoeFeedForward* f) {
  if (f == nullptr) return fail(MMOE_ERR_INVALID_ARGUMENT, "feed-forward: arguments are NULL");
  if (f->type != MMOE_BF16 && f->type != MMOE_FP16) return fail(MMOE_ERR_INVALID_ARGUMENT, "feed-forward: type=%d (supported: BF16, FP16)", f->type);
  if (f->hidden < 8 || f->hidden % 8 != 0 || f->hidden > kMostChannels)
    return fail(MMOE_ERR_INVALID_ARGUMENT, "feed-forward: hidden=%d must be a positive multiple of 8, at most %d", f->hidden, kMostChannels);
  if (f->intermediate < 8 || f->intermediate % 8 != 0 || f->intermediate > kMostChannels)
    return fail(MMOE_ERR_INVALID_ARGUMENT, "feed-forward: intermediate=%d must be a positive multiple of 8, at most %d", f->intermediate, kMostChannels);
  if (f->num_tokens < 0 || f->num_tokens > kMostTokens)
    return fail(MMOE_ERR_INVALID_ARGUMENT, "feed-forward: num_tokens=%d outside [0, %d]", f->num_tokens, kMostTokens);
  if (!(f->clamp > 0.f)) return fail(MMOE_ERR_INVALID_ARGUMENT, "feed-forward: clamp must be positive");
  if (f->x_stride < f->hidden || f->x_stride % 8 != 0)
    return fail(MMOE_ERR_INVALID_ARGUMENT, "feed-forward: x_stride must be a multiple of 8 and at least hidden=%d", f->hidden);
  if (f->w13 == nullptr || f->w2 == nullptr || (f->num_tokens > 0 && (f->x == nullptr || f->status == nullptr)))
    return fail(MMOE_ERR_INVALID_ARGUMENT, "feed-forward: x, w13, w2 and status must not be NULL");
  if (!aligned16(f->x) || !aligned16(f->w13) || !aligned16(f->w2) || !aligned16(f->h) || !aligned16(f->preact) || !aligned16(f->y))
    return fail(MMOE_ERR_INVALID_ARGUMENT, "feed-forward: pointers must be 16-byte aligned");
  return MMOE_OK;
}

int run_dense(const mmoe::DenseProduct* p, int parts, const char* what, void* stream) {
  const cudaError_t e = mmoe::launch_dense(p, parts, static_cast<cudaStream_t>(stream));
  return e == cudaSuccess ? MMOE_OK : e == cudaErrorNotReady ? fail(MMOE_ERR_NOT_PREPARED, "%s: mmoe_dense_prepare() has not run on this device", what) : cuda_fail(e, what);
}

int int8_product(const MmoeInt8Product* a, bool gated, void* stream) {
  const char* what = gated ? "int8 gated projection" : "int8 projection";
  if (a == nullptr) return fail(MMOE_ERR_INVALID_ARGUMENT, "%s: arguments are NULL", what);
  if (a->num_tokens < 0 || a->num_tokens > kMostTokens) return fail(MMOE_ERR_INVALID_ARGUMENT, "%s: num_tokens=%d outside [0, %d]", what, a->num_tokens, kMostTokens);
  // 131072 products of magnitude up to 128 * 128 would reach 2^31; quantised values end at 127
  if (a->width < 16 || a->width % 16 != 0 || a->width >= 131072) return fail(MMOE_ERR_INVALID_ARGUMENT, "%s: width=%d must be a multiple of 16 in [16, 131072)", what, a->width);
  if (a->channels < 1 || a->channels > kMostChannels) return fail(MMOE_ERR_INVALID_ARGUMENT, "%s: channels=%d outside [1, %d]", what, a->channels, kMostChannels);
  if (a->out_type != MMOE_BF16 && a->out_type != MMOE_FP16 && a->out_type != MMOE_FP32) return fail(MMOE_ERR_INVALID_ARGUMENT, "%s: out_type=%d", what, a->out_type);
  if (gated && !(a->clamp > 0.f)) return fail(MMOE_ERR_INVALID_ARGUMENT, "%s: clamp must be positive", what);
  if (a->x_stride < a->width || a->x_stride % 16 != 0) return fail(MMOE_ERR_INVALID_ARGUMENT, "%s: x_stride must be a multiple of 16 and at least width=%d", what, a->width);
  if (a->num_tokens == 0) return MMOE_OK;
  if (a->x == nullptr || a->x_scales == nullptr || a->w == nullptr || a->w_scales == nullptr || a->out == nullptr || a->status == nullptr)
    return fail(MMOE_ERR_INVALID_ARGUMENT, "%s: pointers must not be NULL", what);
  if (!aligned16(a->x) || !aligned16(a->w) || !aligned16(a->out)) return fail(MMOE_ERR_INVALID_ARGUMENT, "%s: pointers must be 16-byte aligned", what);
  mmoe::DenseProduct p = {};
  p.a = {a->x, a->x_stride, false};
  p.b = {a->w, a->width, false};
  p.m = a->num_tokens, p.n = a->channels, p.k = a->width;
  p.type = mmoe::kDenseInt8;
  p.kind = gated ? mmoe::kGated : mmoe::kLinear;
  p.epi.out = a->out, p.epi.ld_out = a->channels, p.epi.out_type = a->out_type;
  p.epi.inter = a->channels, p.epi.clamp = a->clamp;
  p.epi.row_scale = a->x_scales, p.epi.col_scale = a->w_scales;
  p.epi.bias = gated ? nullptr : a->bias;
  p.status = a->status, p.timeout_ms = a->timeout_ms;
  return run_dense(&p, 1, what, stream);
}

}  // namespace

extern "C" {

int mmoe_dense_prepare(void* stream) {
  int dev = 0, major = 0, minor = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess) e = cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, dev);
  if (e == cudaSuccess) e = cudaDeviceGetAttribute(&minor, cudaDevAttrComputeCapabilityMinor, dev);
  if (e != cudaSuccess) return cuda_fail(e, "dense_prepare");
  if (major != 10 || minor != 0) return fail(MMOE_ERR_ARCH, "device %d has compute capability %d.%d, need 10.0", dev, major, minor);
  cudaStreamCaptureStatus cap = cudaStreamCaptureStatusNone;
  e = cudaStreamIsCapturing(static_cast<cudaStream_t>(stream), &cap);
  if (e != cudaSuccess) return cuda_fail(e, "dense_prepare");
  if (cap != cudaStreamCaptureStatusNone) return fail(MMOE_ERR_NOT_PREPARED, "mmoe_dense_prepare() must run before stream capture");
  e = mmoe::prepare_dense();
  if (e == cudaSuccess) e = mmoe::prepare_grouped();
  if (e == cudaSuccess) e = mmoe::prepare_fp8();
  if (e == cudaSuccess) e = mmoe::prepare_grouped_few();
  return e == cudaSuccess ? MMOE_OK : cuda_fail(e, "dense_prepare");
}

int mmoe_feed_forward(const MmoeFeedForward* f, void* stream) {
  int rc = check_feed_forward(f);
  if (rc != MMOE_OK || f->num_tokens == 0) return rc;
  if (f->h == nullptr || f->y == nullptr) return fail(MMOE_ERR_INVALID_ARGUMENT, "feed-forward: h and y must not be NULL");
  mmoe::DenseProduct p = {};
  p.m = f->num_tokens, p.type = f->type;
  p.status = f->status, p.timeout_ms = f->timeout_ms;
  p.a = {f->x, f->x_stride, false};
  p.b = {f->w13, f->hidden, false};
  p.n = f->intermediate, p.k = f->hidden, p.kind = mmoe::kGated;
  p.epi.out = f->h, p.epi.ld_out = f->intermediate, p.epi.out_type = f->type;
  p.epi.inter = f->intermediate, p.epi.clamp = f->clamp, p.epi.preact = f->preact;
  rc = run_dense(&p, 1, "feed-forward, gated product", stream);
  if (rc != MMOE_OK) return rc;
  p.a = {f->h, f->intermediate, false};
  p.b = {f->w2, f->intermediate, false};
  p.n = f->hidden, p.k = f->intermediate, p.kind = mmoe::kLinear;
  p.epi = {};
  p.epi.out = f->y, p.epi.ld_out = f->hidden, p.epi.out_type = f->type;
  return run_dense(&p, 1, "feed-forward, second product", stream);
}

int mmoe_feed_forward_grad(const MmoeFeedForward* f, const void* dy, void* dpre, void* dx, void* dw13, void* dw2, void* stream) {
  int rc = check_feed_forward(f);
  if (rc != MMOE_OK) return rc;
  if (f->num_tokens == 0) {          // the weights' gradients are zero
    const size_t bytes = 2 * (size_t)f->hidden * f->intermediate;
    cudaError_t e = dw13 != nullptr ? cudaMemsetAsync(dw13, 0, 2 * bytes, static_cast<cudaStream_t>(stream)) : cudaSuccess;
    if (e == cudaSuccess && dw2 != nullptr) e = cudaMemsetAsync(dw2, 0, bytes, static_cast<cudaStream_t>(stream));
    return e == cudaSuccess ? MMOE_OK : cuda_fail(e, "feed-forward gradient of no tokens");
  }
  const bool inner = dx != nullptr || dw13 != nullptr;
  if (dy == nullptr || (inner && (dpre == nullptr || f->preact == nullptr)) || (dw2 != nullptr && f->h == nullptr))
    return fail(MMOE_ERR_INVALID_ARGUMENT, "feed-forward gradient: dy, and dpre, preact and h where they are needed, must not be NULL");
  for (const void* q : {dy, static_cast<const void*>(dpre), static_cast<const void*>(dx), static_cast<const void*>(dw13), static_cast<const void*>(dw2)})
    if (!aligned16(q)) return fail(MMOE_ERR_INVALID_ARGUMENT, "feed-forward gradient: pointers must be 16-byte aligned");
  const int h = f->hidden, i = f->intermediate, m = f->num_tokens;
  const auto product = [&](mmoe::DenseOperand a, mmoe::DenseOperand b, int rows, int cols, int k, void* out, int64_t ld) {
    mmoe::DenseProduct p = {};
    p.a = a, p.b = b, p.m = rows, p.n = cols, p.k = k, p.type = f->type, p.kind = mmoe::kLinear;
    p.status = f->status, p.timeout_ms = f->timeout_ms;
    p.epi.out = out, p.epi.ld_out = ld, p.epi.out_type = f->type;
    return p;
  };
  mmoe::DenseProduct through = product({dy, h, false}, {f->w2, i, true}, m, i, h, dpre, 2 * (int64_t)i);
  through.kind = mmoe::kGatedGrad;
  through.epi.inter = i, through.epi.clamp = f->clamp, through.epi.preact = f->preact;
  const mmoe::DenseProduct to_x = product({dpre, 2 * (int64_t)i, false}, {f->w13, h, true}, m, h, 2 * i, dx, h);
  const mmoe::DenseProduct to_w13 = product({dpre, 2 * (int64_t)i, true}, {f->x, f->x_stride, true}, 2 * i, h, m, dw13, h);
  const mmoe::DenseProduct to_w2 = product({dy, h, true}, {f->h, i, true}, h, i, m, dw2, i);
  // Launches of up to two products that need nothing of each other: what leads to g and u with dw2, then dx with dw13.  Few tokens: the
  // products of few tokens by themselves, then both weights' gradients.
  const char* what = "feed-forward gradient";
  mmoe::DenseProduct group[mmoe::kMaxParts];
  int n = 0;
  const auto flush = [&] {
    if (rc == MMOE_OK && n > 0) rc = run_dense(group, n, what, stream);
    n = 0;
  };
  const auto add = [&](const mmoe::DenseProduct& p) {
    const bool alone = mmoe::dense_few_tokens(p);
    if (alone) {
      if (rc == MMOE_OK) rc = run_dense(&p, 1, what, stream);
      return;
    }
    group[n++] = p;
    if (n == mmoe::kMaxParts) flush();
  };
  if (inner) add(through);
  if (inner && mmoe::dense_few_tokens(through)) {
    if (dx != nullptr) add(to_x);
    if (dw13 != nullptr) add(to_w13);
    if (dw2 != nullptr) add(to_w2);
  } else {
    if (dw2 != nullptr) add(to_w2);
    flush();                                 // dx and dw13 read what the first has written
    if (dx != nullptr) add(to_x);
    if (dw13 != nullptr) add(to_w13);
  }
  flush();
  return rc;
}

int mmoe_quantize_int8(const void* x, int32_t type, int64_t x_stride, void* q, float* scales, int32_t num_tokens, int32_t width, void* stream) {
  if (num_tokens < 0 || width <= 0) return fail(MMOE_ERR_INVALID_ARGUMENT, "int8 quantiser: num_tokens=%d must be >= 0 and width=%d positive", num_tokens, width);
  if (type != MMOE_BF16 && type != MMOE_FP16) return fail(MMOE_ERR_INVALID_ARGUMENT, "int8 quantiser: type=%d (supported: BF16, FP16)", type);
  constexpr int32_t kMost = INT32_MAX - 4095;          // the places of a block's threads in a row, a step past its end, are 32-bit numbers
  if (num_tokens > kMost || width > kMost)
    return fail(MMOE_ERR_INVALID_ARGUMENT, "int8 quantiser: num_tokens=%d and width=%d: at most %d", num_tokens, width, kMost);
  if (x_stride < width) return fail(MMOE_ERR_INVALID_ARGUMENT, "int8 quantiser: x_stride must be at least width=%d", width);
  if (num_tokens == 0) return MMOE_OK;
  if (x == nullptr || q == nullptr || scales == nullptr) return fail(MMOE_ERR_INVALID_ARGUMENT, "int8 quantiser: pointers must not be NULL");
  const cudaError_t e = mmoe::launch_quantize_int8(x, type, x_stride, static_cast<int8_t*>(q), scales, num_tokens, width, static_cast<cudaStream_t>(stream));
  return e == cudaSuccess ? MMOE_OK : cuda_fail(e, "int8 quantiser launch");
}

int mmoe_int8_projection(const MmoeInt8Product* p, void* stream) { return int8_product(p, false, stream); }

int mmoe_int8_gated_projection(const MmoeInt8Product* p, void* stream) { return int8_product(p, true, stream); }

int mmoe_dense_read_status(int32_t* status, int32_t* words8, void* stream) {
  if (status == nullptr) return fail(MMOE_ERR_INVALID_ARGUMENT, "status is NULL");
  int32_t host[8];
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  cudaError_t e = cudaMemcpyAsync(host, status, sizeof host, cudaMemcpyDeviceToHost, s);
  if (e == cudaSuccess) e = cudaMemsetAsync(status, 0, sizeof host, s);
  if (e == cudaSuccess) e = cudaStreamSynchronize(s);
  if (e != cudaSuccess) return cuda_fail(e, "reading the status words");
  if (words8 != nullptr) memcpy(words8, host, sizeof host);
  if (host[mmoe::kStatusTimeout] != 0)
    return fail(MMOE_ERR_DEVICE_TIMEOUT, "device wait expired: kernel %d role %d block %d", host[mmoe::kStatusKernel],
                host[mmoe::kStatusRole], host[mmoe::kStatusBlock]);
  if (host[mmoe::kStatusBadIndex] != 0)
    return fail(MMOE_ERR_INVALID_ARGUMENT, "%d launches with ends of groups that fall or pass the last row: no row was taken to be an expert's",
                host[mmoe::kStatusBadIndex]);
  return MMOE_OK;
}

}  // extern "C"
