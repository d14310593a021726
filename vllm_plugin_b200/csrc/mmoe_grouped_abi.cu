// extern "C" entry points of the experts' products (declared in include/mmoe.h): argument checks and the products of a call.  Nothing here
// allocates device memory or synchronises.
#include "mmoe_dense_abi.h"
#include "mmoe_grouped.cuh"

namespace {

bool aligned(const void* p, uintptr_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

// tiles and rows of all experts are 32-bit numbers
constexpr int32_t kMostGroupedChannels = 1 << 20;

int check_grouping(const char* what, int32_t rows, int32_t experts, const int32_t* ends) {
  if (rows < 0 || rows > kMostTokens) return fail(MMOE_ERR_INVALID_ARGUMENT, "%s: num_rows=%d outside [0, %d]", what, rows, kMostTokens);
  if (experts < 1 || experts > mmoe::kMaxExperts) return fail(MMOE_ERR_INVALID_ARGUMENT, "%s: num_experts=%d outside [1, %d]", what, experts, mmoe::kMaxExperts);
  if (ends == nullptr || !aligned(ends, 4)) return fail(MMOE_ERR_INVALID_ARGUMENT, "%s: ends must not be NULL and on 4 bytes", what);
  return MMOE_OK;
}

int check_width(const char* what, const char* name, int32_t width, int32_t step) {
  if (width < step || width % step != 0 || width > kMostGroupedChannels)
    return fail(MMOE_ERR_INVALID_ARGUMENT, "%s: %s=%d must be a positive multiple of %d, at most %d", what, name, width, step, kMostGroupedChannels);
  return MMOE_OK;
}

int check_type(const char* what, int32_t type) {
  return type == MMOE_BF16 || type == MMOE_FP16 ? MMOE_OK : fail(MMOE_ERR_INVALID_ARGUMENT, "%s: type=%d (supported: BF16, FP16)", what, type);
}

int check_rows(const char* what, const void* x, int64_t stride, int32_t width, int64_t step, int32_t rows, const int32_t* status) {
  if (stride < width || stride % step != 0 || stride > (int64_t)1 << 36)
    return fail(MMOE_ERR_INVALID_ARGUMENT, "%s: x_stride must be a multiple of %d and at least the width %d", what, static_cast<int>(step), width);
  if (rows > 0 && (x == nullptr || status == nullptr)) return fail(MMOE_ERR_INVALID_ARGUMENT, "%s: x and status must not be NULL", what);
  return MMOE_OK;
}

int run_grouped(const mmoe::GroupedProduct& p, const char* what, void* stream) {
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  const cudaError_t e = p.type == mmoe::kGroupedE4m3 ? mmoe::launch_fp8(p, s) : mmoe::launch_grouped(p, s);
  return e == cudaSuccess ? MMOE_OK : e == cudaErrorNotReady ? fail(MMOE_ERR_NOT_PREPARED, "%s: mmoe_dense_prepare() has not run on this device", what) : cuda_fail(e, what);
}

int clear(void* p, size_t bytes, const char* what, void* stream) {
  const cudaError_t e = p != nullptr ? cudaMemsetAsync(p, 0, bytes, static_cast<cudaStream_t>(stream)) : cudaSuccess;
  return e == cudaSuccess ? MMOE_OK : cuda_fail(e, what);
}

// what the products of a call have in common
mmoe::GroupedProduct product_of(int32_t type, int32_t rows, int32_t experts, const int32_t* ends, int32_t* status, int32_t timeout_ms) {
  mmoe::GroupedProduct p = {};
  p.type = type, p.kind = mmoe::kLinear, p.rows = rows, p.experts = experts, p.ends = ends, p.status = status, p.timeout_ms = timeout_ms;
  p.epi.out_type = type;
  return p;
}

// out[t, n] = sum_k x[t, k] w[e][n, k], or (k_rows) w[e][k, n]
int to_rows(mmoe::GroupedProduct p, const void* x, int64_t ld, int32_t k, const void* w, bool k_rows, int32_t n, void* out, bool zero_behind, const char* what, void* stream) {
  p.x = x, p.x_ld = ld, p.k = k, p.w = w, p.w_k_rows = k_rows, p.n = n, p.zero_behind = zero_behind;
  p.epi.out = out, p.epi.ld_out = n;
  return run_grouped(p, what, stream);
}

// out[e][n, k] = sum of e's rows of left[t, n] x[t, k]
int to_weights(mmoe::GroupedProduct p, const void* left, int64_t left_ld, int32_t n, const void* x, int64_t ld, int32_t k, void* out, const char* what, void* stream) {
  p.kind = mmoe::kGroupedWeights, p.left = left, p.left_ld = left_ld, p.n = n, p.x = x, p.x_ld = ld, p.k = k;
  p.epi.out = out, p.epi.ld_out = k;
  return run_grouped(p, what, stream);
}

int check_projection(const MmoeGroupedProduct* a, const char* what) {
  if (a == nullptr) return fail(MMOE_ERR_INVALID_ARGUMENT, "%s: arguments are NULL", what);
  int rc = check_type(what, a->type);
  if (rc == MMOE_OK) rc = check_grouping(what, a->num_rows, a->num_experts, a->ends);
  if (rc == MMOE_OK) rc = check_width(what, "width", a->width, 8);
  if (rc == MMOE_OK) rc = check_width(what, "channels", a->channels, 8);
  if (rc == MMOE_OK) rc = check_rows(what, a->x, a->x_stride, a->width, 8, a->num_rows, a->status);
  if (rc != MMOE_OK) return rc;
  if (a->w == nullptr) return fail(MMOE_ERR_INVALID_ARGUMENT, "%s: w must not be NULL", what);
  if (!aligned16(a->x) || !aligned16(a->w) || !aligned16(a->out)) return fail(MMOE_ERR_INVALID_ARGUMENT, "%s: pointers must be 16-byte aligned", what);
  return MMOE_OK;
}

int check_feed_forward(const MmoeGroupedFeedForward* f, const char* what) {
  if (f == nullptr) return fail(MMOE_ERR_INVALID_ARGUMENT, "%s: arguments are NULL", what);
  int rc = check_type(what, f->type);
  if (rc == MMOE_OK) rc = check_grouping(what, f->num_rows, f->num_experts, f->ends);
  if (rc == MMOE_OK) rc = check_width(what, "hidden", f->hidden, 8);
  if (rc == MMOE_OK) rc = check_width(what, "intermediate", f->intermediate, 8);
  if (rc == MMOE_OK) rc = check_rows(what, f->x, f->x_stride, f->hidden, 8, f->num_rows, f->status);
  if (rc != MMOE_OK) return rc;
  if (!(f->clamp > 0.f)) return fail(MMOE_ERR_INVALID_ARGUMENT, "%s: clamp must be positive", what);
  if (f->w13 == nullptr || f->w2 == nullptr) return fail(MMOE_ERR_INVALID_ARGUMENT, "%s: w13 and w2 must not be NULL", what);
  if (!aligned16(f->x) || !aligned16(f->w13) || !aligned16(f->w2) || !aligned16(f->h) || !aligned16(f->preact) || !aligned16(f->y))
    return fail(MMOE_ERR_INVALID_ARGUMENT, "%s: pointers must be 16-byte aligned", what);
  return MMOE_OK;
}

int fp8_product(const MmoeFp8Product* a, bool gated, void* stream) {
  const char* what = gated ? "fp8 gated projection" : "fp8 projection";
  if (a == nullptr) return fail(MMOE_ERR_INVALID_ARGUMENT, "%s: arguments are NULL", what);
  int rc = MMOE_OK;
  if (a->ends != nullptr || a->num_experts != 1) rc = check_grouping(what, a->num_rows, a->num_experts, a->ends);
  else if (a->num_rows < 0 || a->num_rows > kMostTokens) rc = fail(MMOE_ERR_INVALID_ARGUMENT, "%s: num_rows=%d outside [0, %d]", what, a->num_rows, kMostTokens);
  if (rc == MMOE_OK) rc = check_width(what, "width", a->width, 16);
  if (rc == MMOE_OK) rc = check_width(what, "channels", a->channels, gated ? 8 : 1);
  if (rc == MMOE_OK) rc = check_rows(what, a->x, a->x_stride, a->width, 16, a->num_rows, a->status);
  if (rc != MMOE_OK) return rc;
  if (a->out_type != MMOE_BF16 && a->out_type != MMOE_FP16 && a->out_type != MMOE_FP32) return fail(MMOE_ERR_INVALID_ARGUMENT, "%s: out_type=%d", what, a->out_type);
  if (gated && !(a->clamp > 0.f)) return fail(MMOE_ERR_INVALID_ARGUMENT, "%s: clamp must be positive", what);
  if (a->num_rows == 0) return MMOE_OK;
  if (a->x_scales == nullptr || a->w == nullptr || a->w_scales == nullptr || a->out == nullptr) return fail(MMOE_ERR_INVALID_ARGUMENT, "%s: pointers must not be NULL", what);
  if (!aligned16(a->x) || !aligned16(a->w) || !aligned16(a->out)) return fail(MMOE_ERR_INVALID_ARGUMENT, "%s: x, w and out must be 16-byte aligned", what);
  if (!aligned(a->x_scales, 4) || !aligned(a->w_scales, 4)) return fail(MMOE_ERR_INVALID_ARGUMENT, "%s: scales must be on 4 bytes", what);
  mmoe::GroupedProduct p = product_of(mmoe::kGroupedE4m3, a->num_rows, a->num_experts, a->ends, a->status, a->timeout_ms);
  p.kind = gated ? mmoe::kGated : mmoe::kLinear;
  p.n = a->channels, p.k = a->width, p.w = a->w, p.x = a->x, p.x_ld = a->x_stride, p.x_scales = a->x_scales, p.w_scales = a->w_scales;
  p.epi.out = a->out, p.epi.ld_out = a->channels, p.epi.out_type = a->out_type, p.epi.inter = a->channels, p.epi.clamp = a->clamp;
  p.zero_behind = true;
  return run_grouped(p, what, stream);
}

}  // namespace

extern "C" {

int mmoe_grouped_projection(const MmoeGroupedProduct* a, void* stream) {
  const char* what = "grouped projection";
  const int rc = check_projection(a, what);
  if (rc != MMOE_OK || a->num_rows == 0) return rc;
  if (a->out == nullptr) return fail(MMOE_ERR_INVALID_ARGUMENT, "%s: out must not be NULL", what);
  return to_rows(product_of(a->type, a->num_rows, a->num_experts, a->ends, a->status, a->timeout_ms), a->x, a->x_stride, a->width, a->w, false, a->channels, a->out, true,
                 what, stream);
}

int mmoe_grouped_projection_grad(const MmoeGroupedProduct* a, const void* dy, void* dx, void* dw, void* stream) {
  const char* what = "grouped projection, gradient";
  int rc = check_projection(a, what);
  if (rc != MMOE_OK) return rc;
  if (!aligned16(dy) || !aligned16(dx) || !aligned16(dw) || (a->num_rows > 0 && dy == nullptr))
    return fail(MMOE_ERR_INVALID_ARGUMENT, "%s: dy must not be NULL, pointers must be 16-byte aligned", what);
  if (a->num_rows == 0) return clear(dw, 2 * (size_t)a->num_experts * a->channels * a->width, what, stream);
  const mmoe::GroupedProduct p = product_of(a->type, a->num_rows, a->num_experts, a->ends, a->status, a->timeout_ms);
  if (dx != nullptr) rc = to_rows(p, dy, a->channels, a->channels, a->w, true, a->width, dx, true, what, stream);
  if (rc == MMOE_OK && dw != nullptr) rc = to_weights(p, dy, a->channels, a->channels, a->x, a->x_stride, a->width, dw, what, stream);
  return rc;
}

int mmoe_grouped_feed_forward(const MmoeGroupedFeedForward* f, void* stream) {
  const char* what = "grouped feed-forward";
  int rc = check_feed_forward(f, what);
  if (rc != MMOE_OK || f->num_rows == 0) return rc;
  if (f->h == nullptr || f->y == nullptr) return fail(MMOE_ERR_INVALID_ARGUMENT, "%s: h and y must not be NULL", what);
  const mmoe::GroupedProduct p = product_of(f->type, f->num_rows, f->num_experts, f->ends, f->status, f->timeout_ms);
  mmoe::GroupedProduct first = p;
  first.kind = mmoe::kGated, first.epi.inter = f->intermediate, first.epi.clamp = f->clamp, first.epi.preact = f->preact;
  rc = to_rows(first, f->x, f->x_stride, f->hidden, f->w13, false, f->intermediate, f->h, false, what, stream);
  if (rc == MMOE_OK) rc = to_rows(p, f->h, f->intermediate, f->intermediate, f->w2, false, f->hidden, f->y, true, what, stream);
  return rc;
}

int mmoe_grouped_feed_forward_grad(const MmoeGroupedFeedForward* f, const void* dy, void* dpre, void* dx, void* dw13, void* dw2, void* stream) {
  const char* what = "grouped feed-forward, gradient";
  int rc = check_feed_forward(f, what);
  if (rc != MMOE_OK) return rc;
  const int32_t h = f->hidden, i = f->intermediate;
  if (f->num_rows == 0) {            // the weights' gradients are zero
    const size_t bytes = 2 * (size_t)f->num_experts * h * i;
    rc = clear(dw13, 2 * bytes, what, stream);
    return rc == MMOE_OK ? clear(dw2, bytes, what, stream) : rc;
  }
  const bool inner = dx != nullptr || dw13 != nullptr;
  if (dy == nullptr || (inner && (dpre == nullptr || f->preact == nullptr)) || (dw2 != nullptr && f->h == nullptr))
    return fail(MMOE_ERR_INVALID_ARGUMENT, "%s: dy, and dpre, preact and h where they are needed, must not be NULL", what);
  for (const void* q : {dy, static_cast<const void*>(dpre), static_cast<const void*>(dx), static_cast<const void*>(dw13), static_cast<const void*>(dw2)})
    if (!aligned16(q)) return fail(MMOE_ERR_INVALID_ARGUMENT, "%s: pointers must be 16-byte aligned", what);
  const mmoe::GroupedProduct p = product_of(f->type, f->num_rows, f->num_experts, f->ends, f->status, f->timeout_ms);
  if (inner) {
    mmoe::GroupedProduct through = p;
    through.kind = mmoe::kGatedGrad, through.epi.inter = i, through.epi.clamp = f->clamp, through.epi.preact = f->preact;
    through.x = dy, through.x_ld = h, through.k = h, through.w = f->w2, through.w_k_rows = true, through.n = i;
    through.epi.out = dpre, through.epi.ld_out = 2 * (int64_t)i;
    rc = run_grouped(through, what, stream);
  }
  if (rc == MMOE_OK && dw2 != nullptr) rc = to_weights(p, dy, h, h, f->h, i, i, dw2, what, stream);
  if (rc == MMOE_OK && dx != nullptr) rc = to_rows(p, dpre, 2 * (int64_t)i, 2 * i, f->w13, true, h, dx, true, what, stream);
  if (rc == MMOE_OK && dw13 != nullptr) rc = to_weights(p, dpre, 2 * (int64_t)i, 2 * i, f->x, f->x_stride, h, dw13, what, stream);
  return rc;
}

int mmoe_quantize_fp8(const void* x, int32_t type, int64_t x_stride, void* q, float* scales, int32_t num_rows, int32_t width, void* stream) {
  const char* what = "fp8 quantiser";
  int rc = check_type(what, type);
  if (rc != MMOE_OK) return rc;
  constexpr int32_t kMost = INT32_MAX - 4095;
  if (num_rows < 0 || num_rows > kMost || width <= 0 || width > kMost)
    return fail(MMOE_ERR_INVALID_ARGUMENT, "%s: num_rows=%d must be >= 0 and width=%d positive, at most %d", what, num_rows, width, kMost);
  if ((uint64_t)num_rows * (((uint32_t)width + 127) / 128) > UINT32_MAX)
    return fail(MMOE_ERR_INVALID_ARGUMENT, "%s: num_rows=%d of width=%d have more than 2^32 - 1 groups of 128", what, num_rows, width);
  if (x_stride < width) return fail(MMOE_ERR_INVALID_ARGUMENT, "%s: x_stride must be at least width=%d", what, width);
  if (num_rows == 0) return MMOE_OK;
  if (x == nullptr || q == nullptr || scales == nullptr) return fail(MMOE_ERR_INVALID_ARGUMENT, "%s: pointers must not be NULL", what);
  if (!aligned(x, 2) || !aligned(scales, 4)) return fail(MMOE_ERR_INVALID_ARGUMENT, "%s: x must be on 2 bytes and scales on 4", what);
  const cudaError_t e = mmoe::launch_quantize_fp8(x, type, x_stride, static_cast<uint8_t*>(q), scales, num_rows, width, static_cast<cudaStream_t>(stream));
  return e == cudaSuccess ? MMOE_OK : cuda_fail(e, what);
}

int mmoe_fp8_projection(const MmoeFp8Product* p, void* stream) { return fp8_product(p, false, stream); }

int mmoe_fp8_gated_projection(const MmoeFp8Product* p, void* stream) { return fp8_product(p, true, stream); }

}  // extern "C"
