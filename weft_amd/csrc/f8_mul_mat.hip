// weft_ggml_mul_mat_f8: the checks of a call, and which kernels it takes.
#include <algorithm>

#include "f8.h"
#include "runtime.h"

namespace weft {
namespace {

hipError_t fail(hipError_t e) {
  set_error(e);
  return e;
}

// The work buffer.  An activation that arrives as plain rows is quantized into it: codes of
// whole blocks (zeros past k), then scales, block-major; then come the sums of K's ranges.
struct Plan {
  int64_t pitch = 0;  // bytes of a row of codes; 0: the activation arrives quantized, or the product's kernel does it
  size_t scales = 0;  // where the scales begin
  size_t sums = 0;    // where the sums do, 16-byte aligned
  size_t size = 0;
};

bool plan_of(const weft_ggml_tensor* w, const weft_ggml_tensor* x, Plan* out) {
  const int64_t k = w->ne[0], n = w->ne[1], m = x->ne[1];
  if (k < 1 || n < 0 || m < 0 || k > INT32_MAX / 2 || n > INT32_MAX || m > INT32_MAX || x->ne[0] != k) return false;
  Plan p;
  if (x->type != WEFT_GGML_TYPE_F8_E4M3 && !f8_few_quantizes(m, k)) {
    p.pitch = f8_blocks(k) * kF8Block;
    p.scales = (size_t)m * (size_t)p.pitch;
    p.size = p.scales + (size_t)m * (size_t)f8_blocks(k) * sizeof(float);
  }
  if (m > kF8Few && n > 0) {
    p.sums = (p.size + 15) / 16 * 16;
    const size_t bytes = f8_many_work(m, n, k);
    if (bytes > 0) p.size = p.sums + bytes;
  }
  if (m == 0 || n == 0) p.size = 0;
  *out = p;
  return true;
}

bool activation(int32_t t) {
  return t == WEFT_GGML_TYPE_F32 || t == WEFT_GGML_TYPE_F16 || t == WEFT_GGML_TYPE_F8_E4M3;
}

size_t unit_of(int32_t t) {
  return t == WEFT_GGML_TYPE_F32 ? 4 : t == WEFT_GGML_TYPE_F16 ? 2 : 1;
}

// a matrix whose rows of contiguous elements lie any whole elements apart
bool matrix(const weft_ggml_tensor* t, int64_t k, int64_t rows) {
  const size_t unit = unit_of(t->type);
  return t->ne[0] == k && t->ne[1] == rows && t->ne[2] == 1 && t->ne[3] == 1 && t->nb[0] == unit &&
         t->nb[1] % unit == 0 && t->nb[1] < ((size_t)1 << 40) && aligned(t->data, unit);
}

bool scales_of(const weft_ggml_tensor* t, int64_t k, int64_t rows) {
  return t->ne[0] == f8_blocks(k) && t->ne[1] == rows && t->ne[2] == 1 && t->ne[3] == 1 && t->nb[0] % 4 == 0 &&
         t->nb[1] % 4 == 0 && t->nb[0] < ((size_t)1 << 40) && t->nb[1] < ((size_t)1 << 40) && aligned(t->data, 4);
}

F8Rows rows_of(const weft_ggml_tensor* codes, const weft_ggml_tensor* scales) {
  return {static_cast<const uint8_t*>(codes->data), static_cast<const float*>(scales->data),
          (long long)codes->nb[1], (long long)(scales->nb[1] / 4), (long long)(scales->nb[0] / 4)};
}

hipError_t mul_mat_f8(const weft_ggml_tensor* w, const weft_ggml_tensor* w_scales, const weft_ggml_tensor* x,
                      const weft_ggml_tensor* x_scales, const weft_ggml_tensor* dst, void* wdata, size_t wsize) {
  if (w == nullptr || w_scales == nullptr || x == nullptr || dst == nullptr) return fail(hipErrorInvalidValue);
  if (w->type != WEFT_GGML_TYPE_F8_E4M3 || w_scales->type != WEFT_GGML_TYPE_F32 || !activation(x->type) ||
      (dst->type != WEFT_GGML_TYPE_F32 && dst->type != WEFT_GGML_TYPE_F16) ||
      (x_scales != nullptr && x_scales->type != WEFT_GGML_TYPE_F32))
    return fail(hipErrorNotSupported);
  Plan plan;
  if (!plan_of(w, x, &plan)) return fail(hipErrorInvalidValue);
  const int64_t k = w->ne[0], n = w->ne[1], m = x->ne[1];
  const bool quantized = x->type == WEFT_GGML_TYPE_F8_E4M3;
  if (!matrix(w, k, n) || !matrix(x, k, m) || !matrix(dst, n, m) || !scales_of(w_scales, k, f8_blocks(n)) ||
      quantized != (x_scales != nullptr) || (quantized && !scales_of(x_scales, k, m)))
    return fail(hipErrorInvalidValue);
  if (m == 0 || n == 0) return hipSuccess;
  for (const weft_ggml_tensor* t : {w, w_scales, x, dst})
    if (t->data == nullptr) return fail(hipErrorInvalidValue);
  if (quantized && x_scales->data == nullptr) return fail(hipErrorInvalidValue);
  if (wsize < plan.size || (plan.size > 0 && (wdata == nullptr || !aligned(wdata, 16)))) return fail(hipErrorInvalidValue);
  F8Product p{};
  p.w = rows_of(w, w_scales);
  p.y = static_cast<uint8_t*>(dst->data);
  p.y_row = (long long)dst->nb[1];
  p.n = (int)n;
  p.m = (int)m;
  p.k = (int)k;
  p.half_out = dst->type == WEFT_GGML_TYPE_F16;
  if (quantized) {
    p.x = rows_of(x, x_scales);
  } else if (plan.pitch == 0) {
    f8_few(p, static_cast<const uint8_t*>(x->data), x->type == WEFT_GGML_TYPE_F16, (long long)x->nb[1]);
    return pending_error();
  } else {
    uint8_t* codes = static_cast<uint8_t*>(wdata);
    float* scales = reinterpret_cast<float*>(codes + plan.scales);
    f8_quantize_rows(static_cast<const uint8_t*>(x->data), x->type == WEFT_GGML_TYPE_F16, (long long)x->nb[1], codes,
                     plan.pitch, (int)plan.pitch, scales, 1, m, m, (int)k);
    p.x = {codes, scales, plan.pitch, 1, m};
  }
  if (m <= kF8Few)
    f8_few(p);
  else
    f8_many(p, reinterpret_cast<float*>(static_cast<uint8_t*>(wdata) + plan.sums));
  return pending_error();
}

}  // namespace
}  // namespace weft

extern "C" size_t weft_ggml_mul_mat_f8_work_size(const weft_ggml_tensor* w, const weft_ggml_tensor* x) {
  weft::Plan plan;
  if (w == nullptr || x == nullptr || !weft::activation(x->type) || !weft::plan_of(w, x, &plan)) return 0;
  return plan.size;
}

extern "C" int weft_ggml_mul_mat_f8(const weft_ggml_tensor* w, const weft_ggml_tensor* w_scales,
                                    const weft_ggml_tensor* x, const weft_ggml_tensor* x_scales,
                                    const weft_ggml_tensor* dst, void* wdata, size_t wsize) {
  return (int)weft::mul_mat_f8(w, w_scales, x, x_scales, dst, wdata, wsize);
}
