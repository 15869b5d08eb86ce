// layer_norm.cpp -- entry points of layer norm, forward and backward, on the
// caller's device tensors (kernels/layer_norm.hip).
#include <cmath>

#include "device_ops.hpp"

namespace lchip {
namespace {

constexpr const char* kOp = "layer norm";

Status checkConfig(const lcLayerNormConfig* c) {
  if (c == nullptr) {
    return fail(Status::kInvalidValue, "layer norm: null config");
  }
  if (c->n == 0) {
    return fail(Status::kInvalidValue, "layer norm: zero width");
  }
  if (!validDtype(c->dtype) || !validDtype(c->weight_dtype) ||
      (c->weight_dtype != c->dtype && c->weight_dtype != LC_DTYPE_F32)) {
    return fail(Status::kInvalidValue, "layer norm: dtype f32, bf16 or f16, weights in the same or f32");
  }
  if (!std::isfinite(c->eps) || c->eps < 0.0f) {
    return fail(Status::kInvalidValue, "layer norm: eps must be finite and not negative");
  }
  if (c->n > (std::size_t{1} << 28) || c->rows > (std::size_t{1} << 40)) {
    return fail(Status::kNotSupported, "layer norm: shape too large");
  }
  return Status::kSuccess;
}

int chunkOf(lcDataType t) { return static_cast<int>(16 / bytesOf(t)); }

std::size_t partBytes(const lcLayerNormConfig& c) {
  const int groups = kern::layerNormGroups(static_cast<std::int64_t>(c.rows), static_cast<int>(c.n), true,
                                           chunkOf(c.dtype));
  return static_cast<std::size_t>(groups) * 2 * c.n * sizeof(float);
}

// A matrix's base and row stride (null stride pointers are not used: strides
// arrive by value).
Status takeRows(const lcLayerNormConfig& c, const char* name, const void* p, std::int64_t stride, bool written,
                bool* aligned, std::int64_t* out) {
  const std::string who = std::string(kOp) + ": " + name;
  *out = c.rows == 1 ? 0 : stride;
  if (c.rows == 0) {
    return Status::kSuccess;
  }
  if (p == nullptr) {
    return fail(Status::kInvalidValue, who + " is null");
  }
  const std::size_t bytes = bytesOf(c.dtype);
  const std::uintptr_t base = reinterpret_cast<std::uintptr_t>(p);
  if (base % bytes != 0) {
    return fail(Status::kInvalidValue, who + " is not aligned to its elements");
  }
  if (*out < 0 || (written && c.rows > 1 && *out < static_cast<std::int64_t>(c.n))) {
    return fail(Status::kInvalidValue, who + (written ? " is written and has overlapping rows"
                                                      : " has a negative stride"));
  }
  if (*out > (std::int64_t{1} << 46) / static_cast<std::int64_t>(c.rows)) {
    return fail(Status::kNotSupported, who + " has a stride too large");
  }
  if (base % 16 != 0 || *out % chunkOf(c.dtype) != 0 || c.n % chunkOf(c.dtype) != 0) {
    *aligned = false;
  }
  return Status::kSuccess;
}

bool onChunk(const void* p) { return reinterpret_cast<std::uintptr_t>(p) % 16 == 0; }

Status checkWeight(const lcLayerNormConfig& c, const char* name, const void* p) {
  if (reinterpret_cast<std::uintptr_t>(p) % bytesOf(c.weight_dtype) != 0) {
    return fail(Status::kInvalidValue, std::string(kOp) + ": " + name + " is not aligned to its elements");
  }
  return Status::kSuccess;
}

void fillArgs(const lcLayerNormConfig& c, kern::LayerNormArgs* a) {
  a->rows = static_cast<std::int64_t>(c.rows);
  a->n = static_cast<int>(c.n);
  a->wide = c.weight_dtype == LC_DTYPE_F32 ? 1 : 0;
  a->eps = c.eps;
}

Status forward(const lcLayerNormConfig* cfg, const void* x, std::int64_t x_stride, const void* weight,
               const void* bias, void* y, std::int64_t y_stride, float* mean, float* rstd, lcStream stream) {
  LC_TRY(checkConfig(cfg));
  const lcLayerNormConfig& c = *cfg;
  kern::LayerNormArgs a{};
  bool aligned = true;
  LC_TRY(takeRows(c, "x", x, x_stride, false, &aligned, &a.sx));
  LC_TRY(takeRows(c, "y", y, y_stride, true, &aligned, &a.sy));
  LC_TRY(checkWeight(c, "weight", weight));
  LC_TRY(checkWeight(c, "bias", bias));
  if ((mean == nullptr) != (rstd == nullptr)) {
    return fail(Status::kInvalidValue, "layer norm: mean and rstd are stored together or not at all");
  }
  DeviceCall call;
  LC_TRY(call.open(kOp, c.trusted_pointers != 0));
  if (c.rows == 0) {
    return Status::kSuccess;
  }
  const struct {
    const void* p;
    const char* name;
  } pointers[] = {{x, "x"}, {y, "y"}, {weight, "weight"}, {bias, "bias"}, {mean, "mean"}, {rstd, "rstd"}};
  for (const auto& p : pointers) {
    LC_TRY(call.onDevice(p.p, p.name));
  }
  fillArgs(c, &a);
  a.x = x;
  a.y = y;
  a.w = weight;
  a.b = bias;
  a.weights_aligned = onChunk(weight) && onChunk(bias) ? 1 : 0;
  a.mean = mean;
  a.rstd = rstd;
  LC_HIP_TRY(kern::layerNorm(a, dtypeOf(c.dtype), false, aligned, static_cast<hipStream_t>(stream)));
  return Status::kSuccess;
}

Status backward(const lcLayerNormConfig* cfg, const void* dy, std::int64_t dy_stride, const void* x,
                std::int64_t x_stride, const void* weight, const float* mean, const float* rstd, void* dx,
                std::int64_t dx_stride, void* dweight, void* dbias, void* workspace, std::size_t workspace_bytes,
                lcStream stream) {
  LC_TRY(checkConfig(cfg));
  const lcLayerNormConfig& c = *cfg;
  kern::LayerNormArgs a{};
  bool aligned = true;
  LC_TRY(takeRows(c, "dy", dy, dy_stride, false, &aligned, &a.sy));
  LC_TRY(takeRows(c, "x", x, x_stride, false, &aligned, &a.sx));
  LC_TRY(takeRows(c, "dx", dx, dx_stride, true, &aligned, &a.sdx));
  LC_TRY(checkWeight(c, "weight", weight));
  LC_TRY(checkWeight(c, "dweight", dweight));
  LC_TRY(checkWeight(c, "dbias", dbias));
  if (c.rows != 0 && (mean == nullptr || rstd == nullptr)) {
    return fail(Status::kInvalidValue, "layer norm: the backward pass needs the forward's mean and rstd");
  }
  DeviceCall call;
  LC_TRY(call.open(kOp, c.trusted_pointers != 0));
  const std::size_t need = partBytes(c);
  if (need != 0 && (workspace == nullptr || workspace_bytes < need)) {
    return fail(Status::kInvalidValue, "layer norm: the workspace needs " + std::to_string(need) + " bytes, " +
                                           std::to_string(workspace == nullptr ? 0 : workspace_bytes) + " given");
  }
  if (reinterpret_cast<std::uintptr_t>(workspace) % 16 != 0) {
    return fail(Status::kInvalidValue, "layer norm: the workspace is not 16-byte aligned");
  }
  const struct {
    const void* p;
    const char* name;
  } pointers[] = {{dy, "dy"},     {x, "x"},   {weight, "weight"},   {mean, "mean"},
                  {rstd, "rstd"}, {dx, "dx"}, {dweight, "dweight"}, {dbias, "dbias"},
                  {workspace, "the workspace"}};
  for (const auto& p : pointers) {
    LC_TRY(call.onDevice(p.p, p.name));
  }
  fillArgs(c, &a);
  a.x = x;
  a.dy = dy;
  a.w = weight;
  a.weights_aligned = onChunk(weight) ? 1 : 0;
  a.mean = const_cast<float*>(mean);
  a.rstd = const_cast<float*>(rstd);
  a.dx = dx;
  a.dw = dweight;
  a.db = dbias;
  a.part = static_cast<float*>(workspace);
  LC_HIP_TRY(kern::layerNorm(a, dtypeOf(c.dtype), true, aligned, static_cast<hipStream_t>(stream)));
  return Status::kSuccess;
}

}  // namespace
}  // namespace lchip

extern "C" {

lcError_t lcLayerNormWorkspaceSize(const lcLayerNormConfig* cfg, size_t* bytes) {
  using namespace lchip;
  if (bytes == nullptr) {
    return toLc(fail(Status::kInvalidValue, "layer norm: null output"));
  }
  *bytes = 0;
  const Status st = checkConfig(cfg);
  if (st == Status::kSuccess) {
    *bytes = partBytes(*cfg);
  }
  return toLc(st);
}

lcError_t lcLayerNormForward(const lcLayerNormConfig* cfg, const void* x, int64_t x_stride, const void* weight,
                             const void* bias, void* y, int64_t y_stride, float* mean, float* rstd, lcStream stream) {
  return lchip::toLc(lchip::forward(cfg, x, x_stride, weight, bias, y, y_stride, mean, rstd, stream));
}

lcError_t lcLayerNormBackward(const lcLayerNormConfig* cfg, const void* dy, int64_t dy_stride, const void* x,
                              int64_t x_stride, const void* weight, const float* mean, const float* rstd, void* dx,
                              int64_t dx_stride, void* dweight, void* dbias, void* workspace, size_t workspace_bytes,
                              lcStream stream) {
  return lchip::toLc(lchip::backward(cfg, dy, dy_stride, x, x_stride, weight, mean, rstd, dx, dx_stride, dweight,
                                     dbias, workspace, workspace_bytes, stream));
}

}  // extern "C"
