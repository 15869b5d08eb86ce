// device_ops.cpp -- checks shared by the entry points on device tensors.
#include "device_ops.hpp"

#include <algorithm>

namespace lchip {

DeviceCall::~DeviceCall() {
  if (ctx_ != nullptr && before_ >= 0 && before_ != ctx_->device) {
    (void)hipSetDevice(before_);
  }
}

Status DeviceCall::open(const char* op, bool trusted) {
  op_ = op;
  trusted_ = trusted;
  if (hipGetDevice(&before_) != hipSuccess) {
    (void)hipGetLastError();
    before_ = -1;
  }
  return requireHip(LC_DEVICE_HIP, op, &ctx_);
}

Status DeviceCall::onDevice(const void* p, const char* what) const {
  if (p == nullptr || trusted_) {
    return Status::kSuccess;
  }
  hipPointerAttribute_t attr{};
  const bool known = hipPointerGetAttributes(&attr, p) == hipSuccess;
  if (!known) {
    (void)hipGetLastError();  // a failed query must not be taken for a launch's
  }
  if (!known || (attr.type != hipMemoryTypeDevice && attr.type != hipMemoryTypeManaged) ||
      (attr.type == hipMemoryTypeDevice && attr.device != ctx_->device)) {
    return fail(Status::kInvalidValue, std::string(op_) + ": " + what + " is not memory of device " +
                                           std::to_string(ctx_->device));
  }
  return Status::kSuccess;
}

Status takeTensor(const char* op, const char* name, const lcDeviceTensor* t, std::size_t batch, std::size_t heads,
                  std::size_t rows, std::size_t d, lcDataType type, bool written, kern::XTensor* out, bool* aligned) {
  const std::string who = std::string(op) + ": " + name;
  if (t == nullptr) {
    return fail(Status::kInvalidValue, who + " is null");
  }
  *out = {t->data, t->stride_batch, t->stride_head, t->stride_row};
  if (batch == 0 || heads == 0 || rows == 0) {
    return Status::kSuccess;
  }
  if (t->data == nullptr) {
    return fail(Status::kInvalidValue, who + " has values and a null base");
  }
  const std::size_t bytes = bytesOf(type);
  const std::uintptr_t base = reinterpret_cast<std::uintptr_t>(t->data);
  if (base % bytes != 0) {
    return fail(Status::kInvalidValue, who + " is not aligned to its elements");
  }
  // A dimension of one has a stride that means nothing.
  if (batch == 1) out->sb = 0;
  if (heads == 1) out->sh = 0;
  if (rows == 1) out->ss = 0;
  if (out->sb < 0 || out->sh < 0 || out->ss < 0) {
    return fail(Status::kInvalidValue, who + " has a negative stride");
  }
  const std::int64_t most = std::int64_t{1} << 46;  // elements: no address product overflows
  if (out->sb > most || out->sh > most ||
      out->ss > static_cast<std::int64_t>(((std::size_t{1} << 31) - 4096) / (128 * bytes))) {
    return fail(Status::kNotSupported, who + " has a stride too large");
  }
  if (written) {
    // From the smallest stride up, each step must pass all that lies inside it
    // (the padding behind a block's last row may hold the next block's rows).
    struct Dim {
      std::int64_t stride;
      std::size_t n;
    } dims[] = {{out->sb, batch}, {out->sh, heads}, {out->ss, rows}};
    std::sort(dims, dims + 3, [](const Dim& x, const Dim& y) { return x.stride < y.stride; });
    std::int64_t extent = static_cast<std::int64_t>(d);
    for (const Dim& x : dims) {
      if (x.n == 1) {
        continue;
      }
      if (x.stride < extent) {
        return fail(Status::kInvalidValue, who + " is written and has overlapping rows");
      }
      // No product of a stride that a real tensor can have overflows.
      if (x.stride > (std::int64_t{1} << 60) / static_cast<std::int64_t>(x.n)) {
        return fail(Status::kNotSupported, who + " has a stride too large");
      }
      extent += x.stride * static_cast<std::int64_t>(x.n - 1);
    }
  }
  const std::int64_t ec = static_cast<std::int64_t>(16 / bytes);
  if (base % 16 != 0 || out->sb % ec != 0 || out->sh % ec != 0 || out->ss % ec != 0 ||
      static_cast<std::int64_t>(d) % ec != 0) {
    *aligned = false;
  }
  return Status::kSuccess;
}

int splitCount(std::size_t blocks, std::size_t tiles, std::size_t slots, double fixed, double join) {
  if (blocks == 0 || tiles <= 1) {
    return 1;
  }
  int best = 1;
  double least = 0.0;
  const std::size_t most = std::min<std::size_t>(tiles, 32);
  for (std::size_t s = 1; s <= most; ++s) {
    const std::size_t share = (tiles + s - 1) / s;
    if (s > 1 && share == (tiles + s - 2) / (s - 1)) {
      continue;  // no shorter than with one share less
    }
    const double rounds = static_cast<double>((blocks * s + slots - 1) / slots);
    const double cost = rounds * (static_cast<double>(share) + fixed) + (s > 1 ? join : 0.0);
    if (s == 1 || cost < least) {
      least = cost;
      best = static_cast<int>(s);
    }
  }
  return best;
}

}  // namespace lchip

extern "C" lcError_t lcHipDeviceIndex(int* out) {
  using namespace lchip;
  if (out == nullptr) {
    return toLc(fail(Status::kInvalidValue, "device index: null output"));
  }
  *out = -1;
  DeviceCall call;
  const Status st = call.open("device index", false);
  if (st == Status::kSuccess) {
    *out = call.device();
  }
  return toLc(st);
}

extern "C" lcError_t lcHipBackendStream(lcStream* out) {
  using namespace lchip;
  if (out == nullptr) {
    return toLc(fail(Status::kInvalidValue, "backend stream: null output"));
  }
  HipContext* ctx = nullptr;
  const Status st = requireHip(LC_DEVICE_HIP, "backend stream", &ctx);
  *out = st == Status::kSuccess ? ctx->stream : nullptr;
  return toLc(st);
}
