// device_ops.hpp -- what the entry points on the caller's device tensors share:
// they run on the caller's stream, allocate nothing and synchronise nothing.
#pragma once

#include <string>

#include "kernels.hpp"
#include "ops_internal.hpp"

namespace lchip {

constexpr float kLog2e = 1.4426950408889634f;  // the softmax runs on exp2

// The scope of such a call: the library's device is current inside it and the
// caller's is again afterwards.
class DeviceCall {
 public:
  DeviceCall() = default;
  DeviceCall(const DeviceCall&) = delete;
  DeviceCall& operator=(const DeviceCall&) = delete;
  ~DeviceCall();
  Status open(const char* op, bool trusted);
  // kInvalidValue unless p is memory of the library's device (not asked where
  // the caller vouches for its pointers).  Null passes: the callers have refused
  // it where the tensor has values.
  Status onDevice(const void* p, const char* what) const;
  int device() const { return ctx_->device; }

 private:
  HipContext* ctx_ = nullptr;
  const char* op_ = "";
  bool trusted_ = false;
  int before_ = -1;
};

inline kern::DType dtypeOf(lcDataType t) {
  return t == LC_DTYPE_F32 ? kern::DType::kF32 : t == LC_DTYPE_BF16 ? kern::DType::kBF16 : kern::DType::kF16;
}
inline std::size_t bytesOf(lcDataType t) { return t == LC_DTYPE_F32 ? 4 : 2; }

// A [batch, heads, rows, d] tensor as the kernels take it.  kInvalidValue for a
// null base of a tensor with values, a base off its elements' alignment or a
// negative stride; kNotSupported for a row stride whose tile of 128 rows passes
// 2^31 bytes (the kernels' offsets within a tile).  `written`: also kInvalidValue where two of its rows share memory.
// Clears *aligned unless 16-byte accesses suit it.
Status takeTensor(const char* op, const char* name, const lcDeviceTensor* t, std::size_t batch, std::size_t heads,
                  std::size_t rows, std::size_t d, lcDataType type, bool written, kern::XTensor* out, bool* aligned);

// The workgroups that should share the tiles of one row block, when `blocks` of
// them are there, each has `tiles` and the chip runs `slots` workgroups at once.
// A workgroup's time is its tiles plus `fixed` (its start and its end, in tiles);
// the chip's is that times the rounds of workgroups, and a last round that is
// nearly empty costs as much as a full one.  The join of more than one share
// costs `join` tiles.  At most 32 shares.
int splitCount(std::size_t blocks, std::size_t tiles, std::size_t slots, double fixed, double join);

}  // namespace lchip
