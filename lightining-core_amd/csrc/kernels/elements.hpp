// elements.hpp -- loads, stores and conversions of fp32, bf16 and fp16 rows in
// 16-byte chunks, for kernels that take all three.
#pragma once

#include "kcommon.hpp"

namespace lchip::k {

struct F32 {};

template <typename T>
struct Elem {
  using type = uint16_t;
  static constexpr int kChunk = 8;  // elements of a 16-byte chunk
};
template <>
struct Elem<F32> {
  using type = float;
  static constexpr int kChunk = 4;
};

template <typename T>
__device__ __forceinline__ float to_f32(typename Elem<T>::type v);
template <>
__device__ __forceinline__ float to_f32<F32>(float v) {
  return v;
}
template <>
__device__ __forceinline__ float to_f32<BF16>(uint16_t v) {
  return __builtin_bit_cast(float, static_cast<uint32_t>(v) << 16);
}
template <>
__device__ __forceinline__ float to_f32<F16>(uint16_t v) {
  return static_cast<float>(__builtin_bit_cast(_Float16, v));
}
template <typename T>
__device__ __forceinline__ typename Elem<T>::type from_f32(float v) {
  return to_half_bits<T>(v);
}
template <>
__device__ __forceinline__ float from_f32<F32>(float v) {
  return v;
}

// Value i of a 16-byte chunk.
template <typename T>
__device__ __forceinline__ float chunk_value(u32x4 c, int i) {
  if constexpr (Elem<T>::kChunk == 4) {
    const uint32_t w = c[i];
    return __builtin_bit_cast(float, w);
  } else {
    const uint32_t w = c[i >> 1];
    return to_f32<T>(static_cast<uint16_t>((i & 1) ? w >> 16 : w));
  }
}

__device__ __forceinline__ u32x4 zero_chunk() {
  u32x4 z;
  z[0] = 0;
  z[1] = 0;
  z[2] = 0;
  z[3] = 0;
  return z;
}

// Chunk `chunk` of a row of d values, zero past its end.  VEC: rows are 16-byte
// aligned and d is a whole number of chunks.
template <typename T, bool VEC>
__device__ __forceinline__ u32x4 load_chunk(const typename Elem<T>::type* row, int chunk, int d) {
  constexpr int EC = Elem<T>::kChunk;
  const int at = chunk * EC;
  u32x4 r = zero_chunk();
  if constexpr (VEC) {
    if (at < d) {
      r = *reinterpret_cast<const u32x4*>(row + at);
    }
  } else if (at + EC <= d) {
    // One load all the same: the hardware takes any alignment of an element.
    __builtin_memcpy(&r, __builtin_assume_aligned(row + at, sizeof(*row)), 16);
  } else {
#pragma unroll
    for (int i = 0; i < EC; ++i) {
      if (at + i < d) {
        if constexpr (EC == 4) {
          r[i] = __builtin_bit_cast(uint32_t, row[at + i]);
        } else {
          r[i >> 1] |= static_cast<uint32_t>(row[at + i]) << (16 * (i & 1));
        }
      }
    }
  }
  return r;
}

// The same of an aligned row without a branch around the load, for many chunks
// that are needed at once: past the end it reads the row's first chunk and
// drops it, as it does the whole row when `on` is false.
__device__ __forceinline__ u32x4 load_chunk_flat(const void* row, int at_bytes, int row_bytes, bool on) {
  const bool in = at_bytes < row_bytes;
  const u32x4 v = *reinterpret_cast<const u32x4*>(static_cast<const char*>(row) + (in ? at_bytes : 0));
  u32x4 r;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    r[i] = in && on ? v[i] : 0u;
  }
  return r;
}

// A buffer descriptor of `bytes` bytes from p (wave-uniform): loads at offsets
// past its end return zero.
__device__ __forceinline__ u32x4 buffer_of(const void* p, int bytes) {
  const uint64_t a = reinterpret_cast<uint64_t>(p);
  u32x4 r;
  r[0] = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(a));
  r[1] = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(a >> 32)) & 0xffffu;
  r[2] = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(bytes));
  r[3] = 0x00027000u;
  return r;
}

// 16 bytes of each lane from offset voff of the buffer to LDS at lds + 16 lane;
// zeros where the offset is past the buffer's end.  In asm for the reason given
// at load_lds16_sbase (kcommon.hpp): the compiler's own copies make every later
// LDS wait a full one.  The caller waits with wait_vmcnt.  The s_nop is the five
// wait states that a VMEM read of an SGPR needs after a VALU wrote it (the
// descriptor may come from v_readfirstlane), and the one that an LDS copy needs
// after a write of M0.
__device__ __forceinline__ void load_lds16_buffer(uint32_t voff, u32x4 buffer, uint32_t lds) {
  asm volatile("s_nop 4\n\tbuffer_load_dwordx4 %0, %1, 0 offen lds"
               :
               : "v"(voff), "s"(buffer), "{m0}"(lds)
               : "memory");
}

// v summed over lanes l and l ^ 32.
__device__ __forceinline__ float add_xor32(float v) {
  const uint32_t u = __builtin_bit_cast(uint32_t, v);
  const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  const uint32_t a = r[0];
  const uint32_t b = r[1];
  return __builtin_bit_cast(float, a) + __builtin_bit_cast(float, b);
}

}  // namespace lchip::k
