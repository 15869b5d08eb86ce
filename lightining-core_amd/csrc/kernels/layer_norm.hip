// layer_norm.hip -- layer norm of rows of n values and its gradients.
//   y = (x - mu) r w + b,  mu = mean(x),  r = 1 / sqrt(mean((x - mu)^2) + eps)
//   dx = r (g - mean(g) - h mean(g h)),  g = dy w,  h = (x - mu) r
//   dw = sum over rows of dy h,  db = sum over rows of dy
// Both directions are bound by memory: x (and dy) are read once and held in
// registers, in fp32 statistics over the deviations from the mean (a second
// pass over registers, not a difference of large sums).  The sum of x rounds, so
// that mean misses by an amount that goes with |mean| and not with the row's
// spread; the deviations' own sum, taken beside their squares', puts it right: a
// constant row has that very mean and a variance of zero.  LANES threads share a
// row (16, a wave, or a workgroup), each with CH chunks of 16 bytes; they walk
// rows with the weights in registers.  Rows too wide for that are read again
// from the caches.  dw and db are summed per thread over the rows of its
// columns, then over workgroups in a fixed order: no atomics.
#include <hip/hip_runtime.h>

#include "../kernels.hpp"
#include "elements.hpp"
#include "kcommon.hpp"

namespace lchip::k {
namespace {

using kern::LayerNormArgs;

constexpr int kThreads = 256;

// v summed over the LANES threads of a row, in one order for all of them.
// `slot`: LDS of the workgroup's waves, a different one for consecutive calls.
template <int LANES>
__device__ __forceinline__ float row_sum(float v, float* slot) {
  constexpr int W = LANES < 64 ? LANES : 64;
#pragma unroll
  for (int x = W / 2; x > 0; x >>= 1) {
    v += __shfl_xor(v, x);
  }
  if constexpr (LANES > 64) {
    if ((threadIdx.x & 63) == 0) {
      slot[threadIdx.x >> 6] = v;
    }
    __syncthreads();
    v = 0.0f;
#pragma unroll
    for (int w = 0; w < LANES / 64; ++w) {
      v += slot[w];
    }
  }
  return v;
}

// The same for two sums at once.
template <int LANES>
__device__ __forceinline__ void row_sums(float& v, float& u, float* slot_v, float* slot_u) {
  constexpr int W = LANES < 64 ? LANES : 64;
#pragma unroll
  for (int x = W / 2; x > 0; x >>= 1) {
    v += __shfl_xor(v, x);
    u += __shfl_xor(u, x);
  }
  if constexpr (LANES > 64) {
    if ((threadIdx.x & 63) == 0) {
      slot_v[threadIdx.x >> 6] = v;
      slot_u[threadIdx.x >> 6] = u;
    }
    __syncthreads();
    v = 0.0f;
    u = 0.0f;
#pragma unroll
    for (int w = 0; w < LANES / 64; ++w) {
      v += slot_v[w];
      u += slot_u[w];
    }
  }
}

// mean, and deviations d from it with their sum and their squares' sum: how far
// the deviations' mean is from zero.  Returns 1 / sqrt(var + eps).
__device__ __forceinline__ float put_right(float sum, float squares, float n, float eps, float& mean, float& off) {
  off = sum / n;
  mean += off;
  const float var = fmaf(-off, off, squares / n);
  return 1.0f / sqrtf((var < 0.0f ? 0.0f : var) + eps);
}

// Value i of the weights, which are in x's type or fp32.
template <typename T>
__device__ __forceinline__ float weight_at(const void* w, int wide, int i) {
  return wide ? static_cast<const float*>(w)[i] : to_f32<T>(static_cast<const typename Elem<T>::type*>(w)[i]);
}
// Chunk `chunk` of the weights (as many as x's chunk holds), `none` where there
// are none; zeros past their end.
template <typename T, bool VEC>
__device__ __forceinline__ void load_weights(const void* w, const LayerNormArgs& a, int chunk, float none,
                                             float (&v)[Elem<T>::kChunk]) {
  constexpr int EC = Elem<T>::kChunk;
  const int at = chunk * EC;
#pragma unroll
  for (int i = 0; i < EC; ++i) {
    v[i] = at + i < a.n ? none : 0.0f;
  }
  if (w == nullptr || at >= a.n) {
    return;
  }
  if (VEC && a.weights_aligned) {
    if (a.wide) {
#pragma unroll
      for (int j = 0; j < EC / 4; ++j) {
        const float4 f = *reinterpret_cast<const float4*>(static_cast<const float*>(w) + at + 4 * j);
        v[4 * j] = f.x;
        v[4 * j + 1] = f.y;
        v[4 * j + 2] = f.z;
        v[4 * j + 3] = f.w;
      }
    } else {
      const u32x4 c = *reinterpret_cast<const u32x4*>(static_cast<const typename Elem<T>::type*>(w) + at);
#pragma unroll
      for (int i = 0; i < EC; ++i) {
        v[i] = chunk_value<T>(c, i);
      }
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < EC; ++i) {
    if (at + i < a.n) {
      v[i] = weight_at<T>(w, a.wide, at + i);
    }
  }
}
template <typename T>
__device__ __forceinline__ void put_weight(void* w, int wide, int i, float v) {
  if (wide) {
    static_cast<float*>(w)[i] = v;
  } else {
    static_cast<typename Elem<T>::type*>(w)[i] = from_f32<T>(v);
  }
}

// A chunk of values to a row of n, in x's type.
template <typename T, bool VEC>
__device__ __forceinline__ void store_chunk(typename Elem<T>::type* row, int chunk, int n,
                                            const float (&v)[Elem<T>::kChunk]) {
  constexpr int EC = Elem<T>::kChunk;
  const int at = chunk * EC;
  if (at + EC <= n) {
    u32x4 c;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (EC == 4) {
        c[i] = __builtin_bit_cast(uint32_t, v[i]);
      } else {
        c[i] = pack2<T>(v[2 * i], v[2 * i + 1]);
      }
    }
    if constexpr (VEC) {
      *reinterpret_cast<u32x4*>(row + at) = c;
    } else {
      __builtin_memcpy(__builtin_assume_aligned(row + at, sizeof(*row)), &c, 16);
    }
  } else if constexpr (!VEC) {
#pragma unroll
    for (int i = 0; i < EC; ++i) {
      if (at + i < n) {
        row[at + i] = from_f32<T>(v[i]);
      }
    }
  }
}

template <typename T, bool VEC, int LANES, int CH>
__global__ __launch_bounds__(kThreads) void ln_fwd_kernel(LayerNormArgs a) {
  using E = typename Elem<T>::type;
  constexpr int EC = Elem<T>::kChunk;
  constexpr int RPB = kThreads / LANES;  // rows of a workgroup at a time
  __shared__ float sums[6][kThreads / 64];
  const int lane = threadIdx.x % LANES;
  const int64_t step = static_cast<int64_t>(gridDim.x) * RPB;
  float w[CH][EC], bias[CH][EC];
  const float n = static_cast<float>(a.n);
  int flip = 0;
  // All threads of a workgroup make the same number of rounds (barriers).
  int64_t row = static_cast<int64_t>(blockIdx.x) * RPB + threadIdx.x / LANES;
  const int64_t rounds = (a.rows - static_cast<int64_t>(blockIdx.x) * RPB + step - 1) / step;
  const E* const x0 = static_cast<const E*>(a.x);
  u32x4 raw[CH];
  auto fetch = [&](int64_t r) {
    const E* xr = x0 + (r < a.rows ? r : 0) * a.sx;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      raw[c] = load_chunk<T, VEC>(xr, c * LANES + lane, a.n);
    }
  };
  fetch(row);
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    load_weights<T, VEC>(a.w, a, c * LANES + lane, 1.0f, w[c]);
    load_weights<T, VEC>(a.b, a, c * LANES + lane, 0.0f, bias[c]);
  }
  for (int64_t k = 0; k < rounds; ++k, row += step) {
    float x[CH][EC];
    float s = 0.0f;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
#pragma unroll
      for (int i = 0; i < EC; ++i) {
        x[c][i] = chunk_value<T>(raw[c], i);
        s += x[c][i];
      }
    }
    if (k + 1 < rounds) {
      fetch(row + step);
    }
    float mean = row_sum<LANES>(s, sums[flip]) / n;
    s = 0.0f;
    float s1 = 0.0f;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
#pragma unroll
      for (int i = 0; i < EC; ++i) {
        x[c][i] = (c * LANES + lane) * EC + i < a.n ? x[c][i] - mean : 0.0f;
        s1 += x[c][i];
        s = fmaf(x[c][i], x[c][i], s);
      }
    }
    row_sums<LANES>(s, s1, sums[flip + 1], sums[flip + 2]);
    float off;
    const float rstd = put_right(s1, s, n, a.eps, mean, off);
    flip ^= 3;
    if (row < a.rows) {
      E* yr = static_cast<E*>(a.y) + row * a.sy;
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        float y[EC];
#pragma unroll
        for (int i = 0; i < EC; ++i) {
          y[i] = fmaf((x[c][i] - off) * rstd, w[c][i], bias[c][i]);
        }
        store_chunk<T, VEC>(yr, c * LANES + lane, a.n, y);
      }
      if (lane == 0 && a.mean != nullptr) {
        a.mean[row] = mean;
        a.rstd[row] = rstd;
      }
    }
  }
}

// Rows of any width: a workgroup a row, x read three times (twice from cache).
template <typename T, bool VEC>
__global__ __launch_bounds__(kThreads) void ln_fwd_wide_kernel(LayerNormArgs a) {
  using E = typename Elem<T>::type;
  constexpr int EC = Elem<T>::kChunk;
  __shared__ float sums[3][kThreads / 64];
  const float n = static_cast<float>(a.n);
  const int chunks = (a.n + EC - 1) / EC;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const E* xr = static_cast<const E*>(a.x) + row * a.sx;
    E* yr = static_cast<E*>(a.y) + row * a.sy;
    float s = 0.0f;
    for (int c = threadIdx.x; c < chunks; c += kThreads) {
      const u32x4 v = load_chunk<T, VEC>(xr, c, a.n);
#pragma unroll
      for (int i = 0; i < EC; ++i) {
        s += chunk_value<T>(v, i);
      }
    }
    __syncthreads();
    const float first = row_sum<kThreads>(s, sums[0]) / n;
    s = 0.0f;
    float s1 = 0.0f;
    for (int c = threadIdx.x; c < chunks; c += kThreads) {
      const u32x4 v = load_chunk<T, VEC>(xr, c, a.n);
#pragma unroll
      for (int i = 0; i < EC; ++i) {
        const float d = c * EC + i < a.n ? chunk_value<T>(v, i) - first : 0.0f;
        s1 += d;
        s = fmaf(d, d, s);
      }
    }
    row_sums<kThreads>(s, s1, sums[1], sums[2]);
    float mean = first, off;
    const float rstd = put_right(s1, s, n, a.eps, mean, off);
    for (int c = threadIdx.x; c < chunks; c += kThreads) {
      const u32x4 v = load_chunk<T, VEC>(xr, c, a.n);
      float y[EC];
#pragma unroll
      for (int i = 0; i < EC; ++i) {
        const int at = c * EC + i;
        const float w = a.w != nullptr && at < a.n ? weight_at<T>(a.w, a.wide, at) : 1.0f;
        const float b = a.b != nullptr && at < a.n ? weight_at<T>(a.b, a.wide, at) : 0.0f;
        y[i] = fmaf((chunk_value<T>(v, i) - first - off) * rstd, w, b);
      }
      store_chunk<T, VEC>(yr, c, a.n, y);
    }
    if (threadIdx.x == 0 && a.mean != nullptr) {
      a.mean[row] = mean;
      a.rstd[row] = rstd;
    }
  }
}

// dx, and each workgroup's share of dw and db in part [gridDim.x][2][n].
template <typename T, bool VEC, int LANES, int CH>
__global__ __launch_bounds__(kThreads) void ln_bwd_kernel(LayerNormArgs a) {
  using E = typename Elem<T>::type;
  constexpr int EC = Elem<T>::kChunk;
  constexpr int RPB = kThreads / LANES;
  __shared__ float sums[4][kThreads / 64];
  // Columns of the workgroup's row groups, joined at the end.
  __shared__ float cols[RPB > 1 ? RPB : 1][RPB > 1 ? LANES * EC : 1];
  const int lane = threadIdx.x % LANES;
  const int group = threadIdx.x / LANES;
  const int64_t step = static_cast<int64_t>(gridDim.x) * RPB;
  float w[CH][EC], dw[CH][EC], db[CH][EC];
#pragma unroll
  for (int c = 0; c < CH; ++c) {
#pragma unroll
    for (int i = 0; i < EC; ++i) {
      dw[c][i] = 0.0f;
      db[c][i] = 0.0f;
    }
  }
  const float n = static_cast<float>(a.n);
  int flip = 0;
  int64_t row = static_cast<int64_t>(blockIdx.x) * RPB + group;
  const int64_t rounds = (a.rows - static_cast<int64_t>(blockIdx.x) * RPB + step - 1) / step;
  u32x4 xr[CH], gr[CH];
  float mean = 0.0f, rstd = 0.0f;
  auto fetch = [&](int64_t r) {
    const int64_t at = r < a.rows ? r : 0;
    const E* xp = static_cast<const E*>(a.x) + at * a.sx;
    const E* gp = static_cast<const E*>(a.dy) + at * a.sy;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      xr[c] = load_chunk<T, VEC>(xp, c * LANES + lane, a.n);
      gr[c] = load_chunk<T, VEC>(gp, c * LANES + lane, a.n);
    }
    mean = a.mean[at];
    rstd = a.rstd[at];
  };
  fetch(row);
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    load_weights<T, VEC>(a.w, a, c * LANES + lane, 1.0f, w[c]);
  }
  for (int64_t k = 0; k < rounds; ++k, row += step) {
    const bool in = row < a.rows;
    const float mu = mean;
    const float r = rstd;
    float h[CH][EC], g[CH][EC];
    float s0 = 0.0f, s1 = 0.0f;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
#pragma unroll
      for (int i = 0; i < EC; ++i) {
        const bool on = in && (c * LANES + lane) * EC + i < a.n;
        const float dy = on ? chunk_value<T>(gr[c], i) : 0.0f;
        h[c][i] = on ? (chunk_value<T>(xr[c], i) - mu) * r : 0.0f;
        dw[c][i] = fmaf(dy, h[c][i], dw[c][i]);
        db[c][i] += dy;
        g[c][i] = dy * w[c][i];
        s0 += g[c][i];
        s1 = fmaf(g[c][i], h[c][i], s1);
      }
    }
    if (k + 1 < rounds) {
      fetch(row + step);
    }
    const float m0 = row_sum<LANES>(s0, sums[flip]) / n;
    const float m1 = row_sum<LANES>(s1, sums[flip + 1]) / n;
    flip ^= 2;
    if (in) {
      E* dxr = static_cast<E*>(a.dx) + row * a.sdx;
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        float d[EC];
#pragma unroll
        for (int i = 0; i < EC; ++i) {
          d[i] = r * (g[c][i] - m0 - h[c][i] * m1);
        }
        store_chunk<T, VEC>(dxr, c * LANES + lane, a.n, d);
      }
    }
  }
  float* const out = a.part + static_cast<size_t>(blockIdx.x) * 2 * a.n;
#pragma unroll
  for (int which = 0; which < 2; ++which) {
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      if constexpr (RPB > 1) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < EC; ++i) {
          cols[group][lane * EC + i] = which == 0 ? dw[c][i] : db[c][i];
        }
        __syncthreads();
        for (int j = threadIdx.x; j < LANES * EC; j += kThreads) {
          const int at = c * LANES * EC + j;
          if (at < a.n) {
            float v = 0.0f;
#pragma unroll
            for (int q = 0; q < RPB; ++q) {
              v += cols[q][j];
            }
            out[static_cast<size_t>(which) * a.n + at] = v;
          }
        }
      } else {
#pragma unroll
        for (int i = 0; i < EC; ++i) {
          const int at = (c * LANES + lane) * EC + i;
          if (at < a.n) {
            out[static_cast<size_t>(which) * a.n + at] = which == 0 ? dw[c][i] : db[c][i];
          }
        }
      }
    }
  }
}

template <typename T, bool VEC>
__global__ __launch_bounds__(kThreads) void ln_bwd_wide_kernel(LayerNormArgs a) {
  using E = typename Elem<T>::type;
  constexpr int EC = Elem<T>::kChunk;
  __shared__ float sums[2][kThreads / 64];
  const float n = static_cast<float>(a.n);
  const int chunks = (a.n + EC - 1) / EC;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const E* xr = static_cast<const E*>(a.x) + row * a.sx;
    const E* gr = static_cast<const E*>(a.dy) + row * a.sy;
    E* dxr = static_cast<E*>(a.dx) + row * a.sdx;
    const float mu = a.mean[row];
    const float r = a.rstd[row];
    float s0 = 0.0f, s1 = 0.0f;
    for (int c = threadIdx.x; c < chunks; c += kThreads) {
      const u32x4 xv = load_chunk<T, VEC>(xr, c, a.n);
      const u32x4 gv = load_chunk<T, VEC>(gr, c, a.n);
#pragma unroll
      for (int i = 0; i < EC; ++i) {
        if (c * EC + i < a.n) {
          const float w = a.w != nullptr ? weight_at<T>(a.w, a.wide, c * EC + i) : 1.0f;
          const float g = chunk_value<T>(gv, i) * w;
          s0 += g;
          s1 = fmaf(g, (chunk_value<T>(xv, i) - mu) * r, s1);
        }
      }
    }
    __syncthreads();
    const float m0 = row_sum<kThreads>(s0, sums[0]) / n;
    const float m1 = row_sum<kThreads>(s1, sums[1]) / n;
    for (int c = threadIdx.x; c < chunks; c += kThreads) {
      const u32x4 xv = load_chunk<T, VEC>(xr, c, a.n);
      const u32x4 gv = load_chunk<T, VEC>(gr, c, a.n);
      float d[EC];
#pragma unroll
      for (int i = 0; i < EC; ++i) {
        const int at = c * EC + i;
        const float w = a.w != nullptr && at < a.n ? weight_at<T>(a.w, a.wide, at) : 1.0f;
        d[i] = r * (chunk_value<T>(gv, i) * w - m0 - (chunk_value<T>(xv, i) - mu) * r * m1);
      }
      store_chunk<T, VEC>(dxr, c, a.n, d);
    }
  }
}

// Wide rows' dw and db: grid (column blocks, row slabs), part [gridDim.y][2][n].
template <typename T, bool VEC>
__global__ __launch_bounds__(kThreads) void ln_cols_wide_kernel(LayerNormArgs a) {
  using E = typename Elem<T>::type;
  constexpr int EC = Elem<T>::kChunk;
  const int chunk = blockIdx.x * kThreads + threadIdx.x;
  if (chunk * EC >= a.n) {
    return;
  }
  const int64_t per = (a.rows + gridDim.y - 1) / gridDim.y;
  const int64_t first = blockIdx.y * per;
  const int64_t last = min(first + per, a.rows);
  float dw[EC] = {}, db[EC] = {};
  for (int64_t row = first; row < last; ++row) {
    const u32x4 xv = load_chunk<T, VEC>(static_cast<const E*>(a.x) + row * a.sx, chunk, a.n);
    const u32x4 gv = load_chunk<T, VEC>(static_cast<const E*>(a.dy) + row * a.sy, chunk, a.n);
    const float mu = a.mean[row];
    const float r = a.rstd[row];
#pragma unroll
    for (int i = 0; i < EC; ++i) {
      const float g = chunk_value<T>(gv, i);
      dw[i] = fmaf(g, (chunk_value<T>(xv, i) - mu) * r, dw[i]);
      db[i] += g;
    }
  }
  float* const out = a.part + static_cast<size_t>(blockIdx.y) * 2 * a.n;
#pragma unroll
  for (int i = 0; i < EC; ++i) {
    const int at = chunk * EC + i;
    if (at < a.n) {
      out[at] = dw[i];
      out[static_cast<size_t>(a.n) + at] = db[i];
    }
  }
}

// dw and db from the partial sums [parts][2][n]: 64 columns a workgroup, 16
// threads a column, each over every 16th part, then in thread order.
template <typename T>
__global__ __launch_bounds__(1024) void ln_cols_kernel(LayerNormArgs a, int parts) {
  __shared__ float s[16][64];
  const int col = threadIdx.x & 63;
  const int k = threadIdx.x >> 6;
  const int at = blockIdx.x * 64 + col;
  float v = 0.0f;
  if (at < a.n) {
    const float* p = a.part + static_cast<size_t>(blockIdx.y) * a.n + at;
#pragma unroll 8
    for (int i = k; i < parts; i += 16) {
      v += p[static_cast<size_t>(i) * 2 * a.n];
    }
  }
  s[k][col] = v;
  __syncthreads();
  if (k == 0 && at < a.n) {
    v = s[0][col];
#pragma unroll
    for (int i = 1; i < 16; ++i) {
      v += s[i][col];
    }
    void* const out = blockIdx.y == 0 ? a.dw : a.db;
    if (out != nullptr) {
      put_weight<T>(out, a.wide, at, v);
    }
  }
}

// Values of a row that a thread keeps in registers at most.
constexpr int kHeld = 32;

template <typename T, bool VEC>
hipError_t launch(const LayerNormArgs& a, bool backward, hipStream_t stream) {
  constexpr int EC = Elem<T>::kChunk;
  const unsigned groups = static_cast<unsigned>(kern::layerNormGroups(a.rows, a.n, backward, EC));
#define LC_LN(LANES, CH)                                                              \
  do {                                                                                \
    if (backward) {                                                                   \
      ln_bwd_kernel<T, VEC, LANES, CH><<<groups, kThreads, 0, stream>>>(a);           \
    } else {                                                                          \
      ln_fwd_kernel<T, VEC, LANES, CH><<<groups, kThreads, 0, stream>>>(a);           \
    }                                                                                 \
  } while (0)
#define LC_LN_CH(LANES)                       \
  do {                                        \
    const int ch = (a.n + LANES * EC - 1) / (LANES * EC); \
    if (ch <= 1) {                            \
      LC_LN(LANES, 1);                        \
    } else if (ch <= 2) {                     \
      LC_LN(LANES, 2);                        \
    } else if (ch <= 4) {                     \
      LC_LN(LANES, 4);                        \
    } else if constexpr (EC == 4) {           \
      LC_LN(LANES, 8);                        \
    }                                         \
  } while (0)
  // No rows: nothing but the sums' zeros is left to write.
  switch (a.rows == 0 ? -1 : kern::layerNormLanes(a.rows, a.n, EC)) {
    case -1:
      break;
    case 16:
      LC_LN_CH(16);
      break;
    case 64:
      LC_LN_CH(64);
      break;
    case 256:
      LC_LN_CH(256);
      break;
    default:
      if (backward) {
        ln_bwd_wide_kernel<T, VEC>
            <<<static_cast<unsigned>(a.rows < 2048 ? a.rows : 2048), kThreads, 0, stream>>>(a);
        const unsigned blocks = static_cast<unsigned>((a.n + kThreads * EC - 1) / (kThreads * EC));
        ln_cols_wide_kernel<T, VEC><<<dim3(blocks, groups), kThreads, 0, stream>>>(a);
      } else {
        ln_fwd_wide_kernel<T, VEC><<<groups, kThreads, 0, stream>>>(a);
      }
  }
#undef LC_LN_CH
#undef LC_LN
  hipError_t e = hipGetLastError();
  if (e == hipSuccess && backward && (a.dw != nullptr || a.db != nullptr)) {
    ln_cols_kernel<T><<<dim3(static_cast<unsigned>((a.n + 63) / 64), 2), 1024, 0, stream>>>(a, static_cast<int>(groups));
    e = hipGetLastError();
  }
  return e;
}

template <typename T>
hipError_t launch_type(const LayerNormArgs& a, bool backward, bool aligned, hipStream_t stream) {
  return aligned ? launch<T, true>(a, backward, stream) : launch<T, false>(a, backward, stream);
}

}  // namespace
}  // namespace lchip::k

namespace lchip::kern {

// Threads that share a row (0: rows too wide to be held in registers).  A wave
// reads 64 chunks at once; fewer lanes for rows that would leave most of it
// idle, a workgroup where a wave's registers do not hold the row or too few
// rows are there to fill the chip with one wave each.
int layerNormLanes(int64_t rows, int n, int chunk) {
  if (n > 256 * k::kHeld) {
    return 0;
  }
  if (n <= 16 * 2 * chunk) {
    return 16;
  }
  if (n > 64 * k::kHeld || (rows < 1024 && n > 64 * 2 * chunk)) {
    return 256;
  }
  return 64;
}

// Workgroups of a launch; for the backward pass also the partial sums of each
// column.
int layerNormGroups(int64_t rows, int n, bool backward, int chunk) {
  const int lanes = layerNormLanes(rows, n, chunk);
  const int64_t per = lanes == 0 ? 1 : k::kThreads / lanes;
  int64_t most = backward ? 512 : 2048;
  if (backward && lanes == 0) {
    most = 32;
  }
  const int64_t want = (rows + per - 1) / per;
  return static_cast<int>(want < most ? want : most);
}

hipError_t layerNorm(const LayerNormArgs& a, DType type, bool backward, bool aligned, hipStream_t stream) {
  switch (type) {
    case DType::kF32:
      return k::launch_type<k::F32>(a, backward, aligned, stream);
    case DType::kBF16:
      return k::launch_type<k::BF16>(a, backward, aligned, stream);
    default:
      return k::launch_type<k::F16>(a, backward, aligned, stream);
  }
}

}  // namespace lchip::kern
