// cross_attention.hip -- attention of queries of one length over keys and
// values of another, forward and backward, for fp32, bf16 and fp16.
//
// One problem is a (batch row, key/value head) pair: the `group` query heads
// that share the head give R = group * q_len rows, against the row's own
// number of keys.  All three kernels have one shape: a wave owns 32 rows of
// one side (queries for O and dQ, keys for dK and dV), one per MFMA column, and
// the other side streams through LDS in tiles.  Scores are computed with the
// streamed side as MFMA rows, so a lane holds scores of its own row only, and
// the second product takes them from the accumulator registers as its B
// operand; its A operand is the streamed tile read transposed
// (ds_read_b64_tr_b16, which hands a lane four consecutive rows of a column).
//   forward  S^T = K Q^T, O^T += V^T P^T
//   dQ       S^T = K Q^T, dP^T = V dO^T, dQ^T += K^T dS^T
//   dK, dV   S = Q K^T, dP = dO V^T, dV^T += dO^T P, dK^T += Q^T dS
// with P = exp(scale S - lse), dS = P o (dP - delta), delta = rowsum(dO o O).
// The two backward kernels compute the scores twice (14 products of the
// algorithm's 10) so that every gradient has one writer: no atomics, the same
// bits every time.
#include <hip/hip_runtime.h>

#include "../kernels.hpp"
#include "elements.hpp"
#include "kcommon.hpp"

namespace lchip::k {
namespace {

using kern::XAttnArgs;
using kern::XAttnStep;
using kern::XTensor;

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

typedef short s16x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ float fast_exp2(float x) { return __builtin_amdgcn_exp2f(x); }

template <typename T>
__device__ __forceinline__ u32x4 negated(u32x4 v) {
  const uint32_t sign = Elem<T>::kChunk == 4 ? 0x80000000u : 0x80008000u;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[i] ^= sign;
  }
  return v;
}

// acc += A B over one row fragment: 2 * kChunk values of k, of which lane half
// h holds chunk h.
template <typename T>
__device__ __forceinline__ floatx16 mma_rows(u32x4 a, u32x4 b, floatx16 acc) {
  if constexpr (Elem<T>::kChunk == 8) {
    return mfma32x32x16<T>(a, b, acc);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      acc = mfma32x32x2f32(chunk_value<T>(a, i), chunk_value<T>(b, i), acc);
    }
    return acc;
  }
}

// A tile of rows of DP values (d zero padded) in LDS.  16-byte chunk c of row r
// sits at c ^ swz(r): 16 consecutive rows at one chunk, and four consecutive
// rows over 32 columns (the transposed read), each cover all banks once.
template <typename T, int DP>
struct Tile {
  using E = typename Elem<T>::type;
  static constexpr int EC = Elem<T>::kChunk;
  static constexpr int CPR = DP / EC;
  static constexpr int RB = CPR * 16;
  static constexpr int NS = CPR / 2;  // row fragments of a row
  static constexpr int DT = DP / 32;  // 32-column blocks
  static __device__ __forceinline__ int swz(int row) {
    if constexpr (CPR == 8) {
      return (((row >> 1) & 1) << 2) | ((row >> 2) & 3);
    } else {
      return ((row & 3) << 2) | ((row >> 2) & 3);
    }
  }
  static __device__ __forceinline__ int at(int row, int chunk) { return row * RB + ((chunk ^ swz(row)) << 4); }
  // Row fragment s of rows row0 .. row0 + 31 (row0 a multiple of 16).
  static __device__ __forceinline__ u32x4 rows(const char* lds, int row0, int s, int lane) {
    const int r = lane & 31;
    return *reinterpret_cast<const u32x4*>(lds + row0 * RB + at(r, 2 * s + (lane >> 5)));
  }
  // acc[t] += X^T p over the 32 tile rows from row0: column block t of the tile
  // against p, whose register i belongs to row 8 (i / 4) + 4 (lane / 32) + i % 4.
  // 16-bit: pk holds the 32 rows' values packed in that order.
  static __device__ __forceinline__ void transposed(const char* lds, int row0, const u32x4 (&pk)[2], int lane,
                                                    floatx16 (&acc)[DT]) {
    typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
    const int r = 4 * (lane >> 5) + ((lane & 15) >> 2);
    const int c = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
    const int b = (lane & 1) * 8;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
#pragma unroll
      for (int t = 0; t < DT; ++t) {
        const char* p0 = lds + (row0 + 16 * j) * RB + at(r, 4 * t + c) + b;
        const char* p1 = lds + (row0 + 16 * j) * RB + at(r + 8, 4 * t + c) + b;
        const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)p0);
        const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)p1);
        const u32x2 l = __builtin_bit_cast(u32x2, lo);
        const u32x2 h = __builtin_bit_cast(u32x2, hi);
        u32x4 a;
        a[0] = l[0];
        a[1] = l[1];
        a[2] = h[0];
        a[3] = h[1];
        acc[t] = mfma32x32x16<T>(a, pk[j], acc[t]);
      }
    }
  }
  // fp32: p's registers are the B operand as they are.
  static __device__ __forceinline__ void transposed(const char* lds, int row0, const floatx16& p, int lane,
                                                    floatx16 (&acc)[DT]) {
    const int col = lane & 31;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int r = 8 * (i >> 2) + 4 * (lane >> 5) + (i & 3);
#pragma unroll
      for (int t = 0; t < DT; ++t) {
        const float a = *reinterpret_cast<const float*>(lds + row0 * RB + at(r, 8 * t + (col >> 2)) + (col & 3) * 4);
        acc[t] = mfma32x32x2f32(a, p[i], acc[t]);
      }
    }
  }
};

// 16 values (a 32 x 32 block's share of a lane) to 16 bits, in register order.
template <typename T>
__device__ __forceinline__ void pack_block(const floatx16& p, u32x4 (&pk)[2]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    pk[i >> 2][i & 3] = pack2<T>(p[2 * i], p[2 * i + 1]);
  }
}

// Two waves per SIMD, so that one computes probabilities while the other's
// products run; wide fp32 rows and element-wise loads need the registers of one.
template <typename T, int DP, bool VEC>
constexpr int waves_per_simd() {
  return DP == 128 && (Elem<T>::kChunk == 4 || !VEC) ? 1 : 2;
}

// The rows of a [rows, d] matrix with a row stride, moved tile by tile into LDS
// through registers: 256 threads, NL chunks each.  Rows past `rows` and columns
// past d arrive as zeros (a buffer load past its range returns zero), so no
// address past the matrix is ever read and nothing there reaches a product.
// The range is taken anew for each tile, so that 32-bit offsets never span more
// than a tile.  Aligned rows (VEC) are fetched a tile ahead; others, an element
// at a time, as they are needed.
template <typename T, int DP, int KT, bool VEC>
struct Stream {
  using E = typename Elem<T>::type;
  using TL = Tile<T, DP>;
  static constexpr int NL = KT * TL::CPR / 256;
  static constexpr int RPI = 256 / TL::CPR;  // rows between a thread's chunks
  static_assert(NL * 256 == KT * TL::CPR, "tile");
  static constexpr int kOutside = 0x7fffffff;
  u32x4 reg[NL];
  const E* base;
  int64_t stride;
  int rows;
  int d;
  int row;  // this thread's first row and chunk of a tile
  int chunk;
  __device__ __forceinline__ void init(const void* p, int64_t stride_, int rows_, int d_, int tid) {
    base = static_cast<const E*>(p);
    stride = stride_;
    rows = rows_;
    d = d_;
    row = tid / TL::CPR;
    chunk = tid % TL::CPR;
  }
  __device__ __forceinline__ void load(int tile) {
    const E* tp = base + static_cast<int64_t>(tile) * KT * stride;
    const int left = rows - tile * KT;
    const int rb = static_cast<int>(stride) * static_cast<int>(sizeof(E));
    // The last byte a tile may touch: its last row's last value.
    const int bytes = (min(left, KT) - 1) * rb + d * static_cast<int>(sizeof(E));
    auto rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<E*>(tp), 0, bytes, 0x00027000);
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      const int r = row + i * RPI;
      if constexpr (VEC) {
        const int off = (r < left && chunk * TL::EC < d) ? r * rb + chunk * 16 : kOutside;
        reg[i] = __builtin_amdgcn_raw_buffer_load_b128(rsrc, off, 0, 0);
      } else {
        u32x4 v = zero_chunk();
#pragma unroll
        for (int e = 0; e < TL::EC; ++e) {
          const int at = chunk * TL::EC + e;
          const int off = (r < left && at < d) ? r * rb + at * static_cast<int>(sizeof(E)) : kOutside;
          if constexpr (TL::EC == 4) {
            v[e] = __builtin_amdgcn_raw_buffer_load_b32(rsrc, off, 0, 0);
          } else {
            const uint32_t w = __builtin_amdgcn_raw_buffer_load_b16(rsrc, off, 0, 0);
            v[e >> 1] |= w << (16 * (e & 1));
          }
        }
        reg[i] = v;
      }
    }
  }
  __device__ __forceinline__ void store(char* lds) const {
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      *reinterpret_cast<u32x4*>(lds + TL::at(row + i * RPI, chunk)) = reg[i];
    }
  }
};

// Row r of a problem's R = group * q_len query rows: head and position.
struct QueryRow {
  int head;
  int pos;
};
__device__ __forceinline__ QueryRow query_row(int r, int q_len, int first_head) {
  const int g = r / q_len;
  return {first_head + g, r - g * q_len};
}

// This lane's row as MFMA B fragments (column lane % 32, chunks by lane half).
template <typename T, int DP, bool VEC>
__device__ __forceinline__ void load_fragments(const typename Elem<T>::type* row, bool valid, int d, int half,
                                               u32x4 (&f)[Tile<T, DP>::NS]) {
#pragma unroll
  for (int s = 0; s < Tile<T, DP>::NS; ++s) {
    f[s] = valid ? load_chunk<T, VEC>(row, 2 * s + half, d) : zero_chunk();
  }
}

// Four values d0 .. d0 + 3 of a row of d, as they come from an accumulator.
template <typename T, bool VEC>
__device__ __forceinline__ void store4(typename Elem<T>::type* row, int d0, int d, float a, float b, float c,
                                       float e) {
  if constexpr (VEC) {
    if (d0 < d) {
      if constexpr (Elem<T>::kChunk == 4) {
        *reinterpret_cast<float4*>(row + d0) = make_float4(a, b, c, e);
      } else {
        u32x2 w;
        w[0] = pack2<T>(a, b);
        w[1] = pack2<T>(c, e);
        *reinterpret_cast<u32x2*>(row + d0) = w;
      }
    }
  } else {
    const float v[4] = {a, b, c, e};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (d0 + i < d) {
        row[d0 + i] = from_f32<T>(v[i]);
      }
    }
  }
}

// A lane's column of DT 32 x 32 accumulators, times f, to a row of d values.
template <typename T, int DT, bool VEC>
__device__ __forceinline__ void store_column(typename Elem<T>::type* row, int d, int half, const floatx16 (&acc)[DT],
                                             float f) {
#pragma unroll
  for (int t = 0; t < DT; ++t) {
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      store4<T, VEC>(row, t * 32 + 8 * g + 4 * half, d, acc[t][4 * g] * f, acc[t][4 * g + 1] * f,
                     acc[t][4 * g + 2] * f, acc[t][4 * g + 3] * f);
    }
  }
}

// The same to a partial row of DP floats.
template <int DT>
__device__ __forceinline__ void store_partial(float* row, int half, const floatx16 (&acc)[DT], float f) {
#pragma unroll
  for (int t = 0; t < DT; ++t) {
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      *reinterpret_cast<float4*>(row + t * 32 + 8 * g + 4 * half) =
          make_float4(acc[t][4 * g] * f, acc[t][4 * g + 1] * f, acc[t][4 * g + 2] * f, acc[t][4 * g + 3] * f);
    }
  }
}

// The keys of batch row b, held to the padded length whatever the array says.
__device__ __forceinline__ int keys_of(const XAttnArgs& a, int b) {
  return a.lengths == nullptr ? a.kv_len : min(max(a.lengths[b], 0), a.kv_len);
}

// Split z's share of n tiles.
__device__ __forceinline__ void tile_range(int n, int splits, int z, int* first, int* last) {
  const int per = (n + splits - 1) / splits;
  *first = min(n, z * per);
  *last = min(n, *first + per);
}

template <typename T>
constexpr int tile_keys() {
  return Elem<T>::kChunk == 4 ? 32 : 64;
}

// ---------------------------------------------------------------------------
// Forward: grid (problems, 128-row blocks, key splits), four waves of 32 rows.
template <typename T, int DP, bool VEC>
__global__ __launch_bounds__(256, (waves_per_simd<T, DP, VEC>())) void xattn_fwd_kernel(XAttnArgs a) {
  using TL = Tile<T, DP>;
  using E = typename Elem<T>::type;
  constexpr int KT = tile_keys<T>();
  constexpr int NB = KT / 32;
  constexpr int TB = KT * TL::RB;
  extern __shared__ __attribute__((aligned(16))) char smem[];  // K tiles at 0, TB; V tiles at 2 TB, 3 TB
  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int half = lane >> 5;
  const int b = blockIdx.x / a.kv_heads;
  const int hk = blockIdx.x - b * a.kv_heads;
  const int group = a.heads / a.kv_heads;
  const int R = group * a.q_len;
  const int r = blockIdx.y * 128 + (tid >> 6) * 32 + (lane & 31);
  const bool valid = r < R;
  const QueryRow qr = query_row(valid ? r : 0, a.q_len, hk * group);
  const int len = keys_of(a, b);
  int t0, t1;
  tile_range((len + KT - 1) / KT, a.splits, blockIdx.z, &t0, &t1);

  Stream<T, DP, KT, VEC> ks, vs;
  ks.init(static_cast<const E*>(a.k.p) + b * a.k.sb + hk * a.k.sh, a.k.ss, len, a.d, tid);
  vs.init(static_cast<const E*>(a.v.p) + b * a.v.sb + hk * a.v.sh, a.v.ss, len, a.d, tid);
  if (VEC && t0 < t1) {
    ks.load(t0);
    vs.load(t0);
  }
  u32x4 qf[TL::NS];
  load_fragments<T, DP, VEC>(
      static_cast<const E*>(a.q.p) + b * a.q.sb + qr.head * a.q.sh + static_cast<int64_t>(qr.pos) * a.q.ss, valid, a.d,
      half, qf);
  if (a.negate) {
#pragma unroll
    for (int s = 0; s < TL::NS; ++s) {
      qf[s] = negated<T>(qf[s]);
    }
  }
  floatx16 o[TL::DT];
#pragma unroll
  for (int t = 0; t < TL::DT; ++t) {
    o[t] = zero16();
  }
  // Scores and m in exp2 units.  m follows the running maximum lazily: O and l
  // are rescaled only when a tile's maximum passes it by more than 8 (p <= 256).
  float m = -INFINITY;
  float l = 0.0f;
  const float c = a.c;
  for (int t = t0; t < t1; ++t) {
    char* kl = smem + ((t - t0) & 1) * TB;
    char* vl = kl + 2 * TB;
    if (!VEC) {
      ks.load(t);
      vs.load(t);
    }
    ks.store(kl);
    vs.store(vl);
    __syncthreads();
    if (VEC && t + 1 < t1) {
      ks.load(t + 1);
      vs.load(t + 1);
    }
    floatx16 s[NB];
#pragma unroll
    for (int n = 0; n < NB; ++n) {
      s[n] = zero16();
#pragma unroll
      for (int f = 0; f < TL::NS; ++f) {
        s[n] = mma_rows<T>(TL::rows(kl, n * 32, f, lane), qf[f], s[n]);
      }
    }
    float top = -INFINITY;
    if ((t + 1) * KT > len) {
      const int lim = len - t * KT - 4 * half;
#pragma unroll
      for (int n = 0; n < NB; ++n) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          if (n * 32 + 8 * (i >> 2) + (i & 3) >= lim) {
            s[n][i] = -INFINITY;
          }
        }
      }
    }
#pragma unroll
    for (int n = 0; n < NB; ++n) {
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        top = fmaxf(top, s[n][i]);
      }
    }
    top = max_xor32(top) * c;
    if (__any(top > m + 8.0f)) {
      const float next = fmaxf(m, top);
      const float f = m == -INFINITY ? 0.0f : fast_exp2(m - next);
      m = next;
      l *= f;
#pragma unroll
      for (int t2 = 0; t2 < TL::DT; ++t2) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          o[t2][i] *= f;
        }
      }
    }
    const float ref = m == -INFINITY ? 0.0f : m;
#pragma unroll
    for (int n = 0; n < NB; ++n) {
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        s[n][i] = fast_exp2(fmaf(s[n][i], c, -ref));
      }
      if constexpr (TL::EC == 8) {
        // P goes to 16 bits for the matrix cores (an error of half a step per
        // key, averaged over the keys); l sums the rounded values, so the
        // weights of a row still add up to one.
        u32x4 pk[2];
        pack_block<T>(s[n], pk);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          l = add_pair<T>(pk[i >> 2][i & 3], l);
        }
        TL::transposed(vl, n * 32, pk, lane, o);
      } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          l += s[n][i];
        }
        TL::transposed(vl, n * 32, s[n], lane, o);
      }
    }
  }
  l = add_xor32(l);
  if (!valid) {
    return;
  }
  const size_t row = static_cast<size_t>(blockIdx.x) * R + r;
  if (a.splits > 1) {
    const size_t prow = static_cast<size_t>(blockIdx.z) * gridDim.x * R + row;
    store_partial<TL::DT>(a.part + prow * DP, half, o, 1.0f);
    if (half == 0) {
      float* ml = a.stats + prow * 2;
      ml[0] = m;
      ml[1] = l;
    }
    return;
  }
  const float inv = l > 0.0f || l != l ? 1.0f / l : 0.0f;
  store_column<T, TL::DT, VEC>(static_cast<E*>(a.o.p) + b * a.o.sb + qr.head * a.o.sh +
                                   static_cast<int64_t>(qr.pos) * a.o.ss,
                               a.d, half, o, inv);
  if (a.lse != nullptr && half == 0) {
    a.lse[(static_cast<size_t>(b) * a.heads + qr.head) * a.q_len + qr.pos] =
        l > 0.0f || l != l ? m * kLn2 + logf(l) : -INFINITY;
  }
}

// Joins the key splits of the forward: one wave per row, in split order.
template <typename T, int DP>
__global__ __launch_bounds__(256) void xattn_join_kernel(XAttnArgs a) {
  using E = typename Elem<T>::type;
  constexpr int PL = DP / 64;
  const int lane = threadIdx.x & 63;
  const int group = a.heads / a.kv_heads;
  const int R = group * a.q_len;
  const size_t rows = static_cast<size_t>(a.batch) * a.kv_heads * R;
  const size_t row = static_cast<size_t>(blockIdx.x) * 4 + (threadIdx.x >> 6);
  if (row >= rows) {
    return;
  }
  const int problem = static_cast<int>(row / R);
  const int b = problem / a.kv_heads;
  const QueryRow qr = query_row(static_cast<int>(row - static_cast<size_t>(problem) * R), a.q_len,
                                (problem - b * a.kv_heads) * group);
  float m = -INFINITY;
  for (int z = 0; z < a.splits; ++z) {
    m = fmaxf(m, a.stats[(z * rows + row) * 2]);
  }
  float l = 0.0f;
  float o[PL] = {};
  for (int z = 0; z < a.splits; ++z) {
    const float* ml = a.stats + (z * rows + row) * 2;
    const float w = ml[0] == -INFINITY ? 0.0f : fast_exp2(ml[0] - m);
    l = fmaf(w, ml[1], l);
#pragma unroll
    for (int i = 0; i < PL; ++i) {
      o[i] = fmaf(w, a.part[(z * rows + row) * DP + i * 64 + lane], o[i]);
    }
  }
  const bool any = l > 0.0f || l != l;
  const float inv = any ? 1.0f / l : 0.0f;
  E* out = static_cast<E*>(a.o.p) + b * a.o.sb + qr.head * a.o.sh + static_cast<int64_t>(qr.pos) * a.o.ss;
#pragma unroll
  for (int i = 0; i < PL; ++i) {
    if (i * 64 + lane < a.d) {
      out[i * 64 + lane] = from_f32<T>(o[i] * inv);
    }
  }
  if (a.lse != nullptr && lane == 0) {
    a.lse[(static_cast<size_t>(b) * a.heads + qr.head) * a.q_len + qr.pos] = any ? m * kLn2 + logf(l) : -INFINITY;
  }
}

// ---------------------------------------------------------------------------
// fp16 gradients: dS can be far below fp16's range (dO carries no fixed scale,
// and P shares one among thousands of keys), so it is rounded with dO's rows
// scaled by a power of two to a largest value in [1/8, 1/4), and the gradient
// is scaled back at the end.  |dS| <= 2 d / 4 max|V| then stays inside the type
// for values up to 1000.
constexpr int kNoExponent = -126;  // a row of zeros: it sets no scale
__device__ __forceinline__ int exponent_of(float amax) {
  // Infinities and NaN stay what they are at any scale.
  return amax > 0.0f ? (amax < INFINITY ? __builtin_amdgcn_frexp_expf(amax) + 2 : 0) : kNoExponent;
}
__device__ __forceinline__ float power_of_two(int e) { return __builtin_amdgcn_ldexpf(1.0f, e); }

// dQ: as the forward, with dO's rows beside Q's.  Writes each query row's delta
// (and, for fp16, the exponent of its dO) for the dK / dV kernel.
template <typename T, int DP, bool VEC>
__global__ __launch_bounds__(256, (waves_per_simd<T, DP, VEC>())) void xattn_dq_kernel(XAttnArgs a) {
  using TL = Tile<T, DP>;
  using E = typename Elem<T>::type;
  constexpr int KT = tile_keys<T>();
  constexpr int NB = KT / 32;
  constexpr int TB = KT * TL::RB;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int half = lane >> 5;
  const int b = blockIdx.x / a.kv_heads;
  const int hk = blockIdx.x - b * a.kv_heads;
  const int group = a.heads / a.kv_heads;
  const int R = group * a.q_len;
  const int r = blockIdx.y * 128 + (tid >> 6) * 32 + (lane & 31);
  const bool valid = r < R;
  const QueryRow qr = query_row(valid ? r : 0, a.q_len, hk * group);
  const int len = keys_of(a, b);
  int t0, t1;
  tile_range((len + KT - 1) / KT, a.splits, blockIdx.z, &t0, &t1);

  Stream<T, DP, KT, VEC> ks, vs;
  ks.init(static_cast<const E*>(a.k.p) + b * a.k.sb + hk * a.k.sh, a.k.ss, len, a.d, tid);
  vs.init(static_cast<const E*>(a.v.p) + b * a.v.sb + hk * a.v.sh, a.v.ss, len, a.d, tid);
  if (VEC && t0 < t1) {
    ks.load(t0);
    vs.load(t0);
  }
  const int64_t pos = qr.pos;
  u32x4 qf[TL::NS], gf[TL::NS];
  load_fragments<T, DP, VEC>(static_cast<const E*>(a.go.p) + b * a.go.sb + qr.head * a.go.sh + pos * a.go.ss, valid,
                             a.d, half, gf);
  float delta = 0.0f;
  float amax = 0.0f;
  {
    load_fragments<T, DP, VEC>(static_cast<const E*>(a.o.p) + b * a.o.sb + qr.head * a.o.sh + pos * a.o.ss, valid, a.d,
                               half, qf);
#pragma unroll
    for (int s = 0; s < TL::NS; ++s) {
#pragma unroll
      for (int i = 0; i < TL::EC; ++i) {
        const float g = chunk_value<T>(gf[s], i);
        delta = fmaf(g, chunk_value<T>(qf[s], i), delta);
        amax = fmaxf(amax, fabsf(g));
      }
    }
    delta = add_xor32(delta);
    amax = max_xor32(amax);
  }
  load_fragments<T, DP, VEC>(static_cast<const E*>(a.q.p) + b * a.q.sb + qr.head * a.q.sh + pos * a.q.ss, valid, a.d,
                             half, qf);
  if (a.negate) {
#pragma unroll
    for (int s = 0; s < TL::NS; ++s) {
      qf[s] = negated<T>(qf[s]);
    }
  }
  const size_t lrow = (static_cast<size_t>(b) * a.heads + qr.head) * a.q_len + qr.pos;
  const float lse2 = valid ? a.lse[lrow] * kLog2e : 0.0f;
  const int ex = exponent_of(amax);
  if (valid && half == 0 && blockIdx.z == 0) {
    a.delta[2 * lrow] = delta;
    a.delta[2 * lrow + 1] = static_cast<float>(ex);
  }
  float down = 1.0f;
  if constexpr (__is_same(T, F16)) {
    down = power_of_two(-ex);
  }
  floatx16 dq[TL::DT];
#pragma unroll
  for (int t = 0; t < TL::DT; ++t) {
    dq[t] = zero16();
  }
  const float c = a.c;
  for (int t = t0; t < t1; ++t) {
    char* kl = smem + ((t - t0) & 1) * TB;
    char* vl = kl + 2 * TB;
    if (!VEC) {
      ks.load(t);
      vs.load(t);
    }
    ks.store(kl);
    vs.store(vl);
    __syncthreads();
    if (VEC && t + 1 < t1) {
      ks.load(t + 1);
      vs.load(t + 1);
    }
    const int lim = len - t * KT - 4 * half;
    const bool tail = (t + 1) * KT > len;
#pragma unroll
    for (int n = 0; n < NB; ++n) {
      floatx16 s = zero16();
      floatx16 dp = zero16();
#pragma unroll
      for (int f = 0; f < TL::NS; ++f) {
        s = mma_rows<T>(TL::rows(kl, n * 32, f, lane), qf[f], s);
        dp = mma_rows<T>(TL::rows(vl, n * 32, f, lane), gf[f], dp);
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float p = fast_exp2(fmaf(s[i], c, -lse2));
        s[i] = p * (dp[i] - delta) * down;
      }
      if (tail) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          if (n * 32 + 8 * (i >> 2) + (i & 3) >= lim) {
            s[i] = 0.0f;
          }
        }
      }
      if constexpr (TL::EC == 8) {
        u32x4 pk[2];
        pack_block<T>(s, pk);
        TL::transposed(kl, n * 32, pk, lane, dq);
      } else {
        TL::transposed(kl, n * 32, s, lane, dq);
      }
    }
  }
  if (!valid) {
    return;
  }
  // A softmax over one key is constant: its gradient is zero, not the rounding
  // difference between dP and delta.
  float f = len > 1 ? a.scale : 0.0f;
  if constexpr (__is_same(T, F16)) {
    f *= power_of_two(ex);
  }
  if (a.splits > 1) {
    const size_t prow = (static_cast<size_t>(blockIdx.z) * gridDim.x + blockIdx.x) * R + r;
    store_partial<TL::DT>(a.part + prow * DP, half, dq, f);
    return;
  }
  store_column<T, TL::DT, VEC>(static_cast<E*>(a.dq.p) + b * a.dq.sb + qr.head * a.dq.sh + pos * a.dq.ss, a.d, half,
                               dq, f);
}

// dK and dV: grid (problems, 128-key blocks, splits of the query tiles), four
// waves of 32 keys; Q and dO stream.
template <typename T, int DP, bool VEC>
__global__ __launch_bounds__(256, 1) void xattn_dkv_kernel(XAttnArgs a) {
  using TL = Tile<T, DP>;
  using E = typename Elem<T>::type;
  constexpr int KT = tile_keys<T>();
  constexpr int NB = KT / 32;
  constexpr int TB = KT * TL::RB;
  extern __shared__ __attribute__((aligned(16))) char smem[];  // Q, dO tiles, then lse, delta and exponents
  float* const st = reinterpret_cast<float*>(smem + 4 * TB);   // [2][3][KT]
  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int half = lane >> 5;
  const int b = blockIdx.x / a.kv_heads;
  const int hk = blockIdx.x - b * a.kv_heads;
  const int group = a.heads / a.kv_heads;
  const int key = blockIdx.y * 128 + (tid >> 6) * 32 + (lane & 31);
  const int len = keys_of(a, b);
  const bool valid = key < len;
  // Tiles: those of the group's heads, one after the other.
  const int per_head = (a.q_len + KT - 1) / KT;
  int t0, t1;
  tile_range(blockIdx.y * 128 < len ? group * per_head : 0, a.splits, blockIdx.z, &t0, &t1);

  Stream<T, DP, KT, VEC> qs, gs;
  float rl = 0.0f, rd = 0.0f, re = 0.0f;
  auto load = [&](int t) {
    const int g = t / per_head;
    const int tile = t - g * per_head;
    const int head = hk * group + g;
    qs.init(static_cast<const E*>(a.q.p) + b * a.q.sb + head * a.q.sh, a.q.ss, a.q_len, a.d, tid);
    gs.init(static_cast<const E*>(a.go.p) + b * a.go.sb + head * a.go.sh, a.go.ss, a.q_len, a.d, tid);
    qs.load(tile);
    gs.load(tile);
    if (tid < KT) {
      const int pos = tile * KT + tid;
      const bool in = pos < a.q_len;
      const size_t row = (static_cast<size_t>(b) * a.heads + head) * a.q_len + (in ? pos : 0);
      // A row past the end has probabilities of zero.
      rl = in ? a.lse[row] * kLog2e : INFINITY;
      rd = in ? a.delta[2 * row] : 0.0f;
      re = in ? a.delta[2 * row + 1] : kNoExponent;
    }
  };
  if (VEC && t0 < t1) {
    load(t0);
  }
  u32x4 kf[TL::NS], vf[TL::NS];
  const int64_t krow = valid ? key : 0;
  load_fragments<T, DP, VEC>(static_cast<const E*>(a.k.p) + b * a.k.sb + hk * a.k.sh + krow * a.k.ss, valid, a.d, half,
                             kf);
  load_fragments<T, DP, VEC>(static_cast<const E*>(a.v.p) + b * a.v.sb + hk * a.v.sh + krow * a.v.ss, valid, a.d, half,
                             vf);
  if (a.negate) {
#pragma unroll
    for (int s = 0; s < TL::NS; ++s) {
      kf[s] = negated<T>(kf[s]);
    }
  }
  floatx16 dk[TL::DT], dv[TL::DT];
#pragma unroll
  for (int t = 0; t < TL::DT; ++t) {
    dk[t] = zero16();
    dv[t] = zero16();
  }
  int ex = kNoExponent;  // fp16: dk is held at 2^-ex
  const float c = a.c;
  for (int t = t0; t < t1; ++t) {
    const int buf = (t - t0) & 1;
    char* ql = smem + buf * TB;
    char* gl = ql + 2 * TB;
    float* sl = st + buf * 3 * KT;
    if (!VEC) {
      load(t);
    }
    qs.store(ql);
    gs.store(gl);
    if (tid < KT) {
      sl[tid] = rl;
      sl[KT + tid] = rd;
      sl[2 * KT + tid] = re;
    }
    __syncthreads();
    if (VEC && t + 1 < t1) {
      load(t + 1);
    }
    float down = 1.0f;
    if constexpr (__is_same(T, F16)) {
      float e = lane < KT ? sl[2 * KT + lane] : kNoExponent;
#pragma unroll
      for (int x = 32; x > 0; x >>= 1) {
        e = fmaxf(e, __shfl_xor(e, x));
      }
      const int et = __builtin_amdgcn_readfirstlane(static_cast<int>(e));
      if (et > ex) {
        const float f = power_of_two(ex - et);
        ex = et;
#pragma unroll
        for (int t2 = 0; t2 < TL::DT; ++t2) {
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            dk[t2][i] *= f;
          }
        }
      }
      down = power_of_two(-ex);
    }
#pragma unroll
    for (int n = 0; n < NB; ++n) {
      floatx16 s = zero16();
      floatx16 dp = zero16();
#pragma unroll
      for (int f = 0; f < TL::NS; ++f) {
        s = mma_rows<T>(TL::rows(ql, n * 32, f, lane), kf[f], s);
        dp = mma_rows<T>(TL::rows(gl, n * 32, f, lane), vf[f], dp);
      }
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int r0 = n * 32 + 8 * g + 4 * half;
        const float4 l4 = *reinterpret_cast<const float4*>(sl + r0);
        const float4 d4 = *reinterpret_cast<const float4*>(sl + KT + r0);
        const float lv[4] = {l4.x, l4.y, l4.z, l4.w};
        const float dl[4] = {d4.x, d4.y, d4.z, d4.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float p = fast_exp2(fmaf(s[4 * g + i], c, -lv[i]));
          s[4 * g + i] = p;
          dp[4 * g + i] = p * (dp[4 * g + i] - dl[i]) * down;
        }
      }
      if constexpr (TL::EC == 8) {
        u32x4 pk[2];
        pack_block<T>(s, pk);
        TL::transposed(gl, n * 32, pk, lane, dv);
        pack_block<T>(dp, pk);
        TL::transposed(ql, n * 32, pk, lane, dk);
      } else {
        TL::transposed(gl, n * 32, s, lane, dv);
        TL::transposed(ql, n * 32, dp, lane, dk);
      }
    }
  }
  if (key >= a.kv_len) {
    return;
  }
  // Keys past the row's length have gradients of zero.
  float fk = valid && len > 1 ? a.scale : 0.0f;
  const float fv = valid ? 1.0f : 0.0f;
  if constexpr (__is_same(T, F16)) {
    fk *= power_of_two(ex);
  }
  if (!valid) {
#pragma unroll
    for (int t = 0; t < TL::DT; ++t) {
      dk[t] = zero16();
      dv[t] = zero16();
    }
  }
  if (a.splits > 1) {
    const size_t plane = static_cast<size_t>(gridDim.x) * a.kv_len;
    const size_t prow = static_cast<size_t>(blockIdx.z) * 2 * plane + static_cast<size_t>(blockIdx.x) * a.kv_len + key;
    store_partial<TL::DT>(a.part + prow * DP, half, dk, fk);
    store_partial<TL::DT>(a.part + (prow + plane) * DP, half, dv, fv);
    return;
  }
  const int64_t at = key;
  store_column<T, TL::DT, VEC>(static_cast<E*>(a.dk.p) + b * a.dk.sb + hk * a.dk.sh + at * a.dk.ss, a.d, half, dk, fk);
  store_column<T, TL::DT, VEC>(static_cast<E*>(a.dv.p) + b * a.dv.sb + hk * a.dv.sh + at * a.dv.ss, a.d, half, dv, fv);
}

// Sums the splits' partial rows [splits][planes][rows][DP] in split order into
// strided [batch, heads, len, d] tensors, one per plane: a wave per row.
template <typename T, int DP>
__global__ __launch_bounds__(256) void xattn_sum_kernel(const float* __restrict__ part, XTensor first, XTensor second,
                                                        int planes, int splits, int batch, int heads, int len, int d) {
  using E = typename Elem<T>::type;
  constexpr int PL = DP / 64;
  const int lane = threadIdx.x & 63;
  const size_t rows = static_cast<size_t>(batch) * heads * len;
  const size_t row = static_cast<size_t>(blockIdx.x) * 4 + (threadIdx.x >> 6);
  if (row >= rows) {
    return;
  }
  const int problem = static_cast<int>(row / len);
  const int64_t pos = static_cast<int64_t>(row - static_cast<size_t>(problem) * len);
  const int b = problem / heads;
  const XTensor x = blockIdx.y == 0 ? first : second;
  float s[PL] = {};
  for (int z = 0; z < splits; ++z) {
    const float* p = part + ((static_cast<size_t>(z) * planes + blockIdx.y) * rows + row) * DP + lane;
#pragma unroll
    for (int i = 0; i < PL; ++i) {
      s[i] += p[i * 64];
    }
  }
  E* out = static_cast<E*>(x.p) + b * x.sb + (problem - b * heads) * x.sh + pos * x.ss;
#pragma unroll
  for (int i = 0; i < PL; ++i) {
    if (i * 64 + lane < d) {
      out[i * 64 + lane] = from_f32<T>(s[i]);
    }
  }
}

template <typename T, int DP>
constexpr size_t tiles_bytes() {
  return 4u * tile_keys<T>() * Tile<T, DP>::RB;
}

// A launch with `lds` bytes of dynamic LDS, which a kernel has to be allowed
// once.
template <typename K>
hipError_t launch_lds(K kernel, hipError_t allowed, dim3 grid, size_t lds, const XAttnArgs& a, hipStream_t stream) {
  if (allowed != hipSuccess) {
    return allowed;
  }
  kernel<<<grid, 256, lds, stream>>>(a);
  return hipGetLastError();
}
#define LC_XATTN_ALLOW(kernel, lds)                                                                   \
  hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, \
                      static_cast<int>(lds))

template <typename T, int DP, bool VEC>
hipError_t launch(XAttnStep step, const XAttnArgs& a, hipStream_t stream) {
  const unsigned problems = static_cast<unsigned>(a.batch * a.kv_heads);
  const int rows = a.heads / a.kv_heads * a.q_len;
  const unsigned z = static_cast<unsigned>(a.splits);
  constexpr size_t lds = tiles_bytes<T, DP>();
  const dim3 by_rows(problems, static_cast<unsigned>((rows + 127) / 128), z);
  if (step == XAttnStep::kForward) {
    static const hipError_t allowed = LC_XATTN_ALLOW((xattn_fwd_kernel<T, DP, VEC>), lds);
    return launch_lds(xattn_fwd_kernel<T, DP, VEC>, allowed, by_rows, lds, a, stream);
  }
  if (step == XAttnStep::kGradQ) {
    static const hipError_t allowed = LC_XATTN_ALLOW((xattn_dq_kernel<T, DP, VEC>), lds);
    return launch_lds(xattn_dq_kernel<T, DP, VEC>, allowed, by_rows, lds, a, stream);
  }
  constexpr size_t more = lds + 6 * tile_keys<T>() * sizeof(float);
  static const hipError_t allowed = LC_XATTN_ALLOW((xattn_dkv_kernel<T, DP, VEC>), more);
  return launch_lds(xattn_dkv_kernel<T, DP, VEC>, allowed, dim3(problems, static_cast<unsigned>((a.kv_len + 127) / 128), z),
                    more, a, stream);
}
#undef LC_XATTN_ALLOW

template <typename T>
hipError_t launch_type(XAttnStep step, const XAttnArgs& a, bool vec, hipStream_t stream) {
  if (a.d <= 64) {
    return vec ? launch<T, 64, true>(step, a, stream) : launch<T, 64, false>(step, a, stream);
  }
  return vec ? launch<T, 128, true>(step, a, stream) : launch<T, 128, false>(step, a, stream);
}

template <typename T>
hipError_t join_type(const XAttnArgs& a, hipStream_t stream) {
  const size_t rows = static_cast<size_t>(a.batch) * a.heads * a.q_len;
  const dim3 grid(static_cast<unsigned>((rows + 3) / 4));
  if (a.d <= 64) {
    xattn_join_kernel<T, 64><<<grid, 256, 0, stream>>>(a);
  } else {
    xattn_join_kernel<T, 128><<<grid, 256, 0, stream>>>(a);
  }
  return hipGetLastError();
}

template <typename T>
hipError_t sum_type(const float* part, const XTensor& x, const XTensor* second, int splits, int batch, int heads,
                    int len, int d, hipStream_t stream) {
  const size_t rows = static_cast<size_t>(batch) * heads * len;
  const int planes = second != nullptr ? 2 : 1;
  const dim3 grid(static_cast<unsigned>((rows + 3) / 4), planes);
  const XTensor& y = second != nullptr ? *second : x;
  if (d <= 64) {
    xattn_sum_kernel<T, 64><<<grid, 256, 0, stream>>>(part, x, y, planes, splits, batch, heads, len, d);
  } else {
    xattn_sum_kernel<T, 128><<<grid, 256, 0, stream>>>(part, x, y, planes, splits, batch, heads, len, d);
  }
  return hipGetLastError();
}

}  // namespace
}  // namespace lchip::k

namespace lchip::kern {

hipError_t crossAttention(XAttnStep step, const XAttnArgs& a, DType type, bool aligned, hipStream_t stream) {
  switch (type) {
    case DType::kF32:
      return k::launch_type<k::F32>(step, a, aligned, stream);
    case DType::kBF16:
      return k::launch_type<k::BF16>(step, a, aligned, stream);
    default:
      return k::launch_type<k::F16>(step, a, aligned, stream);
  }
}

hipError_t crossAttentionJoin(const XAttnArgs& a, DType type, hipStream_t stream) {
  switch (type) {
    case DType::kF32:
      return k::join_type<k::F32>(a, stream);
    case DType::kBF16:
      return k::join_type<k::BF16>(a, stream);
    default:
      return k::join_type<k::F16>(a, stream);
  }
}

hipError_t crossAttentionSum(const float* part, const XTensor& x, const XTensor* second, int splits, int batch,
                             int heads, int len, int d, DType type, hipStream_t stream) {
  switch (type) {
    case DType::kF32:
      return k::sum_type<k::F32>(part, x, second, splits, batch, heads, len, d, stream);
    case DType::kBF16:
      return k::sum_type<k::BF16>(part, x, second, splits, batch, heads, len, d, stream);
    default:
      return k::sum_type<k::F16>(part, x, second, splits, batch, heads, len, d, stream);
  }
}

}  // namespace lchip::kern
