// cross_attention.hip -- attention of queries of one length over keys and
// values of another, forward and backward, for fp32, bf16 and fp16.
//
// One problem is a (batch row, key/value head) pair: the `group` query heads
// that share the head give R = group * q_len rows, against the row's own
// number of keys.  All three parts have one shape: a wave owns 32 rows of
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
// The backward pass computes the scores twice (14 products of the algorithm's
// 10) so that every gradient has one writer: no atomics, the same bits every
// time.  dQ and dK / dV are different workgroups of one launch, so that the one
// fills the chip where the other has too few.
#include <hip/hip_runtime.h>

#include "../kernels.hpp"
#include "elements.hpp"
#include "kcommon.hpp"

namespace lchip::k {
namespace {

using kern::XAttnArgs;
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

// The rows of a [rows, d] matrix with a row stride, moved into LDS tile by tile
// by NW waves.  Rows past `rows` and columns past d arrive as zeros (a buffer
// load past its range returns zero), so no address past the matrix is ever read
// and nothing there reaches a product.  The range is taken anew for each tile,
// so that 32-bit offsets never span more than a tile.  Aligned rows (VEC) are
// copied by the LDS DMA, 1 KB an instruction: it fills LDS in lane order, so the
// swizzle is made by choosing which chunk a lane fetches.  Other rows go through
// registers, an element at a time.
template <typename T, int DP, int KT, bool VEC, int NW>
struct Stream {
  using E = typename Elem<T>::type;
  using TL = Tile<T, DP>;
  static constexpr int kCopies = KT * TL::RB / 1024;  // of the whole tile
  static constexpr int NI = kCopies / NW;             // of one wave
  static constexpr int RPI = 64 / TL::CPR;            // rows of a copy
  static_assert(NI * NW == kCopies, "tile");
  static constexpr int kOutside = 0x7fffffff;
  const E* base;
  int64_t stride;
  int rows;
  int d;
  int lane;
  int wave;
  int off[VEC ? NI : 1];  // byte offsets of this lane's chunks in a tile
  __device__ __forceinline__ void init(const void* p, int64_t stride_, int rows_, int d_, int wave_, int lane_) {
    base = static_cast<const E*>(p);
    stride = stride_;
    rows = rows_;
    d = d_;
    lane = lane_;
    wave = wave_;
    if constexpr (VEC) {
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        const int r = row_of(i);
        const int c = (lane % TL::CPR) ^ TL::swz(r);
        off[i] = c * TL::EC < d ? r * static_cast<int>(stride) * static_cast<int>(sizeof(E)) + c * 16 : kOutside;
      }
    }
  }
  // Another matrix of the same strides and lengths.
  __device__ __forceinline__ void rebase(const void* p) { base = static_cast<const E*>(p); }
  // The row of a tile that this lane's copy i holds a chunk of.
  __device__ __forceinline__ int row_of(int i) const { return (wave + NW * i) * RPI + lane / TL::CPR; }
  // Starts moving tile `tile` to lds (16-byte aligned).
  __device__ __forceinline__ void stage(int tile, char* lds) const {
    const E* tp = base + static_cast<int64_t>(tile) * KT * stride;
    const int left = rows - tile * KT;
    const int rb = static_cast<int>(stride) * static_cast<int>(sizeof(E));
    // The last byte a tile may touch: its last row's last value.
    const int bytes = (min(left, KT) - 1) * rb + d * static_cast<int>(sizeof(E));
    if constexpr (VEC) {
      const u32x4 buffer = buffer_of(tp, bytes);
      const uint32_t to = lds_addr(lds) + static_cast<uint32_t>(wave) * 1024u;
      if (left >= KT) {
#pragma unroll
        for (int i = 0; i < NI; ++i) {
          load_lds16_buffer(static_cast<uint32_t>(off[i]), buffer, to + i * (NW * 1024u));
        }
      } else {
#pragma unroll
        for (int i = 0; i < NI; ++i) {
          load_lds16_buffer(static_cast<uint32_t>(row_of(i) < left ? off[i] : kOutside), buffer,
                            to + i * (NW * 1024u));
        }
      }
    } else {
      auto rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<E*>(tp), 0, bytes, 0x00027000);
#pragma unroll 1
      for (int i = 0; i < NI; ++i) {
        const int r = row_of(i);
        const int chunk = lane % TL::CPR;
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
        *reinterpret_cast<u32x4*>(lds + TL::at(r, chunk)) = v;
      }
    }
  }
};

// This wave's LDS reads so far have returned (the empty asm keeps the compiler
// from moving one behind the wait): what they read may be overwritten.
__device__ __forceinline__ void reads_done() {
  asm volatile("" ::: "memory");
  wait_lgkmcnt<0>();
}

// Everything staged before has arrived, for every wave, and every wave is done
// reading what it read before.
__device__ __forceinline__ void arrive() {
  reads_done();
  wait_vmcnt<0>();
  stage_barrier();
}

// Row r of a problem's R = group * q_len query rows: head and position.
struct QueryRow {
  int head;
  int pos;
};
__device__ __forceinline__ QueryRow query_row(int r, int q_len, int first_head) {
  const int g = r / q_len;
  return {first_head + g, r - g * q_len};
}

// A row as MFMA B fragments (column lane % 32, chunks by lane half); a row that
// is not valid may be read and counts as zeros.
template <typename T, int DP, bool VEC>
__device__ __forceinline__ void load_fragments(const typename Elem<T>::type* row, bool valid, int d, int half,
                                               u32x4 (&f)[Tile<T, DP>::NS]) {
#pragma unroll
  for (int s = 0; s < Tile<T, DP>::NS; ++s) {
    if constexpr (VEC) {
      f[s] = load_chunk_flat(row, (2 * s + half) * 16, d * static_cast<int>(sizeof(typename Elem<T>::type)), valid);
    } else {
      f[s] = load_chunk<T, VEC>(row, 2 * s + half, valid ? d : 0);
    }
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

// Two waves per SIMD, so that one computes probabilities while the other's
// products run; wide fp32 rows and element-wise loads need the registers of one.
template <typename T, int DP, bool VEC>
constexpr int waves_per_simd() {
  return DP == 128 && (Elem<T>::kChunk == 4 || !VEC) ? 1 : 2;
}

// The softmax state of a wave's 32 query rows (one a lane, in both lane halves)
// over tiles of KT keys.  Scores and m in exp2 units.  m follows the running
// maximum lazily: O and l are rescaled only when a tile's maximum passes it by
// more than 8 (probabilities up to 256).  fp16: m is 7 below the maximum it was
// taken from, so that P, which goes to fp16, lies between 2^7 and 2^15 at its
// largest and is normal down to 2^-21 of that: a tail of very many keys far
// below the maximum, whose values count together, keeps its bits.
template <typename T, int DP, int KT>
struct FwdState {
  using TL = Tile<T, DP>;
  static constexpr int NB = KT / 32;
  static constexpr float kBelow = __is_same(T, F16) ? 7.0f : 0.0f;
  u32x4 qf[TL::NS];
  floatx16 o[TL::DT];
  float m;
  float l;
  float c;
  int len;
  int lane;

  __device__ __forceinline__ void init(float c_, int len_, int lane_) {
    c = c_;
    len = len_;
    lane = lane_;
    m = -INFINITY;
    l = 0.0f;
#pragma unroll
    for (int t = 0; t < TL::DT; ++t) {
      o[t] = zero16();
    }
  }
  __device__ __forceinline__ void scores(const char* kl, floatx16 (&s)[NB]) const {
#pragma unroll
    for (int n = 0; n < NB; ++n) {
      s[n] = zero16();
#pragma unroll
      for (int f = 0; f < TL::NS; ++f) {
        s[n] = mma_rows<T>(TL::rows(kl, n * 32, f, lane), qf[f], s[n]);
      }
    }
  }
  // Hides the keys past the row's length and moves m; returns what to subtract.
  __device__ __forceinline__ float reference(int t, floatx16 (&s)[NB]) {
    if ((t + 1) * KT > len) {
      const int lim = len - t * KT - 4 * (lane >> 5);
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
    float top = -INFINITY;
#pragma unroll
    for (int n = 0; n < NB; ++n) {
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        top = fmaxf(top, s[n][i]);
      }
    }
    top = fmaf(max_xor32(top), c, -kBelow);
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
    return m == -INFINITY ? 0.0f : m;
  }
  // Probabilities of a tile, in place; l sums them unrounded.
  __device__ __forceinline__ void probabilities(floatx16 (&s)[NB], float ref) {
#pragma unroll
    for (int n = 0; n < NB; ++n) {
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        s[n][i] = fast_exp2(fmaf(s[n][i], c, -ref));
        l += s[n][i];
      }
    }
  }
  // O += P V.  P goes to 16 bits for the matrix cores (an error of half a step a
  // key, averaged over the keys).
  __device__ __forceinline__ void values(const char* vl, const floatx16 (&s)[NB]) {
#pragma unroll
    for (int n = 0; n < NB; ++n) {
      if constexpr (TL::EC == 8) {
        u32x4 pk[2];
        pack_block<T>(s[n], pk);
        TL::transposed(vl, n * 32, pk, lane, o);
      } else {
        TL::transposed(vl, n * 32, s[n], lane, o);
      }
    }
  }
  // The same two with the next tile's scores between the exponentials: a product
  // runs for 32 cycles while the wave issues the exponentials behind it (the
  // scheduling barriers keep that order).
  __device__ __forceinline__ void probabilities_and_scores(floatx16 (&s)[NB], float ref, const char* kn,
                                                           floatx16 (&next)[NB]) {
    constexpr int NQ = NB * TL::NS;
    constexpr int EPM = NB * 16 / NQ;
    u32x4 kf[3];
    kf[0] = TL::rows(kn, 0, 0, lane);
    kf[1] = TL::rows(kn, 1 / TL::NS * 32, 1 % TL::NS, lane);
#pragma unroll
    for (int g = 0; g < NQ; ++g) {
      if (g + 2 < NQ) {
        kf[(g + 2) % 3] = TL::rows(kn, (g + 2) / TL::NS * 32, (g + 2) % TL::NS, lane);
      }
      const int n = g / TL::NS;
      const int f = g % TL::NS;
      next[n] = mma_rows<T>(kf[g % 3], qf[f], f == 0 ? zero16() : next[n]);
#pragma unroll
      for (int e = 0; e < EPM; ++e) {
        const int idx = g * EPM + e;
        const float p = fast_exp2(fmaf(s[idx >> 4][idx & 15], c, -ref));
        s[idx >> 4][idx & 15] = p;
        l += p;
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  }
};

// A row's result from its unnormalised o, m and l.
__device__ __forceinline__ bool any_keys(float l) { return l > 0.0f || l != l; }

// Forward: grid (problems, 128-row blocks, key splits), four waves of 32 rows.
// K runs two tiles ahead of the probabilities, V one.
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
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int half = lane >> 5;
  const int b = blockIdx.x / a.kv_heads;
  const int hk = blockIdx.x - b * a.kv_heads;
  const int group = a.heads / a.kv_heads;
  const int R = group * a.q_len;
  const int r = blockIdx.y * 128 + wave * 32 + (lane & 31);
  const bool valid = r < R;
  const QueryRow qr = query_row(valid ? r : 0, a.q_len, hk * group);
  const int len = keys_of(a, b);
  int t0, t1;
  tile_range((len + KT - 1) / KT, a.splits, blockIdx.z, &t0, &t1);

  Stream<T, DP, KT, VEC, 4> ks, vs;
  ks.init(static_cast<const E*>(a.k.p) + b * a.k.sb + hk * a.k.sh, a.k.ss, len, a.d, wave, lane);
  vs.init(static_cast<const E*>(a.v.p) + b * a.v.sb + hk * a.v.sh, a.v.ss, len, a.d, wave, lane);
  if (t0 < t1) {
    ks.stage(t0, smem);
    vs.stage(t0, smem + 2 * TB);
    if (t0 + 1 < t1) {
      ks.stage(t0 + 1, smem + TB);
    }
  }
  FwdState<T, DP, KT> w;
  w.init(a.c, len, lane);
  load_fragments<T, DP, VEC>(
      static_cast<const E*>(a.q.p) + b * a.q.sb + qr.head * a.q.sh + static_cast<int64_t>(qr.pos) * a.q.ss, valid, a.d,
      half, w.qf);
  if (a.negate) {
#pragma unroll
    for (int s = 0; s < TL::NS; ++s) {
      w.qf[s] = negated<T>(w.qf[s]);
    }
  }
  floatx16 sa[NB], sb[NB];
  if (t0 < t1) {
    arrive();
    w.scores(smem, sa);
    arrive();  // K buffer 0 is filled again next
  }
  auto step = [&](int t, floatx16 (&cur)[NB], floatx16 (&next)[NB]) {
    const int at = (t - t0) & 1;
    if (t + 2 < t1) {
      ks.stage(t + 2, smem + at * TB);
    }
    if (t + 1 < t1) {
      vs.stage(t + 1, smem + (3 - at) * TB);
    }
    const float ref = w.reference(t, cur);
    // Past the last tile the scores are of a stale tile and go unused.
    w.probabilities_and_scores(cur, ref, smem + (1 - at) * TB, next);
    // The products of one wave go before the other wave's exponentials (2048 x
    // 4096 keys, 64 heads of 128: 254 -> 244 us).
    __builtin_amdgcn_s_setprio(1);
    w.values(smem + (2 + at) * TB, cur);
    __builtin_amdgcn_s_setprio(0);
    arrive();
  };
  for (int t = t0; t < t1; t += 2) {
    step(t, sa, sb);
    if (t + 1 < t1) {
      step(t + 1, sb, sa);
    }
  }
  const float l = add_xor32(w.l);
  if (!valid) {
    return;
  }
  const size_t row = static_cast<size_t>(blockIdx.x) * R + r;
  if (a.splits > 1) {
    const size_t prow = static_cast<size_t>(blockIdx.z) * gridDim.x * R + row;
    store_partial<TL::DT>(a.part + prow * DP, half, w.o, 1.0f);
    if (half == 0) {
      float* ml = a.stats + prow * 2;
      ml[0] = w.m;
      ml[1] = l;
    }
    return;
  }
  const float inv = any_keys(l) ? 1.0f / l : 0.0f;
  store_column<T, TL::DT, VEC>(static_cast<E*>(a.o.p) + b * a.o.sb + qr.head * a.o.sh +
                                   static_cast<int64_t>(qr.pos) * a.o.ss,
                               a.d, half, w.o, inv);
  if (a.lse != nullptr && half == 0) {
    a.lse[(static_cast<size_t>(b) * a.heads + qr.head) * a.q_len + qr.pos] =
        any_keys(l) ? w.m * kLn2 + logf(l) : -INFINITY;
  }
}

// Forward of few rows: grid (problems, 32-row blocks, key splits).  The four
// waves have the same 32 rows and take the split's tiles in turn, each with
// tiles of its own in LDS and no barrier until their states are joined; K's
// buffer is filled again as soon as the scores have read it, V's after O.
template <typename T, int DP, bool VEC>
__global__ __launch_bounds__(256, 1) void xattn_few_kernel(XAttnArgs a) {
  using TL = Tile<T, DP>;
  using E = typename Elem<T>::type;
  constexpr int KT = tile_keys<T>();
  constexpr int NB = KT / 32;
  constexpr int TB = KT * TL::RB;
  constexpr int SW = DP + 4;  // floats of a row of O in LDS
  using St = Stream<T, DP, KT, VEC, 1>;
  static_assert(4 * 32 * (SW + 2) * sizeof(float) <= 8u * TB, "the states fit where the tiles were");
  extern __shared__ __attribute__((aligned(16))) char smem[];  // four waves' K and V tiles, then their states
  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int half = lane >> 5;
  const int b = blockIdx.x / a.kv_heads;
  const int hk = blockIdx.x - b * a.kv_heads;
  const int group = a.heads / a.kv_heads;
  const int R = group * a.q_len;
  const int r = blockIdx.y * 32 + (lane & 31);
  const bool valid = r < R;
  const QueryRow qr = query_row(valid ? r : 0, a.q_len, hk * group);
  const int len = keys_of(a, b);
  int t0, t1;
  tile_range((len + KT - 1) / KT, a.splits, blockIdx.z, &t0, &t1);
  char* const kl = smem + wave * 2 * TB;
  char* const vl = kl + TB;

  St ks, vs;
  ks.init(static_cast<const E*>(a.k.p) + b * a.k.sb + hk * a.k.sh, a.k.ss, len, a.d, 0, lane);
  vs.init(static_cast<const E*>(a.v.p) + b * a.v.sb + hk * a.v.sh, a.v.ss, len, a.d, 0, lane);
  FwdState<T, DP, KT> w;
  w.init(a.c, len, lane);
  load_fragments<T, DP, VEC>(
      static_cast<const E*>(a.q.p) + b * a.q.sb + qr.head * a.q.sh + static_cast<int64_t>(qr.pos) * a.q.ss, valid, a.d,
      half, w.qf);
  if (a.negate) {
#pragma unroll
    for (int s = 0; s < TL::NS; ++s) {
      w.qf[s] = negated<T>(w.qf[s]);
    }
  }
  int t = t0 + wave;
  if (t < t1) {
    ks.stage(t, kl);
    vs.stage(t, vl);
  }
  for (; t < t1; t += 4) {
    // V's copies are the younger ones.
    wait_vmcnt<VEC ? St::NI : 0>();
    asm volatile("" ::: "memory");
    floatx16 s[NB];
    w.scores(kl, s);
    reads_done();
    const bool more = t + 4 < t1;
    if (more) {
      ks.stage(t + 4, kl);
    }
    const float ref = w.reference(t, s);
    w.probabilities(s, ref);
    if (more) {
      wait_vmcnt<VEC ? St::NI : 0>();
    } else {
      wait_vmcnt<0>();
    }
    asm volatile("" ::: "memory");
    w.values(vl, s);
    reads_done();
    if (more) {
      vs.stage(t + 4, vl);
    }
  }
  const float lw = add_xor32(w.l);
  __syncthreads();
  float* const so = reinterpret_cast<float*>(smem);
  float* const sm = so + 4 * 32 * SW;  // [wave][m or l][row]
  store_partial<TL::DT>(so + (wave * 32 + (lane & 31)) * SW, half, w.o, 1.0f);
  if (half == 0) {
    sm[wave * 64 + lane] = w.m;
    sm[wave * 64 + 32 + lane] = lw;
  }
  __syncthreads();
  // Eight threads a row join the waves' states.
  const int row = tid >> 3;
  const int d0 = (tid & 7) * 4;
  const int r1 = blockIdx.y * 32 + row;
  if (r1 >= R) {
    return;
  }
  float m = -INFINITY;
#pragma unroll
  for (int x = 0; x < 4; ++x) {
    m = fmaxf(m, sm[x * 64 + row]);
  }
  float l = 0.0f;
  float f[4];
#pragma unroll
  for (int x = 0; x < 4; ++x) {
    const float mx = sm[x * 64 + row];
    f[x] = mx == -INFINITY ? 0.0f : fast_exp2(mx - m);
    l = fmaf(f[x], sm[x * 64 + 32 + row], l);
  }
  const QueryRow q1 = query_row(r1, a.q_len, hk * group);
  const size_t prow = (static_cast<size_t>(blockIdx.z) * gridDim.x + blockIdx.x) * R + r1;
  const float inv = a.splits > 1 ? 1.0f : any_keys(l) ? 1.0f / l : 0.0f;
  E* const out = static_cast<E*>(a.o.p) + b * a.o.sb + q1.head * a.o.sh + static_cast<int64_t>(q1.pos) * a.o.ss;
#pragma unroll
  for (int j = 0; j < TL::DT; ++j) {
    float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const float4 p = *reinterpret_cast<const float4*>(so + (x * 32 + row) * SW + j * 32 + d0);
      v[0] = fmaf(f[x], p.x, v[0]);
      v[1] = fmaf(f[x], p.y, v[1]);
      v[2] = fmaf(f[x], p.z, v[2]);
      v[3] = fmaf(f[x], p.w, v[3]);
    }
    if (a.splits > 1) {
      *reinterpret_cast<float4*>(a.part + prow * DP + j * 32 + d0) = make_float4(v[0], v[1], v[2], v[3]);
    } else {
      store4<T, VEC>(out, j * 32 + d0, a.d, v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv);
    }
  }
  if ((tid & 7) != 0) {
    return;
  }
  if (a.splits > 1) {
    a.stats[prow * 2] = m;
    a.stats[prow * 2 + 1] = l;
  } else if (a.lse != nullptr) {
    a.lse[(static_cast<size_t>(b) * a.heads + q1.head) * a.q_len + q1.pos] =
        any_keys(l) ? m * kLn2 + logf(l) : -INFINITY;
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
#pragma unroll 4
  for (int z = 0; z < a.splits; ++z) {
    m = fmaxf(m, a.stats[(z * rows + row) * 2]);
  }
  float l = 0.0f;
  float o[PL] = {};
#pragma unroll 4
  for (int z = 0; z < a.splits; ++z) {
    const float* ml = a.stats + (z * rows + row) * 2;
    const float w = ml[0] == -INFINITY ? 0.0f : fast_exp2(ml[0] - m);
    l = fmaf(w, ml[1], l);
#pragma unroll
    for (int i = 0; i < PL; ++i) {
      o[i] = fmaf(w, a.part[(z * rows + row) * DP + i * 64 + lane], o[i]);
    }
  }
  const bool any = any_keys(l);
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
// fp16 gradients: dS goes to fp16 for the matrix cores, and nothing bounds it
// on either side (dO carries no fixed scale, V may be large, and P shares one
// among thousands of keys).  dQ's accumulators belong to one query row a lane
// and dK's to one key, so each lane holds its own at a power of two, 2^e, of the
// true gradient: the first block's largest |dS| of the row or key comes to
// [2^7, 2^8), and e falls when a later one would pass 2^15.  What the largest
// value so far leaves normal reaches down to 2^-21 of it.  (A scale from dO
// alone lets dS overflow for large V: two keys of 20000 and 0, 128 columns.)
// 64 heads of 2048 x 1500 x 128: the pass takes 411 us, in bf16, without this, 368.
struct Lift {
  int e = 126;               // nothing seen: values below 2^-111 pass as they are
  float up = 0x1p126f;       // 2^e
  float most = 0x1p-111f;    // 2^(15 - e)
  // ds *= 2^e for the lane's e, after `acc` has followed e.  `on`: the lane's
  // column is one whose gradient is kept.
  template <int DT>
  __device__ __forceinline__ void apply(floatx16& ds, bool on, floatx16 (&acc)[DT]) {
    float top = 0.0f;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      top = fmaxf(top, fabsf(ds[i]));
    }
    top = max_xor32(top);
    top = on ? top : 0.0f;
    if (__any(top >= most)) {
      const int next = top >= most ? 8 - __builtin_amdgcn_frexp_expf(top) : e;
      const float f = __builtin_amdgcn_ldexpf(1.0f, next - e);
      e = next;
      up = __builtin_amdgcn_ldexpf(1.0f, e);
      most = __builtin_amdgcn_ldexpf(1.0f, 15 - e);
#pragma unroll
      for (int t = 0; t < DT; ++t) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          acc[t][i] *= f;
        }
      }
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      ds[i] *= up;
    }
  }
  // 2^-e, by which the gradient is scaled back.
  __device__ __forceinline__ float down() const { return __builtin_amdgcn_ldexpf(1.0f, -e); }
};

// The statistics of ROWS query rows (block `blk`): delta = dO . O and lse in exp2
// units, 16 threads a row.  All loads are issued before the first is used: few
// workgroups run at once beside the LDS that short rows need.
template <typename T, bool VEC, int ROWS>
__device__ __forceinline__ void delta_rows(const XAttnArgs& a, int blk) {
  using E = typename Elem<T>::type;
  constexpr int EC = Elem<T>::kChunk;
  constexpr int N = ROWS / 16;
  constexpr int NC = kern::kXAttnMaxDim / (16 * EC);
  const int b = blockIdx.x / a.kv_heads;
  const int hk = blockIdx.x - b * a.kv_heads;
  const int group = a.heads / a.kv_heads;
  const int R = group * a.q_len;
  const int r0 = blk * ROWS + static_cast<int>(threadIdx.x >> 4);
  u32x4 gv[N][NC], ov[N][NC];
  size_t row[N];
  float lse[N];
#pragma unroll
  for (int n = 0; n < N; ++n) {
    const bool in = r0 + 16 * n < R;
    const QueryRow qr = query_row(in ? r0 + 16 * n : 0, a.q_len, hk * group);
    const int64_t pos = qr.pos;
    const E* g = static_cast<const E*>(a.go.p) + b * a.go.sb + qr.head * a.go.sh + pos * a.go.ss;
    const E* o = static_cast<const E*>(a.o.p) + b * a.o.sb + qr.head * a.o.sh + pos * a.o.ss;
    row[n] = (static_cast<size_t>(b) * a.heads + qr.head) * a.q_len + qr.pos;
#pragma unroll
    for (int j = 0; j < NC; ++j) {
      const int c = (threadIdx.x & 15) + 16 * j;
      if constexpr (VEC) {
        gv[n][j] = load_chunk_flat(g, c * 16, a.d * static_cast<int>(sizeof(E)), in);
        ov[n][j] = load_chunk_flat(o, c * 16, a.d * static_cast<int>(sizeof(E)), in);
      } else {
        gv[n][j] = load_chunk<T, VEC>(g, c, a.d);
        ov[n][j] = load_chunk<T, VEC>(o, c, a.d);
      }
    }
    lse[n] = a.lse[row[n]];
  }
#pragma unroll
  for (int n = 0; n < N; ++n) {
    float delta = 0.0f;
#pragma unroll
    for (int j = 0; j < NC; ++j) {
#pragma unroll
      for (int i = 0; i < EC; ++i) {
        delta = fmaf(chunk_value<T>(gv[n][j], i), chunk_value<T>(ov[n][j], i), delta);
      }
    }
#pragma unroll
    for (int x = 8; x > 0; x >>= 1) {
      delta += __shfl_xor(delta, x);
    }
    if ((threadIdx.x & 15) == 0 && r0 + 16 * n < R) {
      *reinterpret_cast<float2*>(a.delta + 2 * row[n]) = make_float2(delta, lse[n] * kLog2e);
    }
  }
}

// dQ of 128 rows (block `blk`) over share z of the keys: as the forward, with
// dO's rows beside Q's.  DELTA: the rows' delta = sum over the keys of P dP
// instead (of all keys, splits_q being ignored).
template <typename T, int DP, bool VEC, bool DELTA>
__device__ __forceinline__ void dq_part(const XAttnArgs& a, char* smem, int blk, int z) {
  using TL = Tile<T, DP>;
  using E = typename Elem<T>::type;
  constexpr int KT = tile_keys<T>();
  constexpr int NB = KT / 32;
  constexpr int TB = KT * TL::RB;
  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int half = lane >> 5;
  const int b = blockIdx.x / a.kv_heads;
  const int hk = blockIdx.x - b * a.kv_heads;
  const int group = a.heads / a.kv_heads;
  const int R = group * a.q_len;
  const int r = blk * 128 + wave * 32 + (lane & 31);
  const bool valid = r < R;
  const QueryRow qr = query_row(valid ? r : 0, a.q_len, hk * group);
  const int len = keys_of(a, b);
  int t0, t1;
  tile_range((len + KT - 1) / KT, DELTA ? 1 : a.splits_q, z, &t0, &t1);

  Stream<T, DP, KT, VEC, 4> ks, vs;
  ks.init(static_cast<const E*>(a.k.p) + b * a.k.sb + hk * a.k.sh, a.k.ss, len, a.d, wave, lane);
  vs.init(static_cast<const E*>(a.v.p) + b * a.v.sb + hk * a.v.sh, a.v.ss, len, a.d, wave, lane);
  if (t0 < t1) {
    ks.stage(t0, smem);
    vs.stage(t0, smem + 2 * TB);
  }
  const int64_t pos = qr.pos;
  u32x4 qf[TL::NS], gf[TL::NS];
  load_fragments<T, DP, VEC>(static_cast<const E*>(a.go.p) + b * a.go.sb + qr.head * a.go.sh + pos * a.go.ss, valid,
                             a.d, half, gf);
  load_fragments<T, DP, VEC>(static_cast<const E*>(a.q.p) + b * a.q.sb + qr.head * a.q.sh + pos * a.q.ss, valid, a.d,
                             half, qf);
  if (a.negate) {
#pragma unroll
    for (int s = 0; s < TL::NS; ++s) {
      qf[s] = negated<T>(qf[s]);
    }
  }
  const size_t lrow = (static_cast<size_t>(b) * a.heads + qr.head) * a.q_len + qr.pos;
  float2 st = make_float2(0.0f, 0.0f);
  if (valid) {
    if constexpr (DELTA) {
      st.y = a.lse[lrow] * kLog2e;
    } else {
      st = *reinterpret_cast<const float2*>(a.delta + 2 * lrow);
    }
  }
  const float delta = st.x;
  const float lse2 = st.y;
  Lift lift;  // fp16
  float sum = 0.0f;
  floatx16 dq[TL::DT];
#pragma unroll
  for (int t = 0; t < TL::DT; ++t) {
    dq[t] = zero16();
  }
  const float c = a.c;
  if (t0 < t1) {
    arrive();
  }
  for (int t = t0; t < t1; ++t) {
    const int at = (t - t0) & 1;
    const char* kl = smem + at * TB;
    const char* vl = kl + 2 * TB;
    if (t + 1 < t1) {
      ks.stage(t + 1, smem + (1 - at) * TB);
      vs.stage(t + 1, smem + (3 - at) * TB);
    }
    const int lim = len - t * KT - 4 * half;
    const bool tail = (t + 1) * KT > len;
#pragma unroll 1
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
        s[i] = DELTA ? p * dp[i] : p * (dp[i] - delta);
      }
      if (tail) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          if (n * 32 + 8 * (i >> 2) + (i & 3) >= lim) {
            s[i] = 0.0f;
          }
        }
      }
      if constexpr (DELTA) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          sum += s[i];
        }
      } else if constexpr (TL::EC == 8) {
        if constexpr (__is_same(T, F16)) {
          lift.apply(s, valid, dq);
        }
        u32x4 pk[2];
        pack_block<T>(s, pk);
        __builtin_amdgcn_s_setprio(1);
        TL::transposed(kl, n * 32, pk, lane, dq);
        __builtin_amdgcn_s_setprio(0);
      } else {
        TL::transposed(kl, n * 32, s, lane, dq);
      }
    }
    arrive();
  }
  if constexpr (DELTA) {
    sum = add_xor32(sum);
    if (valid && half == 0) {
      *reinterpret_cast<float2*>(a.delta + 2 * lrow) = make_float2(sum, lse2);
    }
    return;
  }
  if (!valid) {
    return;
  }
  // A softmax over one key is constant: its gradient is zero, not the rounding
  // difference between dP and delta.
  float f = len > 1 ? a.scale : 0.0f;
  if constexpr (__is_same(T, F16)) {
    f *= lift.down();
  }
  if (a.splits_q > 1) {
    const size_t prow = (static_cast<size_t>(z) * gridDim.x + blockIdx.x) * R + r;
    store_partial<TL::DT>(a.part_q + prow * DP, half, dq, f);
    return;
  }
  store_column<T, TL::DT, VEC>(static_cast<E*>(a.dq.p) + b * a.dq.sb + qr.head * a.dq.sh + pos * a.dq.ss, a.d, half,
                               dq, f);
}

constexpr int kQueryTile = 32;
template <typename T, int DP>
constexpr size_t dkv_lds_bytes() {
  return (4 * kQueryTile + 128) * Tile<T, DP>::RB + 4 * kQueryTile * sizeof(float);
}

// fp16: P goes to fp16 as 2^15 P, at most half its largest number, so that it is
// normal down to 2^-29 (as P alone to 2^-14: among 16384 keys most are not).
template <typename T>
constexpr int probability_lift() {
  return __is_same(T, F16) ? 15 : 0;
}

// dK and dV of 128 keys (block `blk`), four waves of 32, over share z of the
// query tiles; Q and dO stream.  The workgroup's own rows of V stay in LDS: in
// registers beside K's and two accumulators they would leave room for one wave
// on a SIMD, whose products then wait for its exponentials (16-bit, 64 heads of
// 2048 x 1500 x 128: 465 us against 358).
template <typename T, int DP, bool VEC>
__device__ __forceinline__ void dkv_part(const XAttnArgs& a, char* smem, int blk, int z) {
  using TL = Tile<T, DP>;
  using E = typename Elem<T>::type;
  constexpr int KT = kQueryTile;
  constexpr int TB = KT * TL::RB;
  // LDS: Q and dO tiles, then lse and delta, then V.
  float* const st = reinterpret_cast<float*>(smem + 4 * TB);   // [2][2][KT]
  char* const own = smem + 4 * TB + 4 * KT * sizeof(float);
  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int half = lane >> 5;
  const int b = blockIdx.x / a.kv_heads;
  const int hk = blockIdx.x - b * a.kv_heads;
  const int group = a.heads / a.kv_heads;
  const int key = blk * 128 + wave * 32 + (lane & 31);
  const int len = keys_of(a, b);
  const bool valid = key < len;
  // Tiles: those of the group's heads, one after the other.
  const int per_head = (a.q_len + KT - 1) / KT;
  int t0, t1;
  tile_range(blk * 128 < len ? group * per_head : 0, a.splits_kv, z, &t0, &t1);

  Stream<T, DP, KT, VEC, 4> qs, gs;
  qs.init(a.q.p, a.q.ss, a.q_len, a.d, wave, lane);
  gs.init(a.go.p, a.go.ss, a.q_len, a.d, wave, lane);
  float rl = 0.0f, rd = 0.0f;
  // Starts moving tile t; its rows' statistics stay in registers until `keep`.
  auto stage = [&](int t, int buf) {
    const int g = t / per_head;
    const int tile = t - g * per_head;
    const int head = hk * group + g;
    if (tid < KT) {
      const int pos = tile * KT + tid;
      const bool in = pos < a.q_len;
      const size_t row = (static_cast<size_t>(b) * a.heads + head) * a.q_len + (in ? pos : 0);
      const float* dr = a.delta + 2 * row;
      // A row past the end has probabilities of zero.
      rl = in ? dr[1] - probability_lift<T>() : INFINITY;
      rd = in ? dr[0] : 0.0f;
    }
    qs.rebase(static_cast<const E*>(a.q.p) + b * a.q.sb + head * a.q.sh);
    gs.rebase(static_cast<const E*>(a.go.p) + b * a.go.sb + head * a.go.sh);
    qs.stage(tile, smem + buf * TB);
    gs.stage(tile, smem + (2 + buf) * TB);
  };
  auto keep = [&](int buf) {
    if (tid < KT) {
      float* sl = st + buf * 2 * KT;
      sl[tid] = rl;
      sl[KT + tid] = rd;
    }
  };
  u32x4 kf[TL::NS];
  const int64_t krow = valid ? key : 0;
  const E* const vbase = static_cast<const E*>(a.v.p) + b * a.v.sb + hk * a.v.sh;
  if (t0 < t1) {
    stage(t0, 0);
    Stream<T, DP, 128, VEC, 4> vs;
    vs.init(vbase, a.v.ss, len, a.d, wave, lane);
    vs.stage(blk, own);
  }
  load_fragments<T, DP, VEC>(static_cast<const E*>(a.k.p) + b * a.k.sb + hk * a.k.sh + krow * a.k.ss, valid, a.d, half,
                             kf);
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
  Lift lift;  // fp16
  const float c = a.c;
  if (t0 < t1) {
    keep(0);
    arrive();
  }
  for (int t = t0; t < t1; ++t) {
    const int buf = (t - t0) & 1;
    const char* ql = smem + buf * TB;
    const char* gl = ql + 2 * TB;
    const float* sl = st + buf * 2 * KT;
    if (t + 1 < t1) {
      stage(t + 1, 1 - buf);
    }
    floatx16 s = zero16();
    floatx16 dp = zero16();
#pragma unroll
    for (int f = 0; f < TL::NS; ++f) {
      s = mma_rows<T>(TL::rows(ql, 0, f, lane), kf[f], s);
      dp = mma_rows<T>(TL::rows(gl, 0, f, lane), TL::rows(own, wave * 32, f, lane), dp);
    }
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int r0 = 8 * g + 4 * half;
      const float4 l4 = *reinterpret_cast<const float4*>(sl + r0);
      const float4 d4 = *reinterpret_cast<const float4*>(sl + KT + r0);
      const float lv[4] = {l4.x, l4.y, l4.z, l4.w};
      const float dl[4] = {d4.x, d4.y, d4.z, d4.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float p = fast_exp2(fmaf(s[4 * g + i], c, -lv[i]));
        s[4 * g + i] = p;
        dp[4 * g + i] = p * (dp[4 * g + i] - dl[i]);
      }
    }
    if constexpr (TL::EC == 8) {
      u32x4 pk[2];
      pack_block<T>(s, pk);
      // As in the forward: 383 -> 375 us for the whole pass at 2048 x 1500.
      __builtin_amdgcn_s_setprio(1);
      TL::transposed(gl, 0, pk, lane, dv);
      if constexpr (__is_same(T, F16)) {
        lift.apply(dp, valid, dk);
      }
      u32x4 pd[2];
      pack_block<T>(dp, pd);
      TL::transposed(ql, 0, pd, lane, dk);
      __builtin_amdgcn_s_setprio(0);
    } else {
      TL::transposed(gl, 0, s, lane, dv);
      TL::transposed(ql, 0, dp, lane, dk);
    }
    if (t + 1 < t1) {
      keep(1 - buf);
    }
    arrive();
  }
  if (key >= a.kv_len) {
    return;
  }
  // Keys past the row's length have gradients of zero.
  float fk = valid && len > 1 ? a.scale : 0.0f;
  float fv = valid ? 1.0f : 0.0f;
  if constexpr (__is_same(T, F16)) {
    constexpr float kDown = 1.0f / (1 << probability_lift<T>());
    fk *= lift.down() * kDown;
    fv *= kDown;
  }
  if (!valid) {
#pragma unroll
    for (int t = 0; t < TL::DT; ++t) {
      dk[t] = zero16();
      dv[t] = zero16();
    }
  }
  if (a.splits_kv > 1) {
    const size_t plane = static_cast<size_t>(gridDim.x) * a.kv_len;
    const size_t prow = static_cast<size_t>(z) * 2 * plane + static_cast<size_t>(blockIdx.x) * a.kv_len + key;
    store_partial<TL::DT>(a.part_kv + prow * DP, half, dk, fk);
    store_partial<TL::DT>(a.part_kv + (prow + plane) * DP, half, dv, fv);
    return;
  }
  const int64_t at = key;
  store_column<T, TL::DT, VEC>(static_cast<E*>(a.dk.p) + b * a.dk.sb + hk * a.dk.sh + at * a.dk.ss, a.d, half, dk, fk);
  store_column<T, TL::DT, VEC>(static_cast<E*>(a.dv.p) + b * a.dv.sb + hk * a.dv.sh + at * a.dv.ss, a.d, half, dv, fv);
}

// The whole backward pass: grid (problems, workgroups), the dK / dV ones (the
// longer ones) first.
template <typename T, int DP, bool VEC>
__global__ __launch_bounds__(256, (VEC && (Elem<T>::kChunk == 8 || DP == 64) ? 2 : 1)) void xattn_bwd_kernel(
    XAttnArgs a) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int kv_blocks = (a.kv_len + 127) / 128;
  const int y = blockIdx.y;
  if (y < kv_blocks * a.splits_kv) {
    dkv_part<T, DP, VEC>(a, smem, y % kv_blocks, y / kv_blocks);
  } else {
    const int q_blocks = (a.heads / a.kv_heads * a.q_len + 127) / 128;
    const int i = y - kv_blocks * a.splits_kv;
    dq_part<T, DP, VEC, false>(a, smem, i % q_blocks, i / q_blocks);
  }
}

// Parts of a 128-row block, a workgroup each, where delta comes from `out`: fp32;
// 16-bit types whose blocks would not fill the chip (else one).
constexpr int kDeltaParts = 8;
constexpr int kDeltaPartsFew = 4;

// Every query row's delta: grid (problems, 128-row blocks, parts).  16-bit
// types take it from the probabilities instead of from `out` where the batch row
// has few keys of its own, however far it is padded: a 16-bit `out` has lost 2^-9
// of itself, and with few keys it is of the values' own size (dQ and dK of 18
// keys were 1.7 times as far from 64 bits as a rounding of the exact ones is).
// Two more products, for short keys only.  us, one kernel for either kind of
// row: 64 heads of 2048 rows of 128 from `out` 15 (a kernel without LDS 14), 64
// heads of 512 x 100 x 64 from the probabilities 6.7.
template <typename T, int DP, bool VEC>
__global__ __launch_bounds__(256, (waves_per_simd<T, DP, VEC>())) void xattn_delta_kernel(XAttnArgs a) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  if constexpr (Elem<T>::kChunk == 4) {
    delta_rows<T, VEC, 128 / kDeltaParts>(a, blockIdx.y * kDeltaParts + blockIdx.z);
  } else if (keys_of(a, blockIdx.x / a.kv_heads) <= kern::kXAttnShortKeys) {
    if (blockIdx.z == 0) {
      dq_part<T, DP, VEC, true>(a, smem, blockIdx.y, 0);
    }
  } else if (gridDim.z == 1) {
    delta_rows<T, VEC, 128>(a, blockIdx.y);
  } else {
    delta_rows<T, VEC, 128 / kDeltaPartsFew>(a, blockIdx.y * kDeltaPartsFew + blockIdx.z);
  }
}

// Sums the shares' partial rows in their order, a wave per row: blockIdx.y 0 dQ
// from part_q [splits_q][rows][DP], 1 and 2 dK and dV from part_kv
// [splits_kv][2][rows][DP]; `from` where the first is not wanted.
template <typename T, int DP>
__global__ __launch_bounds__(256) void xattn_sum_kernel(XAttnArgs a, int from) {
  using E = typename Elem<T>::type;
  constexpr int PL = DP / 64;
  const int lane = threadIdx.x & 63;
  const int which = blockIdx.y + from;
  const int heads = which == 0 ? a.heads : a.kv_heads;
  const int len = which == 0 ? a.q_len : a.kv_len;
  const size_t rows = static_cast<size_t>(a.batch) * heads * len;
  const size_t row = static_cast<size_t>(blockIdx.x) * 4 + (threadIdx.x >> 6);
  if (row >= rows) {
    return;
  }
  const int problem = static_cast<int>(row / len);
  const int64_t pos = static_cast<int64_t>(row - static_cast<size_t>(problem) * len);
  const int b = problem / heads;
  const XTensor& x = which == 0 ? a.dq : which == 1 ? a.dk : a.dv;
  const int splits = which == 0 ? a.splits_q : a.splits_kv;
  const size_t step = (which == 0 ? 1 : 2) * rows * DP;
  const float* p = (which == 0 ? a.part_q : a.part_kv) + ((which == 2 ? rows : 0) + row) * DP + lane;
  float s[PL] = {};
#pragma unroll 8
  for (int z = 0; z < splits; ++z) {
#pragma unroll
    for (int i = 0; i < PL; ++i) {
      s[i] += p[z * step + i * 64];
    }
  }
  E* out = static_cast<E*>(x.p) + b * x.sb + (problem - b * heads) * x.sh + pos * x.ss;
#pragma unroll
  for (int i = 0; i < PL; ++i) {
    if (i * 64 + lane < a.d) {
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
hipError_t launch_forward(const XAttnArgs& a, hipStream_t stream) {
  const unsigned problems = static_cast<unsigned>(a.batch * a.kv_heads);
  const unsigned rows = static_cast<unsigned>(a.heads / a.kv_heads * a.q_len);
  const unsigned z = static_cast<unsigned>(a.splits);
  constexpr size_t lds = tiles_bytes<T, DP>();
  if (a.few) {
    static const hipError_t allowed = LC_XATTN_ALLOW((xattn_few_kernel<T, DP, VEC>), 2 * lds);
    return launch_lds(xattn_few_kernel<T, DP, VEC>, allowed, dim3(problems, (rows + 31) / 32, z), 2 * lds, a, stream);
  }
  static const hipError_t allowed = LC_XATTN_ALLOW((xattn_fwd_kernel<T, DP, VEC>), lds);
  return launch_lds(xattn_fwd_kernel<T, DP, VEC>, allowed, dim3(problems, (rows + 127) / 128, z), lds, a, stream);
}

template <typename T, int DP, bool VEC>
hipError_t launch_backward(const XAttnArgs& a, hipStream_t stream) {
  const size_t rows_q = static_cast<size_t>(a.batch) * a.heads * a.q_len;
  const size_t rows_kv = static_cast<size_t>(a.batch) * a.kv_heads * a.kv_len;
  const unsigned q_blocks = static_cast<unsigned>((a.heads / a.kv_heads * a.q_len + 127) / 128);
  const unsigned problems = static_cast<unsigned>(a.batch * a.kv_heads);
  if (rows_q != 0) {
    constexpr bool k16 = Elem<T>::kChunk == 8;
    // LDS where a row may take delta from the probabilities.
    constexpr size_t most = k16 ? tiles_bytes<T, DP>() : 0;
    const size_t lds = a.lengths != nullptr || a.kv_len <= kern::kXAttnShortKeys ? most : 0;
    static const hipError_t allowed = LC_XATTN_ALLOW((xattn_delta_kernel<T, DP, VEC>), most);
    // A workgroup for each CU at least (2 x 2 heads of keys, 308 rows each: 5.1 -> 3.3 us).
    const dim3 grid(problems, q_blocks, !k16 ? kDeltaParts : problems * q_blocks < 256 ? kDeltaPartsFew : 1);
    const hipError_t e = launch_lds(xattn_delta_kernel<T, DP, VEC>, allowed, grid, lds, a, stream);
    if (e != hipSuccess) {
      return e;
    }
  }
  const unsigned blocks = static_cast<unsigned>((a.kv_len + 127) / 128 * a.splits_kv) +
                          q_blocks * static_cast<unsigned>(a.splits_q);
  constexpr size_t tiles = tiles_bytes<T, DP>();
  constexpr size_t own = dkv_lds_bytes<T, DP>();
  constexpr size_t lds = tiles > own ? tiles : own;
  if (blocks != 0) {
    static const hipError_t allowed = LC_XATTN_ALLOW((xattn_bwd_kernel<T, DP, VEC>), lds);
    const hipError_t e = launch_lds(xattn_bwd_kernel<T, DP, VEC>, allowed,
                                    dim3(static_cast<unsigned>(a.batch * a.kv_heads), blocks), lds, a, stream);
    if (e != hipSuccess) {
      return e;
    }
  }
  const bool sum_q = a.splits_q > 1;
  const bool sum_kv = a.splits_kv > 1;
  if (sum_q || sum_kv) {
    const size_t rows = sum_q && (!sum_kv || rows_q > rows_kv) ? rows_q : rows_kv;
    const dim3 grid(static_cast<unsigned>((rows + 3) / 4), (sum_q ? 1 : 0) + (sum_kv ? 2 : 0));
    xattn_sum_kernel<T, DP><<<grid, 256, 0, stream>>>(a, sum_q ? 0 : 1);
  }
  return hipGetLastError();
}
#undef LC_XATTN_ALLOW

template <typename T>
hipError_t launch_type(bool backward, const XAttnArgs& a, bool vec, hipStream_t stream) {
  if (a.d <= 64) {
    if (backward) {
      return vec ? launch_backward<T, 64, true>(a, stream) : launch_backward<T, 64, false>(a, stream);
    }
    return vec ? launch_forward<T, 64, true>(a, stream) : launch_forward<T, 64, false>(a, stream);
  }
  if (backward) {
    return vec ? launch_backward<T, 128, true>(a, stream) : launch_backward<T, 128, false>(a, stream);
  }
  return vec ? launch_forward<T, 128, true>(a, stream) : launch_forward<T, 128, false>(a, stream);
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

}  // namespace
}  // namespace lchip::k

namespace lchip::kern {

namespace {
hipError_t launch(bool backward, const XAttnArgs& a, DType type, bool aligned, hipStream_t stream) {
  switch (type) {
    case DType::kF32:
      return k::launch_type<k::F32>(backward, a, aligned, stream);
    case DType::kBF16:
      return k::launch_type<k::BF16>(backward, a, aligned, stream);
    default:
      return k::launch_type<k::F16>(backward, a, aligned, stream);
  }
}
}  // namespace

hipError_t crossAttentionForward(const XAttnArgs& a, DType type, bool aligned, hipStream_t stream) {
  return launch(false, a, type, aligned, stream);
}

hipError_t crossAttentionBackward(const XAttnArgs& a, DType type, bool aligned, hipStream_t stream) {
  return launch(true, a, type, aligned, stream);
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

}  // namespace lchip::kern
