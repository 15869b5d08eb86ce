// kv_cache.hip -- an 8-bit paged cache of keys and values, and attention of a
// few query rows over it.
//
// A page holds 64 tokens of every key/value head as e4m3 codes with one fp32
// scale for a page and head: keys [page, head, token, d], values
// [page, head, d, token].  Values are kept transposed because the second
// product contracts over tokens: both products then take their matrix operand
// from 16 consecutive bytes of a lane, straight from memory to registers, with
// no pass through LDS.  e4m3 is exact in bf16, so the products run on bf16
// matrix cores; queries and probabilities enter as one, two or three bf16 terms
// (bf16, fp16, fp32 queries), which cost matrix-core time that a kernel bound by
// the cache's bytes has to spare.
#include <hip/hip_runtime.h>

#include "../kernels.hpp"
#include "elements.hpp"
#include "kcommon.hpp"

namespace lchip::k {
namespace {

using kern::KvAttnArgs;
using kern::KvStoreArgs;

constexpr int kPage = kern::kKvPage;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kE4m3Max = 448.0f;

__device__ __forceinline__ float fast_exp2(float x) { return __builtin_amdgcn_exp2f(x); }

// Eight values d0 .. d0 + 7 of a row (all inside the row).
template <typename T, bool VEC>
__device__ __forceinline__ void load8(const typename Elem<T>::type* row, int d0, float (&v)[8]) {
  if constexpr (VEC) {
    constexpr int EC = Elem<T>::kChunk;
#pragma unroll
    for (int c = 0; c < 8 / EC; ++c) {
      const u32x4 x = *reinterpret_cast<const u32x4*>(row + d0 + c * EC);
#pragma unroll
      for (int i = 0; i < EC; ++i) {
        v[c * EC + i] = chunk_value<T>(x, i);
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      v[i] = to_f32<T>(row[d0 + i]);
    }
  }
}

// Four values to four e4m3 codes, round to nearest even.
__device__ __forceinline__ uint32_t codes4(float a, float b, float c, float d) {
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  w = __builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
  return static_cast<uint32_t>(w);
}

// One workgroup writes a page's head: thread (token quad, 8 columns) holds four
// tokens of K and of V, so that a page is read once, its scale is known before
// any code is made, and V's codes come out as dwords of four tokens.  Tokens
// past the row's length are zero codes.  fmaxf leaves a NaN out of the maximum:
// one bad value does not cost its page the other 64 d - 1.
template <typename T, bool VEC>
__global__ __launch_bounds__(256) void kv_store_kernel(KvStoreArgs a) {
  using E = typename Elem<T>::type;
  __shared__ float tops[2][4];
  const int b = blockIdx.z;
  const int h = blockIdx.x;
  const int p = blockIdx.y;
  const int len = min(max(a.lengths == nullptr ? a.kv_len : a.lengths[b], 0), a.kv_len);
  const int left = min(len - p * kPage, kPage);
  if (left <= 0) {
    return;
  }
  const int page = a.table[static_cast<int64_t>(b) * a.table_stride + p];
  if (page < 0 || page >= a.pages) {
    return;
  }
  const int tid = threadIdx.x;
  const int quad = tid & 15;
  const int d0 = (tid >> 4) * 8;
  const bool on = d0 < a.d;
  float kv[2][4][8];
  float top[2] = {0.0f, 0.0f};
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    const kern::XTensor& t = x == 0 ? a.k : a.v;
    const E* base = static_cast<const E*>(t.p) + b * t.sb + h * t.sh + static_cast<int64_t>(p) * kPage * t.ss;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int tok = quad * 4 + i;
      if (on && tok < left) {
        load8<T, VEC>(base + tok * t.ss, d0, kv[x][i]);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          kv[x][i][j] = 0.0f;
        }
      }
    }
  }
#pragma unroll
  for (int x = 0; x < 2; ++x) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        top[x] = fmaxf(top[x], fabsf(kv[x][i][j]));
      }
    }
#pragma unroll
    for (int s = 32; s > 0; s >>= 1) {
      top[x] = fmaxf(top[x], __shfl_xor(top[x], s));
    }
    if ((tid & 63) == 0) {
      tops[x][tid >> 6] = top[x];
    }
  }
  __syncthreads();
  float scale[2];
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    const float m = fmaxf(fmaxf(tops[x][0], tops[x][1]), fmaxf(tops[x][2], tops[x][3]));
    // At least the smallest normal number: a page of zeros divides by it.
    scale[x] = fmaxf(m / kE4m3Max, 1.1754943508222875e-38f);
  }
  const size_t head = static_cast<size_t>(page) * a.heads + h;
  if (tid < 2) {
    (tid == 0 ? a.k_scales : a.v_scales)[head] = scale[tid];
  }
  if (!on) {
    return;
  }
  uint8_t* const kp = a.k_pages + head * kPage * a.d;
  uint8_t* const vp = a.v_pages + head * kPage * a.d;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float q[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      q[j] = kv[0][i][j] / scale[0];
    }
    u32x2 w;
    w[0] = codes4(q[0], q[1], q[2], q[3]);
    w[1] = codes4(q[4], q[5], q[6], q[7]);
    *reinterpret_cast<u32x2*>(kp + (quad * 4 + i) * a.d + d0) = w;
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    *reinterpret_cast<uint32_t*>(vp + (d0 + j) * kPage + quad * 4) =
        codes4(kv[1][0][j] / scale[1], kv[1][1][j] / scale[1], kv[1][2][j] / scale[1], kv[1][3][j] / scale[1]);
  }
}

// Eight e4m3 codes (two dwords) as bf16, exactly.
__device__ __forceinline__ u32x4 widen(uint32_t lo, uint32_t hi) {
  u32x4 r;
  r[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, false));
  r[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, true));
  r[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, false));
  r[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, true));
  return r;
}

// v in NT bf16 terms: each rounds what the ones before it left.
template <int NT>
__device__ __forceinline__ void terms(const float (&v)[8], u32x4 (&t)[NT]) {
  float r[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    r[i] = v[i];
  }
#pragma unroll
  for (int n = 0; n < NT; ++n) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t w = pack2<BF16>(r[2 * i], r[2 * i + 1]);
      t[n][i] = w;
      if (n + 1 < NT) {
        r[2 * i] -= __builtin_bit_cast(float, w << 16);
        r[2 * i + 1] -= __builtin_bit_cast(float, w & 0xffff0000u);
      }
    }
  }
}

// bf16 terms of queries and of probabilities.  A bf16 query is one term; its
// probabilities take two, so that the output's own rounding is what is left of
// the error.
template <typename T>
struct Terms;
template <>
struct Terms<BF16> {
  static constexpr int kQ = 1, kP = 2;
};
template <>
struct Terms<F16> {
  static constexpr int kQ = 2, kP = 2;
};
template <>
struct Terms<F32> {
  static constexpr int kQ = 3, kP = 3;
};

// 16 bytes of a page, zero where not `in`.  ONCE: nothing else in the call reads
// them, so they need not stay in the caches (32 x 8 heads of 6144 tokens: 80.8 ->
// 73.3 us; three blocks of rows that share the pages: 27.8 -> 31.9 us).
template <bool ONCE>
__device__ __forceinline__ u32x4 load_page(const uint8_t* page, int at, bool in) {
  const u32x4* const p = reinterpret_cast<const u32x4*>(page + (in ? at : 0));
  u32x4 v;
  if constexpr (ONCE) {
    v = __builtin_nontemporal_load(p);
  } else {
    v = *p;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[i] = in ? v[i] : 0u;
  }
  return v;
}

constexpr int kWaves = 4;

// Grid (problems, key splits, blocks of 16 rows); a split's pages go to the
// workgroup's waves in turn, whose states are joined through LDS.  Scores are
// S^T = K Q^T on 16 x 16 x 32 MFMAs: the row order of K is chosen so that lane
// group g = lane / 16 holds the scores of tokens 16 g .. 16 g + 15 of its query
// (lane % 16), the very tokens whose values the same lane loads.
// WHOLE: d is 64 NC, no part of a row is padding.  ONCE: one block of 16 rows
// reads the pages.
template <typename T, int NC, bool WHOLE, bool ONCE>
__global__ __launch_bounds__(256, 2) void kv_attn_kernel(KvAttnArgs a) {
  using E = typename Elem<T>::type;
  constexpr int DW = NC * 64;
  constexpr int NQ = Terms<T>::kQ;
  constexpr int NP = Terms<T>::kP;
  __shared__ float sm[kWaves][2][16];
  __shared__ __attribute__((aligned(16))) float so[kWaves][16][DW + 4];
  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int g = lane >> 4;
  const int m16 = lane & 15;
  const int b = blockIdx.x / a.kv_heads;
  const int hk = blockIdx.x - b * a.kv_heads;
  const int group = a.heads / a.kv_heads;
  const int R = group * a.q_len;
  const int r = blockIdx.z * 16 + m16;
  const bool valid = r < R;
  const int rr = valid ? r : 0;
  const int head = hk * group + rr / a.q_len;
  const int pos = rr % a.q_len;
  const int len = min(max(a.lengths == nullptr ? a.kv_len : a.lengths[b], 0), a.kv_len);
  const int np = (len + kPage - 1) / kPage;
  const int per = (np + a.splits - 1) / a.splits;
  const int first = min(np, static_cast<int>(blockIdx.y) * per);
  const int last = min(np, first + per);

  // Query terms: MFMA (c, u) contracts over d = 64 c + 16 g + 8 u + i.
  u32x4 qf[NC][2][NQ];
  {
    const E* q = static_cast<const E*>(a.q.p) + b * a.q.sb + head * a.q.sh + static_cast<int64_t>(pos) * a.q.ss;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        float v[8];
        const int d0 = 64 * c + 16 * g + 8 * u;
        if (valid && d0 < a.d) {
          if (a.aligned) {
            load8<T, true>(q, d0, v);
          } else {
            load8<T, false>(q, d0, v);
          }
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            v[i] = 0.0f;
          }
        }
        terms<NQ>(v, qf[c][u]);
      }
    }
  }
  floatx4 o[DW / 16];
#pragma unroll
  for (int t = 0; t < DW / 16; ++t) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      o[t][i] = 0.0f;
    }
  }
  float m = -INFINITY;
  float l = 0.0f;
  bool bad = false;

  u32x4 kr[4][NC], vr[DW / 16];
  const int32_t* const table = a.table + static_cast<int64_t>(b) * a.table_stride;
  const size_t head_bytes = static_cast<size_t>(kPage) * a.d;
  // A table entry outside the pool is never followed: page 0 is read in its
  // place and the rows come out as NaN.
  auto page_of = [&](int p) {
    const int id = table[p];
    const bool in = id >= 0 && id < a.pages;
    bad = bad || !in;
    return static_cast<size_t>(in ? id : 0) * a.kv_heads + hk;
  };
  auto load_k = [&](size_t ph) {
    const uint8_t* kp = a.k_pages + ph * head_bytes;
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const int key = 16 * (m16 >> 2) + 4 * t + (m16 & 3);
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        const int d0 = 64 * c + 16 * g;
        kr[t][c] = load_page<ONCE>(kp, key * a.d + d0, WHOLE || d0 < a.d);
      }
    }
  };
  auto load_v = [&](size_t ph) {
    const uint8_t* vp = a.v_pages + ph * head_bytes;
#pragma unroll
    for (int t = 0; t < DW / 16; ++t) {
      vr[t] = load_page<ONCE>(vp, (t * 16 + m16) * kPage + 16 * g, WHOLE || t * 16 < a.d);
    }
  };
  int p = first + wave;
  size_t ph = 0;
  if (p < last) {
    ph = page_of(p);
    load_k(ph);
    load_v(ph);
  }
  for (; p < last; p += kWaves) {
    const float kscale = a.k_scales[ph] * a.c;
    const float vscale = a.v_scales[ph];
    floatx4 s[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        s[t][i] = 0.0f;
      }
#pragma unroll
      for (int c = 0; c < NC; ++c) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const u32x4 kw = widen(kr[t][c][2 * u], kr[t][c][2 * u + 1]);
#pragma unroll
          for (int n = 0; n < NQ; ++n) {
            s[t] = mfma16x16x32<BF16>(kw, qf[c][u][n], s[t]);
          }
        }
      }
    }
    // K's registers are free: the next page's keys load during the rest.
    const bool more = p + kWaves < last;
    if (more) {
      ph = page_of(p + kWaves);
      load_k(ph);
    }
    const int left = len - p * kPage;
    float top = -INFINITY;
#pragma unroll
    for (int t = 0; t < 4; ++t) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        s[t][i] = 16 * g + 4 * t + i < left ? s[t][i] * kscale : -INFINITY;
        top = fmaxf(top, s[t][i]);
      }
    }
    top = max_xor32(top);
    top = fmaxf(top, __shfl_xor(top, 16));
    if (__any(top > m)) {
      const float next = fmaxf(m, top);
      const float f = m == -INFINITY ? 0.0f : fast_exp2(m - next);
      m = next;
      l *= f;
#pragma unroll
      for (int t = 0; t < DW / 16; ++t) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          o[t][i] *= f;
        }
      }
    }
    const float ref = m == -INFINITY ? 0.0f : m;
    u32x4 pt[2][NP];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      float v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float e = fast_exp2(s[2 * u + (i >> 2)][i & 3] - ref);
        l += e;
        v[i] = e * vscale;
      }
      terms<NP>(v, pt[u]);
    }
    // Codes behind the last token may be anything: a NaN there must not meet its
    // probability of zero.  (Every page is masked, 4 instructions a load: behind a
    // branch around it the compiler, clang 22 of ROCm 7.2.0, wrote a term of the
    // probabilities into v46, which still held codes of V that it widened 50
    // instructions later.  tests/test_asm_kv_values.py looks for that in the
    // compiled kernels.)
    u32x4 keep;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const int n = min(max(left - 16 * g - 4 * w, 0), 4);
      keep[w] = n == 4 ? 0xffffffffu : (1u << (8 * n)) - 1u;
    }
#pragma unroll
    for (int t = 0; t < DW / 16; ++t) {
      const u32x4 v = vr[t] & keep;
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const u32x4 vw = widen(v[2 * u], v[2 * u + 1]);
#pragma unroll
        for (int n = 0; n < NP; ++n) {
          o[t] = mfma16x16x32<BF16>(vw, pt[u][n], o[t]);
        }
      }
    }
    if (more) {
      load_v(ph);
    }
  }
  l += __shfl_xor(l, 16);
  l = add_xor32(l);
  if (bad) {
    l = NAN;
  }
  if (g == 0) {
    sm[wave][0][m16] = m;
    sm[wave][1][m16] = l;
  }
#pragma unroll
  for (int t = 0; t < DW / 16; ++t) {
    *reinterpret_cast<floatx4*>(&so[wave][m16][t * 16 + 4 * g]) = o[t];
  }
  __syncthreads();
  // Thread (row, 16 threads a row) joins the waves' states.
  const int row = tid >> 4;
  const int d1 = tid & 15;
  const int r1 = blockIdx.z * 16 + row;
  if (r1 >= R) {
    return;
  }
  float mm = -INFINITY;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    mm = fmaxf(mm, sm[w][0][row]);
  }
  float ll = 0.0f;
  float f[kWaves];
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    const float mw = sm[w][0][row];
    f[w] = mw == -INFINITY ? 0.0f : fast_exp2(mw - mm);
    ll = fmaf(f[w], sm[w][1][row], ll);
  }
  float v[DW / 16];
#pragma unroll
  for (int j = 0; j < DW / 16; ++j) {
    v[j] = 0.0f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      v[j] = fmaf(f[w], so[w][row][j * 16 + d1], v[j]);
    }
  }
  if (a.splits > 1) {
    const size_t prow = (static_cast<size_t>(blockIdx.y) * gridDim.x + blockIdx.x) * R + r1;
#pragma unroll
    for (int j = 0; j < DW / 16; ++j) {
      a.part[prow * DW + j * 16 + d1] = v[j];
    }
    if (d1 == 0) {
      a.stats[prow * 2] = mm;
      a.stats[prow * 2 + 1] = ll;
    }
    return;
  }
  const int head1 = hk * group + r1 / a.q_len;
  const int pos1 = r1 % a.q_len;
  const bool any = ll > 0.0f || ll != ll;
  const float inv = any ? 1.0f / ll : 0.0f;
  E* out = static_cast<E*>(a.o.p) + b * a.o.sb + head1 * a.o.sh + static_cast<int64_t>(pos1) * a.o.ss;
#pragma unroll
  for (int j = 0; j < DW / 16; ++j) {
    if (j * 16 < a.d) {
      out[j * 16 + d1] = from_f32<T>(v[j] * inv);
    }
  }
  if (a.lse != nullptr && d1 == 0) {
    a.lse[(static_cast<size_t>(b) * a.heads + head1) * a.q_len + pos1] = any ? mm * kLn2 + logf(ll) : -INFINITY;
  }
}

template <typename T>
hipError_t store_type(const KvStoreArgs& a, bool aligned, hipStream_t stream) {
  // Heads first: of tokens whose rows hold all heads, workgroups that run at once
  // then read neighbouring parts.
  const dim3 grid(static_cast<unsigned>(a.heads), static_cast<unsigned>((a.kv_len + kPage - 1) / kPage),
                  static_cast<unsigned>(a.batch));
  if (aligned) {
    kv_store_kernel<T, true><<<grid, 256, 0, stream>>>(a);
  } else {
    kv_store_kernel<T, false><<<grid, 256, 0, stream>>>(a);
  }
  return hipGetLastError();
}

template <typename T>
hipError_t attn_type(const KvAttnArgs& a, hipStream_t stream) {
  const int R = a.heads / a.kv_heads * a.q_len;
  const dim3 grid(static_cast<unsigned>(a.batch * a.kv_heads), static_cast<unsigned>(a.splits),
                  static_cast<unsigned>((R + 15) / 16));
#define LC_KV_ATTN(NC)                                                \
  do {                                                                \
    if (a.d == 64 * NC && grid.z == 1) {                              \
      kv_attn_kernel<T, NC, true, true><<<grid, 256, 0, stream>>>(a);  \
    } else if (a.d == 64 * NC) {                                      \
      kv_attn_kernel<T, NC, true, false><<<grid, 256, 0, stream>>>(a); \
    } else if (grid.z == 1) {                                         \
      kv_attn_kernel<T, NC, false, true><<<grid, 256, 0, stream>>>(a); \
    } else {                                                          \
      kv_attn_kernel<T, NC, false, false><<<grid, 256, 0, stream>>>(a); \
    }                                                                 \
  } while (0)
  if (a.d <= 64) {
    LC_KV_ATTN(1);
  } else {
    LC_KV_ATTN(2);
  }
#undef LC_KV_ATTN
  return hipGetLastError();
}

}  // namespace
}  // namespace lchip::k

namespace lchip::kern {

hipError_t kvStore(const KvStoreArgs& a, DType type, bool aligned, hipStream_t stream) {
  switch (type) {
    case DType::kF32:
      return k::store_type<k::F32>(a, aligned, stream);
    case DType::kBF16:
      return k::store_type<k::BF16>(a, aligned, stream);
    default:
      return k::store_type<k::F16>(a, aligned, stream);
  }
}

hipError_t kvAttention(const KvAttnArgs& a, DType type, hipStream_t stream) {
  switch (type) {
    case DType::kF32:
      return k::attn_type<k::F32>(a, stream);
    case DType::kBF16:
      return k::attn_type<k::BF16>(a, stream);
    default:
      return k::attn_type<k::F16>(a, stream);
  }
}

}  // namespace lchip::kern
