// cross_attention.cpp -- entry points of cross attention, forward and backward,
// on the caller's device tensors (kernels/cross_attention.hip).
#include <algorithm>
#include <cmath>

#include "device_ops.hpp"

namespace lchip {
namespace {

constexpr const char* kOp = "cross attention";
constexpr std::size_t kMostRows = std::size_t{1} << 30;
constexpr std::size_t kMostProblems = std::size_t{1} << 24;
// Workgroups that the shares are cut for, on 256 CUs: two a CU, of the few-row
// forward one.  Where a CU holds only one of the former (fp32 rows wider than 64,
// rows that no vector load suits), a round of workgroups takes two rounds' time.
constexpr std::size_t kSlots = 512;
constexpr std::size_t kFewSlots = 256;
// The forward's waves share the keys of 32 rows, instead of taking 32 rows each,
// up to so many 32-row blocks in all: the keys need no second launch to be
// joined and each wave's chain of tiles is a quarter as long.  Beyond, reading a
// tile for 32 rows instead of 128 costs more.  Wide 16-bit tiles fill a CU's LDS
// with one such workgroup, the others with half.  us, rows per wave -> shared
// keys: 16 heads of 300 x 1400 x 128 (160 blocks) 27.2 -> 17.7, 32 of 500 x 1000
// x 128 (512) 30.4 -> 26.2, 32 of 700 x 1400 x 128 (704) 39.1 -> 47.2; 32 of 1000
// x 1400 x 64 (1024) 37.8 -> 26.9, 32 of 1200 x 500 x 64 (1216) 15.6 -> 19.6; fp32
// 32 of 700 x 1400 x 128 201 -> 167.
constexpr std::size_t kFewBlocksWide = 512;
constexpr std::size_t kFewBlocks = 1024;
// A workgroup's start and end, and a join, in tiles' time (splitCount).
constexpr double kFixed = 2.0;
constexpr double kJoin = 3.0;
// The backward pass's work is counted in products of 32 x 32 blocks: dQ has three
// for a block, dK and dV four.  A workgroup gets at most kShare of what each
// place on the chip has to do in all, so that the short ones fill what the long
// ones leave, and no less than kLeast, below which its start and its partial
// result cost more than its work.
constexpr double kShare = 0.8;
constexpr std::size_t kMostShares = 32;
constexpr double kLeast = 40.0;     // 16-bit types
constexpr double kLeastF32 = 12.0;  // fp32 products take eight times as long

// How the kernels share the work of a problem, and the workspace that it
// takes: a function of the shape alone, so that the size a caller asks for is
// the one its call needs.
struct Plan {
  bool few = false;
  int splits_fwd = 1, splits_q = 1, splits_kv = 1;
  std::size_t rows_q = 0, rows_kv = 0;  // rows of all problems
  std::size_t width = 0;                // floats of a partial row
  std::size_t forwardBytes() const {
    return splits_fwd > 1 ? static_cast<std::size_t>(splits_fwd) * rows_q * (width + 2) * sizeof(float) : 0;
  }
  std::size_t deltaBytes() const { return roundUp(rows_q * 2 * sizeof(float), 256); }
  std::size_t partialQ() const { return splits_q > 1 ? static_cast<std::size_t>(splits_q) * rows_q * width : 0; }
  std::size_t partialKv() const {
    return splits_kv > 1 ? static_cast<std::size_t>(splits_kv) * 2 * rows_kv * width : 0;
  }
  std::size_t backwardBytes() const { return deltaBytes() + (partialQ() + partialKv()) * sizeof(float); }
};

Plan planOf(const lcCrossAttentionConfig& c) {
  Plan p;
  const std::size_t problems = c.batch * c.kv_heads;
  const std::size_t group = c.heads / c.kv_heads;
  const std::size_t tile = static_cast<std::size_t>(kern::kXAttnTile(dtypeOf(c.dtype)));
  const std::size_t block = kern::kXAttnRows;
  p.rows_q = c.batch * c.heads * c.q_len;
  p.rows_kv = problems * c.kv_len;
  p.width = static_cast<std::size_t>(kern::kXAttnWidth(static_cast<int>(c.head_dim)));
  const std::size_t q_blocks = problems * ((group * c.q_len + block - 1) / block);
  const std::size_t kv_tiles = (c.kv_len + tile - 1) / tile;
  const std::size_t few_rows = kern::kXAttnFewRows;
  const bool wide = c.dtype != LC_DTYPE_F32 && c.head_dim > 64;
  p.few = problems * ((group * c.q_len + few_rows - 1) / few_rows) <= (wide ? kFewBlocksWide : kFewBlocks);
  p.splits_fwd = p.few ? splitCount(problems * ((group * c.q_len + few_rows - 1) / few_rows), (kv_tiles + 3) / 4,
                                    kFewSlots, kFixed, kJoin)
                       : splitCount(q_blocks, kv_tiles, kSlots, kFixed, kJoin);
  const std::size_t q_tile = kern::kXAttnQueryTile;
  const std::size_t kv_blocks = problems * ((c.kv_len + block - 1) / block);
  const std::size_t q_tiles = group * ((c.q_len + q_tile - 1) / q_tile);
  const double work_q = 3.0 * static_cast<double>(tile / 32 * kv_tiles);  // of one block
  const double work_kv = 4.0 * static_cast<double>(q_tiles);
  const double all = work_q * static_cast<double>(q_blocks) + work_kv * static_cast<double>(kv_blocks);
  const double most = std::max(c.dtype == LC_DTYPE_F32 ? kLeastF32 : kLeast, kShare * all / static_cast<double>(kSlots));
  const auto shares = [most](double work, std::size_t tiles) {
    const std::size_t want = static_cast<std::size_t>(std::ceil(work / most));
    return static_cast<int>(std::max<std::size_t>(1, std::min({want, tiles, kMostShares})));
  };
  p.splits_q = shares(work_q, kv_tiles);
  p.splits_kv = shares(work_kv, q_tiles);
  return p;
}

Status checkConfig(const lcCrossAttentionConfig* c) {
  if (c == nullptr) {
    return fail(Status::kInvalidValue, "cross attention: null config");
  }
  if (c->heads == 0 || c->kv_heads == 0 || c->head_dim == 0) {
    return fail(Status::kInvalidValue, "cross attention: zero heads or head_dim");
  }
  if (c->heads % c->kv_heads != 0) {
    return fail(Status::kInvalidValue, "cross attention: heads must be a multiple of kv_heads");
  }
  if (!validDtype(c->dtype)) {
    return fail(Status::kInvalidValue, "cross attention: dtype must be f32, bf16 or f16");
  }
  if (!std::isfinite(c->scale * kLog2e)) {
    return fail(Status::kInvalidValue, "cross attention: scale is not finite in exp2 units");
  }
  if (c->head_dim > kern::kXAttnMaxDim) {
    return fail(Status::kNotSupported, "cross attention: head_dim <= 128");
  }
  // Row indices are 32-bit, and a launch has less than 2^32 threads a dimension:
  // 256 a problem.
  const std::size_t most = kMostRows;
  if (c->batch > most || c->heads > most || c->q_len > most || c->kv_len > most ||
      c->batch * c->kv_heads >= kMostProblems || (c->heads / c->kv_heads) * c->q_len > most / 512 ||
      c->kv_len > most / 512) {
    return fail(Status::kNotSupported, "cross attention: shape too large");
  }
  return Status::kSuccess;
}

void fillArgs(const lcCrossAttentionConfig& c, kern::XAttnArgs* a) {
  a->batch = static_cast<int>(c.batch);
  a->heads = static_cast<int>(c.heads);
  a->kv_heads = static_cast<int>(c.kv_heads);
  a->q_len = static_cast<int>(c.q_len);
  a->kv_len = static_cast<int>(c.kv_len);
  a->d = static_cast<int>(c.head_dim);
  a->scale = c.scale != 0.0f ? c.scale : 1.0f / std::sqrt(static_cast<float>(c.head_dim));
  a->c = std::fabs(a->scale) * kLog2e;
  a->negate = a->scale < 0.0f ? 1 : 0;
}

Status checkWorkspace(const void* workspace, std::size_t have, std::size_t need) {
  if (need == 0) {
    return Status::kSuccess;
  }
  if (workspace == nullptr || have < need) {
    return fail(Status::kInvalidValue, "cross attention: the workspace needs " + std::to_string(need) + " bytes, " +
                                           std::to_string(workspace == nullptr ? 0 : have) + " given");
  }
  if (reinterpret_cast<std::uintptr_t>(workspace) % 16 != 0) {
    return fail(Status::kInvalidValue, "cross attention: the workspace is not 16-byte aligned");
  }
  return Status::kSuccess;
}

Status forward(const lcCrossAttentionConfig* cfg, const lcDeviceTensor* q, const lcDeviceTensor* k,
               const lcDeviceTensor* v, const std::int32_t* kv_lengths, const lcDeviceTensor* out, float* lse,
               void* workspace, std::size_t workspace_bytes, lcStream stream) {
  LC_TRY(checkConfig(cfg));
  const lcCrossAttentionConfig& c = *cfg;
  kern::XAttnArgs a{};
  bool aligned = true;
  LC_TRY(takeTensor(kOp, "q", q, c.batch, c.heads, c.q_len, c.head_dim, c.dtype, false, &a.q, &aligned));
  LC_TRY(takeTensor(kOp, "k", k, c.batch, c.kv_heads, c.kv_len, c.head_dim, c.dtype, false, &a.k, &aligned));
  LC_TRY(takeTensor(kOp, "v", v, c.batch, c.kv_heads, c.kv_len, c.head_dim, c.dtype, false, &a.v, &aligned));
  LC_TRY(takeTensor(kOp, "out", out, c.batch, c.heads, c.q_len, c.head_dim, c.dtype, true, &a.o, &aligned));
  fillArgs(c, &a);
  const Plan plan = planOf(c);
  DeviceCall call;
  LC_TRY(call.open(kOp, c.trusted_pointers != 0));
  if (plan.rows_q == 0) {
    return Status::kSuccess;
  }
  LC_TRY(checkWorkspace(workspace, workspace_bytes, plan.forwardBytes()));
  LC_TRY(call.onDevice(a.q.p, "q"));
  LC_TRY(call.onDevice(a.k.p, "k"));
  LC_TRY(call.onDevice(a.v.p, "v"));
  LC_TRY(call.onDevice(a.o.p, "out"));
  LC_TRY(call.onDevice(kv_lengths, "kv_lengths"));
  LC_TRY(call.onDevice(lse, "lse"));
  a.lse = lse;
  a.lengths = kv_lengths;
  a.splits = plan.splits_fwd;
  a.few = plan.few ? 1 : 0;
  if (a.splits > 1) {
    LC_TRY(call.onDevice(workspace, "the workspace"));
    a.part = static_cast<float*>(workspace);
    a.stats = a.part + static_cast<std::size_t>(a.splits) * plan.rows_q * plan.width;
  }
  traceOpDispatch(TraceOp::kAttentionForward, Device::kHIP, Device::kHIP, false, c.q_len * c.kv_len * c.head_dim);
  const hipStream_t s = static_cast<hipStream_t>(stream);
  LC_HIP_TRY(kern::crossAttentionForward(a, dtypeOf(c.dtype), aligned, s));
  if (a.splits > 1) {
    LC_HIP_TRY(kern::crossAttentionJoin(a, dtypeOf(c.dtype), s));
  }
  return Status::kSuccess;
}

Status backward(const lcCrossAttentionConfig* cfg, const lcDeviceTensor* dout, const lcDeviceTensor* q,
                const lcDeviceTensor* k, const lcDeviceTensor* v, const lcDeviceTensor* out, const float* lse,
                const std::int32_t* kv_lengths, const lcDeviceTensor* dq, const lcDeviceTensor* dk,
                const lcDeviceTensor* dv, void* workspace, std::size_t workspace_bytes, lcStream stream) {
  LC_TRY(checkConfig(cfg));
  const lcCrossAttentionConfig& c = *cfg;
  kern::XAttnArgs a{};
  bool aligned = true;
  const std::size_t b = c.batch, d = c.head_dim;
  LC_TRY(takeTensor(kOp, "dout", dout, b, c.heads, c.q_len, d, c.dtype, false, &a.go, &aligned));
  LC_TRY(takeTensor(kOp, "q", q, b, c.heads, c.q_len, d, c.dtype, false, &a.q, &aligned));
  LC_TRY(takeTensor(kOp, "k", k, b, c.kv_heads, c.kv_len, d, c.dtype, false, &a.k, &aligned));
  LC_TRY(takeTensor(kOp, "v", v, b, c.kv_heads, c.kv_len, d, c.dtype, false, &a.v, &aligned));
  LC_TRY(takeTensor(kOp, "out", out, b, c.heads, c.q_len, d, c.dtype, false, &a.o, &aligned));
  LC_TRY(takeTensor(kOp, "dq", dq, b, c.heads, c.q_len, d, c.dtype, true, &a.dq, &aligned));
  LC_TRY(takeTensor(kOp, "dk", dk, b, c.kv_heads, c.kv_len, d, c.dtype, true, &a.dk, &aligned));
  LC_TRY(takeTensor(kOp, "dv", dv, b, c.kv_heads, c.kv_len, d, c.dtype, true, &a.dv, &aligned));
  fillArgs(c, &a);
  const Plan plan = planOf(c);
  if (plan.rows_q != 0 && lse == nullptr) {
    return fail(Status::kInvalidValue, "cross attention: the backward pass needs the forward's lse");
  }
  DeviceCall call;
  LC_TRY(call.open(kOp, c.trusted_pointers != 0));
  LC_TRY(checkWorkspace(workspace, workspace_bytes, plan.backwardBytes()));
  const struct {
    const void* p;
    const char* name;
  } pointers[] = {{a.go.p, "dout"}, {a.q.p, "q"},   {a.k.p, "k"},   {a.v.p, "v"},
                  {a.o.p, "out"},   {lse, "lse"},   {a.dq.p, "dq"}, {a.dk.p, "dk"},
                  {a.dv.p, "dv"},   {kv_lengths, "kv_lengths"},     {workspace, "the workspace"}};
  for (const auto& x : pointers) {
    LC_TRY(call.onDevice(x.p, x.name));
  }
  a.lse = const_cast<float*>(lse);
  a.lengths = kv_lengths;
  a.delta = static_cast<float*>(workspace);
  a.part_q = reinterpret_cast<float*>(static_cast<char*>(workspace) + plan.deltaBytes());
  a.part_kv = a.part_q + plan.partialQ();
  a.splits_q = plan.splits_q;
  a.splits_kv = plan.splits_kv;
  LC_HIP_TRY(kern::crossAttentionBackward(a, dtypeOf(c.dtype), aligned, static_cast<hipStream_t>(stream)));
  return Status::kSuccess;
}

}  // namespace
}  // namespace lchip

extern "C" {

lcError_t lcCrossAttentionWorkspaceSize(const lcCrossAttentionConfig* cfg, int backward, size_t* bytes) {
  using namespace lchip;
  if (bytes == nullptr) {
    return toLc(fail(Status::kInvalidValue, "cross attention: null output"));
  }
  *bytes = 0;
  const Status st = checkConfig(cfg);
  if (st == Status::kSuccess) {
    const Plan plan = planOf(*cfg);
    *bytes = backward != 0 ? plan.backwardBytes() : plan.forwardBytes();
  }
  return toLc(st);
}

lcError_t lcCrossAttentionForward(const lcCrossAttentionConfig* cfg, const lcDeviceTensor* q, const lcDeviceTensor* k,
                                  const lcDeviceTensor* v, const int32_t* kv_lengths, const lcDeviceTensor* out,
                                  float* lse, void* workspace, size_t workspace_bytes, lcStream stream) {
  return lchip::toLc(lchip::forward(cfg, q, k, v, kv_lengths, out, lse, workspace, workspace_bytes, stream));
}

lcError_t lcCrossAttentionBackward(const lcCrossAttentionConfig* cfg, const lcDeviceTensor* dout,
                                   const lcDeviceTensor* q, const lcDeviceTensor* k, const lcDeviceTensor* v,
                                   const lcDeviceTensor* out, const float* lse, const int32_t* kv_lengths,
                                   const lcDeviceTensor* dq, const lcDeviceTensor* dk, const lcDeviceTensor* dv,
                                   void* workspace, size_t workspace_bytes, lcStream stream) {
  return lchip::toLc(lchip::backward(cfg, dout, q, k, v, out, lse, kv_lengths, dq, dk, dv, workspace, workspace_bytes,
                                     stream));
}

}  // extern "C"
