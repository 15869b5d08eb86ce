// kv_cache.cpp -- entry points of the 8-bit paged key/value cache
// (kernels/kv_cache.hip).
#include <algorithm>
#include <cmath>

#include "device_ops.hpp"

namespace lchip {
namespace {

constexpr const char* kOp = "kv cache";
constexpr std::size_t kMost = std::size_t{1} << 30;
constexpr std::size_t kMostProblems = std::size_t{1} << 24;
// Workgroups of four waves that run at once.
constexpr std::size_t kSlots = 512;
constexpr std::size_t kRows = 16;  // query rows of a workgroup

Status checkCache(const lcKvCache* c) {
  if (c == nullptr) {
    return fail(Status::kInvalidValue, "kv cache: null cache");
  }
  if (c->kv_heads == 0 || c->head_dim == 0) {
    return fail(Status::kInvalidValue, "kv cache: zero heads or head_dim");
  }
  if (c->head_dim % 16 != 0 || c->head_dim > 128) {
    return fail(Status::kNotSupported, "kv cache: head_dim a multiple of 16, at most 128");
  }
  if (c->pages > kMost || c->kv_heads > 65535) {
    return fail(Status::kNotSupported, "kv cache: pool too large");
  }
  if (c->pages != 0) {
    if (c->k_pages == nullptr || c->v_pages == nullptr || c->k_scales == nullptr || c->v_scales == nullptr) {
      return fail(Status::kInvalidValue, "kv cache: null pages or scales");
    }
    if (reinterpret_cast<std::uintptr_t>(c->k_pages) % 16 != 0 ||
        reinterpret_cast<std::uintptr_t>(c->v_pages) % 16 != 0) {
      return fail(Status::kInvalidValue, "kv cache: pages must be 16-byte aligned");
    }
    if (reinterpret_cast<std::uintptr_t>(c->k_scales) % 4 != 0 ||
        reinterpret_cast<std::uintptr_t>(c->v_scales) % 4 != 0) {
      return fail(Status::kInvalidValue, "kv cache: scales must be aligned to their elements");
    }
  }
  return Status::kSuccess;
}

Status checkTable(const lcKvCache& c, const std::int32_t* table, std::size_t batch, std::size_t width,
                  std::int64_t stride) {
  if (batch == 0 || width == 0) {
    return Status::kSuccess;
  }
  if (table == nullptr) {
    return fail(Status::kInvalidValue, "kv cache: null block table");
  }
  if (batch > 1 && (stride < 0 || stride > (std::int64_t{1} << 40))) {
    return fail(Status::kInvalidValue, "kv cache: the block table's stride");
  }
  if (c.pages == 0) {
    return fail(Status::kInvalidValue, "kv cache: a block table and a pool without pages");
  }
  return Status::kSuccess;
}

Status poolOnDevice(const DeviceCall& call, const lcKvCache& c) {
  LC_TRY(call.onDevice(c.k_pages, "k_pages"));
  LC_TRY(call.onDevice(c.v_pages, "v_pages"));
  LC_TRY(call.onDevice(c.k_scales, "k_scales"));
  return call.onDevice(c.v_scales, "v_scales");
}

Status store(const lcKvCache* cache, std::size_t batch, std::size_t kv_len, lcDataType dtype, const lcDeviceTensor* k,
             const lcDeviceTensor* v, const std::int32_t* table, std::size_t width, std::int64_t stride,
             const std::int32_t* lengths, lcStream stream) {
  LC_TRY(checkCache(cache));
  const lcKvCache& c = *cache;
  if (!validDtype(dtype)) {
    return fail(Status::kInvalidValue, "kv cache: dtype must be f32, bf16 or f16");
  }
  if (batch > 65535 || kv_len > std::size_t{65535} * kern::kKvPage) {
    return fail(Status::kNotSupported, "kv cache: shape too large");
  }
  kern::KvStoreArgs a{};
  bool aligned = true;
  LC_TRY(takeTensor(kOp, "k", k, batch, c.kv_heads, kv_len, c.head_dim, dtype, false, &a.k, &aligned));
  LC_TRY(takeTensor(kOp, "v", v, batch, c.kv_heads, kv_len, c.head_dim, dtype, false, &a.v, &aligned));
  const std::size_t need = (kv_len + kern::kKvPage - 1) / kern::kKvPage;
  if (width < need) {
    return fail(Status::kInvalidValue, "kv cache: the block table holds " + std::to_string(width) + " pages a row, " +
                                           std::to_string(need) + " needed");
  }
  LC_TRY(checkTable(c, table, batch, need, stride));
  DeviceCall call;
  LC_TRY(call.open(kOp, c.trusted_pointers != 0));
  if (batch == 0 || kv_len == 0) {
    return Status::kSuccess;
  }
  LC_TRY(call.onDevice(a.k.p, "k"));
  LC_TRY(call.onDevice(a.v.p, "v"));
  LC_TRY(call.onDevice(table, "the block table"));
  LC_TRY(call.onDevice(lengths, "kv_lengths"));
  LC_TRY(poolOnDevice(call, c));
  a.lengths = lengths;
  a.table = table;
  a.table_stride = batch > 1 ? stride : 0;
  a.k_pages = static_cast<std::uint8_t*>(c.k_pages);
  a.v_pages = static_cast<std::uint8_t*>(c.v_pages);
  a.k_scales = c.k_scales;
  a.v_scales = c.v_scales;
  a.batch = static_cast<int>(batch);
  a.heads = static_cast<int>(c.kv_heads);
  a.kv_len = static_cast<int>(kv_len);
  a.d = static_cast<int>(c.head_dim);
  a.pages = static_cast<int>(c.pages);
  LC_HIP_TRY(kern::kvStore(a, dtypeOf(dtype), aligned, static_cast<hipStream_t>(stream)));
  return Status::kSuccess;
}

struct AttnPlan {
  int splits = 1;
  std::size_t rows = 0;
  std::size_t width = 0;
  std::size_t bytes() const {
    return splits > 1 ? static_cast<std::size_t>(splits) * rows * (width + 2) * sizeof(float) : 0;
  }
};

Status checkAttn(const lcKvCache* cache, const lcKvAttentionConfig* cfg, AttnPlan* plan) {
  LC_TRY(checkCache(cache));
  if (cfg == nullptr) {
    return fail(Status::kInvalidValue, "kv cache: null config");
  }
  if (cfg->heads == 0 || cfg->heads % cache->kv_heads != 0) {
    return fail(Status::kInvalidValue, "kv cache: heads must be a multiple of the cache's kv_heads");
  }
  if (!validDtype(cfg->dtype)) {
    return fail(Status::kInvalidValue, "kv cache: dtype must be f32, bf16 or f16");
  }
  if (!std::isfinite(cfg->scale * kLog2e)) {
    return fail(Status::kInvalidValue, "kv cache: scale is not finite in exp2 units");
  }
  const std::size_t group = cfg->heads / cache->kv_heads;
  // 256 threads a problem, and a launch has less than 2^32 a dimension.
  if (cfg->batch > kMost || cfg->heads > kMost || cfg->q_len > kMost || cfg->batch * cache->kv_heads >= kMostProblems ||
      group * cfg->q_len > kRows * 65535 || cfg->table_width > kMost / kern::kKvPage) {
    return fail(Status::kNotSupported, "kv cache: shape too large");
  }
  plan->rows = cfg->batch * cfg->heads * cfg->q_len;
  plan->width = static_cast<std::size_t>(kern::kXAttnWidth(static_cast<int>(cache->head_dim)));
  const std::size_t blocks = cfg->batch * cache->kv_heads * ((group * cfg->q_len + kRows - 1) / kRows);
  // A split has at least a page for each of its four waves.  Rows differ in
  // length and the host does not know by how much: tables that are split to fill
  // the chip are split twice as often when they are long, so that short rows'
  // workgroups make room.  us, once -> twice, 32 rows x 8 heads of 128 pages: 64
  // to 128 in use 76 -> 71, one row of 128 among rows of 16 63 -> 42, all in use
  // 86 -> 88.  Where the blocks fill the chip unsplit a second share only adds a
  // join and its workspace: 64 x 8 heads of 64 pages 83 -> 87, half in use 69 ->
  // 71; 64 rows of 16 x 32 heads 183 -> 307, of 512 x 4 x 32 94 -> 122.
  const std::size_t quads = (cfg->table_width + 3) / 4;
  const int splits = splitCount(blocks, quads, kSlots, 1.0, 3.0);
  plan->splits = splits > 1 && quads >= 8u * splits ? 2 * splits : splits;
  return Status::kSuccess;
}

Status attention(const lcKvCache* cache, const lcKvAttentionConfig* cfg, const lcDeviceTensor* q,
                 const std::int32_t* table, std::int64_t stride, const std::int32_t* lengths,
                 const lcDeviceTensor* out, float* lse, void* workspace, std::size_t workspace_bytes,
                 lcStream stream) {
  AttnPlan plan;
  LC_TRY(checkAttn(cache, cfg, &plan));
  const lcKvCache& c = *cache;
  kern::KvAttnArgs a{};
  bool q_aligned = true;
  bool o_aligned = true;
  LC_TRY(takeTensor(kOp, "q", q, cfg->batch, cfg->heads, cfg->q_len, c.head_dim, cfg->dtype, false, &a.q, &q_aligned));
  LC_TRY(takeTensor(kOp, "out", out, cfg->batch, cfg->heads, cfg->q_len, c.head_dim, cfg->dtype, true, &a.o,
                    &o_aligned));
  LC_TRY(checkTable(c, table, cfg->batch, cfg->table_width, stride));
  DeviceCall call;
  LC_TRY(call.open(kOp, c.trusted_pointers != 0));
  if (plan.rows == 0) {
    return Status::kSuccess;
  }
  if (plan.bytes() != 0) {
    if (workspace == nullptr || workspace_bytes < plan.bytes()) {
      return fail(Status::kInvalidValue, "kv cache: the workspace needs " + std::to_string(plan.bytes()) + " bytes, " +
                                             std::to_string(workspace == nullptr ? 0 : workspace_bytes) + " given");
    }
    if (reinterpret_cast<std::uintptr_t>(workspace) % 16 != 0) {
      return fail(Status::kInvalidValue, "kv cache: the workspace is not 16-byte aligned");
    }
    LC_TRY(call.onDevice(workspace, "the workspace"));
  }
  LC_TRY(call.onDevice(a.q.p, "q"));
  LC_TRY(call.onDevice(a.o.p, "out"));
  LC_TRY(call.onDevice(lse, "lse"));
  LC_TRY(call.onDevice(table, "the block table"));
  LC_TRY(call.onDevice(lengths, "kv_lengths"));
  LC_TRY(poolOnDevice(call, c));
  a.lse = lse;
  a.lengths = lengths;
  a.table = table;
  a.table_stride = cfg->batch > 1 ? stride : 0;
  a.k_pages = static_cast<const std::uint8_t*>(c.k_pages);
  a.v_pages = static_cast<const std::uint8_t*>(c.v_pages);
  a.k_scales = c.k_scales;
  a.v_scales = c.v_scales;
  a.batch = static_cast<int>(cfg->batch);
  a.heads = static_cast<int>(cfg->heads);
  a.kv_heads = static_cast<int>(c.kv_heads);
  a.q_len = static_cast<int>(cfg->q_len);
  a.kv_len = static_cast<int>(cfg->table_width * kern::kKvPage);
  a.d = static_cast<int>(c.head_dim);
  a.pages = static_cast<int>(c.pages);
  const float scale = cfg->scale != 0.0f ? cfg->scale : 1.0f / std::sqrt(static_cast<float>(c.head_dim));
  a.c = scale * kLog2e;
  a.aligned = q_aligned ? 1 : 0;
  a.splits = plan.splits;
  a.part = static_cast<float*>(workspace);
  a.stats = a.splits > 1 ? a.part + static_cast<std::size_t>(a.splits) * plan.rows * plan.width : nullptr;
  traceOpDispatch(TraceOp::kAttentionForward, Device::kHIP, Device::kHIP, false,
                  cfg->q_len * cfg->table_width * kern::kKvPage * c.head_dim);
  const hipStream_t s = static_cast<hipStream_t>(stream);
  LC_HIP_TRY(kern::kvAttention(a, dtypeOf(cfg->dtype), s));
  if (a.splits > 1) {
    kern::XAttnArgs j{};
    j.o = a.o;
    j.lse = a.lse;
    j.batch = a.batch;
    j.heads = a.heads;
    j.kv_heads = a.kv_heads;
    j.q_len = a.q_len;
    j.d = a.d;
    j.splits = a.splits;
    j.part = a.part;
    j.stats = a.stats;
    LC_HIP_TRY(kern::crossAttentionJoin(j, dtypeOf(cfg->dtype), s));
  }
  return Status::kSuccess;
}

}  // namespace
}  // namespace lchip

extern "C" {

lcError_t lcKvCacheStore(const lcKvCache* cache, size_t batch, size_t kv_len, lcDataType dtype,
                         const lcDeviceTensor* k, const lcDeviceTensor* v, const int32_t* block_table,
                         size_t table_width, int64_t table_stride, const int32_t* kv_lengths, lcStream stream) {
  return lchip::toLc(lchip::store(cache, batch, kv_len, dtype, k, v, block_table, table_width, table_stride,
                                  kv_lengths, stream));
}

lcError_t lcKvCacheAttentionWorkspaceSize(const lcKvCache* cache, const lcKvAttentionConfig* cfg, size_t* bytes) {
  using namespace lchip;
  if (bytes == nullptr) {
    return toLc(fail(Status::kInvalidValue, "kv cache: null output"));
  }
  *bytes = 0;
  AttnPlan plan;
  const Status st = checkAttn(cache, cfg, &plan);
  if (st == Status::kSuccess) {
    *bytes = plan.bytes();
  }
  return toLc(st);
}

lcError_t lcKvCacheAttention(const lcKvCache* cache, const lcKvAttentionConfig* cfg, const lcDeviceTensor* q,
                             const int32_t* block_table, int64_t table_stride, const int32_t* kv_lengths,
                             const lcDeviceTensor* out, float* lse, void* workspace, size_t workspace_bytes,
                             lcStream stream) {
  return lchip::toLc(lchip::attention(cache, cfg, q, block_table, table_stride, kv_lengths, out, lse, workspace,
                                      workspace_bytes, stream));
}

}  // extern "C"
