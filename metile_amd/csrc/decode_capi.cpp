// extern "C" boundary of the decode-step operators around the projections: block tables and slot
// maps, cache append, paged attention and residual norms. Argument checks and launches only; no
// allocation of device memory, no synchronisation, no exceptions across the ABI.
#include "../../include/metile_amd.h"

#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdint>
#include <string>

#include "capi_internal.h"
#include "paged.h"
#include "residual_norm.h"

namespace {

constexpr int64_t kInt31 = (int64_t)1 << 31;
constexpr int kMaxHeads = 65536;

int refuse(const char* op, const char* what) {
  return mt::set_last_error(MT_ERR_INVALID_ARGUMENT, std::string(op) + ": " + what);
}

int launched(const char* op, hipError_t e) {
  if (e == hipSuccess) return MT_OK;
  return mt::set_last_error(MT_ERR_HIP, std::string(op) + ": " + hipGetErrorString(e));
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// Strides of `bytes`-wide elements that are whole 16-byte steps and not negative.
bool stride16(int64_t stride, int bytes) {
  return stride >= 0 && stride < kInt31 * 256 && stride * bytes % 16 == 0;
}

int check_cache(const char* op, const mt_paged_cache* c) {
  if (!c) return refuse(op, "null cache");
  if (c->dtype != MT_BF16 && c->dtype != MT_F16 && c->dtype != MT_FP8)
    return refuse(op, "cache dtype must be MT_BF16, MT_F16 or MT_FP8");
  if (c->pages < 1 || c->page_size < 1 || (int64_t)c->pages * c->page_size >= kInt31)
    return refuse(op, "pages and page_size must be positive and hold fewer than 2^31 tokens");
  if (c->heads < 1 || c->heads > kMaxHeads) return refuse(op, "cache heads must be positive");
  if (c->dim < 16 || c->dim > 256 || c->dim % 16)
    return refuse(op, "head dim must be a multiple of 16 up to 256");
  const int bytes = c->dtype == MT_FP8 ? 1 : 2;
  for (int i = 0; i < 3; ++i)
    if (!stride16(c->key_strides[i], bytes) || !stride16(c->value_strides[i], bytes))
      return refuse(op, "cache strides must be multiples of 16 bytes");
  for (int i = 0; i < 2; ++i)  // the kernels multiply page numbers and slots with 32-bit strides
    if (c->key_strides[i] * bytes > UINT32_MAX || c->value_strides[i] * bytes > UINT32_MAX)
      return refuse(op, "page and token strides of a cache must be below 4 GiB");
  if (!c->key || !c->value) return refuse(op, "null cache pointer");
  if (!aligned16(c->key) || !aligned16(c->value))
    return refuse(op, "cache must be 16-byte aligned");
  const float scales[2] = {c->key_scale, c->value_scale};
  for (float s : scales)
    if (!(s > 0.0f) || !std::isnormal(s) || !std::isnormal(1.0f / s))
      return refuse(op, "cache scales must be positive and normal");
  if (c->dtype != MT_FP8 && (c->key_scale != 1.0f || c->value_scale != 1.0f))
    return refuse(op, "a 16-bit cache has scales of 1");
  return MT_OK;
}

// Units of the longest request that the table holds.
int64_t most_units(int64_t most, int window) {
  if (window > 0 && window + (mt::kAttentionUnit - 1ll) < most)
    most = window + (mt::kAttentionUnit - 1ll);
  const int64_t n = (most + mt::kAttentionUnit - 1) / mt::kAttentionUnit;
  return (n > 0 ? n : 1) + mt::kAttentionRowCost;
}

constexpr int64_t kMostUnits = kInt31 - 65536;  // the kernel adds up to its waves in 32 bits

struct AttentionPlan {
  int workgroups;
  size_t bytes;
};

int plan_attention(const char* op, const mt_paged_cache* c, int requests, int heads, int width,
                   int window, AttentionPlan* plan) {
  if (const int st = check_cache(op, c)) return st;
  if (requests < 1) return refuse(op, "requests must be positive");
  if (heads < 1 || heads > kMaxHeads || heads % c->heads)
    return refuse(op, "query heads must be a positive multiple of the cache's");
  // (64 less than 2^31: the kernel counts to the end of the last unit in 32 bits)
  if (width < 1 || (int64_t)width * c->page_size > kInt31 - 64)
    return refuse(op, "block table width must be positive and hold fewer than 2^31 - 64 tokens");
  if (window < 0) return refuse(op, "window must not be negative");
  const int group = heads / c->heads, head_tiles = (group + 15) / 16;
  const int64_t units = most_units((int64_t)width * c->page_size, window);
  const int64_t rows = (int64_t)c->heads * head_tiles;
  if (units * rows > kMostUnits || units * rows * requests > kMostUnits)
    return refuse(op, "requests, heads and table width make more than 2^31 - 2^16 units of work");
  plan->workgroups =
      mt::paged_attention_workgroups(mt::current_device_cus(), c->dim,
                                     units * rows * requests);
  plan->bytes = mt::kWorkspaceCounterBytes +
                (size_t)plan->workgroups * 2 * mt::paged_attention_slot_floats(group, c->dim) * 4;
  return MT_OK;
}

}  // namespace

extern "C" {

int mt_paged_tables(const mt_paged_tables_args* args, void* stream) {
  const char* op = "mt_paged_tables";
  if (!args) return refuse(op, "null arguments");
  const mt_paged_tables_args& in = *args;
  if (in.requests < 0 || in.tokens < 0 || in.free_count < 0)
    return refuse(op, "counts must not be negative");
  if (in.page_size < 1 || in.width < 1 || (int64_t)in.width * in.page_size >= kInt31)
    return refuse(op, "page_size and width must be positive and hold fewer than 2^31 tokens");
  if (in.requests > 1 && in.table_stride < in.width) return refuse(op, "block table rows overlap");
  if ((in.requests && (!in.cached || !in.new_tokens || !in.block_tables || !in.lengths)) ||
      (in.free_count && !in.free_pages) ||
      (in.tokens && (!in.slots || !in.positions || !in.token_requests)) || !in.starts || !in.taken)
    return refuse(op, "null pointer");
  mt::PagedTablesArgs a{};
  a.cached = in.cached;
  a.fresh = in.new_tokens;
  a.tables = in.block_tables;
  a.table_stride = in.table_stride;
  a.free_pages = in.free_pages;
  a.free_start = in.free_start;
  a.slots = in.slots;
  a.positions = in.positions;
  a.requests = in.token_requests;
  a.starts = in.starts;
  a.lengths = in.lengths;
  a.taken = in.taken;
  a.num_requests = in.requests;
  a.width = in.width;
  a.page_size = in.page_size;
  a.free_count = in.free_count;
  a.tokens = in.tokens;
  return launched(op, mt::launch_paged_tables(a, mt::current_device_cus(),
                                              static_cast<hipStream_t>(stream)));
}

int mt_paged_append(const mt_paged_cache* cache, const mt_paged_append_args* args, void* stream) {
  const char* op = "mt_paged_append";
  if (const int st = check_cache(op, cache)) return st;
  if (!args) return refuse(op, "null arguments");
  const mt_paged_append_args& in = *args;
  if (in.dtype != MT_BF16 && in.dtype != MT_F16)
    return refuse(op, "dtype must be MT_BF16 or MT_F16");
  if (cache->dtype != MT_FP8 && cache->dtype != in.dtype)
    return refuse(op, "a 16-bit cache must have the rows' dtype");
  if (in.tokens < 0 || in.tokens >= kInt31 ||
      in.tokens * cache->heads * (cache->dim / 8) >= kInt31)
    return refuse(op, "tokens must not be negative, and tokens * heads * dim / 8 below 2^31");
  if (in.tokens == 0) return MT_OK;
  if (!in.key || !in.value || !in.slots) return refuse(op, "null pointer");
  if (!aligned16(in.key) || !aligned16(in.value) || !stride16(in.key_strides[0], 2) ||
      !stride16(in.key_strides[1], 2) || !stride16(in.value_strides[0], 2) ||
      !stride16(in.value_strides[1], 2))
    return refuse(op, "rows and their strides must be multiples of 16 bytes");
  const bool fp8 = cache->dtype == MT_FP8;
  const int bytes = fp8 ? 1 : 2;
  mt::PagedAppendArgs a{};
  for (int i = 0; i < 2; ++i) {
    mt::PagedSide& s = a.side[i];
    const int64_t* strides = i ? cache->value_strides : cache->key_strides;
    const int64_t* row_strides = i ? in.value_strides : in.key_strides;
    s.cache = static_cast<unsigned char*>(i ? cache->value : cache->key);
    s.page_stride = (uint32_t)(strides[0] * bytes);
    s.slot_stride = (uint32_t)(strides[1] * bytes);
    s.head_stride = strides[2] * bytes;
    s.rows = static_cast<const unsigned char*>(i ? in.value : in.key);
    s.row_stride = row_strides[0] * 2;
    s.row_head_stride = row_strides[1] * 2;
    s.scale = i ? cache->value_scale : cache->key_scale;
    s.inv_scale = 1.0f / s.scale;
  }
  a.slots = in.slots;
  a.tokens = in.tokens;
  a.pages = cache->pages;
  a.page_size = cache->page_size;
  a.heads = cache->heads;
  a.dim = cache->dim;
  a.by_row = mt::div_magic((uint32_t)(cache->heads * (cache->dim / 8)));
  a.by_head = mt::div_magic((uint32_t)(cache->dim / 8));
  a.by_page = mt::div_magic((uint32_t)cache->page_size);
  return launched(op, mt::launch_paged_append(a, in.dtype, fp8, static_cast<hipStream_t>(stream)));
}

size_t mt_paged_attention_workspace_bytes(const mt_paged_cache* cache, int requests, int heads,
                                          int width, int window) {
  AttentionPlan plan;
  if (plan_attention("mt_paged_attention_workspace_bytes", cache, requests, heads, width, window,
                     &plan))
    return 0;
  return plan.bytes;
}

int mt_paged_attention(const mt_paged_cache* cache, const mt_paged_attention_args* args,
                       void* workspace, size_t workspace_bytes, void* stream) {
  const char* op = "mt_paged_attention";
  if (!args) return refuse(op, "null arguments");
  const mt_paged_attention_args& in = *args;
  AttentionPlan plan;
  if (const int st =
          plan_attention(op, cache, in.requests, in.heads, in.width, in.window, &plan))
    return st;
  if (in.dtype != MT_BF16 && in.dtype != MT_F16)
    return refuse(op, "dtype must be MT_BF16 or MT_F16");
  if (cache->dtype != MT_FP8 && cache->dtype != in.dtype)
    return refuse(op, "a 16-bit cache must have the query's dtype");
  const float scale_log2 = in.scale * cache->key_scale * 1.4426950408889634f;
  if (!std::isfinite(scale_log2)) return refuse(op, "scale must be finite");
  if (!in.query || !in.block_tables || !in.lengths || !in.out) return refuse(op, "null pointer");
  if (!aligned16(in.query) || !aligned16(in.out) || !stride16(in.query_strides[0], 2) ||
      !stride16(in.query_strides[1], 2))
    return refuse(op, "query, its strides and out must be multiples of 16 bytes");
  if (in.requests > 1 && in.table_stride < 0)
    return refuse(op, "block table rows must be in order");
  if (!workspace || workspace_bytes < plan.bytes)
    return mt::set_last_error(MT_ERR_WORKSPACE,
                              std::string(op) + ": workspace smaller than required");
  const bool fp8 = cache->dtype == MT_FP8;
  const int64_t bytes = fp8 ? 1 : 2;
  mt::PagedAttentionArgs a{};
  a.query = static_cast<const uint16_t*>(in.query);
  a.q_row_stride = in.query_strides[0];
  a.q_head_stride = in.query_strides[1];
  a.key = static_cast<const unsigned char*>(cache->key);
  a.value = static_cast<const unsigned char*>(cache->value);
  a.k_page = (uint32_t)(cache->key_strides[0] * bytes);
  a.k_slot = (uint32_t)(cache->key_strides[1] * bytes);
  a.k_head = cache->key_strides[2] * bytes;
  a.v_page = (uint32_t)(cache->value_strides[0] * bytes);
  a.v_slot = (uint32_t)(cache->value_strides[1] * bytes);
  a.v_head = cache->value_strides[2] * bytes;
  a.tables = in.block_tables;
  a.table_stride = in.table_stride;
  a.lengths = in.lengths;
  a.out = static_cast<uint16_t*>(in.out);
  a.lse = in.lse;
  a.counters = static_cast<uint32_t*>(workspace);
  a.partial = reinterpret_cast<float*>(static_cast<unsigned char*>(workspace) +
                                       mt::kWorkspaceCounterBytes);
  a.requests = in.requests;
  a.kv_heads = cache->heads;
  a.group = in.heads / cache->heads;
  a.head_tiles = (a.group + 15) / 16;
  a.dim = cache->dim;
  a.pages = cache->pages;
  a.page_size = cache->page_size;
  a.width = in.width;
  a.window = in.window;
  a.scale_log2 = scale_log2;
  a.value_scale = cache->value_scale;
  return launched(op, mt::launch_paged_attention(a, in.dtype, fp8, plan.workgroups,
                                                 static_cast<hipStream_t>(stream)));
}

int mt_residual_norm(const mt_residual_norm_args* args, void* stream) {
  const char* op = "mt_residual_norm";
  if (!args) return refuse(op, "null arguments");
  const mt_residual_norm_args& in = *args;
  if (in.dtype != MT_BF16 && in.dtype != MT_F16)
    return refuse(op, "dtype must be MT_BF16 or MT_F16");
  if (in.residual_dtype != in.dtype && in.residual_dtype != MT_F32)
    return refuse(op, "residual_dtype must be dtype or MT_F32");
  if (in.kind != MT_NORM_RMS && in.kind != MT_NORM_LAYER)
    return refuse(op, "kind must be MT_NORM_RMS or MT_NORM_LAYER");
  if (in.width < 1 || in.width > mt::kNormMaxWidth) return refuse(op, "width must be 1 to 65536");
  if (in.rows < 0) return refuse(op, "rows must not be negative");
  if (!(in.eps >= 0.0f) || !std::isfinite(in.eps))
    return refuse(op, "eps must be finite and >= 0");
  if (!std::isfinite(in.residual_scale)) return refuse(op, "residual_scale must be finite");
  if (in.gate && (in.gate_rows < 1 || in.gate_stride < 0))
    return refuse(op, "gate_rows must be positive and gate_stride not negative");
  if (in.rows == 0) return MT_OK;
  if (!in.residual || !in.weight || !in.normed) return refuse(op, "null pointer");
  mt::ResidualNormArgs a{};
  a.residual = in.residual;
  a.block = static_cast<const uint16_t*>(in.block);
  a.weight = static_cast<const uint16_t*>(in.weight);
  a.bias = static_cast<const uint16_t*>(in.bias);
  a.post_weight = static_cast<const uint16_t*>(in.post_weight);
  a.post_bias = static_cast<const uint16_t*>(in.post_bias);
  a.gate = static_cast<const uint16_t*>(in.gate);
  a.residual_out = in.residual_out;
  a.normed = static_cast<uint16_t*>(in.normed);
  a.residual_stride = in.residual_stride;
  a.block_stride = in.block_stride;
  a.gate_stride = in.gate_stride;
  a.rows = in.rows;
  a.width = in.width;
  a.gate_rows = in.gate ? in.gate_rows : 1;
  a.gate_scalar = in.gate_scalar;
  a.scale = in.residual_scale;
  a.eps = in.eps;
  return launched(op, mt::launch_residual_norm(a, in.dtype, in.residual_dtype == MT_F32,
                                               in.kind == MT_NORM_LAYER, mt::current_device_cus(),
                                               static_cast<hipStream_t>(stream)));
}

}  // extern "C"
