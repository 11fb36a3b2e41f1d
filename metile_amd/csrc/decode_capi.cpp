// extern "C" boundary of the serving operators around the projections: block tables and slot maps,
// cache append, paged attention of one token and of chunks, copies, forks, freeing and compaction of
// pages, residual norms and log probabilities of tokens. Argument checks and launches only; no
// allocation of device memory, no synchronisation, no exceptions across the ABI.
#include "../../include/metile_amd.h"

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cfloat>
#include <cmath>
#include <cstdint>
#include <cstring>
#include <string>

#include "capi_internal.h"
#include "chunk_attention.h"
#include "common.h"
#include "paged.h"
#include "paged_pages.h"
#include "residual_norm.h"
#include "token_logprobs.h"

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

// ---- chunks ----

struct ChunkCall {
  mt::ChunkPlan plan;
  size_t plan_bytes, bytes;
};

int plan_chunks(const char* op, const mt_paged_cache* c, int tokens, int requests, int heads, int width,
                int window, ChunkCall* call) {
  if (const int st = check_cache(op, c)) return st;
  if (tokens < 1 || requests < 1) return refuse(op, "tokens and requests must be positive");
  if (heads < 1 || heads > kMaxHeads || heads % c->heads)
    return refuse(op, "query heads must be a positive multiple of the cache's");
  if (width < 1 || (int64_t)width * c->page_size > kInt31 - 64)
    return refuse(op, "block table width must be positive and hold fewer than 2^31 - 64 tokens");
  if (window < 0) return refuse(op, "window must not be negative");
  if ((int64_t)tokens * heads >= kInt31 ||
      (int64_t)tokens * heads / mt::kChunkTile + (int64_t)requests * c->heads >= (1 << 24) - (1 << 16))
    return refuse(op, "tokens * heads must be below 2^31, and tokens * heads / 128 + requests * cache "
                      "heads below 2^24 - 2^16");
  call->plan = mt::plan_chunk_attention(tokens, requests, c->heads, heads / c->heads, c->dim,
                                        (int64_t)width * c->page_size, window,
                                        mt::current_device_cus());
  const size_t ints = mt::kPlanHead + 3 * ((size_t)requests + 1);
  call->plan_bytes = (ints * 4 + 255) / 256 * 256;
  call->bytes = call->plan_bytes +
                (size_t)call->plan.parts * c->heads * mt::chunk_part_floats(c->dim) * 4;
  return MT_OK;
}

// ---- pages ----

// A page of one side of a cache as nested runs of 16-byte units.
mt::PageShape page_shape(const int64_t* strides, const mt_paged_cache* c) {
  const int64_t bytes = c->dtype == MT_FP8 ? 1 : 2;
  struct {
    uint32_t n;
    int64_t s;
  } level[2] = {{(uint32_t)c->page_size, strides[1] * bytes}, {(uint32_t)c->heads, strides[2] * bytes}};
  if (level[1].s > level[0].s) std::swap(level[0], level[1]);  // the outer one first
  mt::PageShape p{(uint32_t)(c->dim * bytes / 16), 1, 1, 0, 0, strides[0] * bytes};
  for (int i = 1; i >= 0; --i) {
    if (level[i].n == 1) continue;
    if (p.n1 == 1 && level[i].s == (int64_t)p.run * 16) {
      p.run *= level[i].n;
    } else if (p.n1 == 1) {
      p.n1 = level[i].n;
      p.s1 = level[i].s;
    } else {
      p.n0 = level[i].n;
      p.s0 = level[i].s;
    }
  }
  return p;
}

bool same_shape(const mt_paged_cache* a, const mt_paged_cache* b) {
  return a->pages == b->pages && a->page_size == b->page_size && a->heads == b->heads &&
         a->dim == b->dim && (a->dtype == MT_FP8) == (b->dtype == MT_FP8) &&
         !memcmp(a->key_strides, b->key_strides, sizeof a->key_strides) &&
         !memcmp(a->value_strides, b->value_strides, sizeof a->value_strides);
}

int check_table(const char* op, int requests, int width, int64_t stride, int page_size) {
  if (requests < 0 || requests >= 1 << 24)
    return refuse(op, "requests must not be negative, and below 2^24");
  if (page_size < 1 || width < 1 || (int64_t)width * page_size >= kInt31)
    return refuse(op, "page_size and width must be positive and hold fewer than 2^31 tokens");
  if (requests > 1 && stride < width) return refuse(op, "block table rows overlap");
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

size_t mt_paged_chunk_attention_workspace_bytes(const mt_paged_cache* cache, int tokens, int requests,
                                                int heads, int width, int window) {
  ChunkCall call;
  if (plan_chunks("mt_paged_chunk_attention_workspace_bytes", cache, tokens, requests, heads, width,
                  window, &call))
    return 0;
  return call.bytes;
}

int mt_paged_chunk_attention(const mt_paged_cache* cache, const mt_paged_chunk_attention_args* args,
                             void* workspace, size_t workspace_bytes, void* stream) {
  const char* op = "mt_paged_chunk_attention";
  if (!args) return refuse(op, "null arguments");
  const mt_paged_chunk_attention_args& in = *args;
  ChunkCall call;
  if (const int st = plan_chunks(op, cache, in.tokens, in.requests, in.heads, in.width, in.window, &call))
    return st;
  if (in.dtype != MT_BF16 && in.dtype != MT_F16)
    return refuse(op, "dtype must be MT_BF16 or MT_F16");
  if (cache->dtype != MT_FP8 && cache->dtype != in.dtype)
    return refuse(op, "a 16-bit cache must have the query's dtype");
  const float scale_log2 = in.scale * cache->key_scale * 1.4426950408889634f;
  if (!std::isfinite(scale_log2)) return refuse(op, "scale must be finite");
  if (!in.query || !in.block_tables || !in.lengths || !in.starts || !in.out)
    return refuse(op, "null pointer");
  if (!aligned16(in.query) || !aligned16(in.out) || !stride16(in.query_strides[0], 2) ||
      !stride16(in.query_strides[1], 2))
    return refuse(op, "query, its strides and out must be multiples of 16 bytes");
  if (in.requests > 1 && in.table_stride < 0)
    return refuse(op, "block table rows must be in order");
  if (!workspace || workspace_bytes < call.bytes)
    return mt::set_last_error(MT_ERR_WORKSPACE,
                              std::string(op) + ": workspace smaller than required");
  if (!aligned16(workspace)) return refuse(op, "workspace must be 16-byte aligned");
  const bool fp8 = cache->dtype == MT_FP8;
  const int64_t bytes = fp8 ? 1 : 2;
  mt::ChunkAttentionArgs a{};
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
  a.starts = in.starts;
  a.out = static_cast<uint16_t*>(in.out);
  a.lse = in.lse;
  a.plan = static_cast<int32_t*>(workspace);
  a.parts = reinterpret_cast<float*>(static_cast<unsigned char*>(workspace) + call.plan_bytes);
  a.tokens = in.tokens;
  a.requests = in.requests;
  a.kv_heads = cache->heads;
  a.group = in.heads / cache->heads;
  a.dim = cache->dim;
  a.pages = cache->pages;
  a.page_size = cache->page_size;
  a.width = in.width;
  a.window = in.window;
  a.target = call.plan.target;
  a.slots = call.plan.slots;
  a.most_tiles = call.plan.tiles;
  a.most_parts = call.plan.parts;
  // A scale below zero is the query's; one of zero stands for the smallest, whose products are as
  // good as none (zero times -inf, a masked score, would be no number).
  a.scale_log2 = std::max(std::fabs(scale_log2), FLT_MIN);
  a.flip = scale_log2 < 0.0f ? 0x80008000u : 0u;
  a.value_scale = cache->value_scale;
  a.narrow = true;
  for (const int64_t* strides : {cache->key_strides, cache->value_strides})
    a.narrow &= ((cache->pages - 1) * strides[0] + (cache->page_size - 1) * strides[1] + cache->dim) *
                    bytes <= (int64_t)UINT32_MAX;
  return launched(op, mt::launch_chunk_attention(a, in.dtype, fp8, static_cast<hipStream_t>(stream)));
}

int mt_paged_copy(const mt_paged_cache* const* caches, int num_caches, const mt_paged_copy_args* args,
                  void* stream) {
  const char* op = "mt_paged_copy";
  if (!args || (num_caches > 0 && !caches)) return refuse(op, "null arguments");
  if (num_caches < 0 || args->count < 0) return refuse(op, "counts must not be negative");
  for (int i = 0; i < num_caches; ++i)
    if (const int st = check_cache(op, caches[i])) return st;
  if (args->count == 0 || num_caches == 0) return MT_OK;
  if (!args->sources || !args->targets) return refuse(op, "null pointer");
  for (int i = 0; i < num_caches; ++i)
    if ((int64_t)caches[i]->page_size * caches[i]->heads * (caches[i]->dim / 8) >= kInt31)
      return refuse(op, "a page must be less than 2^31 chunks of eight values");
  for (int i = 0; i < num_caches;) {
    mt::PagedCopyArgs a{};
    int sides = 0;
    const mt_paged_cache* first = caches[i];
    for (; i < num_caches && sides < mt::kCopySides && same_shape(first, caches[i]); ++i) {
      a.side[sides++] = static_cast<unsigned char*>(caches[i]->key);
      a.side[sides++] = static_cast<unsigned char*>(caches[i]->value);
    }
    a.shape[0] = page_shape(first->key_strides, first);
    a.shape[1] = page_shape(first->value_strides, first);
    a.sources = args->sources;
    a.targets = args->targets;
    a.count = args->count;
    a.pages = first->pages;
    if (const int st = launched(op, mt::launch_paged_copy(a, sides, mt::current_device_cus(),
                                                          static_cast<hipStream_t>(stream))))
      return st;
  }
  return MT_OK;
}

int mt_paged_fork(const mt_paged_fork_args* args, void* stream) {
  const char* op = "mt_paged_fork";
  if (!args) return refuse(op, "null arguments");
  const mt_paged_fork_args& in = *args;
  if (const int st = check_table(op, in.requests, in.width, in.table_stride, in.page_size)) return st;
  if (in.forks < 0 || in.forks >= 1 << 23 || in.free_count < 0)
    return refuse(op, "counts must not be negative, and forks below 2^23");
  if (!in.taken || (in.free_count && !in.free_pages) || (in.requests && (!in.block_tables || !in.lengths)) ||
      (in.forks && (!in.sources || !in.targets || !in.copy_sources || !in.copy_targets)))
    return refuse(op, "null pointer");
  if (in.forks == 0)  // nothing is taken (by a kernel: a call may be captured)
    return launched(op, mt::launch_zero_int(in.taken, static_cast<hipStream_t>(stream)));
  mt::PagedForkArgs a{in.block_tables, in.table_stride, in.lengths, in.sources, in.targets, in.tokens,
                      in.free_pages, in.free_start, in.copy_sources, in.copy_targets, in.taken,
                      in.requests, in.width, in.free_count, in.page_size, in.forks};
  return launched(op, mt::launch_paged_fork(a, static_cast<hipStream_t>(stream)));
}

size_t mt_paged_free_workspace_bytes(int pages) {
  return pages < 1 ? 0 : mt::paged_free_work(pages);
}

int mt_paged_free(const mt_paged_free_args* args, void* workspace, size_t workspace_bytes,
                  void* stream) {
  const char* op = "mt_paged_free";
  if (!args) return refuse(op, "null arguments");
  const mt_paged_free_args& in = *args;
  if (const int st = check_table(op, in.requests, in.width, in.table_stride, in.page_size)) return st;
  if (in.pages < 1 || in.free_count < 0)
    return refuse(op, "pages must be positive and free_count not negative");
  if (!in.freed || !in.free_start || (in.free_count && !in.free_pages) ||
      (in.requests && (!in.block_tables || !in.lengths || !in.kept)))
    return refuse(op, "null pointer");
  if (!workspace || workspace_bytes < mt::paged_free_work(in.pages))
    return mt::set_last_error(MT_ERR_WORKSPACE,
                              std::string(op) + ": workspace smaller than required");
  if (!aligned16(workspace)) return refuse(op, "workspace must be 16-byte aligned");
  mt::PagedFreeArgs a{in.block_tables, in.table_stride, in.lengths, in.kept, in.free_pages,
                      in.free_start, in.freed, static_cast<unsigned char*>(workspace), in.requests,
                      in.width, in.free_count, in.page_size, in.pages};
  return launched(op, mt::launch_paged_free(a, static_cast<hipStream_t>(stream)));
}

size_t mt_paged_compact_workspace_bytes(int pages) {
  return pages < 1 ? 0 : mt::paged_compact_work(pages);
}

int mt_paged_compact(const mt_paged_compact_args* args, void* workspace, size_t workspace_bytes,
                     void* stream) {
  const char* op = "mt_paged_compact";
  if (!args) return refuse(op, "null arguments");
  const mt_paged_compact_args& in = *args;
  if (const int st = check_table(op, in.requests, in.width, in.table_stride, in.page_size)) return st;
  if (in.pages < 1 || in.free_count < 0)
    return refuse(op, "pages must be positive and free_count not negative");
  if (in.most_moves < std::min<int64_t>(in.pages / 2, (int64_t)in.requests * in.width))
    return refuse(op, "most_moves must be at least min(pages / 2, requests * width)");
  if (!in.moves || !in.free_start || (in.free_count && (!in.free_pages || !in.new_free)) ||
      (in.most_moves && (!in.sources || !in.targets)) ||
      (in.requests && (!in.block_tables || !in.lengths || !in.new_tables)))
    return refuse(op, "null pointer");
  if (!workspace || workspace_bytes < mt::paged_compact_work(in.pages))
    return mt::set_last_error(MT_ERR_WORKSPACE,
                              std::string(op) + ": workspace smaller than required");
  if (!aligned16(workspace)) return refuse(op, "workspace must be 16-byte aligned");
  mt::PagedCompactArgs a{in.block_tables, in.table_stride, in.lengths, in.free_pages, in.free_start,
                         in.new_tables, in.new_free, in.sources, in.targets, in.moves,
                         static_cast<unsigned char*>(workspace), in.requests, in.width, in.free_count,
                         in.page_size, in.pages, in.most_moves};
  return launched(op, mt::launch_paged_compact(a, static_cast<hipStream_t>(stream)));
}

size_t mt_token_logprobs_workspace_bytes(int rows, int vocab, int top) {
  if (rows < 1 || vocab < 1 || vocab > 1 << 24 || top < 0 || top > mt::kLogprobsMostTop) return 0;
  const mt::LogprobsPlan plan = mt::plan_token_logprobs(rows, vocab, mt::current_device_cus());
  return plan.num_parts == 1 ? 0 : (size_t)rows * plan.num_parts * mt::logprobs_part_bytes(top);
}

int mt_token_logprobs(const mt_token_logprobs_args* args, void* workspace, size_t workspace_bytes,
                      void* stream) {
  const char* op = "mt_token_logprobs";
  if (!args) return refuse(op, "null arguments");
  const mt_token_logprobs_args& in = *args;
  if (in.dtype != MT_BF16 && in.dtype != MT_F16 && in.dtype != MT_F32)
    return refuse(op, "dtype must be MT_BF16, MT_F16 or MT_F32");
  if (in.rows < 0) return refuse(op, "rows must not be negative");
  if (in.vocab < 1 || in.vocab > 1 << 24) return refuse(op, "vocab must be 1 to 2^24");
  if (in.top < 0 || in.top > std::min(in.vocab, mt::kLogprobsMostTop))
    return refuse(op, "top must be 0 to 32, and at most vocab");
  const float inverse = 1.0f / in.temperature;
  if (!(in.temperature >= 1e-6f && in.temperature <= 1e6f))
    return refuse(op, "temperature must be 1e-6 to 1e6");
  if (in.row_stride < 0) return refuse(op, "row_stride must not be negative");
  if (in.rows == 0) return MT_OK;
  if (!in.logits || !in.entropies || (in.tokens && (!in.logprobs || !in.ranks)) ||
      (in.top && (!in.top_logprobs || !in.top_tokens)))
    return refuse(op, "null pointer");
  const mt::LogprobsPlan plan =
      mt::plan_token_logprobs(in.rows, in.vocab, mt::current_device_cus());
  const size_t need = mt_token_logprobs_workspace_bytes(in.rows, in.vocab, in.top);
  if (need && (!workspace || workspace_bytes < need))
    return mt::set_last_error(MT_ERR_WORKSPACE,
                              std::string(op) + ": workspace smaller than required");
  if (need && !aligned16(workspace)) return refuse(op, "workspace must be 16-byte aligned");
  mt::LogprobsArgs a{in.logits, in.row_stride, in.tokens, in.logprobs, in.entropies, in.ranks,
                     in.top_logprobs, in.top_tokens, static_cast<unsigned char*>(workspace), in.rows,
                     in.vocab, in.top, plan.threads, plan.part_batches, plan.num_parts, inverse};
  return launched(op, mt::launch_token_logprobs(a, in.dtype, static_cast<hipStream_t>(stream)));
}

}  // extern "C"
