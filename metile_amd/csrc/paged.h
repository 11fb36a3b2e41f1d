// Host-visible launch interfaces of the paged key-value cache: block tables and slot maps, the
// append of a step's keys and values, and decode attention over the pages.
#pragma once

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace mt {

// Division of n in [0, 2^31) by a constant d in [1, 2^31): n / d = (2 n * mul) >> (32 + shift),
// exact, since mul = ceil(2^(31 + shift) / d) with shift = ceil(log2 d) errs by less than d <=
// 2^shift.
struct DivMagic {
  uint32_t mul, shift;
};
inline DivMagic div_magic(uint32_t d) {
  uint32_t s = 0;
  while ((1ull << s) < d) ++s;
  return {(uint32_t)(((1ull << (31 + s)) + d - 1) / d), s};
}
__device__ __forceinline__ uint32_t div_by(uint32_t n, DivMagic m) {
  return __umulhi(2 * n, m.mul) >> m.shift;
}

struct PagedTablesArgs {
  const int32_t* cached;   // [R] tokens already in the cache
  const int32_t* fresh;    // [R] new tokens of the step
  int32_t* tables;         // [R, width], rows `table_stride` entries apart
  int64_t table_stride;
  const int32_t* free_pages;  // [free_count]
  const int32_t* free_start;  // first entry of free_pages to take, or null for 0
  int64_t* slots;          // [tokens]
  int32_t* positions;      // [tokens]
  int32_t* requests;       // [tokens]
  int32_t* starts;         // [R + 1]
  int32_t* lengths;        // [R]
  int32_t* taken;          // [1] pages the step takes
  int32_t num_requests, width, page_size, free_count, tokens;
};
hipError_t launch_paged_tables(const PagedTablesArgs& a, int cus, hipStream_t stream);

// One side (keys or values) of a cache and of the rows written to it. Strides in bytes.
struct PagedSide {
  unsigned char* cache;
  uint32_t page_stride, slot_stride;
  int64_t head_stride;
  const unsigned char* rows;
  int64_t row_stride, row_head_stride;
  float scale, inv_scale;  // of an 8-bit cache
};
struct PagedAppendArgs {
  PagedSide side[2];
  const int64_t* slots;
  int64_t tokens;
  int32_t pages, page_size, heads, dim;
  DivMagic by_row, by_head, by_page;  // chunks of a token, chunks of a head, slots of a page
};
hipError_t launch_paged_append(const PagedAppendArgs& a, int dtype, bool fp8, hipStream_t stream);

struct PagedAttentionArgs {
  const uint16_t* query;           // [R, heads, dim], last dimension contiguous
  int64_t q_row_stride, q_head_stride;  // elements
  const unsigned char* key;
  const unsigned char* value;
  uint32_t k_page, k_slot, v_page, v_slot;  // bytes
  int64_t k_head, v_head;
  const int32_t* tables;           // [R, width], rows `table_stride` entries apart
  int64_t table_stride;
  const int32_t* lengths;          // [R]
  uint16_t* out;                   // [R, heads, dim] contiguous
  float* lse;                      // [R, heads] or null
  float* partial;
  uint32_t* counters;
  int32_t requests, kv_heads, group, head_tiles;  // group: query heads of a kv head
  int32_t dim, pages, page_size, width, window;   // window 0: none
  float scale_log2, value_scale;
  DivMagic by_page, by_waves, by_rows;  // slots of a page, waves of the call, rows of a request
};
// Work is counted in units of 32 tokens of a row, plus kAttentionRowCost a row for what every row
// costs; a workgroup takes kAttentionLeast at least (one a wave).
constexpr int kAttentionUnit = 32;
constexpr int kAttentionRowCost = 4;
constexpr int kAttentionLeast = 4;
// Workgroups of a call of `units` at most, and floats of one partial slot (two slots a workgroup).
int paged_attention_workgroups(int cus, int dim, int64_t units);
size_t paged_attention_slot_floats(int group, int dim);
hipError_t launch_paged_attention(const PagedAttentionArgs& a, int dtype, bool fp8, int workgroups,
                                  hipStream_t stream);

}  // namespace mt
