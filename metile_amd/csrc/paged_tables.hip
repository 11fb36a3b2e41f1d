// Block tables and slot maps of a step, from the requests' lengths.
//
// With len = cached + new, a request needs ceil(len / P) - ceil(cached / P) more pages; it takes
// them from the free list behind those of the requests before it. Token t of the step belongs to
// the last request whose first token is at most t. Both are prefix sums over the requests:
// integer work on a few kilobytes, bound by latency for ordinary steps and by the 16 bytes
// written a token for large ones. So that one launch does it, every workgroup scans all requests
// itself (4096 at a time, sums carried on) into LDS, then looks its own tokens up there. A token
// that opens a page of its own writes the page's table entry.
#include "common.h"
#include "paged.h"

namespace mt {
namespace {

constexpr int kThreads = 256;
constexpr int kItems = 16;
constexpr int kChunk = kThreads * kItems;  // requests scanned at a time

// Sums stop at the largest int instead of wrapping (still associative for counts >= 0).
__device__ __forceinline__ uint32_t add_sat(uint32_t a, uint32_t b) {
  const uint32_t s = a + b;
  return s < 0x7fffffffu ? s : 0x7fffffffu;
}

__device__ __forceinline__ uint32_t ceil_pages(uint32_t tokens, DivMagic by_page, uint32_t page) {
  const uint32_t q = div_by(tokens, by_page);
  return q + (q * page != tokens);
}

__device__ __forceinline__ uint32_t count_of(int32_t v) { return v > 0 ? (uint32_t)v : 0u; }

__global__ __launch_bounds__(kThreads) void paged_tables_kernel(PagedTablesArgs a,
                                                                DivMagic by_page, int per_block) {
  __shared__ uint32_t lds_start[kChunk];
  __shared__ uint32_t lds_first[kChunk];
  __shared__ uint32_t lds_wave[2][kThreads / 64];

  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const uint32_t page = (uint32_t)a.page_size;
  const uint32_t most = (uint32_t)a.width * page;  // the host checks that it fits 31 bits
  const uint32_t t_begin = (uint32_t)blockIdx.x * (uint32_t)per_block;
  const uint32_t t_end = min((uint32_t)a.tokens, t_begin + (uint32_t)per_block);
  const int64_t free_start = a.free_start ? *a.free_start : 0;
  uint32_t tokens_before = 0, pages_before = 0;

  for (int base = 0; base < a.num_requests; base += kChunk) {
    const int count = min(kChunk, a.num_requests - base);
    const int items = (count + kThreads - 1) / kThreads;  // <= kItems
    // a thread's own requests, then the sums before it
    uint32_t tokens = 0, pages = 0;
    for (int i = 0; i < items; ++i) {
      const int r = tid * items + i;
      if (r >= count) break;
      const uint32_t had = count_of(a.cached[base + r]), n = count_of(a.fresh[base + r]);
      const uint32_t len = add_sat(had, n);
      lds_start[r] = tokens;
      lds_first[r] = pages;
      tokens = add_sat(tokens, n);
      pages = add_sat(pages, ceil_pages(min(len, most), by_page, page) -
                                 ceil_pages(min(had, most), by_page, page));
      if (base / kChunk % (int)gridDim.x == (int)blockIdx.x) a.lengths[base + r] = (int32_t)len;
    }
    uint32_t sum_t = tokens, sum_p = pages;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const uint32_t ot = __shfl_up(sum_t, d), op = __shfl_up(sum_p, d);
      if (lane >= d) sum_t = add_sat(sum_t, ot), sum_p = add_sat(sum_p, op);
    }
    if (lane == 63) lds_wave[0][wave] = sum_t, lds_wave[1][wave] = sum_p;
    // exclusive sums within the wave: the lane before's (no subtraction: the sums saturate)
    uint32_t off_t = __shfl_up(sum_t, 1), off_p = __shfl_up(sum_p, 1);
    if (lane == 0) off_t = off_p = 0;
    __syncthreads();
    uint32_t all_t = tokens_before, all_p = pages_before;
#pragma unroll
    for (int w = 0; w < kThreads / 64; ++w) {
      if (w == wave) off_t = add_sat(all_t, off_t), off_p = add_sat(all_p, off_p);
      all_t = add_sat(all_t, lds_wave[0][w]);
      all_p = add_sat(all_p, lds_wave[1][w]);
    }
    for (int i = 0; i < items; ++i) {
      const int r = tid * items + i;
      if (r >= count) break;
      const uint32_t s = add_sat(off_t, lds_start[r]);
      lds_start[r] = s;
      lds_first[r] = add_sat(off_p, lds_first[r]);
      if (base / kChunk % (int)gridDim.x == (int)blockIdx.x) a.starts[base + r] = (int32_t)s;
    }
    __syncthreads();

    // this workgroup's tokens among the chunk's
    const uint32_t from = max(t_begin, tokens_before), to = min(t_end, all_t);
    for (uint32_t t = from + tid; t < to; t += kThreads) {
      int lo = 0, hi = count;  // last r with start <= t: it is not empty
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (lds_start[mid] <= t) lo = mid;
        else hi = mid;
      }
      const int r = base + lo;
      const uint32_t had = count_of(a.cached[r]);
      const uint32_t p = add_sat(had, t - lds_start[lo]);
      int64_t slot = -1;
      if (p < most) {
        const uint32_t column = div_by(p, by_page), in_page = p - column * page;
        const uint32_t have = ceil_pages(min(had, most), by_page, page);
        int32_t* entry = a.tables + (int64_t)r * a.table_stride + column;
        int32_t number;
        if (column >= have) {
          const int64_t k = free_start + lds_first[lo] + (column - have);
          number = k >= 0 && k < a.free_count ? a.free_pages[k] : -1;
          if (in_page == 0) *entry = number;
        } else {
          number = *entry;
        }
        if (number >= 0) slot = (int64_t)number * page + in_page;
      }
      a.slots[t] = slot;
      a.positions[t] = (int32_t)p;
      a.requests[t] = r;
    }
    tokens_before = all_t;
    pages_before = all_p;
    __syncthreads();  // the next chunk overwrites the sums
  }
  if (blockIdx.x == 0 && tid == 0) {
    a.starts[a.num_requests] = (int32_t)tokens_before;
    *a.taken = (int32_t)pages_before;
  }
  for (uint32_t t = max(t_begin, tokens_before) + tid; t < t_end; t += kThreads) {
    a.slots[t] = -1;
    a.positions[t] = 0;
    a.requests[t] = -1;
  }
}

}  // namespace

hipError_t launch_paged_tables(const PagedTablesArgs& a, int cus, hipStream_t stream) {
  // 1024 tokens a workgroup, up to two workgroups a CU
  int blocks = (a.tokens + 1023) / 1024;
  blocks = blocks < 1 ? 1 : blocks > 2 * cus ? 2 * cus : blocks;
  const int per = (int)(((int64_t)a.tokens + blocks - 1) / blocks);
  paged_tables_kernel<<<blocks, kThreads, 0, stream>>>(a, div_magic((uint32_t)a.page_size), per);
  return hipGetLastError();
}

}  // namespace mt
