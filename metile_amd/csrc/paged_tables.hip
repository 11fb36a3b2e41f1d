// Block tables and slot maps of a step, from the requests' lengths.
//
// With len = cached + new, a request needs ceil(len / P) - ceil(cached / P) more pages; it takes
// them from the free list behind those of the requests before it. Token t of the step belongs to
// the last request whose first token is at most t. Both are prefix sums over the requests:
// integer work on a few kilobytes, bound by latency for ordinary steps and by the 16 bytes
// written a token for large ones. So that one launch does it, every workgroup scans all requests
// itself (up to 4096 at a time, sums carried on) into LDS, then looks its own tokens up there. A
// token that opens a page writes the page's table entry. 64 requests of one token each take 2.6 us;
// 4096 of 1 to 1900 tokens (a million, 16.6 MB) 13.4 us, half of it the scan.
#include <algorithm>

#include "common.h"
#include "paged.h"

namespace mt {
namespace {

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

// Inclusive sums over the lanes, stopping likewise.
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t dpp_add_sat(uint32_t v) {
  return add_sat(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xF, false));
}
__device__ __forceinline__ uint32_t wave_scan_sat(uint32_t v) {
  v = dpp_add_sat<0x111, 0xF>(v);  // row_shr:1
  v = dpp_add_sat<0x112, 0xF>(v);
  v = dpp_add_sat<0x114, 0xF>(v);
  v = dpp_add_sat<0x118, 0xF>(v);
  v = dpp_add_sat<kDppRowBcast15, 0xA>(v);
  return dpp_add_sat<kDppRowBcast31, 0xC>(v);
}

// ITEMS: requests of a thread in a scan, TOKENS: consecutive tokens of a thread (see
// launch_paged_tables).
template <int THREADS, int ITEMS, int TOKENS>
__global__ __launch_bounds__(THREADS) void paged_tables_kernel(PagedTablesArgs a,
                                                                DivMagic by_page, int per_block) {
  constexpr int kChunk = THREADS * ITEMS;  // requests scanned at a time
  // a thread's ITEMS requests lie ITEMS + 1 words from the next thread's: all banks are used alike
  constexpr int kPad = ITEMS > 1 ? THREADS : 0;
  __shared__ uint32_t lds_start[kChunk + kPad];
  __shared__ uint32_t lds_first[kChunk + kPad];
  __shared__ uint32_t lds_had[kChunk + kPad];
  auto place_of = [](int r) { return ITEMS > 1 ? r + r / ITEMS : r; };
  __shared__ uint32_t lds_wave[2][THREADS / 64];

  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const uint32_t page = (uint32_t)a.page_size;
  const uint32_t most = (uint32_t)a.width * page;  // the host checks that it fits 31 bits
  const uint32_t t_begin = (uint32_t)blockIdx.x * (uint32_t)per_block;
  const uint32_t t_end = min((uint32_t)a.tokens, t_begin + (uint32_t)per_block);
  const int64_t free_start = a.free_start ? *a.free_start : 0;
  uint32_t tokens_before = 0, pages_before = 0;

  for (int base = 0; base < a.num_requests; base += kChunk) {
    const int count = min(kChunk, a.num_requests - base);
    const bool writes = base / kChunk % (int)gridDim.x == (int)blockIdx.x;
    // counts of new tokens and pages into LDS, read side by side
    uint32_t had[ITEMS], fresh[ITEMS];
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      const int r = base + min(i * THREADS + tid, count - 1);
      had[i] = count_of(a.cached[r]);
      fresh[i] = count_of(a.fresh[r]);
    }
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      const int r = i * THREADS + tid;
      if (r >= count) break;
      const uint32_t len = add_sat(had[i], fresh[i]);
      lds_start[place_of(r)] = fresh[i];
      lds_first[place_of(r)] = ceil_pages(min(len, most), by_page, page) -
                               ceil_pages(min(had[i], most), by_page, page);
      lds_had[place_of(r)] = had[i];
      if (writes) a.lengths[base + r] = (int32_t)len;
    }
    __syncthreads();
    // a thread's own requests, then the sums before it
    const int run = (count + THREADS - 1) / THREADS, begin = tid * run;
    const int end = min(count, begin + run);
    uint32_t own_t[ITEMS], own_p[ITEMS], tokens = 0, pages = 0;
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      if (i >= run) break;
      const int r = min(begin + i, count - 1);
      own_t[i] = lds_start[place_of(r)];
      own_p[i] = lds_first[place_of(r)];
    }
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      if (i >= run) break;
      tokens = add_sat(tokens, begin + i < end ? own_t[i] : 0u);
      pages = add_sat(pages, begin + i < end ? own_p[i] : 0u);
    }
    const uint32_t sum_t = wave_scan_sat(tokens), sum_p = wave_scan_sat(pages);
    if (lane == 63) lds_wave[0][wave] = sum_t, lds_wave[1][wave] = sum_p;
    // exclusive sums within the wave: the lane before's (no subtraction: the sums saturate)
    uint32_t off_t = __shfl_up(sum_t, 1), off_p = __shfl_up(sum_p, 1);
    if (lane == 0) off_t = off_p = 0;
    __syncthreads();
    uint32_t all_t = tokens_before, all_p = pages_before;
#pragma unroll
    for (int w = 0; w < THREADS / 64; ++w) {
      if (w == wave) off_t = add_sat(all_t, off_t), off_p = add_sat(all_p, off_p);
      all_t = add_sat(all_t, lds_wave[0][w]);
      all_p = add_sat(all_p, lds_wave[1][w]);
    }
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      if (i >= run || begin + i >= end) break;
      lds_start[place_of(begin + i)] = off_t;
      lds_first[place_of(begin + i)] = off_p;
      off_t = add_sat(off_t, own_t[i]);
      off_p = add_sat(off_p, own_p[i]);
    }
    __syncthreads();
    if (writes)
      for (int r = tid; r < count; r += THREADS)
        a.starts[base + r] = (int32_t)lds_start[place_of(r)];

    // this workgroup's tokens among the chunk's
    const uint32_t from = max(t_begin, tokens_before), to = min(t_end, all_t);
    for (uint32_t t0 = from + tid * TOKENS; t0 < to; t0 += THREADS * TOKENS) {
      int lo = 0;  // the last r with start <= t: it is not empty
      for (int step = 1 << (31 - __clz(count)); step; step >>= 1) {
        const int mid = lo + step;
        if (mid < count && lds_start[place_of(mid)] <= t0) lo = mid;
      }
      // The tokens' pages: table entries, or the free list's for pages that the step opens.
      // Addresses are chosen, not branches, so that the loads overlap.
      const int32_t* from_where[TOKENS];
      uint32_t position[TOKENS];
      int request[TOKENS];
      bool known[TOKENS], opens[TOKENS];
      uint32_t next = lo + 1 < count ? lds_start[place_of(lo + 1)] : all_t;
      uint32_t had = lds_had[place_of(lo)], start = lds_start[place_of(lo)];
      uint32_t first = lds_first[place_of(lo)];
      uint32_t have = ceil_pages(min(had, most), by_page, page);
#pragma unroll
      for (int k = 0; k < TOKENS; ++k) {
        const uint32_t t = t0 + k;
        if (TOKENS > 1 && t < to && t >= next) {  // on to the next request that is not empty
          do {
            ++lo;
            next = lo + 1 < count ? lds_start[place_of(lo + 1)] : all_t;
          } while (t >= next);
          had = lds_had[place_of(lo)];
          start = lds_start[place_of(lo)];
          first = lds_first[place_of(lo)];
          have = ceil_pages(min(had, most), by_page, page);
        }
        const uint32_t p = add_sat(had, t - start), column = div_by(p, by_page);
        const bool in_table = t < to && p < most, fresh = column >= have;
        const int64_t n = free_start + first + (column - have);
        request[k] = base + lo;
        position[k] = p;
        opens[k] = in_table && fresh && p == column * page;
        known[k] = in_table && (!fresh || (n >= 0 && n < a.free_count));
        from_where[k] = !known[k] ? a.cached
                        : fresh ? a.free_pages + n
                                : a.tables + (int64_t)request[k] * a.table_stride + column;
      }
      int32_t number[TOKENS];
#pragma unroll
      for (int k = 0; k < TOKENS; ++k) number[k] = *from_where[k];
#pragma unroll
      for (int k = 0; k < TOKENS; ++k) {
        const uint32_t t = t0 + k;
        if (t >= to) break;
        const uint32_t column = div_by(position[k], by_page);
        if (!known[k]) number[k] = -1;
        if (opens[k]) a.tables[(int64_t)request[k] * a.table_stride + column] = number[k];
        a.slots[t] = number[k] >= 0 ? (int64_t)number[k] * page + (position[k] - column * page)
                                    : -1;
        a.positions[t] = (int32_t)position[k];
        a.requests[t] = request[k];
      }
    }
    tokens_before = all_t;
    pages_before = all_p;
    __syncthreads();  // the next chunk overwrites the sums
  }
  if (blockIdx.x == 0 && tid == 0) {
    a.starts[a.num_requests] = (int32_t)tokens_before;
    *a.taken = (int32_t)pages_before;
  }
  for (uint32_t t = max(t_begin, tokens_before) + tid; t < t_end; t += THREADS) {
    a.slots[t] = -1;
    a.positions[t] = 0;
    a.requests[t] = -1;
  }
}

template <int THREADS, int ITEMS, int TOKENS>
hipError_t launch(const PagedTablesArgs& a, int64_t most, hipStream_t stream) {
  constexpr int kRun = THREADS * TOKENS;
  const int64_t full = ((int64_t)a.tokens + kRun - 1) / kRun;
  const int64_t blocks = std::max<int64_t>(1, std::min(most, full));
  const int64_t per = ((int64_t)a.tokens + blocks - 1) / blocks;
  paged_tables_kernel<THREADS, ITEMS, TOKENS>
      <<<blocks, THREADS, 0, stream>>>(a, div_magic((uint32_t)a.page_size), (int)per);
  return hipGetLastError();
}

}  // namespace

// A workgroup a CU at most, since each scans all requests: of four waves where these can do that in
// one step, else of sixteen (4096 requests and a million tokens: two workgroups of four waves a CU
// 17 us, one of sixteen 13.4). A token a thread as long as that reaches, then runs of two, which
// share the search for their request (runs of four: 15 us).
hipError_t launch_paged_tables(const PagedTablesArgs& a, int cus, hipStream_t stream) {
  if (a.num_requests <= 256 && a.tokens <= 256 * cus) return launch<256, 1, 1>(a, cus, stream);
  if (a.tokens <= 1024 * cus) return launch<1024, 4, 1>(a, cus, stream);
  return launch<1024, 4, 2>(a, cus, stream);
}

}  // namespace mt
