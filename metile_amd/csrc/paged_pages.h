// Host-visible launch interfaces of what is done to whole pages of a paged key-value cache: copies,
// forks of requests, freeing and compaction.
#pragma once

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "paged.h"

namespace mt {

// A page as nested runs: `run` 16-byte units next to each other, n1 such runs s1 bytes apart, n0 of
// those s0 bytes apart; pages are `page` bytes apart.
struct PageShape {
  uint32_t run, n1, n0;
  int64_t s1, s0, page;
};
constexpr int kCopySides = 64;  // keys or values of caches in one launch
struct PagedCopyArgs {
  unsigned char* side[kCopySides];
  PageShape shape[2];       // of even and odd sides (keys, values)
  const int32_t* sources;   // [count]
  const int32_t* targets;
  int64_t count;
  int32_t pages;
};
hipError_t launch_paged_copy(const PagedCopyArgs& a, int sides, int cus, hipStream_t stream);

hipError_t launch_zero_int(int32_t* to, hipStream_t stream);

struct PagedForkArgs {
  int32_t* tables;  // [requests, width], rows `table_stride` entries apart
  int64_t table_stride;
  int32_t* lengths;
  const int32_t* sources;  // [forks] requests
  const int32_t* targets;
  const int32_t* tokens;   // [forks] or null
  const int32_t* free_pages;
  const int32_t* free_start;  // or null for 0
  int32_t* from;   // [forks] pages to copy
  int32_t* to;
  int32_t* taken;  // [1]
  int32_t requests, width, free_count, page_size, forks;
};
hipError_t launch_paged_fork(const PagedForkArgs& a, hipStream_t stream);

struct PagedFreeArgs {
  const int32_t* tables;
  int64_t table_stride;
  const int32_t* lengths;
  const int32_t* kept;
  int32_t* free_pages;
  const int32_t* free_start;
  int32_t* freed;       // [1]
  unsigned char* work;  // paged_free_work bytes
  int32_t requests, width, free_count, page_size, pages;
};
size_t paged_free_work(int pages);
hipError_t launch_paged_free(const PagedFreeArgs& a, hipStream_t stream);

struct PagedCompactArgs {
  const int32_t* tables;
  int64_t table_stride;
  const int32_t* lengths;
  const int32_t* free_pages;
  const int32_t* free_start;
  int32_t* new_tables;  // [requests, width]
  int32_t* new_free;    // [free_count]
  int32_t* sources;     // [most_moves]
  int32_t* targets;
  int32_t* moves;       // [1]
  unsigned char* work;  // paged_compact_work bytes
  int32_t requests, width, free_count, page_size, pages, most_moves;
};
size_t paged_compact_work(int pages);
hipError_t launch_paged_compact(const PagedCompactArgs& a, hipStream_t stream);

}  // namespace mt
