// What is done to whole pages of a paged cache: copies, forks of requests, freeing and compaction.
//
// Which pages are in use is read from the block tables each time: a page is if any request has it
// among its tokens' pages. So there are no counts of references to keep, a page that requests share is
// freed with the last of them, and calls may come in any order. Marks are bytes, set by plain
// stores of the same value, so that no result goes by the order of threads; lists are made by prefix
// sums over the pages, in ascending order.
#include <algorithm>

#include "common.h"
#include "paged_pages.h"

namespace mt {
namespace {

constexpr int kThreads = 256, kWaves = kThreads / 64;

// ---- copies ----------------------------------------------------------------------------------------

constexpr int kUnroll = 4;

struct CopyMagic {
  DivMagic units, run, n1;
};

// Memory bounds it: 252 MB of 256 forks' pages in 8 layers take 49 us, 5.1 TB/s, as a copy of 1 GiB does. A
// thread moves four 16-byte units, a workgroup's next to each other.
__global__ __launch_bounds__(kThreads) void copy_kernel(PagedCopyArgs a, CopyMagic even, CopyMagic odd,
                                                         uint32_t units, uint32_t total) {
  const bool is_odd = blockIdx.y & 1;
  const PageShape& s = a.shape[is_odd];
  const CopyMagic magic = is_odd ? odd : even;
  unsigned char* base = a.side[blockIdx.y];
  const uint32_t step = gridDim.x * (kThreads * kUnroll);
  for (uint32_t first = blockIdx.x * (kThreads * kUnroll) + threadIdx.x; first < total;) {
    u32x4 v[kUnroll];
    unsigned char* to[kUnroll];
#pragma unroll
    for (int i = 0; i < kUnroll; ++i) {
      const uint32_t n = min(first + i * kThreads, total - 1);
      const uint32_t pair = div_by(n, magic.units), u = n - pair * units;
      const int32_t source = a.sources[pair], target = a.targets[pair];
      const bool here = first + i * kThreads < total && (uint32_t)source < (uint32_t)a.pages &&
                        (uint32_t)target < (uint32_t)a.pages;
      const uint32_t t = div_by(u, magic.run), i0 = div_by(t, magic.n1);
      const int64_t at = (int64_t)(u - t * s.run) * 16 + (int64_t)(t - i0 * s.n1) * s.s1 +
                         (int64_t)i0 * s.s0;
      to[i] = here ? base + (int64_t)target * s.page + at : nullptr;
      if (here) v[i] = *reinterpret_cast<const u32x4*>(base + (int64_t)source * s.page + at);
    }
#pragma unroll
    for (int i = 0; i < kUnroll; ++i)
      if (to[i]) *reinterpret_cast<u32x4*>(to[i]) = v[i];
    if (total - first <= step) break;
    first += step;
  }
}

// ---- forks -----------------------------------------------------------------------------------------

__device__ __forceinline__ int block_sum(int v, int* lds) {
  for (int d = 32; d; d /= 2) v += __shfl_xor(v, d);
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  v = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) v += lds[w];
  __syncthreads();
  return v;
}

struct Fork {
  int source, target, tokens;  // source -1: left out
};
__device__ __forceinline__ Fork fork_of(const PagedForkArgs& a, int i) {
  Fork f{a.sources[i], a.targets[i], 0};
  if ((uint32_t)f.source >= (uint32_t)a.requests || (uint32_t)f.target >= (uint32_t)a.requests) {
    f.source = -1;
    return f;
  }
  const int most = a.width * a.page_size;  // the host checks that it fits 31 bits
  f.tokens = min(max(a.lengths[f.source], 0), most);
  if (a.tokens) f.tokens = min(f.tokens, max(a.tokens[i], 0));
  return f;
}

__global__ void zero_int_kernel(int32_t* to) { *to = 0; }

// Calls of so many forks or more count those before each in a launch of one workgroup before: in the forks'
// own workgroups, which is one launch less, the work grows with their number's square. (us without and with
// that launch: 256 forks 3.4 and 5.7, 2048 6.2 and 7.2, 4096 12.8 and 10.3, 16384 108 and 28.5; 65536 101,
// 8388607 15361.)
constexpr int kForksCounted = 2560;
constexpr int kCountThreads = 1024, kCountRun = 4;  // forks of a thread, next to each other

__device__ __forceinline__ int begun_of(const PagedForkArgs& a, const Fork& f, DivMagic by_page) {
  return f.tokens - (int)div_by(f.tokens, by_page) * a.page_size;
}

// The forks before each that take a page, where the fork's own page will be written.
__global__ __launch_bounds__(kCountThreads) void count_forks_kernel(PagedForkArgs a, DivMagic by_page) {
  __shared__ int lds[2][kCountThreads / 64];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  int carry = 0, turn = 0;
  for (int base = 0; base < a.forks; base += kCountThreads * kCountRun, turn ^= 1) {
    const int first = base + tid * kCountRun;
    int takes[kCountRun], mine = 0;
#pragma unroll
    for (int k = 0; k < kCountRun; ++k) {
      const Fork f = fork_of(a, min(first + k, a.forks - 1));
      takes[k] = begun_of(a, f, by_page) > 0 && first + k < a.forks;
      mine += takes[k];
    }
    int sum = mine;
    for (int d = 1; d < 64; d *= 2) {
      const int x = __shfl_up(sum, d);
      if (lane >= d) sum += x;
    }
    if (lane == 63) lds[turn][wave] = sum;
    __syncthreads();
    int before = carry + sum - mine;
#pragma unroll
    for (int w = 0; w < kCountThreads / 64; ++w) {
      if (w < wave) before += lds[turn][w];
      carry += lds[turn][w];
    }
#pragma unroll
    for (int k = 0; k < kCountRun; ++k) {
      if (first + k < a.forks) a.to[first + k] = before;
      before += takes[k];
    }
  }
}

// A workgroup a fork. Each counts the forks before its own that take a page, unless they have been counted.
// Round trips bound it: a fork 2.5 us, 256 5.1.
template <bool kCounted>
__global__ __launch_bounds__(kThreads) void fork_kernel(PagedForkArgs a, DivMagic by_page) {
  __shared__ int lds[kWaves];
  const int i = blockIdx.x, tid = threadIdx.x;
  const bool last = i == a.forks - 1;
  int before = 0;
  if constexpr (kCounted) {
    before = a.to[i];
    __syncthreads();
  } else {
    for (int j = tid; j < i; j += kThreads) before += begun_of(a, fork_of(a, j), by_page) > 0;
    before = block_sum(before, lds);
  }
  const Fork f = fork_of(a, i);
  const int full = (int)div_by(f.tokens, by_page);
  const bool partial = begun_of(a, f, by_page) > 0;
  if (last && tid == 0) *a.taken = before + partial;
  int32_t fresh = -1, old = -1;
  if (partial) {
    const int64_t n = (a.free_start ? (int64_t)*a.free_start : 0) + before;
    if (n >= 0 && n < a.free_count) fresh = a.free_pages[n];
    if (fresh >= 0) old = a.tables[(int64_t)f.source * a.table_stride + full];
  }
  if (tid == 0) {
    a.from[i] = old;
    a.to[i] = fresh;
  }
  if (f.source < 0) return;
  const int32_t* from = a.tables + (int64_t)f.source * a.table_stride;
  int32_t* to = a.tables + (int64_t)f.target * a.table_stride;
  for (uint32_t c = tid; c < (uint32_t)full; c += kThreads) to[c] = from[c];
  if (tid == 0) {
    if (partial) to[full] = fresh;
    a.lengths[f.target] = f.tokens;
  }
}

// ---- marks -----------------------------------------------------------------------------------------

// Freeing and compaction are bound by launches and round trips, 2 to 5 us each: with marks in memory, whose
// stores from many CUs meet there, every step of them is a launch.

// Pages of a thread. (Free and compact of 24000 pages, us: 9.8 and 15.6, with 16 10.2 and 17.4, with 4 9.6
// and 14.7; of 4000000: 52 and 149, with 16 49 and 157, with 4 60 and 153.)
constexpr int kScan = 8;
constexpr int kScanBlock = kThreads * kScan;    // of a workgroup

__host__ __device__ inline int scan_blocks(int pages) {
  return (int)(((int64_t)pages + kScanBlock - 1) / kScanBlock);
}
size_t padded(int pages) { return (size_t)scan_blocks(pages) * kScanBlock; }

__global__ __launch_bounds__(kThreads) void fill_kernel(u32x4* to, int64_t count) {
  const int64_t step = (int64_t)gridDim.x * kThreads;
  for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < count; i += step)
    to[i] = (u32x4){0, 0, 0, 0};
}

__device__ __forceinline__ int columns_of(int tokens, DivMagic by_page, int page_size, int width) {
  const int n = max(tokens, 0), c = (int)div_by(n, by_page);
  return min(c + (c * page_size != n), width);
}

// A wave a row of a block table, several side by side for long ones, which count columns past 2^31: f(column)
// for those below `end`.
constexpr uint32_t kRowPiece = 1024;  // entries

template <typename F>
__device__ __forceinline__ void each_column(int end, F f) {
  const uint32_t lane = threadIdx.x & 63;
  for (uint32_t c0 = blockIdx.y * kRowPiece; c0 < (uint32_t)end; c0 += gridDim.y * kRowPiece)
    for (uint32_t c = c0 + lane; c < min(c0 + kRowPiece, (uint32_t)end); c += 64) f(c);
}

__global__ __launch_bounds__(kThreads) void mark_free_kernel(PagedFreeArgs a, DivMagic by_page,
                                                              unsigned char* keeps,
                                                              unsigned char* drops) {
  const int r = blockIdx.x * kWaves + (threadIdx.x >> 6);
  if (r >= a.requests) return;
  const int length = a.lengths[r], kept = min(a.kept[r], length);
  const uint32_t keep = columns_of(kept, by_page, a.page_size, a.width);
  const int32_t* row = a.tables + (int64_t)r * a.table_stride;
  each_column(columns_of(length, by_page, a.page_size, a.width), [&](uint32_t c) {
    const int32_t p = row[c];
    if ((uint32_t)p < (uint32_t)a.pages) (c < keep ? keeps : drops)[p] = 1;
  });
}

// A thread's marks, bytes of 0 or 1.
struct __attribute__((aligned(kScan))) Marks {
  uint32_t word[kScan / 4];
  __device__ __forceinline__ bool has(int i) const { return word[i / 4] >> (8 * (i % 4)) & 1; }
  __device__ __forceinline__ int count() const {
    int n = 0;
#pragma unroll
    for (int i = 0; i < kScan / 4; ++i) n += __popc(word[i]);
    return n;
  }
  // Those that `other` does not have.
  __device__ __forceinline__ Marks without(const Marks& other) const {
    Marks m;
#pragma unroll
    for (int i = 0; i < kScan / 4; ++i) m.word[i] = word[i] & ~other.word[i];
    return m;
  }
};
__device__ __forceinline__ Marks marks_of(const unsigned char* marks, int64_t first) {
  return *reinterpret_cast<const Marks*>(marks + first);
}

// Exclusive sums over a workgroup's threads of up to two counts, and their totals.
struct Pair {
  int a, b;
};
__device__ __forceinline__ Pair scan_pair(Pair v, Pair* total, Pair (*lds)) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  Pair s = v;
  for (int d = 1; d < 64; d *= 2) {
    const int x = __shfl_up(s.a, d), y = __shfl_up(s.b, d);
    if (lane >= d) s.a += x, s.b += y;
  }
  if (lane == 63) lds[wave] = s;
  __syncthreads();
  Pair before{0, 0}, all{0, 0};
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    if (w < wave) before.a += lds[w].a, before.b += lds[w].b;
    all.a += lds[w].a, all.b += lds[w].b;
  }
  __syncthreads();
  *total = all;
  return {before.a + s.a - v.a, before.b + s.b - v.b};
}
// Sums of the blocks' counts before this one, and of all. (Every workgroup reads all counts: nothing beside a
// launch in ordinary pools, 7.6 ms a call in one of 2^28 pages, 0.57 s in one of 2^31 - 1.)
__device__ __forceinline__ Pair blocks_before(const Pair* counts, int blocks, Pair* total, Pair* lds) {
  Pair before{0, 0}, all{0, 0};
  for (int i = threadIdx.x; i < blocks; i += kThreads) {
    const Pair c = counts[i];
    all.a += c.a, all.b += c.b;
    if (i < (int)blockIdx.x) before.a += c.a, before.b += c.b;
  }
  int* words = reinterpret_cast<int*>(lds);
  before.a = block_sum(before.a, words);
  before.b = block_sum(before.b, words);
  total->a = block_sum(all.a, words);
  total->b = block_sum(all.b, words);
  return before;
}

__global__ __launch_bounds__(kThreads) void count_free_kernel(const unsigned char* keeps,
                                                               const unsigned char* drops,
                                                               Pair* counts) {
  __shared__ int lds[kWaves];
  const int64_t first = ((int64_t)blockIdx.x * kThreads + threadIdx.x) * kScan;
  const int n = block_sum(marks_of(drops, first).without(marks_of(keeps, first)).count(), lds);
  if (threadIdx.x == 0) counts[blockIdx.x] = {n, 0};
}

__global__ __launch_bounds__(kThreads) void list_free_kernel(PagedFreeArgs a,
                                                              const unsigned char* keeps,
                                                              const unsigned char* drops,
                                                              const Pair* counts) {
  __shared__ Pair lds[kWaves];
  Pair total, in_block;
  const Pair before = blocks_before(counts, gridDim.x, &total, lds);
  const int64_t first = ((int64_t)blockIdx.x * kThreads + threadIdx.x) * kScan;
  const Marks marks = marks_of(drops, first).without(marks_of(keeps, first));
  const Pair mine = scan_pair({marks.count(), 0}, &in_block, lds);
  int64_t at = (int64_t)*a.free_start - total.a + before.a + mine.a;
#pragma unroll
  for (int i = 0; i < kScan; ++i) {
    if (marks.has(i)) {
      if (at >= 0 && at < a.free_count) a.free_pages[at] = (int32_t)(first + i);
      ++at;
    }
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) *a.freed = total.a;
}

// ---- compaction ------------------------------------------------------------------------------------

// No moves yet, and the free list up to its start.
__global__ __launch_bounds__(kThreads) void begin_compact_kernel(PagedCompactArgs a, u32x4* marks,
                                                                  int64_t mark_count) {
  const int64_t step = (int64_t)gridDim.x * kThreads;
  const int64_t first = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  for (int64_t i = first; i < mark_count; i += step) marks[i] = (u32x4){0, 0, 0, 0};
  for (int64_t i = first; i < a.most_moves; i += step) a.sources[i] = a.targets[i] = -1;
  const int start = *a.free_start;
  for (int64_t i = first; i < a.free_count; i += step) a.new_free[i] = i < start ? a.free_pages[i] : -1;
}

__global__ __launch_bounds__(kThreads) void mark_compact_kernel(PagedCompactArgs a, DivMagic by_page,
                                                                 int row_blocks, unsigned char* used,
                                                                 unsigned char* open) {
  if ((int)blockIdx.x >= row_blocks) {  // the free list
    const int64_t step = (int64_t)(gridDim.x - row_blocks) * gridDim.y * kThreads;
    const int64_t start = max(*a.free_start, 0);
    for (int64_t i = start + ((int64_t)(blockIdx.x - row_blocks) * gridDim.y + blockIdx.y) * kThreads +
                     threadIdx.x;
         i < a.free_count; i += step) {
      const int32_t p = a.free_pages[i];
      if ((uint32_t)p < (uint32_t)a.pages) open[p] = 1;
    }
    return;
  }
  const int r = blockIdx.x * kWaves + (threadIdx.x >> 6);
  if (r >= a.requests) return;
  const int32_t* row = a.tables + (int64_t)r * a.table_stride;
  each_column(columns_of(a.lengths[r], by_page, a.page_size, a.width), [&](uint32_t c) {
    const int32_t p = row[c];
    if ((uint32_t)p < (uint32_t)a.pages) used[p] = 1;
  });
}

__global__ __launch_bounds__(kThreads) void count_compact_kernel(const unsigned char* used,
                                                                  const unsigned char* open,
                                                                  Pair* counts) {
  __shared__ int lds[kWaves];
  const int64_t first = ((int64_t)blockIdx.x * kThreads + threadIdx.x) * kScan;
  const Marks u = marks_of(used, first);
  const int n = block_sum(u.count(), lds);
  const int m = block_sum(marks_of(open, first).without(u).count(), lds);
  if (threadIdx.x == 0) counts[blockIdx.x] = {n, m};
}

// With U pages in use, those in use beyond the U lowest of all (in use or free) move, the highest to
// the lowest free page, and so on; `number` says of each page where in the list of moves it is.
__global__ __launch_bounds__(kThreads) void list_compact_kernel(PagedCompactArgs a,
                                                                 const unsigned char* used,
                                                                 const unsigned char* open,
                                                                 const Pair* counts,
                                                                 int32_t* number) {
  __shared__ Pair lds[kWaves];
  Pair total, in_block;
  const Pair before = blocks_before(counts, gridDim.x, &total, lds);
  const int64_t first = ((int64_t)blockIdx.x * kThreads + threadIdx.x) * kScan;
  const Marks u = marks_of(used, first), o = marks_of(open, first).without(u);
  const Pair mine = scan_pair({u.count(), o.count()}, &in_block, lds);
  int used_before = before.a + mine.a, open_before = before.b + mine.b;
  const int in_use = total.a, start = max(*a.free_start, 0);
  if (blockIdx.x == 0 && threadIdx.x == 0 && in_use == 0) *a.moves = 0;
#pragma unroll
  for (int i = 0; i < kScan; ++i) {
    const int32_t page = (int32_t)(first + i);
    const bool is_used = u.has(i), is_open = o.has(i);
    const int rank = used_before + open_before;
    const bool low = rank < in_use;
    if (is_used || is_open) {
      // (moves: as many as there are free pages among the lowest)
      if (rank == in_use - 1) *a.moves = open_before + is_open;
      const int move = is_used ? in_use - 1 - used_before : open_before;
      if (is_used) number[page] = low ? -1 : move;
      if (is_used && !low && move < a.most_moves) a.sources[move] = page;
      if (is_open && low && move < a.most_moves) a.targets[move] = page;
      if (!low && (int64_t)start + rank - in_use < a.free_count)
        a.new_free[start + rank - in_use] = page;
      if (is_used) ++used_before;
      else ++open_before;
    }
  }
}

__global__ __launch_bounds__(kThreads) void apply_compact_kernel(PagedCompactArgs a, DivMagic by_page,
                                                                  const int32_t* number) {
  const int r = blockIdx.x * kWaves + (threadIdx.x >> 6);
  if (r >= a.requests) return;
  const uint32_t columns = columns_of(a.lengths[r], by_page, a.page_size, a.width);
  const int32_t* row = a.tables + (int64_t)r * a.table_stride;
  int32_t* to = a.new_tables + (int64_t)r * a.width;
  each_column(a.width, [&](uint32_t c) {
    int32_t p = row[c];
    if (c < columns && (uint32_t)p < (uint32_t)a.pages) {
      const int move = number[p];
      if (move >= 0) p = a.targets[move];
    }
    to[c] = p;
  });
}

// ---- small pools: one launch -----------------------------------------------------------------------

// One workgroup does it all where it needs no more time than the others' launches, with the marks in
// LDS. (Free and compact, us: 64 requests over 1024 pages 9.0 -> 4.0 and 14.2 -> 5.6, 256 over 8192
// 9.6 -> 6.4 and 15.9 -> 13.7, 64 over 16384 10.1 -> 9.0 and 18.2 -> 16.8; 1024 over 16384 took 15 and
// 27 where the launches take 9.7 and 16.7. The host's part of a call is 17.4 -> 9.4 and 23.5 -> 12.7.)
constexpr int kSmallThreads = 1024, kSmallWaves = kSmallThreads / 64;
constexpr int kSmallPages = 16384, kSmallEntries = 32768, kSmallRequests = 256;
constexpr int kAhead = 4;  // entries that a thread has under way

// f(entry, column) for the columns [from(r), to(r)) of each row, 2^bits threads to a row.
template <typename From, typename To, typename F>
__device__ __forceinline__ void each_entry(const int32_t* tables, int64_t stride, int requests, int bits,
                                           From from, To to, F f) {
  const int threads = 1 << bits, me = threadIdx.x & (threads - 1);
  for (int r = threadIdx.x >> bits; r < requests; r += kSmallThreads >> bits) {
    const int32_t* row = tables + (int64_t)r * stride;
    const int end = to(r);
    for (int c = from(r) + me; c < end; c += threads * kAhead) {
      int32_t p[kAhead];
#pragma unroll
      for (int i = 0; i < kAhead; ++i) p[i] = c + i * threads < end ? row[c + i * threads] : 0;
#pragma unroll
      for (int i = 0; i < kAhead; ++i)
        if (c + i * threads < end) f(p[i], r, c + i * threads);
    }
  }
}

__device__ __forceinline__ void no_marks(unsigned char* marks) {
  for (int i = threadIdx.x; i < kSmallPages / 16; i += kSmallThreads)
    reinterpret_cast<u32x4*>(marks)[i] = (u32x4){0, 0, 0, 0};
}

// The pages of a wave are next to each other, 64 at a time. Sums over the waves before this one, and
// over all, of how many pages have the marks.
struct SmallScan {
  int first, last;  // pages of the wave
  Pair before, all;
};
__device__ __forceinline__ SmallScan scan_marks(const unsigned char* marks, int pages, int mark_a,
                                                int mark_b, Pair* lds) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int per = (pages + kSmallThreads - 1) / kSmallThreads * 64;
  SmallScan s;
  s.first = wave * per;
  s.last = min(s.first + per, pages);
  Pair mine{0, 0};
  for (int p = s.first; p < s.last; p += 64) {
    const int mark = p + lane < s.last ? marks[p + lane] : 0;
    mine.a += __popcll(__ballot(mark == mark_a));
    mine.b += __popcll(__ballot(mark == mark_b));
  }
  if (lane == 0) lds[wave] = mine;
  __syncthreads();
  s.before = s.all = {0, 0};
#pragma unroll
  for (int w = 0; w < kSmallWaves; ++w) {
    if (w < wave) s.before.a += lds[w].a, s.before.b += lds[w].b;
    s.all.a += lds[w].a, s.all.b += lds[w].b;
  }
  return s;
}
__device__ __forceinline__ int lanes_before(uint64_t mask) {
  return __popcll(mask & ((1ull << (threadIdx.x & 63)) - 1));
}

__global__ __launch_bounds__(kSmallThreads) void free_small_kernel(PagedFreeArgs a, DivMagic by_page,
                                                                    int bits) {
  __shared__ __attribute__((aligned(16))) unsigned char marks[kSmallPages];  // 1: dropped, 2: kept
  __shared__ Pair lds[kSmallWaves];
  const int64_t start = *a.free_start;
  no_marks(marks);
  __syncthreads();
  auto used = [&](int r) { return columns_of(a.lengths[r], by_page, a.page_size, a.width); };
  auto kept = [&](int r) {
    return columns_of(min(a.kept[r], a.lengths[r]), by_page, a.page_size, a.width);
  };
  auto none = [](int) { return 0; };
  each_entry(a.tables, a.table_stride, a.requests, bits, kept, used, [&](int32_t p, int, int) {
    if ((uint32_t)p < (uint32_t)a.pages) marks[p] = 1;
  });
  __syncthreads();
  each_entry(a.tables, a.table_stride, a.requests, bits, none, kept, [&](int32_t p, int, int) {
    if ((uint32_t)p < (uint32_t)a.pages) marks[p] = 2;
  });
  __syncthreads();
  const SmallScan s = scan_marks(marks, a.pages, 1, 3, lds);
  int64_t at = start - s.all.a + s.before.a;
  for (int p = s.first; p < s.last; p += 64) {
    const int page = p + (threadIdx.x & 63);
    const bool mine = page < s.last && marks[page] == 1;
    const uint64_t mask = __ballot(mine);
    const int64_t to = at + lanes_before(mask);
    if (mine && to >= 0 && to < a.free_count) a.free_pages[to] = page;
    at += __popcll(mask);
  }
  if (threadIdx.x == 0) *a.freed = s.all.a;
}

// As list_compact_kernel and those around it.
__global__ __launch_bounds__(kSmallThreads) void compact_small_kernel(PagedCompactArgs a,
                                                                       DivMagic by_page, int bits) {
  __shared__ __attribute__((aligned(16))) unsigned char marks[kSmallPages];  // 1: free, 2: in use
  __shared__ uint16_t number[kSmallPages];       // of a page in use: its move, or kStays
  __shared__ uint16_t target_of[kSmallPages / 2];  // of a move
  __shared__ Pair lds[kSmallWaves];
  __shared__ int num_moves;
  constexpr int kStays = 0xffff;
  const int tid = threadIdx.x;
  const int given = *a.free_start, start = max(given, 0);
  if (tid == 0) num_moves = 0;
  no_marks(marks);
  __syncthreads();
  for (int64_t i = (int64_t)start + tid; i < a.free_count; i += kSmallThreads) {
    const int32_t p = a.free_pages[i];
    if ((uint32_t)p < (uint32_t)a.pages) marks[p] = 1;
  }
  for (int i = tid; i < min(given, a.free_count); i += kSmallThreads) a.new_free[i] = a.free_pages[i];
  __syncthreads();
  auto columns = [&](int r) { return columns_of(a.lengths[r], by_page, a.page_size, a.width); };
  auto none = [](int) { return 0; };
  each_entry(a.tables, a.table_stride, a.requests, bits, none, columns, [&](int32_t p, int, int) {
    if ((uint32_t)p < (uint32_t)a.pages) marks[p] = 2;
  });
  __syncthreads();
  const SmallScan s = scan_marks(marks, a.pages, 2, 1, lds);
  const int in_use = s.all.a;
  int used_before = s.before.a, open_before = s.before.b;
  for (int p = s.first; p < s.last; p += 64) {
    const int page = p + (tid & 63), mark = page < s.last ? marks[page] : 0;
    const uint64_t used = __ballot(mark == 2), open = __ballot(mark == 1);
    const int before = used_before + lanes_before(used), opens = open_before + lanes_before(open);
    const int rank = before + opens;
    const bool low = rank < in_use;
    if (mark) {
      if (rank == in_use - 1) num_moves = opens + (mark == 1);
      if (mark == 2) number[page] = low ? kStays : in_use - 1 - before;
      if (mark == 2 && !low) a.sources[in_use - 1 - before] = page;
      if (mark == 1 && low) {
        a.targets[opens] = page;
        target_of[opens] = page;
      }
      if (!low && (int64_t)start + rank - in_use < a.free_count) a.new_free[start + rank - in_use] = page;
    }
    used_before += __popcll(used);
    open_before += __popcll(open);
  }
  __syncthreads();
  const int moves = num_moves;
  if (tid == 0) *a.moves = moves;
  for (int i = moves + tid; i < a.most_moves; i += kSmallThreads) a.sources[i] = a.targets[i] = -1;
  for (int64_t i = (int64_t)start + s.all.b + tid; i < a.free_count; i += kSmallThreads)
    a.new_free[i] = -1;
  each_entry(a.tables, a.table_stride, a.requests, bits, none, columns, [&](int32_t p, int r, int c) {
    if ((uint32_t)p < (uint32_t)a.pages && number[p] != kStays) p = target_of[number[p]];
    a.new_tables[(int64_t)r * a.width + c] = p;
  });
  auto width = [&](int) { return a.width; };
  each_entry(a.tables, a.table_stride, a.requests, bits, columns, width, [&](int32_t p, int r, int c) {
    a.new_tables[(int64_t)r * a.width + c] = p;
  });
}

bool is_small(int pages, int requests, int width) {
  return pages <= kSmallPages && requests <= kSmallRequests &&
         (int64_t)requests * width <= kSmallEntries;
}
// Threads of a row, as many as there are for each.
int row_bits(int requests) {
  int bits = 10;
  while (bits && (kSmallThreads >> bits) < requests) --bits;
  return bits;
}

dim3 row_grid(int requests, int width) {
  const int rows = (requests + kWaves - 1) / kWaves;
  const int pieces = (int)(((int64_t)width + kRowPiece - 1) / (int64_t)kRowPiece);
  return dim3(rows, std::max(1, std::min({pieces, 64, (1 << 20) / std::max(rows, 1)})));
}
unsigned fill_grid(int64_t vectors) {
  return (unsigned)std::max<int64_t>(1, std::min<int64_t>(1024, (vectors + kThreads - 1) / kThreads));
}

}  // namespace

hipError_t launch_paged_copy(const PagedCopyArgs& args, int sides, int cus, hipStream_t stream) {
  const uint32_t units = args.shape[0].run * args.shape[0].n1 * args.shape[0].n0;
  CopyMagic magic[2];
  for (int i = 0; i < 2; ++i)
    magic[i] = {div_magic(units), div_magic(args.shape[i].run), div_magic(args.shape[i].n1)};
  // pairs of a launch, so that units are counted in 31 bits
  const int64_t most = std::max<int64_t>(1, 0x7fffffffll / units);
  for (int64_t at = 0; at < args.count; at += most) {
    PagedCopyArgs a = args;
    a.sources += at;
    a.targets += at;
    const uint32_t total = (uint32_t)std::min(most, args.count - at) * units;
    const uint32_t blocks = (total + kThreads * kUnroll - 1) / (kThreads * kUnroll);
    const uint32_t grid = std::min<uint32_t>(blocks, std::max(1, 32 * cus / sides));
    copy_kernel<<<dim3(grid, sides), kThreads, 0, stream>>>(a, magic[0], magic[1], units, total);
    if (const hipError_t e = hipGetLastError()) return e;
  }
  return hipSuccess;
}

hipError_t launch_zero_int(int32_t* to, hipStream_t stream) {
  zero_int_kernel<<<1, 1, 0, stream>>>(to);
  return hipGetLastError();
}

hipError_t launch_paged_fork(const PagedForkArgs& a, hipStream_t stream) {
  const DivMagic by_page = div_magic((uint32_t)a.page_size);
  if (a.forks >= kForksCounted) {
    count_forks_kernel<<<1, kCountThreads, 0, stream>>>(a, by_page);
    fork_kernel<true><<<a.forks, kThreads, 0, stream>>>(a, by_page);
  } else {
    fork_kernel<false><<<a.forks, kThreads, 0, stream>>>(a, by_page);
  }
  return hipGetLastError();
}

// Marks of the pages that are kept and that are dropped, then the blocks' counts.
size_t paged_free_work(int pages) {
  return 2 * padded(pages) + (size_t)scan_blocks(pages) * sizeof(Pair);
}

hipError_t launch_paged_free(const PagedFreeArgs& a, hipStream_t stream) {
  const DivMagic by_page = div_magic((uint32_t)a.page_size);
  if (is_small(a.pages, a.requests, a.width)) {
    free_small_kernel<<<1, kSmallThreads, 0, stream>>>(a, by_page, row_bits(a.requests));
    return hipGetLastError();
  }
  const size_t marks = padded(a.pages);
  unsigned char *keeps = a.work, *drops = a.work + marks;
  Pair* counts = reinterpret_cast<Pair*>(a.work + 2 * marks);
  fill_kernel<<<fill_grid(marks / 8), kThreads, 0, stream>>>(reinterpret_cast<u32x4*>(a.work),
                                                             (int64_t)marks / 8);
  if (a.requests)
    mark_free_kernel<<<row_grid(a.requests, a.width), kThreads, 0, stream>>>(a, by_page, keeps, drops);
  count_free_kernel<<<scan_blocks(a.pages), kThreads, 0, stream>>>(keeps, drops, counts);
  list_free_kernel<<<scan_blocks(a.pages), kThreads, 0, stream>>>(a, keeps, drops, counts);
  return hipGetLastError();
}

// Marks of the pages in use and of the free ones, the blocks' counts, then each page's move.
size_t paged_compact_work(int pages) {
  return 2 * padded(pages) + (size_t)scan_blocks(pages) * sizeof(Pair) + padded(pages) * 4;
}

hipError_t launch_paged_compact(const PagedCompactArgs& a, hipStream_t stream) {
  const DivMagic by_page = div_magic((uint32_t)a.page_size);
  if (is_small(a.pages, a.requests, a.width) && a.free_count <= 2 * kSmallPages &&
      a.most_moves <= 2 * kSmallPages) {
    compact_small_kernel<<<1, kSmallThreads, 0, stream>>>(a, by_page, row_bits(a.requests));
    return hipGetLastError();
  }
  const size_t marks = padded(a.pages);
  unsigned char *used = a.work, *open = a.work + marks;
  int32_t* number = reinterpret_cast<int32_t*>(a.work + 2 * marks);
  Pair* counts = reinterpret_cast<Pair*>(number + marks);
  const int64_t most = std::max<int64_t>({(int64_t)marks / 8, a.most_moves, a.free_count});
  begin_compact_kernel<<<fill_grid(most), kThreads, 0, stream>>>(
      a, reinterpret_cast<u32x4*>(a.work), (int64_t)marks / 8);
  const dim3 rows = row_grid(a.requests, a.width);
  const int list = (int)std::max<int64_t>(1, std::min<int64_t>(256, a.free_count / 4096));
  mark_compact_kernel<<<dim3(rows.x + list, rows.y), kThreads, 0, stream>>>(a, by_page, rows.x, used,
                                                                            open);
  count_compact_kernel<<<scan_blocks(a.pages), kThreads, 0, stream>>>(used, open, counts);
  list_compact_kernel<<<scan_blocks(a.pages), kThreads, 0, stream>>>(a, used, open, counts, number);
  if (a.requests)
    apply_compact_kernel<<<rows, kThreads, 0, stream>>>(a, by_page, number);
  return hipGetLastError();
}

}  // namespace mt
