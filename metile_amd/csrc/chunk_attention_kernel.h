// The kernels of chunk_attention.hip, a template over types and head size, instantiated in
// chunk_attention_{bf16,f16}{,_fp8}.hip.
//
//   s_j = scale * q . k_j      o = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m)
//
// over the keys j up to a token's own position. The rows of a tile are (token, query head) pairs of
// one request and one key-value head, so that all of them read the same keys. A workgroup takes a
// tile of 128 rows, 32 a wave, through blocks of 64 keys, with a running reference (near the maximum)
// and sum:
//  * keys are the rows of v_mfma_f32_32x32x16 and query rows its columns, so a lane holds scores of
//    one query row. Key rows are dealt to operand rows so that a lane's registers 8 n .. 8 n + 7 hold
//    eight consecutive keys, which are the operand of the second product as they stand: no exchange
//    between lanes but one for the maximum;
//  * values are read from LDS transposed (ds_read_b64_tr_b16: four rows by sixteen columns a group of
//    sixteen lanes); the result has the query row in the lane again, so rescaling is local;
//  * both lie in LDS as 16-bit rows whose 16-byte chunks are exchanged within a row so that every
//    read touches all banks alike. 8-bit caches are converted on the way in.
// Probabilities enter the second product rounded to 16 bits (at most 2^-8 of each in bf16, 2^-11 in
// f16), as the result itself is; a second part of them would add half as many products again. Scores,
// references, sums and results are fp32, and the sums are of the probabilities before that rounding.
//
// What bounds it: the matrix and the vector unit, each busy a little more than half of the time (heads of 128:
// 32 products and 190 vector instructions a wave and block), and beneath them the power: the same launch over
// zeros takes 0.73 of the time. A prompt of 8192 tokens, 32 heads of 128 over 8, in bf16, takes 558 us (986
// TFLOP/s; a library's product of 8192 x 8192 x 8192 reaches 1271), 509 tokens behind 130500 take 1098 us
// (993). 1024 tokens behind 16384 in a stream of 600 calls, in which that product reaches 1412 TFLOP/s: 953 in
// 32 heads of 128 over 8, 787 in 24 of 96 over 3, 673 in 16 of 80, 754 in 32 of 64 over 8, whose products have
// half the steps for the same exponentials, 704 in 20 of 192 over 5 and 833 in 16 of 256 over 1, whose wave
// fills the registers of a SIMD (256 with results in accumulation registers: 1.27 times the time); over 8-bit
// caches 3% less to 1% more. Three waves a SIMD instead of two for heads of 64 were slower (24 parts of prompts
// 54 -> 61 us), as were two and three parts for each slot.
#pragma once

#include <algorithm>

#include "chunk_attention.h"
#include "common.h"

namespace mt {
namespace chunk {

constexpr int kThreads = 256;
constexpr int kTile = kChunkTile, kBlock = kChunkBlock;
constexpr float kTiny = 0x1p-126f;

__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

// A request's new tokens: the packed rows they are, the position of the first (below zero where there
// are more of them than tokens altogether), and its keys.
struct Request {
  int start, count, first, keys;
};
__device__ __forceinline__ Request request_of(const ChunkAttentionArgs& a, int r) {
  Request q;
  const int s = a.starts[r], e = a.starts[r + 1], n = a.lengths[r];
  q.start = min(max(s, 0), a.tokens);
  q.count = max(min(e, a.tokens) - q.start, 0);
  q.keys = min(max(n, 0), a.width * a.page_size);  // the host checks that it fits 31 bits
  q.first = max(n, 0) - q.count;
  return q;
}
__device__ __forceinline__ int tiles_of(const ChunkAttentionArgs& a, const Request& q) {
  return (int)(((int64_t)q.count * a.group + kTile - 1) / kTile);
}
// The blocks of keys that tokens t0 .. t1 of a request see, the first one and how many.
struct Blocks {
  int first, count;
};
__device__ __forceinline__ Blocks blocks_of(const ChunkAttentionArgs& a, const Request& q, int t0,
                                            int t1) {
  const int hi = min(q.first + t1 + 1, q.keys);
  const int lo = a.window ? max(max(q.first + t0 + 1, 0) - a.window, 0) : 0;  // (in 32 bits)
  Blocks b;
  b.first = lo / kBlock;
  b.count = hi > lo ? (hi + kBlock - 1) / kBlock - b.first : 0;
  return b;
}
// Blocks of the tile of a request that has most, or somewhat more.
__device__ __forceinline__ int most_blocks(const ChunkAttentionArgs& a, const Request& q) {
  const int all = blocks_of(a, q, 0, q.count - 1).count;
  if (!a.window) return all;
  const int64_t tile = (int64_t)a.window + (kTile - 1) / a.group + 1;
  return (int)min((int64_t)all, (tile + kBlock - 1) / kBlock + 1);
}

// Parts of each tile of a request whose tiles have up to `most` blocks.
__device__ __forceinline__ int splits_of(int most, int per) {
  return most < kChunkLeastSplit ? 1 : (int)(((int64_t)most + per - 1) / per);
}
// Blocks that a part has at least, of a call with so many.
__device__ __forceinline__ int least_blocks(float total) {
  return (int)fminf(fmaxf(total * (1.0f / 64.0f), (float)kChunkLeastBlocks), 4.0f);
}

// An item: a request's tile, or one part of `splits` of its keys; `part` is where a part is kept.
struct Item {
  int request, splits, in_request, part;  // request -1: none
  Request q;
  __device__ int tile(const ChunkAttentionArgs& a) const {  // the longest first
    return tiles_of(a, q) - 1 - in_request / splits;
  }
};

// Inclusive sums over the lanes: within rows of 16, then across them.
template <int CTRL, int ROWS>
__device__ __forceinline__ int dpp_read_int(int v) {
  return __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xF, false);
}
template <typename T>
__device__ __forceinline__ T wave_scan(T v) {
  auto from = [](T x, auto read) { return __builtin_bit_cast(T, read(__builtin_bit_cast(int, x))); };
  v += from(v, dpp_read_int<0x111, 0xF>);  // row_shr:1
  v += from(v, dpp_read_int<0x112, 0xF>);
  v += from(v, dpp_read_int<0x114, 0xF>);
  v += from(v, dpp_read_int<0x118, 0xF>);
  v += from(v, dpp_read_int<kDppRowBcast15, 0xA>);
  v += from(v, dpp_read_int<kDppRowBcast31, 0xC>);
  return v;
}
__device__ __forceinline__ int readlane(int v, int l) { return __builtin_amdgcn_readlane(v, l); }

// Blocks of a part of one request's tiles, so that the last round of workgroups is not left nearly empty: a
// lane a choice, from twice to a third of an even share, the last one `per`, which is kept unless another
// promises a seventh less. A round takes as long as an item and its start; one that leaves half of the slots
// free (of two a CU) three quarters of that.
__device__ __forceinline__ int best_parts(const ChunkAttentionArgs& a, int lane, float even, int per,
                                          int tiles, int most) {
  constexpr float kStart = 3.0f;  // in blocks
  const int mine = lane == 63 ? per : (int)fmaxf(even * 16.0f / (float)(lane % 40 + 8), kChunkLeastBlocks);
  const int splits = splits_of(most, mine);
  const float items = (float)tiles * (float)splits;
  const float rounds = items * (float)a.kv_heads / (float)a.slots, whole = floorf(rounds);
  const float rest = rounds - whole;
  const float last = rest == 0.0f ? 0.0f : a.dim <= 128 && rest <= 0.5f ? 0.75f : 1.0f;
  float cost = (whole + last) * (ceilf((float)most / (float)splits) + kStart);
  if (splits > 1 && items > (float)a.most_parts) cost = 3.0e38f;
  if (lane == 63) cost *= 0.85f;
  float least = cost;
  for (int d = 32; d; d /= 2) least = fminf(least, __shfl_xor(least, d));
  // (of equal ones the first lane's, which has the fewest parts; `per` has room for its own)
  return readlane(mine, __ffsll((unsigned long long)__ballot(cost == least)) - 1);
}

// Item n, or with JOIN the first part of the n-th tile that has parts, of a call of up to 64 requests: each
// wave counts the work up for itself, a lane a request. `behind` receives the packed row behind the last
// request's.
template <bool JOIN>
__device__ __forceinline__ Item find_here(const ChunkAttentionArgs& a, int n, int* behind) {
  const int lane = threadIdx.x & 63, r = min(lane, a.requests - 1);
  const Request q = request_of(a, r);
  *behind = readlane(min(max(a.starts[r + 1], 0), a.tokens), a.requests - 1);
  const int tiles = lane < a.requests ? tiles_of(a, q) : 0, most = most_blocks(a, q);
  int per;
  if constexpr (JOIN) {
    // (as the attention kernel found it: the parts lie where it put them, however its sums were rounded)
    per = a.plan[0];
  } else {
    // (rounded up, so that there are no more than `target` parts on top of the tiles)
    const float total =
        __builtin_bit_cast(float, readlane(__builtin_bit_cast(int, wave_scan((float)tiles * (float)most)),
                                           63));
    const float even = total * 1.0001f / (float)a.target;  // blocks of an item, if all were the same
    per = max((int)fminf(even + 1.0f, 1073741824.0f), least_blocks(total));
    // (us of 1024 tokens behind 16384 without and with the choice: 14 heads of 64 on 2 129 and 108, 24 of 96 on
    // 3 261 and 221, 20 of 192 on 5 588 and 460; for 2 to 8 requests, a choice a time over all of them, it cost
    // more than it gave: 3 prompts 60 and 77)
    if (a.requests == 1 && even > 16.0f)
      per = best_parts(a, lane, even, per, readlane(tiles, 0), readlane(most, 0));
    if (blockIdx.x == 0 && threadIdx.x == 0) a.plan[0] = per;
  }
  const int splits = splits_of(most, per);
  const int items = tiles * splits, parts = splits > 1 ? items : 0;
  const int count = !JOIN ? items : splits > 1 ? tiles : 0;
  const int sums = wave_scan(count), part_sums = wave_scan(parts);
  const uint64_t later = __ballot(sums > n);
  Item i{-1, 1, 0, 0, {}};
  if (!later) return i;
  const int l = __ffsll((unsigned long long)later) - 1;
  i.request = l;
  i.splits = readlane(splits, l);
  i.in_request = (n - readlane(sums - count, l)) * (JOIN ? i.splits : 1);
  i.part = readlane(part_sums - parts, l) + i.in_request;
  i.q = {readlane(q.start, l), readlane(q.count, l), readlane(q.first, l), readlane(q.keys, l)};
  return i;
}

// The same of a call of more requests, from the sums that the plan holds: the last request whose sum of
// those before it is at most n, 64 at a time, by a whole wave.
template <bool JOIN>
__device__ __forceinline__ Item find_planned(const ChunkAttentionArgs& a, int n, int* behind) {
  const int lane = threadIdx.x & 63;
  const int32_t *items = a.plan + kPlanHead, *parts = items + a.requests + 1;
  const int32_t* sums = JOIN ? parts + a.requests + 1 : items;
  *behind = min(max(a.starts[a.requests], 0), a.tokens);
  Item i{-1, 1, 0, 0, {}};
  if (n >= a.plan[JOIN ? 2 : 1]) return i;
  int lo = 0;
  for (int count = a.requests; count > 1;) {
    const int step = (count + 63) / 64;
    const bool ok = lane * step < count && sums[lo + lane * step] <= n;
    const int last = 63 - __clzll((long long)__ballot(ok));
    lo = uniform(lo + last * step);
    count = min(step, uniform(count) - last * step);
  }
  i.request = lo;
  i.q = request_of(a, lo);
  i.splits = splits_of(most_blocks(a, i.q), a.plan[0]);
  i.in_request = (n - sums[lo]) * (JOIN ? i.splits : 1);
  i.part = parts[lo] + i.in_request;
  return i;
}
template <bool JOIN>
__device__ __forceinline__ Item find(const ChunkAttentionArgs& a, int n, int* behind) {
  return a.requests <= kChunkHere ? find_here<JOIN>(a, n, behind) : find_planned<JOIN>(a, n, behind);
}

template <int DT>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  if constexpr (DT == kBF16)
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2){a, b}, bf16x2));
  else
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2){a, b}, f16x2));
}

template <int DT>
__device__ __forceinline__ u32x4 fp8_eight(u32x2 w) {
  const uint32_t lo = w.x, hi = w.y;
  if constexpr (DT == kBF16)
    return (u32x4){
        __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)lo, 1.0f, false)),
        __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)lo, 1.0f, true)),
        __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)hi, 1.0f, false)),
        __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)hi, 1.0f, true))};
  else
    return (u32x4){
        __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)lo, 1.0f, false)),
        __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)lo, 1.0f, true)),
        __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)hi, 1.0f, false)),
        __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)hi, 1.0f, true))};
}

// Two 16-bit floats, 0 in place of infinities and NaN.
template <int DT>
__device__ __forceinline__ uint32_t finite_pair(uint32_t w) {
  constexpr uint32_t kExponent = DT == kBF16 ? 0x7f80u : 0x7c00u;
  if ((w & kExponent) == kExponent) w &= 0xffff0000u;
  if ((w >> 16 & kExponent) == kExponent) w &= 0x0000ffffu;
  return w;
}

// The larger of the two halves' values, in both.
__device__ __forceinline__ float halves_max(float v) {
  const auto p = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(p[0]), __uint_as_float(p[1]));
}
__device__ __forceinline__ float halves_sum(float v) {
  const auto p = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(p[0]) + __uint_as_float(p[1]);
}

// Where chunk c (16 bytes) of row `row` lies in its row of CHUNKS: sixteen lanes that read one chunk
// of sixteen rows (keys), and thirty-two that read four chunks of four rows (values), touch all banks.
template <int CHUNKS>
__device__ __forceinline__ int key_place(int c, int row) {
  if constexpr (CHUNKS % 16 == 0) return c ^ (row & 15);
  else if constexpr (CHUNKS % 8 == 0) return c ^ ((row >> 1) & 7);
  else return c ^ ((row >> 2) & 3);
}
template <int CHUNKS>
__device__ __forceinline__ int value_place(int c, int row) {
  if constexpr (CHUNKS % 16 == 0) return c ^ ((row & 3) << 2);
  else if constexpr (CHUNKS % 8 == 0) return c ^ ((row >> 1 & 1) << 2);
  else return c;
}

typedef short s16x4 __attribute__((ext_vector_type(4)));

// LDS is addressed as such throughout: a pointer of no address space costs two registers and a check.
typedef __attribute__((address_space(3))) uint16_t Lds;
typedef __attribute__((address_space(3))) u32x4 Lds16;
typedef __attribute__((address_space(3))) u32x2 Lds8;

// Bytes to a token's row of one head.
template <bool GENERAL>
struct Offset {
  typedef uint64_t type;
};
template <>
struct Offset<false> {
  typedef uint32_t type;
};

// DIM: the head's values. With GENERAL, that many or more (the rest count as zero), in caches of any size;
// else the offsets of rows fit 32 bits.
template <int DT, bool FP8, int DIM, bool GENERAL>
__global__ __launch_bounds__(kThreads, DIM <= 128 ? 2 : 1) void attention_kernel(
    ChunkAttentionArgs a) {
  constexpr int kChunks = DIM / 8, kSteps = DIM / 16, kTiles = DIM / 32;
  constexpr int kLoads = kChunks * kBlock / kThreads;  // of a thread, a side
  constexpr int kStage = kBlock * DIM;                 // 16-bit values
  // the narrowest head that is given to this DIM
  constexpr int kLeastDim = DIM == 64 ? 16 : DIM == 96 ? 80 : DIM == 128 ? 112 : DIM == 192 ? 144 : 208;
  // p = 2^(x - base) with base kShift below the largest x when it was set; it is set anew once x
  // passes base + kRoom, so that most blocks need no rescaling. f16 probabilities are scaled up so that
  // small ones stay above its smallest numbers: 2^15 at most.
  constexpr float kShift = DT == kF16 ? 11.0f : 0.0f, kRoom = DT == kF16 ? 15.0f : 8.0f;

  // an array a stage and side: the compiler has to see that reads of one do not wait for loads to another
  __shared__ __attribute__((aligned(16))) uint16_t lds_k0[kStage], lds_v0[kStage], lds_k1[kStage],
      lds_v1[kStage];
  Lds *const keys0 = (Lds*)lds_k0, *const values0 = (Lds*)lds_v0, *const keys1 = (Lds*)lds_k1,
      *const values1 = (Lds*)lds_v1;

  const int tid = threadIdx.x, wave = uniform(tid >> 6);
  int lane = tid & 63, col = lane & 31, half = lane >> 5;
  const int dim = GENERAL ? a.dim : DIM;

  // ---- this workgroup's item: a tile of a request, or a part of its keys, for one head ----
  const int head = (int)(blockIdx.x % (unsigned)a.kv_heads);
  int behind;
  const Item item = find<false>(a, (int)(blockIdx.x / (unsigned)a.kv_heads), &behind);

  // ---- rows that belong to no request, in front of the first one's and behind the last one's (counted in 32
  // unsigned bits: with gridDim.x they may pass 2^31) ----
  {
    const int row_words = a.kv_heads * a.group * (dim / 8);
    const uint32_t front = (uint32_t)min(max(a.starts[0], 0), a.tokens);
    const uint32_t none = front + (uint32_t)(a.tokens - behind);
    for (uint32_t n = blockIdx.x; n < none; n += gridDim.x) {
      const uint32_t row = n < front ? n : n - front + (uint32_t)behind;
      u32x4* to = reinterpret_cast<u32x4*>(a.out) + (int64_t)row * row_words;
      for (int i = tid; i < row_words; i += kThreads) to[i] = (u32x4){0, 0, 0, 0};
      if (a.lse)
        for (int i = tid; i < a.kv_heads * a.group; i += kThreads)
          a.lse[(int64_t)row * a.kv_heads * a.group + i] = -__builtin_inff();
    }
  }

  if (item.request < 0) return;
  const int r = item.request, splits = item.splits;
  const Request q = item.q;
  const int tile = item.tile(a), split = item.in_request % splits;
  if (tile < 0 || (splits > 1 && (uint32_t)item.part >= (uint32_t)a.most_parts)) return;
  const int row0 = tile * kTile, rows = min(kTile, q.count * a.group - row0);
  const Blocks all = blocks_of(a, q, (int)div_by(row0, a.by_group),
                               (int)div_by(row0 + rows - 1, a.by_group));
  const int block0 = uniform(all.first + (int)((int64_t)all.count * split / splits));
  const int block_end = uniform(all.first + (int)((int64_t)all.count * (split + 1) / splits));

  // ---- this lane's row, and what the wave's rows see ----
  const int wave_rows = min(rows - 32 * wave, 32);  // may be none
  const int my_row = row0 + min(32 * wave + col, rows - 1);
  const int my_token = (int)div_by(my_row, a.by_group);
  const int my_head = head * a.group + (my_row - my_token * a.group);
  const bool has_row = 32 * wave + col < rows;
  const int my_end = min(q.first + my_token + 1, q.keys);  // keys below
  const int my_begin = a.window ? max(max(q.first + my_token + 1, 0) - a.window, 0) : 0;
  // (rows are in order of their tokens, so the ends of lanes 0 and 31 bound the wave's; readlane of
  // lanes whose row repeats the last one)
  const int first_end = __builtin_amdgcn_readlane(my_end, 0);
  const int last_end = __builtin_amdgcn_readlane(my_end, 31);
  const int first_begin = __builtin_amdgcn_readlane(my_begin, 0);
  const int last_begin = __builtin_amdgcn_readlane(my_begin, 31);

  // (what depends on these is left for later: entries and rows are on their way at the same time)
  u32x4 query[kSteps];
  {
    const uint16_t* p = a.query + (int64_t)(q.start + my_token) * a.q_row_stride +
                        (int64_t)my_head * a.q_head_stride;
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      const int d = 16 * s + 8 * half;
      query[s] = *reinterpret_cast<const u32x4*>(p + (d < dim ? d : 0));
    }
  }
  auto finish_query = [&]() {
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      query[s] ^= a.flip;
      if (!has_row || 16 * s + 8 * half >= dim) query[s] = (u32x4){0, 0, 0, 0};
    }
  };

  const int32_t* table = a.tables + (int64_t)r * a.table_stride;
  const unsigned char* kbase = a.key + (int64_t)head * a.k_head;
  const unsigned char* vbase = a.value + (int64_t)head * a.v_head;
  const int last_key = max(q.keys - 1, 0);

  // Where a block's tokens are: a lane a token looks up its entry; those that load the row ask for the
  // offset. Tokens past the end stand for the last one, tokens on no page of the cache for page 0;
  // both are masked.
  typedef typename Offset<GENERAL>::type RowOffset;
  struct Place {
    int page;
    uint32_t slot;
  };
  auto look_up = [&](int block) __attribute__((always_inline)) {
    // (blocks past the end may be past 2^31 too)
    const uint32_t token = min((uint32_t)block * kBlock + (uint32_t)lane, (uint32_t)last_key);
    const uint32_t column = div_by(token, a.by_page);
    return Place{table[column], token - column * (uint32_t)a.page_size};
  };
  struct Offsets {
    RowOffset key, value;
    uint64_t on_page;  // of the block's tokens, which are on a page of the cache
  };
  auto offsets_of = [&](const Place& p) __attribute__((always_inline)) {
    const bool ok = (uint32_t)p.page < (uint32_t)a.pages;
    const RowOffset page = ok ? (uint32_t)p.page : 0u, slot = p.slot;
    return Offsets{page * a.k_page + slot * a.k_slot, page * a.v_page + slot * a.v_slot, __ballot(ok)};
  };
  auto of_row = [&](RowOffset offset, int row) {
    const uint32_t lo = (uint32_t)__builtin_amdgcn_ds_bpermute(4 * row, (int)(uint32_t)offset);
    if constexpr (!GENERAL) return lo;
    else
      return (uint64_t)(uint32_t)__builtin_amdgcn_ds_bpermute(4 * row, (int)((uint64_t)offset >> 32))
                 << 32 |
             lo;
  };
  // One side of a block to LDS. Chunk i of this thread: LDS chunk n of the stage is row n / kChunks, place
  // n % kChunks. 8-bit rows wait in registers until they are parked.
  u32x2 held8[2][FP8 ? kLoads : 1];
  auto request = [&](int side, Lds* to, RowOffset offset) __attribute__((always_inline)) {
    const unsigned char* base = side ? vbase : kbase;
    // (chunks of later rows follow from the first one's: not kept, in registers that are short)
    constexpr bool kEven = 64 % kChunks == 0;
    constexpr int kRows = kEven ? 64 / kChunks : 1;  // of a load
    auto place_of = [&](int c, int row) {
      return side ? value_place<kChunks>(c, row) : key_place<kChunks>(c, row);
    };
    uint32_t chunk0 = (uint32_t)place_of(lane % kChunks, lane / kChunks) * (FP8 ? 8 : 16);
    int row0 = wave * kLoads * kRows + lane / kChunks;
    if constexpr (kEven) __asm__("" : "+v"(chunk0), "+v"(row0));
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int n = (wave * kLoads + i) * 64 + lane;
      const int row = kEven ? row0 + i * kRows : n / kChunks;
      const uint32_t chunk = kEven ? chunk0 ^ (uint32_t)place_of(0, i * kRows) * (FP8 ? 8 : 16)
                                   : (uint32_t)place_of(n % kChunks, row) * (FP8 ? 8 : 16);
      const unsigned char* from =
          base + (of_row(offset, row) +
                  (!GENERAL || chunk / (FP8 ? 1 : 2) < (uint32_t)dim ? chunk : 0u));
      if constexpr (FP8) {
        held8[side][i] = *reinterpret_cast<const u32x2*>(from);
      } else {
        __builtin_amdgcn_global_load_lds(
            (const __attribute__((address_space(1))) void*)from,
            (lds_ptr_t)(to + (wave * kLoads + i) * 512), 16, 0, 0);
      }
    }
  };
  auto park = [&](int side, Lds* to) __attribute__((always_inline)) {
    if constexpr (FP8) {
#pragma unroll
      for (int i = 0; i < kLoads; ++i)
        *(Lds16*)(to + ((wave * kLoads + i) * 64 + lane) * 8) =
            fp8_eight<DT>(held8[side][i]);
    }
  };

  float base = -__builtin_inff(), sum = 0.0f;
  f32x16 acc[kTiles];

  // Scores of a block: operand row i is key 16 (i / 16) + 8 (i / 4 % 2) + 4 (i / 8 % 2) + i % 4. Operands
  // are read kAhead products ahead; `between` is done after each product, in this order: left to itself
  // the compiler puts all products first, the waves of a SIMD fall into step, and its matrix and vector
  // units take turns instead of working side by side.
  constexpr int kAhead = 3, kScores = 2 * kSteps, kSums = 4 * kTiles;
  auto score = [&](const Lds* keys, f32x16 (&s)[2], auto between) __attribute__((always_inline)) {
    u32x4 key[kScores];
    auto read = [&](int n) __attribute__((always_inline)) {
      const int row =
          32 * (n & 1) + (col & 16) + ((col >> 2) & 1) * 8 + ((col >> 3) & 1) * 4 + (col & 3);
      const int c = 2 * (n >> 1) + half;
      key[n] = *(const Lds16*)(keys + (row * kChunks + key_place<kChunks>(c, row)) * 8);
    };
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int i = 0; i < 16; ++i) s[u][i] = 0.0f;
#pragma unroll
    for (int n = 0; n < kAhead; ++n) read(n);
#pragma unroll
    for (int n = 0; n < kScores; ++n) {
      if (n + kAhead < kScores) read(n + kAhead);
      // (with GENERAL, steps that the head does not have are skipped)
      if (!GENERAL || 8 * (n & ~1) < kLeastDim || 8 * (n & ~1) < dim)
        s[n & 1] = mfma32<DT>(key[n], query[n >> 1], s[n & 1]);
      between(n);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  // -inf for keys that the row does not see, or that are on no page.
  auto mask = [&](int block, uint64_t on_page, f32x16 (&s)[2]) __attribute__((always_inline)) {
    const int k0 = block * kBlock;
    if (first_end >= k0 + kBlock && last_begin <= k0 && on_page == ~0ull) return;
    const int end = my_end - k0 - 8 * half, begin = my_begin - k0 - 8 * half;
    const uint64_t known = on_page >> (8 * half);
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int j = 32 * u + 16 * (i / 8) + i % 8;  // and 8 of the half
        const bool ok = j < end && j >= begin && (known >> j & 1);
        s[u][i] = ok ? s[u][i] : -__builtin_inff();
      }
  };
  auto largest = [&](const f32x16 (&s)[2]) __attribute__((always_inline)) {
    float top = s[0][0];
#pragma unroll
    for (int i = 1; i < 32; ++i) top = fmaxf(top, s[i / 16][i % 16]);
    return top;
  };
  auto of_row_max = [&](float top) __attribute__((always_inline)) {
    return halves_max(top) * a.scale_log2;
  };
  // A reference near the maximum; what has been summed follows it.
  auto refer = [&](float top) __attribute__((always_inline)) {
    if (__any(top > base + kRoom)) {
      const float next = fmaxf(base, top - kShift);
      const float at = next == -__builtin_inff() ? 0.0f : next;
      const float fix = fmaxf(__builtin_amdgcn_exp2f(base - at), kTiny);
      sum *= fix;
#pragma unroll
      for (int t = 0; t < kTiles; ++t)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[t][i] *= fix;
      base = next;
    }
  };
  // Probabilities of a row's scores `from` to `to` (two at a time).
  auto weigh = [&](const f32x16 (&s)[2], u32x4 (&p)[4], float zero_at, float (&sums)[2], int from,
                   int to) __attribute__((always_inline)) {
#pragma unroll
    for (int i = from; i < to; i += 2) {
      const float p0 = __builtin_amdgcn_exp2f(fmaf(s[i / 16][i % 16], a.scale_log2, -zero_at));
      const float p1 = __builtin_amdgcn_exp2f(fmaf(s[i / 16][i % 16 + 1], a.scale_log2, -zero_at));
      sums[0] += p0;
      sums[1] += p1;
      uint32_t pair = pack2<DT>(p0, p1);
      __asm__ volatile("" : "+v"(pair), "+v"(sums[0]), "+v"(sums[1]));  // (here, and not later)
      p[i / 8][i % 8 / 2] = pair;
    }
  };
  // Values: 4 rows by 16 columns a group of 16 lanes, transposed on the way.
  auto add = [&](auto careful, const Lds* values, const u32x4 (&p)[4], auto between)
      __attribute__((always_inline)) {
    const int in_group = lane & 15;
    u32x4 v[kSums];
    auto read = [&](int n) __attribute__((always_inline)) {
      const int k = n / kTiles, t = n % kTiles;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int row = 16 * k + 8 * half + 4 * e + (in_group >> 2);
        const int c = 4 * t + ((lane >> 4) & 1) * 2 + ((in_group & 3) >> 1);
        const Lds* at =
            values + (row * kChunks + value_place<kChunks>(c, row)) * 8 + 4 * (in_group & 1);
        const u32x2 w = __builtin_bit_cast(
            u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                       (__attribute__((address_space(3))) s16x4*)(at)));
        v[n][2 * e] = w.x;
        v[n][2 * e + 1] = w.y;
      }
    };
#pragma unroll
    for (int n = 0; n < kAhead; ++n) read(n);
#pragma unroll
    for (int n = 0; n < kSums; ++n) {
      if (n + kAhead < kSums) read(n + kAhead);
      if constexpr (decltype(careful)::value != 0) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t x = v[n][j];
          v[n][j] = finite_pair<DT>(x);
        }
      }
      acc[n % kTiles] = mfma32<DT>(v[n], p[n / kTiles], acc[n % kTiles]);
      between(n);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  auto nothing = [](int) {};
  // Values that are not finite: their keys one by one, since products with the zeros of rows that do not
  // see them would make no numbers.
  auto add_odd = [&](const Lds* values, uint64_t on_page, const f32x16 (&s)[2])
      __attribute__((always_inline)) {
    const float zero_at = base == -__builtin_inff() ? 0.0f : base;
    bool odd_row = false;
#pragma unroll 1
    for (int c = 0; c < kChunks; ++c) {
      const u32x4 w = *(const Lds16*)(values + (lane * kChunks + c) * 8);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t x = w[j];
        odd_row |= finite_pair<DT>(x) != x && (8 * value_place<kChunks>(c, lane) < dim);
      }
    }
    uint64_t odd = __ballot(odd_row) & on_page;
#pragma unroll 1
    for (; odd; odd &= odd - 1) {
      const int j = __ffsll((unsigned long long)odd) - 1;
      const int reg = 16 * (j / 32) + 8 * (j / 16 % 2) + j % 8;
      float x = 0.0f;
#pragma unroll
      for (int i = 0; i < 32; ++i) x = i == reg ? s[i / 16][i % 16] : x;
      x = __shfl(x, col + 32 * (j / 8 % 2));
      float w = __builtin_amdgcn_exp2f(fmaf(x, a.scale_log2, -zero_at));
      w = w == 0.0f ? kTiny : w;  // below fp32's range, but not nothing
      const bool seen = !(x == -__builtin_inff());
#pragma unroll
      for (int t = 0; t < kTiles; ++t)
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
          const int d = 32 * t + 2 * i + 4 * half;
          const u32x2 v = *(const Lds8*)(
              values + (j * kChunks + value_place<kChunks>(d / 8, j)) * 8 + (d & 7));
          const uint32_t lo = v.x, hi = v.y;
          const float f[4] = {lo16<DT>(lo), hi16<DT>(lo), lo16<DT>(hi), hi16<DT>(hi)};
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (seen && !(fabsf(f[e]) < __builtin_inff())) acc[t][i + e] += w * f[e];
        }
    }
  };

  // ---- the blocks ----
  // A wave's last block: later ones only pass through it for the others' sake.
  const int wave_end =
      wave_rows > 0 ? min(block_end, (last_end + kBlock - 1) / kBlock) : block0;
  auto clear = [&]() {
    base = -__builtin_inff();
    sum = 0.0f;
#pragma unroll
    for (int t = 0; t < kTiles; ++t)
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[t][i] = 0.0f;
  };
  // While a block's probabilities are taken, the next one's scores are under way; keys are requested two
  // blocks ahead, values one, table entries a block before that. (Blocks past the end stand for the last
  // one: steps have no branches for them.)
  clear();
  if (block0 < block_end) {
    f32x16 s[2];
    float top = 0.0f;
    Place ahead = look_up(block0), second = look_up(block0 + 1), third = look_up(block0 + 2);
    const Offsets first = offsets_of(ahead);
    request(0, keys0, first.key);
    request(1, values0, first.value);
    park(0, keys0);
    park(1, values0);
    Offsets next = offsets_of(second);  // of the block whose values are requested next
    request(0, keys1, next.key);
    park(0, keys1);
    ahead = third;  // of the block whose keys are
    finish_query();
    wait_vmcnt<0>();
    __syncthreads();
    if (block0 < wave_end) {
      score(keys0, s, nothing);
      mask(block0, first.on_page, s);
      top = of_row_max(largest(s));
    }
    // Block `block`, whose values are in `values`, with scores s; the next one's keys in keys_next.
    auto take = [&](auto which, int block, Lds* keys, Lds* values, Lds* keys_next, Lds* values_next)
        __attribute__((always_inline)) {
      constexpr int kNext = decltype(which)::value;  // 1: scores of the next block too, -1: neither
      wait_vmcnt<0>();
      __syncthreads();
      const uint64_t on_page = next.on_page;
      auto request_values = [&]() __attribute__((always_inline)) {
        request(1, values_next, next.value);
      };
      auto request_keys = [&]() __attribute__((always_inline)) {
        next = offsets_of(ahead);
        request(0, keys, next.key);
        ahead = look_up(block + 3);
      };
      if constexpr (kNext <= 0) {
        request_values();
        request_keys();
      }
      if constexpr (kNext >= 0) {
        refer(top);
        const float zero_at = base == -__builtin_inff() ? 0.0f : base;
        float sums[2] = {0.0f, 0.0f};
        u32x4 p[4];
        if constexpr (kNext > 0) {
          f32x16 s_next[2];
          score(keys_next, s_next, [&](int n) __attribute__((always_inline)) {
            // rows are asked for first, the 32 probabilities follow
            constexpr int kFirst = kScores / 4;
            if (n == 0) request_values();
            if (n == kFirst / 2) request_keys();
            if (n >= kFirst)
              weigh(s, p, zero_at, sums, (n - kFirst) * 16 / (kScores - kFirst) * 2,
                    (n + 1 - kFirst) * 16 / (kScores - kFirst) * 2);
          });
          sum += sums[0] + sums[1];
          mask(block + 1, on_page, s_next);
          float tops[2] = {s_next[0][0], s_next[1][0]};
          add(IntConst<0>(), values, p, [&](int n) __attribute__((always_inline)) {
#pragma unroll
            for (int i = n * 32 / kSums; i < (n + 1) * 32 / kSums; ++i)
              tops[i / 16] = fmaxf(tops[i / 16], s_next[i / 16][i % 16]);
          });
          top = of_row_max(fmaxf(tops[0], tops[1]));
          s[0] = s_next[0];
          s[1] = s_next[1];
        } else {
          weigh(s, p, zero_at, sums, 0, 32);
          sum += sums[0] + sums[1];
          add(IntConst<0>(), values, p, nothing);
        }
      }
      park(1, values_next);
      park(0, keys);
    };
    int block = block0;
#pragma unroll 1
    for (; block + 2 < wave_end; block += 2) {
      take(IntConst<1>(), block, keys0, values0, keys1, values1);
      take(IntConst<1>(), block + 1, keys1, values1, keys0, values0);
    }
    bool swapped = false;
    if (block + 1 < wave_end) {
      take(IntConst<1>(), block, keys0, values0, keys1, values1);
      take(IntConst<0>(), block + 1, keys1, values1, keys0, values0);
      block += 2;
    } else if (block < wave_end) {
      take(IntConst<0>(), block, keys0, values0, keys1, values1);
      ++block;
      swapped = true;
    }
#pragma unroll 1
    for (; block < block_end; ++block, swapped = !swapped)
      take(IntConst<-1>(), block, swapped ? keys1 : keys0, swapped ? values1 : values0,
           swapped ? keys0 : keys1, swapped ? values0 : values1);
    wait_vmcnt<0>();  // (rows on their way to LDS that is not this workgroup's any more)
  }
  // A value that is not finite may have met a zero of a row that does not see it: once more, with
  // care (for rows that see it the result stays what it is).
  float odd = 0.0f;
#pragma unroll
  for (int t = 0; t < kTiles; ++t)
#pragma unroll
    for (int i = 0; i < 16; ++i) odd = fmaf(acc[t][i], 0.0f, odd);
  if (__syncthreads_or(odd != 0.0f)) {
    __asm__ volatile("" : "+v"(lane));  // no address of this is to be reckoned, and kept, before
    col = lane & 31, half = lane >> 5;
    clear();
#pragma unroll 1
    for (int block = block0; block < block_end; ++block) {
      const Offsets at = offsets_of(look_up(block));
      request(0, keys0, at.key);
      request(1, values0, at.value);
      park(0, keys0);
      park(1, values0);
      wait_vmcnt<0>();
      __syncthreads();
      if (block < wave_end) {
        f32x16 s[2];
        score(keys0, s, nothing);
        mask(block, at.on_page, s);
        refer(of_row_max(largest(s)));
        u32x4 p[4];
        float sums[2] = {0.0f, 0.0f};
        weigh(s, p, base == -__builtin_inff() ? 0.0f : base, sums, 0, 32);
        sum += sums[0] + sums[1];
        add_odd(values0, at.on_page, s);
        add(IntConst<1>(), values0, p, nothing);
      }
      __syncthreads();
    }
  }
  sum = halves_sum(sum);

  // ---- the result, or this part of it ----
  if (wave_rows <= 0) return;
  if (splits > 1) {
    const int64_t part = (int64_t)item.part * a.kv_heads + head;
    float* to = a.parts + part * (kTile * (DIM + 2));
#pragma unroll
    for (int t = 0; t < kTiles; ++t)
#pragma unroll
      for (int i = 0; i < 16; ++i) to[((wave * kTiles + t) * 16 + i) * 64 + lane] = acc[t][i];
    if (half == 0) {
      // (a sum that is no number has no reference, but is not nothing)
      to[kTile * DIM + 32 * wave + col] = sum != sum && base == -__builtin_inff() ? 0.0f : base;
      to[kTile * (DIM + 1) + 32 * wave + col] = sum;
    }
    return;
  }
  if (!has_row) return;
  const int64_t row = (int64_t)(q.start + my_token) * a.kv_heads * a.group + my_head;
  const float inv = sum == 0.0f ? 0.0f : a.value_scale / sum;
#pragma unroll
  for (int t = 0; t < kTiles; ++t)
#pragma unroll
    for (int i = 0; i < 16; i += 4) {
      const int d = 32 * t + 2 * i + 4 * half;
      if (d < dim)
        *reinterpret_cast<u32x2*>(a.out + row * dim + d) =
            (u32x2){pack2<DT>(acc[t][i] * inv, acc[t][i + 1] * inv),
                    pack2<DT>(acc[t][i + 2] * inv, acc[t][i + 3] * inv)};
    }
  if (a.lse && half == 0)
    a.lse[row] = sum == 0.0f ? -__builtin_inff()
                             : (base + __builtin_amdgcn_logf(sum)) * 0.6931471805599453f;
}

// The parts of a tile whose keys were split, joined in an order that does not change. Workgroup (tile of
// those, head; 32 dimensions; 32 rows): its waves take the parts in turn, in the layout that they were
// stored, and what they have is joined through LDS. With kWaves of 1 there are four to a workgroup, each
// with all parts of 32 rows.
template <int DT, int DIM, int kWaves>
__global__ __launch_bounds__(kWaves == 1 ? 256 : 64 * kWaves) void join_kernel(ChunkAttentionArgs a) {
  constexpr int kTiles = DIM / 32, kPart = kTile * (DIM + 2), kBatch = 4;
  const int lane = threadIdx.x & 63, in_group = uniform(threadIdx.x >> 6);
  const int wave = kWaves == 1 ? 0 : in_group, slab = kWaves == 1 ? in_group : blockIdx.z;
  const int col = lane & 31, half = lane >> 5;
  const int head = (int)(blockIdx.x % (unsigned)a.kv_heads), t = blockIdx.y;
  int behind;
  const Item item = find<true>(a, (int)(blockIdx.x / (unsigned)a.kv_heads), &behind);
  if (item.request < 0) return;
  const Request q = item.q;
  const int splits = item.splits, tile = item.tile(a), part = item.part;
  if (tile < 0 || part < 0 || part + splits > a.most_parts) return;
  const int row0 = tile * kTile, rows = min(kTile, q.count * a.group - row0);
  if (32 * slab >= rows) return;
  const float* from = a.parts + ((int64_t)part * a.kv_heads + head) * kPart;
  const int64_t step = (int64_t)a.kv_heads * kPart;

  float base = -__builtin_inff(), sum = 0.0f;
  float acc[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) acc[i] = 0.0f;
  auto fix_of = [](float from, float to) { return fmaxf(__builtin_amdgcn_exp2f(from - to), kTiny); };
  for (int n0 = wave; n0 < splits; n0 += kBatch * kWaves) {
    float b[kBatch], l[kBatch], v[kBatch][16];
#pragma unroll
    for (int n = 0; n < kBatch; ++n) {
      const float* p = from + min(n0 + n * kWaves, splits - 1) * step;
      b[n] = p[kTile * DIM + 32 * slab + col];
      l[n] = p[kTile * (DIM + 1) + 32 * slab + col];
#pragma unroll
      for (int i = 0; i < 16; ++i) v[n][i] = p[((slab * kTiles + t) * 16 + i) * 64 + lane];
    }
#pragma unroll
    for (int n = 0; n < kBatch; ++n) {
      if (n0 + n * kWaves >= splits || b[n] == -__builtin_inff()) continue;
      const float next = fmaxf(base, b[n]);
      const float old = fix_of(base, next), now = fix_of(b[n], next);
      sum = sum * old + l[n] * now;
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[i] = acc[i] * old + v[n][i] * now;
      base = next;
    }
  }
  const bool has_row = 32 * slab + col < rows;
  const int my_row = row0 + min(32 * slab + col, rows - 1);
  const int token = (int)div_by(my_row, a.by_group);
  const int64_t row = (int64_t)(q.start + token) * a.kv_heads * a.group + head * a.group +
                      (my_row - token * a.group);
  // values 4 g .. 4 g + 3 of a lane
  auto write = [&](int g, float x0, float x1, float x2, float x3) {
    const float inv = sum == 0.0f ? 0.0f : a.value_scale / sum;
    const int d = 32 * t + 8 * g + 4 * half;
    if (has_row && d < a.dim)
      *reinterpret_cast<u32x2*>(a.out + row * a.dim + d) =
          (u32x2){pack2<DT>(x0 * inv, x1 * inv), pack2<DT>(x2 * inv, x3 * inv)};
    if (has_row && a.lse && half == 0 && t == 0 && g == 0)
      a.lse[row] = sum == 0.0f ? -__builtin_inff()
                               : (base + __builtin_amdgcn_logf(sum)) * 0.6931471805599453f;
  };
  if constexpr (kWaves == 1) {
#pragma unroll
    for (int g = 0; g < 4; ++g) write(g, acc[4 * g], acc[4 * g + 1], acc[4 * g + 2], acc[4 * g + 3]);
  } else {
    __shared__ float kept[kWaves][16][64], bases[kWaves][64], sums[kWaves][64];
#pragma unroll
    for (int i = 0; i < 16; ++i) kept[wave][i][lane] = acc[i];
    bases[wave][lane] = base;
    sums[wave][lane] = sum;
    __syncthreads();
    if (wave >= 4) return;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) base = fmaxf(base, bases[w][lane]);
    sum = 0.0f;
    float x[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const float b = bases[w][lane];
      if (b == -__builtin_inff()) continue;
      const float now = fix_of(b, base);
      sum += sums[w][lane] * now;
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] += kept[w][4 * wave + e][lane] * now;
    }
    write(wave, x[0], x[1], x[2], x[3]);
  }
}

template <int DT, bool FP8, int DIM>
hipError_t launch_dim(const ChunkAttentionArgs& a, hipStream_t stream) {
  // Items: no more than there are tiles and, on top of them, even shares; or one request's tiles or parts.
  const int most = a.requests > 1 ? a.most_tiles + a.target : std::max(a.most_tiles, a.most_parts);
  const unsigned items = (unsigned)most * (unsigned)a.kv_heads;
  if (a.dim == DIM && a.narrow)
    attention_kernel<DT, FP8, DIM, false><<<items, kThreads, 0, stream>>>(a);
  else attention_kernel<DT, FP8, DIM, true><<<items, kThreads, 0, stream>>>(a);
  if (a.most_parts > 0) {
    // (a tile that has parts has two or more)
    const int tiles = std::min(a.most_tiles, a.most_parts / 2);
    const int slabs = (int)((std::min<int64_t>(kTile, (int64_t)a.tokens * a.group) + 31) / 32);
    dim3 grid((unsigned)tiles * (unsigned)a.kv_heads, DIM / 32, slabs);
    const int parts = std::min(a.target, a.most_parts) / tiles;  // of a tile
    // (us of a draft of 6 tokens with 4 waves and with 16: 33 parts 16.9 and 17.9, 128 28.0 and 24.7; of
    // 24 parts of prompts, which have one part or few, with 1 and with 4: 49.7 and 55.4)
    if (parts > 64) {
      join_kernel<DT, DIM, 16><<<grid, 1024, 0, stream>>>(a);
    } else if (parts > 4) {
      join_kernel<DT, DIM, 4><<<grid, 256, 0, stream>>>(a);
    } else {
      grid.z = 1;
      join_kernel<DT, DIM, 1><<<grid, 256, 0, stream>>>(a);
    }
  }
  return hipGetLastError();
}

template <int DT, bool FP8>
hipError_t launch_type(const ChunkAttentionArgs& a, hipStream_t stream) {
  if (a.dim <= 64) return launch_dim<DT, FP8, 64>(a, stream);
  if (a.dim <= 96) return launch_dim<DT, FP8, 96>(a, stream);
  if (a.dim <= 128) return launch_dim<DT, FP8, 128>(a, stream);
  if (a.dim <= 192) return launch_dim<DT, FP8, 192>(a, stream);
  return launch_dim<DT, FP8, 256>(a, stream);
}

hipError_t launch_bf16(const ChunkAttentionArgs& a, hipStream_t stream);
hipError_t launch_f16(const ChunkAttentionArgs& a, hipStream_t stream);
hipError_t launch_bf16_fp8(const ChunkAttentionArgs& a, hipStream_t stream);
hipError_t launch_f16_fp8(const ChunkAttentionArgs& a, hipStream_t stream);

}  // namespace chunk
}  // namespace mt
