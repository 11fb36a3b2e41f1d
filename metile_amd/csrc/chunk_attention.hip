// Attention of chunks of new tokens over a paged cache: how the work is split, and the launches.
//
// An item is a tile of 128 rows of one request and key-value head, with all of its keys or, where
// the call has too few tiles to fill the GPU evenly, an equal part of them. The lengths are known on
// the device alone: with `total` blocks of keys over all tiles and `target` items wanted, tiles of more
// than total / target blocks are split. Up to 64 requests are counted up by every wave of the attention
// for itself (a draft of 6 tokens over 2049 keys 25.7 -> 21.4 us without a launch before it), more by
// a launch of one workgroup, in whose sums the attention's then search. A last launch joins the parts, a
// workgroup a tile (that draft 16.9 -> 14.2 us with smaller parts; over 131072 keys 99 -> 44).
#include <algorithm>

#include "chunk_attention.h"
#include "chunk_attention_kernel.h"

namespace mt {
namespace chunk {
namespace {

constexpr int kPlanThreads = 1024;
__device__ __forceinline__ int64_t most31(int64_t v) { return v < 0x7fffffff ? v : 0x7fffffff; }

__global__ __launch_bounds__(kPlanThreads) void plan_kernel(ChunkAttentionArgs a) {
  __shared__ int64_t sums[3][kPlanThreads];
  const int tid = threadIdx.x;
  const int run = (a.requests + kPlanThreads - 1) / kPlanThreads;
  const int begin = min(tid * run, a.requests), end = min(begin + run, a.requests);
  int64_t blocks = 0;
  for (int r = begin; r < end; ++r) {
    const Request q = request_of(a, r);
    blocks += (int64_t)tiles_of(a, q) * most_blocks(a, q);
  }
  sums[0][tid] = blocks;
  __syncthreads();
  for (int step = kPlanThreads / 2; step; step /= 2) {
    if (tid < step) sums[0][tid] += sums[0][tid + step];
    __syncthreads();
  }
  const int64_t total = sums[0][0];
  __syncthreads();
  const int per = (int)most31(max((total + a.target - 1) / a.target, (int64_t)least_blocks((float)total)));
  int64_t items = 0, parts = 0, joins = 0;
  for (int r = begin; r < end; ++r) {
    const Request q = request_of(a, r);
    const int64_t tiles = tiles_of(a, q);
    const int splits = splits_of(most_blocks(a, q), per);
    items += tiles * splits;
    if (splits > 1) parts += tiles * splits, joins += tiles;
  }
  sums[0][tid] = items;
  sums[1][tid] = parts;
  sums[2][tid] = joins;
  __syncthreads();
  for (int step = 1; step < kPlanThreads; step *= 2) {
    const int64_t x = tid >= step ? sums[0][tid - step] : 0;
    const int64_t y = tid >= step ? sums[1][tid - step] : 0;
    const int64_t z = tid >= step ? sums[2][tid - step] : 0;
    __syncthreads();
    sums[0][tid] += x;
    sums[1][tid] += y;
    sums[2][tid] += z;
    __syncthreads();
  }
  items = sums[0][tid] - items;
  parts = sums[1][tid] - parts;
  joins = sums[2][tid] - joins;
  int32_t* item_sums = a.plan + kPlanHead;
  int32_t* part_sums = item_sums + a.requests + 1;
  int32_t* join_sums = part_sums + a.requests + 1;
  for (int r = begin; r < end; ++r) {
    item_sums[r] = (int32_t)most31(items);
    part_sums[r] = (int32_t)most31(parts);
    join_sums[r] = (int32_t)most31(joins);
    const Request q = request_of(a, r);
    const int64_t tiles = tiles_of(a, q);
    const int splits = splits_of(most_blocks(a, q), per);
    items += tiles * splits;
    if (splits > 1) parts += tiles * splits, joins += tiles;
  }
  if (tid == kPlanThreads - 1) {
    a.plan[0] = per;
    a.plan[1] = item_sums[a.requests] = (int32_t)most31(sums[0][tid]);
    part_sums[a.requests] = (int32_t)most31(sums[1][tid]);
    a.plan[2] = join_sums[a.requests] = (int32_t)most31(sums[2][tid]);
  }
}

int padded_dim(int dim) {
  return dim <= 64 ? 64 : dim <= 96 ? 96 : dim <= 128 ? 128 : dim <= 192 ? 192 : 256;
}

}  // namespace
}  // namespace chunk

size_t chunk_part_floats(int dim) { return (size_t)kChunkTile * (chunk::padded_dim(dim) + 2); }

ChunkPlan plan_chunk_attention(int tokens, int requests, int kv_heads, int group, int dim,
                               int64_t most_keys, int window, int cus) {
  ChunkPlan p;
  p.tiles = (int)((int64_t)tokens * group / kChunkTile) + std::min(requests, tokens);
  p.slots = (dim <= 128 ? 2 : 1) * cus;
  p.target = (p.slots + kv_heads - 1) / kv_heads;
  if (window > 0) most_keys = std::min<int64_t>(most_keys, (int64_t)window + kChunkTile);
  const int64_t blocks = (most_keys + kChunkBlock - 1) / kChunkBlock + (window > 0);
  const int64_t splits =
      blocks < kChunkLeastSplit ? 1 : (blocks + kChunkLeastBlocks - 1) / kChunkLeastBlocks;
  p.parts = splits > 1 ? (int)std::min<int64_t>(2 * p.target, splits * p.tiles) : 0;
  return p;
}

hipError_t launch_chunk_attention(const ChunkAttentionArgs& args, int dtype, bool fp8,
                                  hipStream_t stream) {
  ChunkAttentionArgs a = args;
  a.by_page = div_magic((uint32_t)a.page_size);
  a.by_group = div_magic((uint32_t)a.group);
  if (a.requests > kChunkHere) chunk::plan_kernel<<<1, chunk::kPlanThreads, 0, stream>>>(a);
  if (dtype == kBF16) return fp8 ? chunk::launch_bf16_fp8(a, stream) : chunk::launch_bf16(a, stream);
  return fp8 ? chunk::launch_f16_fp8(a, stream) : chunk::launch_f16(a, stream);
}

}  // namespace mt
