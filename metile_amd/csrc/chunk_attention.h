// Host-visible launch interface of the attention of chunks of new tokens over a paged cache.
#pragma once

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "paged.h"

namespace mt {

// Rows (token, query head of a key-value head) of a tile, and keys of a block.
constexpr int kChunkTile = 128;
constexpr int kChunkBlock = 64;
// Tiles of fewer blocks are not split, and a part has at least two (a draft of 6 tokens over 2049 keys, us:
// 15.5 with four, 14.2), or four in calls with so many blocks that there would be more than 64 parts (over
// 32768 keys 24.0 with four, 29.1).
constexpr int kChunkLeastSplit = 4, kChunkLeastBlocks = 2;
// Requests of a call whose work its workgroups count up themselves.
constexpr int kChunkHere = 64;

struct ChunkAttentionArgs {
  const uint16_t* query;                // [tokens, heads, dim], last dimension contiguous
  int64_t q_row_stride, q_head_stride;  // elements
  const unsigned char* key;
  const unsigned char* value;
  uint32_t k_page, k_slot, v_page, v_slot;  // bytes
  int64_t k_head, v_head;
  const int32_t* tables;                // [requests, width], rows `table_stride` entries apart
  int64_t table_stride;
  const int32_t* lengths;               // [requests]
  const int32_t* starts;                // [requests + 1]
  uint16_t* out;                        // [tokens, heads, dim] contiguous
  float* lse;                           // [tokens, heads] or null
  int32_t* plan;                        // kPlanHead + 3 (requests + 1) entries
  float* parts;                         // slots of chunk_part_floats each
  int32_t tokens, requests, kv_heads, group, dim, pages, page_size, width, window;
  int32_t target;                       // items that the work is split into, if it can be
  int32_t slots;                        // workgroups that run at once
  int32_t most_tiles, most_parts;       // of one key-value head
  float scale_log2, value_scale;
  bool narrow;                          // every row of a head begins less than 4 GiB behind its first
  uint32_t flip;                        // sign bits of a query pair to flip
  DivMagic by_page, by_group;
};

// In front of the plan: blocks of a split, then items and tiles with parts of one key-value head. Behind it
// the sums of items, parts and tiles with parts of the requests before each. Calls of up to kChunkHere requests
// have the first alone, from the attention for the join.
constexpr int kPlanHead = 4;
// Floats of a part: 16 a lane and 32 dimensions, then reference and sum of each row.
size_t chunk_part_floats(int dim);

// Bounds of a call's tiles and parts of one key-value head, and the items wanted of it, from shapes.
struct ChunkPlan {
  int tiles, parts, target, slots;
};
ChunkPlan plan_chunk_attention(int tokens, int requests, int kv_heads, int group, int dim,
                               int64_t most_keys, int window, int cus);

hipError_t launch_chunk_attention(const ChunkAttentionArgs& a, int dtype, bool fp8,
                                  hipStream_t stream);

}  // namespace mt
