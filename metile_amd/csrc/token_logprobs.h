// Host-visible launch interface of the log probabilities of tokens.
#pragma once

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace mt {

constexpr int kLogprobsMostTop = 32;

struct LogprobsArgs {
  const void* logits;     // [rows, vocab], rows `row_stride` elements apart
  int64_t row_stride;
  const int64_t* tokens;  // [rows] or null
  float* logprobs;        // [rows] or null with tokens
  float* entropies;       // [rows]
  int32_t* ranks;         // [rows] or null with tokens
  float* top_logprobs;    // [rows, top]
  int64_t* top_tokens;    // [rows, top]
  unsigned char* parts;   // of rows in several parts
  int32_t rows, vocab, top;
  int32_t threads, part_batches, num_parts;  // of a workgroup; batches of a part, parts of a row
  float inv_temperature;
};

// How a call's rows are split: threads of a workgroup, batches of a part, parts of a row.
struct LogprobsPlan {
  int threads, part_batches, num_parts;
};
LogprobsPlan plan_token_logprobs(int rows, int vocab, int cus);
size_t logprobs_part_bytes(int top);
// dtype: kBF16, kF16, or 2 for fp32.
hipError_t launch_token_logprobs(const LogprobsArgs& a, int dtype, hipStream_t stream);

}  // namespace mt
