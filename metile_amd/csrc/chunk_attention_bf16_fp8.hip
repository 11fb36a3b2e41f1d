// Chunk attention of bfloat16 queries over an 8-bit cache.
#include "chunk_attention_kernel.h"

namespace mt {
namespace chunk {
hipError_t launch_bf16_fp8(const ChunkAttentionArgs& a, hipStream_t stream) {
  return launch_type<kBF16, true>(a, stream);
}
}  // namespace chunk
}  // namespace mt
