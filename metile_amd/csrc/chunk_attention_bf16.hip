// Chunk attention of bfloat16 queries over a cache of their type.
#include "chunk_attention_kernel.h"

namespace mt {
namespace chunk {
hipError_t launch_bf16(const ChunkAttentionArgs& a, hipStream_t stream) {
  return launch_type<kBF16, false>(a, stream);
}
}  // namespace chunk
}  // namespace mt
