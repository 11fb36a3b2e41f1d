// Chunk attention of float16 queries over a cache of their type.
#include "chunk_attention_kernel.h"

namespace mt {
namespace chunk {
hipError_t launch_f16(const ChunkAttentionArgs& a, hipStream_t stream) {
  return launch_type<kF16, false>(a, stream);
}
}  // namespace chunk
}  // namespace mt
