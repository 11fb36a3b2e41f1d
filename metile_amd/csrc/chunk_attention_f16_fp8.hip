// Chunk attention of float16 queries over an 8-bit cache.
#include "chunk_attention_kernel.h"

namespace mt {
namespace chunk {
hipError_t launch_f16_fp8(const ChunkAttentionArgs& a, hipStream_t stream) {
  return launch_type<kF16, true>(a, stream);
}
}  // namespace chunk
}  // namespace mt
