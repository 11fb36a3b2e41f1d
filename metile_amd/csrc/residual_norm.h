// Host-visible launch interface of the norms around a model's blocks.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace mt {

constexpr int kNormMaxWidth = 65536;

// Pointers may be null as noted; strides in elements.
struct ResidualNormArgs {
  const void* residual;         // [rows, width], 16-bit or fp32
  const uint16_t* block;        // [rows, width] or null
  const uint16_t* weight;       // [width]
  const uint16_t* bias;         // [width] or null
  const uint16_t* post_weight;  // [width] or null: no norm of the block's output
  const uint16_t* post_bias;    // [width] or null
  const uint16_t* gate;         // or null
  void* residual_out;           // [rows, width] contiguous, residual's type; null: not written
  uint16_t* normed;             // [rows, width] contiguous
  int64_t residual_stride, block_stride, gate_stride;  // of a row (of the gate: of its own rows)
  int32_t rows, width;
  uint32_t first_row;   // of the launch (its own to set)
  int32_t gate_rows;    // rows of the batch that share one row of the gate
  int32_t gate_scalar;  // the gate's rows hold one value each
  float scale, eps;
};
hipError_t launch_residual_norm(const ResidualNormArgs& a, int dtype, bool residual_f32, bool layer,
                                int cus, hipStream_t stream);

}  // namespace mt
