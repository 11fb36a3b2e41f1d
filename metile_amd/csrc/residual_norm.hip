// The norms around a model's blocks in one pass: a block's output through its own norm and gate
// into the scaled residual stream, and the next block's norm of that.
//
//   r = scale * residual + gate * post(block)        normed = pre(r)
//   rms(x) = x / sqrt(mean(x^2) + eps) * w           layer(x) = (x - mean) / sqrt(var + eps) * w
//
// (each + a bias, if there is one.) post and pre are both rms or both layer norms; either input is read once and either output
// written once, with the row held in registers in fp32 between (the pre-norm sees r before its
// rounding to the stream's type; the variance is that of deviations, in a second sum). Memory
// bounds it for many rows, the chain of one read and the row sums for few. A row belongs to
// one wave, or to a workgroup of 4 or 16: threads take eight consecutive values at a time.
#include "common.h"
#include "residual_norm.h"

namespace mt {
namespace {

// Eight values, fewer at a row's end (the others read as zero). Rows need not be aligned to more
// than their type: the loads are byte-addressed.
template <int DT>
__device__ __forceinline__ void read8(const uint16_t* p, int n, float (&x)[8]) {
  if (n >= 8) {
    u32x4 v;
    __builtin_memcpy(&v, p, 16);
    x[0] = lo16<DT>(v.x), x[1] = hi16<DT>(v.x), x[2] = lo16<DT>(v.y), x[3] = hi16<DT>(v.y);
    x[4] = lo16<DT>(v.z), x[5] = hi16<DT>(v.z), x[6] = lo16<DT>(v.w), x[7] = hi16<DT>(v.w);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = j < n ? act_to_f32<DT>(p[j]) : 0.0f;
  }
}
template <int DT>
__device__ __forceinline__ void read8(const float* p, int n, float (&x)[8]) {
  if (n >= 8) {
    __builtin_memcpy(x, p, 32);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = j < n ? p[j] : 0.0f;
  }
}
template <int DT>
__device__ __forceinline__ void write8(uint16_t* p, int n, const float (&x)[8]) {
  if (n >= 8) {
    u32x4 v;
#pragma unroll
    for (int j = 0; j < 4; ++j)
      v[j] = (uint32_t)f32_to_act<DT>(x[2 * j]) | (uint32_t)f32_to_act<DT>(x[2 * j + 1]) << 16;
    __builtin_memcpy(p, &v, 16);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j < n) p[j] = f32_to_act<DT>(x[j]);
  }
}
template <int DT>
__device__ __forceinline__ void write8(float* p, int n, const float (&x)[8]) {
  if (n >= 8) {
    __builtin_memcpy(p, x, 32);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j < n) p[j] = x[j];
  }
}

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
  for (int d = 32; d; d >>= 1) v += __shfl_xor(v, d);
  return v;
}

// Sum over the threads of a row (every one gets it); `turn` alternates the LDS used.
template <int WAVES>
__device__ __forceinline__ float row_sum(float v, float (&lds)[2][WAVES], int& turn) {
  v = wave_sum(v);
  if constexpr (WAVES > 1) {
    const int wave = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0) lds[turn][wave] = v;
    __syncthreads();
    v = 0.0f;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) v += lds[turn][w];
    turn ^= 1;
  }
  return v;
}

template <int DT, typename RT, bool LAYER, int WAVES, int NV>
__global__ __launch_bounds__(WAVES == 1 ? 256 : 64 * WAVES) void residual_norm_kernel(
    ResidualNormArgs a) {
  constexpr int kRowThreads = 64 * WAVES;
  constexpr int kRows = WAVES == 1 ? 4 : 1;  // rows of a workgroup
  __shared__ float lds[2][WAVES];
  int turn = 0;
  const int t = WAVES == 1 ? threadIdx.x & 63 : threadIdx.x;
  const int row = blockIdx.x * kRows + (WAVES == 1 ? threadIdx.x >> 6 : 0);
  if (WAVES == 1 && row >= a.rows) return;
  const int width = a.width;

  const RT* res = static_cast<const RT*>(a.residual) + (int64_t)row * a.residual_stride;
  const uint16_t* blk = a.block ? a.block + (int64_t)row * a.block_stride : nullptr;
  float x[NV][8], b[NV][8];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int e = 8 * (t + i * kRowThreads);
    read8<DT>(res + (e < width ? e : 0), e < width ? width - e : 0, x[i]);
    if (blk) read8<DT>(blk + (e < width ? e : 0), e < width ? width - e : 0, b[i]);
  }

  // in place; values past the row's end stay zero
  auto norm = [&](float (&v)[NV][8], const uint16_t* weight, const uint16_t* bias) {
    if constexpr (LAYER) {
      float s = 0.0f;
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) s += v[i][j];
      const float mean = row_sum<WAVES>(s, lds, turn) / (float)width;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int left = width - 8 * (t + i * kRowThreads);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[i][j] = j < left ? v[i][j] - mean : 0.0f;
      }
    }
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) s = fmaf(v[i][j], v[i][j], s);
    const float mean_sq = row_sum<WAVES>(s, lds, turn) / (float)width;
    const float inv = 1.0f / sqrtf(mean_sq + a.eps);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int e = 8 * (t + i * kRowThreads);
      if (e >= width) continue;
      float w[8];
      read8<DT>(weight + e, width - e, w);
      if (bias) {
        float b[8];
        read8<DT>(bias + e, width - e, b);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[i][j] = fmaf(v[i][j], inv * w[j], b[j]);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[i][j] *= inv * w[j];
      }
    }
  };

  if (blk) {
    if (a.post_weight) norm(b, a.post_weight, a.post_bias);
    if (a.gate) {
      const uint16_t* gate = a.gate + (int64_t)(row / a.gate_rows) * a.gate_stride;
      const float one = a.gate_scalar ? act_to_f32<DT>(gate[0]) : 0.0f;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int e = 8 * (t + i * kRowThreads);
        if (e >= width) continue;
        float w[8];
        if (a.gate_scalar) {
#pragma unroll
          for (int j = 0; j < 8; ++j) w[j] = one;
        } else {
          read8<DT>(gate + e, width - e, w);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) b[i][j] *= w[j];
      }
    }
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) x[i][j] = fmaf(x[i][j], a.scale, b[i][j]);
  } else {
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) x[i][j] *= a.scale;
  }
  RT* out = static_cast<RT*>(a.residual_out);
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int e = 8 * (t + i * kRowThreads);
    if (e >= width) {
#pragma unroll
      for (int j = 0; j < 8; ++j) x[i][j] = 0.0f;
    } else {
      if (out) write8<DT>(out + (int64_t)row * width + e, width - e, x[i]);
#pragma unroll
      for (int j = 0; j < 8; ++j) x[i][j] = e + j < width ? x[i][j] : 0.0f;
    }
  }
  norm(x, a.weight, a.bias);
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int e = 8 * (t + i * kRowThreads);
    if (e < width) write8<DT>(a.normed + (int64_t)row * width + e, width - e, x[i]);
  }
}

template <int DT, typename RT, bool LAYER, int WAVES>
void launch_vectors(const ResidualNormArgs& a, hipStream_t stream) {
  const int rows = WAVES == 1 ? 4 : 1, threads = WAVES == 1 ? 256 : 64 * WAVES;
  const int blocks = (a.rows + rows - 1) / rows;
  const int vectors = (a.width + 512 * WAVES - 1) / (512 * WAVES);
  if (vectors <= 1)
    residual_norm_kernel<DT, RT, LAYER, WAVES, 1><<<blocks, threads, 0, stream>>>(a);
  else if (vectors <= 2)
    residual_norm_kernel<DT, RT, LAYER, WAVES, 2><<<blocks, threads, 0, stream>>>(a);
  else if (vectors <= 4)
    residual_norm_kernel<DT, RT, LAYER, WAVES, 4><<<blocks, threads, 0, stream>>>(a);
  else
    residual_norm_kernel<DT, RT, LAYER, WAVES, 8><<<blocks, threads, 0, stream>>>(a);
}

template <int DT, typename RT, bool LAYER>
void launch_waves(const ResidualNormArgs& a, int cus, hipStream_t stream) {
  const bool many = a.rows >= 8 * cus;
  if (a.width <= (many ? 2048 : 512)) launch_vectors<DT, RT, LAYER, 1>(a, stream);
  else if (a.width <= (many ? 8192 : 2048)) launch_vectors<DT, RT, LAYER, 4>(a, stream);
  else launch_vectors<DT, RT, LAYER, 16>(a, stream);
}

template <int DT, typename RT>
void launch_kind(const ResidualNormArgs& a, bool layer, int cus, hipStream_t stream) {
  if (layer) launch_waves<DT, RT, true>(a, cus, stream);
  else launch_waves<DT, RT, false>(a, cus, stream);
}

}  // namespace

hipError_t launch_residual_norm(const ResidualNormArgs& a, int dtype, bool residual_f32, bool layer,
                                int cus, hipStream_t stream) {
  if (dtype == kBF16) {
    if (residual_f32) launch_kind<kBF16, float>(a, layer, cus, stream);
    else launch_kind<kBF16, uint16_t>(a, layer, cus, stream);
  } else {
    if (residual_f32) launch_kind<kF16, float>(a, layer, cus, stream);
    else launch_kind<kF16, uint16_t>(a, layer, cus, stream);
  }
  return hipGetLastError();
}

}  // namespace mt
