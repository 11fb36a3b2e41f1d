// The norms around a model's blocks in one pass: a block's output through its own norm and gate
// into the scaled residual stream, and the next block's norm of that.
//
//   r = scale * residual + gate * post(block)        normed = pre(r)
//   rms(x) = x / sqrt(mean(x^2) + eps) * w           layer(x) = (x - mean) / sqrt(var + eps) * w
//
// each + a bias, if there is one. post and pre are both rms or both layer norms. Either input is read
// once and either output written once, with the row in fp32 registers between: the pre-norm sees r
// before its rounding to the stream's type, and the variance is that of deviations, in a second
// sum. Memory bounds it for many rows, the chain of one read and the row sums for few. A row belongs
// to 16 lanes up to a wave, or to a workgroup of 2 to 16 waves: threads take eight consecutive values
// at a time.
#include <algorithm>

#include "common.h"
#include "residual_norm.h"

namespace mt {
namespace {

// Eight consecutive values. Rows need not be aligned to more than their type: accesses are
// byte-addressed.
template <int DT>
__device__ __forceinline__ void read8(const uint16_t* p, float (&x)[8]) {
  u32x4 v;
  __builtin_memcpy(&v, p, 16);
  x[0] = lo16<DT>(v.x), x[1] = hi16<DT>(v.x), x[2] = lo16<DT>(v.y), x[3] = hi16<DT>(v.y);
  x[4] = lo16<DT>(v.z), x[5] = hi16<DT>(v.z), x[6] = lo16<DT>(v.w), x[7] = hi16<DT>(v.w);
}
template <int DT>
__device__ __forceinline__ void read8(const float* p, float (&x)[8]) {
  __builtin_memcpy(x, p, 32);
}
template <int DT>
__device__ __forceinline__ void write8(uint16_t* p, const float (&x)[8]) {
  u32x4 v;
#pragma unroll
  for (int j = 0; j < 4; ++j)
    v[j] = (uint32_t)f32_to_act<DT>(x[2 * j]) | (uint32_t)f32_to_act<DT>(x[2 * j + 1]) << 16;
  __builtin_memcpy(p, &v, 16);
}
template <int DT>
__device__ __forceinline__ void write8(float* p, const float (&x)[8]) {
  __builtin_memcpy(p, x, 32);
}

// Sum over 16, 32 or all lanes, the same in every one of them: exchanges within rows of 16 lanes,
// then across them.
template <int LANES>
__device__ __forceinline__ float lanes_sum(float v) {
  v += dpp_read<kDppXor1>(v);
  v += dpp_read<kDppXor2>(v);
  v += dpp_read<kDppHalfMirror>(v);
  v += dpp_read<0x140>(v);  // row_mirror
  if constexpr (LANES == 16) return v;
  if constexpr (LANES == 32) return v + __shfl_xor(v, 16);
  v += dpp_read_rows<kDppRowBcast15, 0xA>(v);
  v += dpp_read_rows<kDppRowBcast31, 0xC>(v);
  return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(v), 63));
}

// Sum over the threads of a row (every one gets it); `turn` alternates the LDS used.
template <int WAVES, int LANES>
__device__ __forceinline__ float row_sum(float v, float (&lds)[2][WAVES], int& turn) {
  v = lanes_sum<LANES>(v);
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

// LANES: of a wave that a row has to itself (16 or 32 only with one wave and vector).
template <int DT, typename RT, bool LAYER, int WAVES, int NV, int LANES>
__global__ __launch_bounds__(WAVES == 1 ? 256 : 64 * WAVES) void residual_norm_kernel(
    ResidualNormArgs a) {
  constexpr int kRowThreads = LANES * WAVES;
  constexpr int kRows = WAVES == 1 ? 256 / LANES : 1;  // rows of a workgroup
  __shared__ float lds[2][WAVES];
  int turn = 0;
  const int t = WAVES == 1 ? threadIdx.x & (LANES - 1) : threadIdx.x;
  const uint32_t row = a.first_row + blockIdx.x * kRows + (WAVES == 1 ? threadIdx.x / LANES : 0);
  if (WAVES == 1 && row >= (uint32_t)a.rows) return;
  const int width = a.width;

  const RT* res = static_cast<const RT*>(a.residual) + (int64_t)row * a.residual_stride;
  const uint16_t* blk = a.block ? a.block + (int64_t)row * a.block_stride : nullptr;

  // Vector n of a row is its values 8 n and on; the last one ends with the row and so overlaps the
  // one before, whose values it computes as well but does not count (`skip` of them). Threads
  // past the last vector repeat it and count nothing.
  int at[NV], skip[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int e = 8 * (t + i * kRowThreads);
    at[i] = min(e, width - 8);
    skip[i] = e < width ? e - at[i] : 8;
  }
  // A row has more than kSure vectors a thread (launch_width sees to it): only those behind can be
  // its last one or past it.
  constexpr int kSure = NV == 3 ? 2 : NV / 2;
  auto counted = [&](float v, int i, int j) {
    return i >= kSure && j < skip[i] ? 0.0f : v;
  };

  float x[NV][8], b[NV][8];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    read8<DT>(res + at[i], x[i]);
    if (blk) read8<DT>(blk + at[i], b[i]);
  }

  auto norm = [&](float (&v)[NV][8], const uint16_t* weight, const uint16_t* bias) {  // in place
    if constexpr (LAYER) {
      float s = 0.0f;
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) s += counted(v[i][j], i, j);
      const float mean = row_sum<WAVES, LANES>(s, lds, turn) / (float)width;
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) v[i][j] -= mean;
    }
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float c = counted(v[i][j], i, j);
        s = fmaf(c, c, s);
      }
    const float mean_sq = row_sum<WAVES, LANES>(s, lds, turn) / (float)width;
    const float inv = 1.0f / sqrtf(mean_sq + a.eps);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      float w[8];
      read8<DT>(weight + at[i], w);
      if (bias) {
        float c[8];
        read8<DT>(bias + at[i], c);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[i][j] = fmaf(v[i][j], inv * w[j], c[j]);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[i][j] *= inv * w[j];
      }
    }
  };

  if (blk) {
    if (a.post_weight) norm(b, a.post_weight, a.post_bias);
    if (a.gate) {
      const uint16_t* gate = a.gate + (int64_t)(row / (uint32_t)a.gate_rows) * a.gate_stride;
      const float one = act_to_f32<DT>(gate[0]);
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        float w[8];
        if (!a.gate_scalar) read8<DT>(gate + at[i], w);
#pragma unroll
        for (int j = 0; j < 8; ++j) b[i][j] *= a.gate_scalar ? one : w[j];
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
  if (out) {
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (skip[i] < 8) write8<DT>(out + (int64_t)row * width + at[i], x[i]);
  }
  norm(x, a.weight, a.bias);
#pragma unroll
  for (int i = 0; i < NV; ++i)
    if (skip[i] < 8) write8<DT>(a.normed + (int64_t)row * width + at[i], x[i]);
}

// Rows of fewer than eight values: a row a thread, value by value.
template <int DT, typename RT, bool LAYER>
__global__ __launch_bounds__(256) void residual_norm_narrow_kernel(ResidualNormArgs a) {
  const uint32_t row = a.first_row + blockIdx.x * 256 + threadIdx.x;
  if (row >= (uint32_t)a.rows) return;
  const int width = a.width;
  auto value = [](const uint16_t* p, int j) { return act_to_f32<DT>(p[j]); };
  auto norm = [&](float (&v)[8], const uint16_t* weight, const uint16_t* bias) {
    float mean = 0.0f, square = 0.0f;
    if constexpr (LAYER) {
#pragma unroll
      for (int j = 0; j < 8; ++j) mean += j < width ? v[j] : 0.0f;
      mean /= (float)width;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      v[j] -= mean;
      square = j < width ? fmaf(v[j], v[j], square) : square;
    }
    const float inv = 1.0f / sqrtf(square / (float)width + a.eps);
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j < width) v[j] = fmaf(v[j], inv * value(weight, j), bias ? value(bias, j) : 0.0f);
  };
  const RT* res = static_cast<const RT*>(a.residual) + (int64_t)row * a.residual_stride;
  float x[8], b[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    x[j] = b[j] = 0.0f;
    if (j >= width) continue;
    if constexpr (sizeof(RT) == 4) x[j] = res[j];
    else x[j] = value(res, j);
    if (a.block) b[j] = value(a.block + (int64_t)row * a.block_stride, j);
  }
  if (a.block && a.post_weight) norm(b, a.post_weight, a.post_bias);
  const uint16_t* gate = a.block && a.gate
                             ? a.gate + (int64_t)(row / (uint32_t)a.gate_rows) * a.gate_stride : nullptr;
  RT* out = static_cast<RT*>(a.residual_out);
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    if (j >= width) continue;
    if (gate) b[j] *= value(gate, a.gate_scalar ? 0 : j);
    x[j] = fmaf(x[j], a.scale, b[j]);
    if (!out) continue;
    if constexpr (sizeof(RT) == 4) out[(int64_t)row * width + j] = x[j];
    else out[(int64_t)row * width + j] = f32_to_act<DT>(x[j]);
  }
  norm(x, a.weight, a.bias);
#pragma unroll
  for (int j = 0; j < 8; ++j)
    if (j < width) a.normed[(int64_t)row * width + j] = f32_to_act<DT>(x[j]);
}

// One launch for every kMostBlocks workgroups (of `rows` rows each): the threads of a launch are
// counted in 32 bits, and those that do not fit are left out without an error.
constexpr int64_t kMostBlocks = 1 << 21;
template <typename K>
void launch_blocks(K kernel, const ResidualNormArgs& args, int rows, int threads,
                   hipStream_t stream) {
  ResidualNormArgs a = args;
  const int64_t blocks = ((int64_t)a.rows + rows - 1) / rows;
  for (int64_t first = 0; first < blocks; first += kMostBlocks) {
    a.first_row = (uint32_t)(first * rows);
    kernel<<<(uint32_t)std::min(blocks - first, kMostBlocks), threads, 0, stream>>>(a);
  }
}

template <int DT, typename RT, bool LAYER, int WAVES, int NV, int LANES = 64>
void launch_rows(const ResidualNormArgs& a, hipStream_t stream) {
  launch_blocks(residual_norm_kernel<DT, RT, LAYER, WAVES, NV, LANES>, a,
                WAVES == 1 ? 256 / LANES : 1, WAVES == 1 ? 256 : 64 * WAVES, stream);
}

// Waves of a row and vectors of a thread, by width and whether there are rows enough to fill the
// CUs with several of them. Few rows: a vector a thread, for the shortest chain (one row of 5120
// takes 2.5 us). Many: two a thread up to 8192 values, so that loads overlap without the registers
// of four costing half the waves, and sums cross as few waves as that allows. us, bf16, rms norm
// without and layer norm with a post-norm:
//   16384 x 4096    1 wave, 8 vectors 126 / 146    4, 2  98 / 98      16, 1  122 / 177
//   16384 x 2048    1, 4   51 / 56                 2, 2  45 / 47       4, 1   42 / 49
//    4096 x 8192    4, 4   51 / 58                 8, 2  45 / 49      16, 1   44 / 56
//    4096 x 896     1, 2   8.4 / 10.0              4, 1   9.4 / 13.1
//   16384 x 1133    1, 3  33 / 37                  2, 2   .. / 45       4, 1   36 / ..
//    4096 x 1536    1, 3  10.7 / 12.5              2, 2   .. / 13.6     4, 1   11.2 / ..
//    1024 x 1536    1, 3   5.7 / 6.7               2, 2   .. / 6.1      4, 1   4.5 / ..
//     768 x 4096    4, 2   7.3 / 8.7              16, 1   8.1 / 11.8
//     512 x 4096    4, 2   6.0 / 7.1              16, 1   5.7 / 8.6
//     768 x 896     1, 2   4.2 / 4.8               4, 1   3.6 / 4.8
// Rows of up to 256 values leave most of a wave idle: 16 lanes take those of up to 128, 32 the others.
//  100001 x 128    a wave  40 / 54    16 lanes  20 / 21
//  100001 x 256    a wave  45 / 60    32 lanes  35 / 37
//       1 x 256    a wave 2.0 / 2.4   32 lanes 2.1 / 2.5
//  100001 x 448    a wave  65 / 70    32 lanes, two vectors each  68 / 69
// (98 us for 16384 x 4096 are 5.5 TB/s; a copy of 1 GiB reaches 5.1 to 5.2.)
template <int DT, typename RT, bool LAYER>
void launch_width(const ResidualNormArgs& a, int cus, hipStream_t stream) {
  const int w = a.width;
  const bool many = w > 2048 ? a.rows > 2 * cus : a.rows >= 4 * cus;
  if (w < 8)
    launch_blocks(residual_norm_narrow_kernel<DT, RT, LAYER>, a, 256, 256, stream);
  else if (w <= 128) launch_rows<DT, RT, LAYER, 1, 1, 16>(a, stream);
  else if (w <= 256) launch_rows<DT, RT, LAYER, 1, 1, 32>(a, stream);
  else if (w <= 512) launch_rows<DT, RT, LAYER, 1, 1>(a, stream);
  else if (w <= 1024 && many) launch_rows<DT, RT, LAYER, 1, 2>(a, stream);
  else if (w <= 1536 && many && LAYER) launch_rows<DT, RT, LAYER, 1, 3>(a, stream);
  else if (w <= 2048 && many && LAYER) launch_rows<DT, RT, LAYER, 2, 2>(a, stream);
  else if (w <= 2048) launch_rows<DT, RT, LAYER, 4, 1>(a, stream);
  else if (w <= 4096 && many) launch_rows<DT, RT, LAYER, 4, 2>(a, stream);
  else if (w <= 8192 && many) launch_rows<DT, RT, LAYER, 8, 2>(a, stream);
  else if (w <= 8192) launch_rows<DT, RT, LAYER, 16, 1>(a, stream);
  else if (w <= 16384) launch_rows<DT, RT, LAYER, 16, 2>(a, stream);
  else if (w <= 32768) launch_rows<DT, RT, LAYER, 16, 4>(a, stream);
  else launch_rows<DT, RT, LAYER, 16, 8>(a, stream);
}

template <int DT, typename RT>
void launch_kind(const ResidualNormArgs& a, bool layer, int cus, hipStream_t stream) {
  if (layer) launch_width<DT, RT, true>(a, cus, stream);
  else launch_width<DT, RT, false>(a, cus, stream);
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
