// A step's keys and values written to their slots of a paged cache.
//
// Each row is read once and written once; nothing else is to do but the conversion to 8-bit
// floats (e4m3: the value over the cache's scale, limited to +-448, rounded to nearest even), so
// memory bounds it. A thread moves eight values (16 bytes in) twice, side by side (16384 tokens of
// 8 heads of 128 into 8 bits, 101 MB: 23.2 us, 4.3 TB/s; four times 25.4, once 25.1); keys and values
// are the two halves of the grid.
#include "common.h"
#include "paged.h"

namespace mt {
namespace {

constexpr int kThreads = 256;
constexpr int kUnroll = 2;

// x / scale, rounded once (the product with the reciprocal, corrected by its exact residue),
// limited to e4m3's largest number; NaN stays.
__device__ __forceinline__ float held(float x, float scale, float inv) {
  float q = x * inv;
  if (fabsf(q) < 512.0f) q = fmaf(fmaf(-q, scale, x), inv, q);
  return q > 448.0f ? 448.0f : q < -448.0f ? -448.0f : q;
}

template <int DT, bool FP8>
__global__ __launch_bounds__(kThreads) void paged_append_kernel(PagedAppendArgs a,
                                                                uint32_t chunks) {
  const PagedSide& s = a.side[blockIdx.y];
  const uint32_t limit = (uint32_t)a.pages * (uint32_t)a.page_size;
  const uint32_t first = blockIdx.x * (kThreads * kUnroll) + threadIdx.x;
  // every row and slot is requested before any is stored; only stores go by the slot
  u32x4 v[kUnroll];
  unsigned char* to[kUnroll];
#pragma unroll
  for (int i = 0; i < kUnroll; ++i) {
    const uint32_t n = min(first + i * kThreads, chunks - 1);
    const uint32_t token = div_by(n, a.by_row);
    const uint32_t rest = n - token * (uint32_t)(a.heads * (a.dim >> 3));
    const uint32_t head = div_by(rest, a.by_head);
    const uint32_t chunk = rest - head * (uint32_t)(a.dim >> 3);
    v[i] = *reinterpret_cast<const u32x4*>(s.rows + (int64_t)token * s.row_stride +
                                           (int64_t)head * s.row_head_stride + chunk * 16);
    const int64_t slot = a.slots[token];
    const bool here = first + i * kThreads < chunks && slot >= 0 && slot < (int64_t)limit;
    const uint32_t page = div_by(here ? (uint32_t)slot : 0u, a.by_page);
    const uint32_t in_page = (uint32_t)slot - page * (uint32_t)a.page_size;
    to[i] = here ? s.cache + (uint64_t)page * s.page_stride + (uint64_t)in_page * s.slot_stride +
                       (int64_t)head * s.head_stride + chunk * (FP8 ? 8 : 16)
                 : nullptr;
  }
#pragma unroll
  for (int i = 0; i < kUnroll; ++i) {
    if (!to[i]) continue;
    if constexpr (!FP8) {
      *reinterpret_cast<u32x4*>(to[i]) = v[i];
    } else {
      uint32_t w[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint32_t x = h ? v[i].z : v[i].x, y = h ? v[i].w : v[i].y;
        int b = __builtin_amdgcn_cvt_pk_fp8_f32(held(lo16<DT>(x), s.scale, s.inv_scale),
                                                held(hi16<DT>(x), s.scale, s.inv_scale), 0, false);
        b = __builtin_amdgcn_cvt_pk_fp8_f32(held(lo16<DT>(y), s.scale, s.inv_scale),
                                            held(hi16<DT>(y), s.scale, s.inv_scale), b, true);
        w[h] = (uint32_t)b;
      }
      *reinterpret_cast<u32x2*>(to[i]) = (u32x2){w[0], w[1]};
    }
  }
}

}  // namespace

hipError_t launch_paged_append(const PagedAppendArgs& a, int dtype, bool fp8, hipStream_t stream) {
  const uint32_t chunks = (uint32_t)(a.tokens * a.heads * (a.dim >> 3));  // host: below 2^31
  const dim3 grid((chunks + kThreads * kUnroll - 1) / (kThreads * kUnroll), 2);
  if (!fp8)  // a copy of 16-bit values, whichever they are
    paged_append_kernel<kBF16, false><<<grid, kThreads, 0, stream>>>(a, chunks);
  else if (dtype == kBF16)
    paged_append_kernel<kBF16, true><<<grid, kThreads, 0, stream>>>(a, chunks);
  else
    paged_append_kernel<kF16, true><<<grid, kThreads, 0, stream>>>(a, chunks);
  return hipGetLastError();
}

}  // namespace mt
