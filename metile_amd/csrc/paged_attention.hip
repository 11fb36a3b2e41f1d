// Decode attention over a paged key-value cache: one new token of each request.
//
//   s_t = scale * q . k_t      o = sum_t exp(s_t - m) v_t / sum_t exp(s_t - m)      m = max_t s_t
//
// in one pass over the pages with a running maximum and sum (in powers of two: the scale holds
// log2 e). A workgroup takes tiles of 128 tokens of one row (request, key-value head, up to 16
// query heads that share it), 32 tokens a wave and tile:
//  * keys: v_mfma_f32_16x16x32 with the keys as rows and the query heads as columns, so a lane
//    holds scores of one head, eight consecutive tokens of it in two tiles (row i of tile t is
//    token 8 (i / 4) + 4 t + i % 4);
//  * values: a lane loads DIM / 16 dimensions of eight consecutive tokens; eight byte permutes
//    a dimension pair turn them into operands with the dimensions as rows, and the lane's own
//    eight probabilities are the other operand as they stand: no exchange between lanes, no LDS.
//    The result has the head in the lane again, so rescaling is local to the lane.
// Probabilities go to the matrix cores as two 16-bit parts (their rounding and the rest of it),
// so the 16-bit rounding of the result is the only one; sums, maxima and results are fp32. (The
// second part is zero or negative as often as not, and an infinite value times it is no number: a
// segment whose sums are not finite is taken again with the first parts alone, which are positive.)
//
// Split: all tiles of all rows, laid end to end, are dealt out in equal contiguous runs to a
// fixed number of workgroups (each finds its place from a scan over the lengths), so ragged
// batches balance by themselves. Parts of a row that several workgroups share are stored with
// their maximum and sum and joined, in order, by the last of them to arrive.
#include "common.h"
#include "paged.h"

namespace mt {
namespace {

constexpr int kWaves = 4;
constexpr int kThreads = 64 * kWaves;
constexpr int kTile = kAttentionTile;
static_assert(kTile == 32 * kWaves, "a wave takes 32 tokens of a tile");

__device__ __forceinline__ int wave_scan(int v, int lane) {  // inclusive
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int o = __shfl_up(v, d);
    if (lane >= d) v += o;
  }
  return v;
}

__device__ __forceinline__ int readlane(int v, int l) { return __builtin_amdgcn_readlane(v, l); }
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

// A request's tokens as they are read: its length, the first token of its window rounded down to
// 32, and its tiles (one for an empty request, which writes its zeros).
struct Span {
  int len, first, base, tiles;
};
__device__ __forceinline__ Span span_of(int length, int most, int window) {
  Span s;
  s.len = length < 0 ? 0 : (length > most ? most : length);
  s.first = window > 0 && s.len > window ? s.len - window : 0;
  s.base = s.first & ~31;
  const int n = (int)(((unsigned)(s.len - s.base) + kTile - 1) / kTile);
  s.tiles = n > 0 ? n : 1;
  return s;
}

template <int DT>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  return (uint32_t)f32_to_act<DT>(a) | (uint32_t)f32_to_act<DT>(b) << 16;
}

// Two 8-bit floats (half HI of a word) as 16-bit ones: exact.
template <int DT, bool HI>
__device__ __forceinline__ uint32_t fp8_pair(uint32_t w) {
  if constexpr (DT == kBF16)
    return __builtin_bit_cast(uint32_t,
                              __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)w, 1.0f, HI));
  else
    return __builtin_bit_cast(uint32_t,
                              __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)w, 1.0f, HI));
}
template <int DT>
__device__ __forceinline__ u32x4 fp8_eight(uint32_t lo, uint32_t hi) {
  return (u32x4){fp8_pair<DT, false>(lo), fp8_pair<DT, true>(lo), fp8_pair<DT, false>(hi),
                 fp8_pair<DT, true>(hi)};
}

template <int DT, bool FP8, int DIM, bool PAGE8>
__global__ __launch_bounds__(kThreads, 2) void paged_attention_kernel(PagedAttentionArgs a,
                                                                      int slot_floats) {
  constexpr int kElt = FP8 ? 1 : 2;
  constexpr int kMfmas = DIM / 32;               // K depth of a score
  constexpr int kLaneDims = DIM / 16;            // value dimensions of a lane
  constexpr int kKeyLoads = kMfmas * kElt / 2;   // 16-byte loads of a key row a lane makes
  constexpr int kValueWords = kLaneDims * kElt / 4;
  // f16 probabilities are scaled up so that small ones, and the second parts, stay above its
  // smallest numbers; the sum carries the same factor.
  constexpr float kShift = DT == kF16 ? 14.0f : 0.0f;

  __shared__ float lds_acc[kWaves][16][DIM];
  __shared__ float lds_m[kWaves][16];
  __shared__ float lds_l[kWaves][16];
  __shared__ int lds_last;

  const int tid = threadIdx.x;
  const int lane = tid & 63, wave = uniform(tid >> 6);
  const int c = lane & 15, g = lane >> 4;
  const int most = a.width * a.page_size;  // the host checks that it fits 31 bits
  const int hr_count = a.kv_heads * a.head_tiles;
  const int hcnt = a.group < 16 ? a.group : 16;

  // ---- this workgroup's run of tiles ----
  const int chunk = (a.requests + 63) >> 6;
  int mine = 0;
  for (int i = 0; i < chunk; ++i) {
    const int r = lane * chunk + i;
    if (r < a.requests) mine += span_of(a.lengths[r], most, a.window).tiles;
  }
  const int inc = wave_scan(mine, lane);
  const int64_t units = (int64_t)readlane(inc, 63) * hr_count;
  const int64_t per = (units + gridDim.x - 1) / gridDim.x;
  int64_t u = (int64_t)blockIdx.x * per;
  if (u >= units) return;
  const int64_t u_end = u + per < units ? u + per : units;
  const int target = (int)(u / hr_count);
  const int owner = __ffsll(__ballot(inc > target)) - 1;
  int prefix = readlane(inc, owner) - readlane(mine, owner);  // tiles of the requests before r
  int piece = owner * chunk;                                  // 64 requests from `piece` on: lens
  int len_lane = 0, r = piece;
  for (;;) {
    len_lane = piece + lane < a.requests ? a.lengths[piece + lane] : 0;
    const int t = piece + lane < a.requests ? span_of(len_lane, most, a.window).tiles : 0;
    const int s = wave_scan(t, lane) + prefix;
    const uint64_t hit = __ballot(s > target);
    if (hit) {
      const int at = __ffsll((unsigned long long)hit) - 1;
      r = piece + at;
      prefix = readlane(s, at) - readlane(t, at);
      break;
    }
    prefix = readlane(s, 63);
    piece += 64;
    if (piece >= a.requests) return;  // only if the lengths changed under the scan
  }
  Span sp = span_of(readlane(len_lane, r - piece), most, a.window);
  int hr, tile;
  int64_t row_u;  // unit of the row's first tile
  {
    const int off = (int)(u - (int64_t)prefix * hr_count);
    hr = off / sp.tiles;
    tile = off - hr * sp.tiles;
    row_u = u - tile;
  }

  const int page_size = a.page_size;

  while (u < u_end && r < a.requests) {
    const int tile_end = sp.tiles - tile <= u_end - u ? sp.tiles : tile + (int)(u_end - u);
    const int kv = hr / a.head_tiles;
    const int head0 = kv * a.group + (hr - kv * a.head_tiles) * 16;
    const int heads = a.group - (hr - kv * a.head_tiles) * 16 < 16
                          ? a.group - (hr - kv * a.head_tiles) * 16 : 16;
    const int32_t* table = a.tables + (int64_t)r * a.table_stride;
    const unsigned char* kbase = a.key + (int64_t)kv * a.k_head;
    const unsigned char* vbase = a.value + (int64_t)kv * a.v_head;
    const int len = sp.len, first = sp.first, last = len - 1;

    // ---- the query heads, as columns: dimensions in the order of the key loads ----
    u32x4 q[kMfmas];
    {
      const bool has = c < heads;
      const uint16_t* row = a.query + (int64_t)r * a.q_row_stride +
                            (int64_t)(head0 + (has ? c : 0)) * a.q_head_stride;
#pragma unroll
      for (int k = 0; k < kMfmas; ++k) {
        const int d = FP8 ? 64 * (k >> 1) + 16 * g + 8 * (k & 1) : 32 * k + 8 * g;
        q[k] = (u32x4){0, 0, 0, 0};
        if (has && d < a.dim) q[k] = *reinterpret_cast<const u32x4*>(row + d);
      }
    }

    float m = -__builtin_inff(), l = 0.0f;
    f32x4 acc[kLaneDims];
#pragma unroll
    for (int e = 0; e < kLaneDims; ++e) acc[e] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};

    u32x4 kf[2][kKeyLoads];
    uint32_t vf[8][kValueWords];
    bool v_ok[PAGE8 ? 1 : 8];

    // Tokens past the end read the last one; tokens of a page that is none of the cache's read
    // page 0. Both are masked.
    auto page_of = [&](int token, bool& ok) {
      const int col = (int)div_by((uint32_t)token, a.by_page);
      const int p = table[col];
      ok = (uint32_t)p < (uint32_t)a.pages;
      return (int2){ok ? p : 0, token - col * page_size};
    };
    auto load_keys = [&](int tok0) {
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        int token = tok0 + 8 * (c >> 2) + 4 * t + (c & 3);
        token = token < last ? token : last;
        bool ok;
        const int2 at = page_of(token, ok);
        const unsigned char* p = kbase + (int64_t)at.x * a.k_page + (int64_t)at.y * a.k_slot;
#pragma unroll
        for (int k = 0; k < kKeyLoads; ++k) {
          const int d = FP8 ? 64 * k + 16 * g : 32 * k + 8 * g;
          kf[t][k] = *reinterpret_cast<const u32x4*>(p + (d < a.dim ? d * kElt : 0));
        }
      }
    };
    auto load_values = [&](int tok0) {
      const int d = kLaneDims * c;
      const unsigned char* p0 = vbase + (d < a.dim ? d * kElt : 0);
      int2 at;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        int token = tok0 + 8 * g + j;
        token = token < last ? token : last;
        if (!PAGE8 || j == 0) {
          at = page_of(token, v_ok[PAGE8 ? 0 : j]);
          if (PAGE8) at.y -= token;
        }
        const int slot = PAGE8 ? at.y + token : at.y;
        const unsigned char* p = p0 + (int64_t)at.x * a.v_page + (int64_t)slot * a.v_slot;
        if constexpr (kValueWords >= 4) {
#pragma unroll
          for (int w = 0; w < kValueWords; w += 4) {
            const u32x4 v = *reinterpret_cast<const u32x4*>(p + 4 * w);
            vf[j][w] = v.x, vf[j][w + 1] = v.y, vf[j][w + 2] = v.z, vf[j][w + 3] = v.w;
          }
        } else if constexpr (kValueWords == 2) {
          const u32x2 v = *reinterpret_cast<const u32x2*>(p);
          vf[j][0] = v.x, vf[j][1] = v.y;
        } else {
          vf[j][0] = *reinterpret_cast<const uint32_t*>(p);
        }
      }
    };

    auto start_of = [&](int t) { return sp.base + t * kTile + wave * 32; };
    bool two_parts = true;
    int tok0;
    bool live;
  again:
    tok0 = start_of(tile);
    live = tile < tile_end && tok0 < len;
    if (live) {
      load_keys(tok0);
      load_values(tok0);
    }
    for (int t = tile; live;) {
      // ---- scores ----
      f32x4 s[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        s[h] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int k = 0; k < kMfmas; ++k) {
          u32x4 key;
          if constexpr (FP8) {
            const u32x4 w = kf[h][k >> 1];
            key = (k & 1) ? fp8_eight<DT>(w.z, w.w) : fp8_eight<DT>(w.x, w.y);
          } else {
            key = kf[h][k];
          }
          if (a.dim != DIM) {  // dimensions that the cache does not have
            const int d = FP8 ? 64 * (k >> 1) + 16 * g + 8 * (k & 1) : 32 * k + 8 * g;
            if (d >= a.dim) key = (u32x4){0, 0, 0, 0};
          }
          s[h] = mfma16<DT>(key, q[k], s[h]);
        }
      }
      const int next = start_of(t + 1);
      const bool more = t + 1 < tile_end && next < len;
      bool ok[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int token = tok0 + 8 * g + j;
        ok[j] = v_ok[PAGE8 ? 0 : j] && token >= first && token < len;
      }
      if (more) load_keys(next);

      // ---- running maximum and sum ----
      float x[8];
      float top = -__builtin_inff();
      bool all = true;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        x[j] = ok[j] ? s[j >> 2][j & 3] * a.scale_log2 : -__builtin_inff();
        top = fmaxf(top, x[j]);
        all = all && ok[j];
      }
      top = fmaxf(top, __shfl_xor(top, 16));
      top = fmaxf(top, __shfl_xor(top, 32));
      if (__any(top > m)) {
        const float m_new = fmaxf(m, top);
        const float base = m_new == -__builtin_inff() ? 0.0f : m_new;
        const float fix = __builtin_amdgcn_exp2f(m - base);
        l *= fix;
#pragma unroll
        for (int e = 0; e < kLaneDims; ++e) acc[e] *= fix;
        m = m_new;
      }
      const float zero_at = (m == -__builtin_inff() ? 0.0f : m) - kShift;
      u32x4 p_hi, p_lo;
#pragma unroll
      for (int j = 0; j < 8; j += 2) {
        const float p0 = __builtin_amdgcn_exp2f(x[j] - zero_at);
        const float p1 = __builtin_amdgcn_exp2f(x[j + 1] - zero_at);
        l += p0;
        l += p1;
        const uint32_t hi = pack2<DT>(p0, p1);
        p_hi[j >> 1] = hi;
        p_lo[j >> 1] = pack2<DT>(p0 - lo16<DT>(hi), p1 - hi16<DT>(hi));
      }

      // ---- values ----
      if (!__all(all)) {  // what masked rows hold must not reach the sums, not even times zero
#pragma unroll
        for (int j = 0; j < 8; ++j)
#pragma unroll
          for (int w = 0; w < kValueWords; ++w) vf[j][w] = ok[j] ? vf[j][w] : 0u;
      }
      if constexpr (!FP8) {
#pragma unroll
        for (int e = 0; e < kLaneDims; ++e) {
          u32x4 v;
#pragma unroll
          for (int j = 0; j < 8; j += 2)
            v[j >> 1] = __builtin_amdgcn_perm(vf[j + 1][e >> 1], vf[j][e >> 1],
                                              (e & 1) ? 0x07060302u : 0x05040100u);
          acc[e] = mfma16<DT>(v, p_hi, acc[e]);
          if (two_parts) acc[e] = mfma16<DT>(v, p_lo, acc[e]);
        }
      } else {
#pragma unroll
        for (int w = 0; w < kValueWords; ++w) {
          // 4x4 byte transposes of tokens 0-3 and 4-7
          uint32_t d[2][4];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint32_t w0 = vf[4 * h][w], w1 = vf[4 * h + 1][w], w2 = vf[4 * h + 2][w],
                           w3 = vf[4 * h + 3][w];
            const uint32_t a01 = __builtin_amdgcn_perm(w1, w0, 0x05010400u);
            const uint32_t b01 = __builtin_amdgcn_perm(w1, w0, 0x07030602u);
            const uint32_t a23 = __builtin_amdgcn_perm(w3, w2, 0x05010400u);
            const uint32_t b23 = __builtin_amdgcn_perm(w3, w2, 0x07030602u);
            d[h][0] = __builtin_amdgcn_perm(a23, a01, 0x05040100u);
            d[h][1] = __builtin_amdgcn_perm(a23, a01, 0x07060302u);
            d[h][2] = __builtin_amdgcn_perm(b23, b01, 0x05040100u);
            d[h][3] = __builtin_amdgcn_perm(b23, b01, 0x07060302u);
          }
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const u32x4 v = fp8_eight<DT>(d[0][e], d[1][e]);
            acc[4 * w + e] = mfma16<DT>(v, p_hi, acc[4 * w + e]);
            if (two_parts) acc[4 * w + e] = mfma16<DT>(v, p_lo, acc[4 * w + e]);
          }
        }
      }
      if (more) load_values(next);
      tok0 = next;
      live = more;
      ++t;
    }
    float finite = 0.0f;
#pragma unroll
    for (int e = 0; e < kLaneDims; ++e)
#pragma unroll
      for (int i = 0; i < 4; ++i) finite = fmaf(acc[e][i], 0.0f, finite);
    if (two_parts && __any(finite != 0.0f)) {
      two_parts = false;
      m = -__builtin_inff();
      l = 0.0f;
#pragma unroll
      for (int e = 0; e < kLaneDims; ++e) acc[e] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
      goto again;
    }
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);

    // ---- the four waves' parts ----
    if (c < hcnt) {
#pragma unroll
      for (int e = 0; e < kLaneDims; ++e)
#pragma unroll
        for (int i = 0; i < 4; ++i) lds_acc[wave][c][kLaneDims * (4 * g + i) + e] = acc[e][i];
      if (g == 0) {
        lds_m[wave][c] = m;
        lds_l[wave][c] = l;
      }
    }
    __syncthreads();
    const bool whole = tile == 0 && tile_end == sp.tiles;
    const int64_t row_end = row_u + sp.tiles;
    const int w_first = whole ? 0 : (int)(row_u / per);
    const int w_last = whole ? 0 : (int)((row_end - 1) / per);
    float* slot = a.partial + ((int64_t)blockIdx.x * 2 + ((int)blockIdx.x == w_first ? 1 : 0)) *
                                  slot_floats;
    for (int i = tid; i < heads * (DIM / 4); i += kThreads) {
      const int h = i / (DIM / 4), d = (i - h * (DIM / 4)) * 4;
      float top = lds_m[0][h];
#pragma unroll
      for (int w = 1; w < kWaves; ++w) top = fmaxf(top, lds_m[w][h]);
      const float base = top == -__builtin_inff() ? 0.0f : top;
      f32x4 o = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
      float sum = 0.0f;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        const float f = __builtin_amdgcn_exp2f(lds_m[w][h] - base);
        sum += lds_l[w][h] * f;
        o += *reinterpret_cast<const f32x4*>(&lds_acc[w][h][d]) * f;
      }
      if (whole) {
        const int64_t row = (int64_t)r * a.kv_heads * a.group + head0 + h;
        const float inv = sum == 0.0f ? 0.0f : a.value_scale / sum;
        if (d < a.dim) {
          u32x2 w;
          w.x = pack2<DT>(o.x * inv, o.y * inv);
          w.y = pack2<DT>(o.z * inv, o.w * inv);
          *reinterpret_cast<u32x2*>(a.out + row * a.dim + d) = w;
        }
        if (a.lse && d == 0)
          a.lse[row] = sum == 0.0f ? -__builtin_inff()
                                   : (top - kShift + __builtin_amdgcn_logf(sum)) *
                                         0.6931471805599453f;
      } else {
        float* to = slot + h * (DIM + 2);
#pragma unroll
        for (int v = 0; v < 4; ++v)
          __hip_atomic_store(to + 2 + d + v, o[v], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        if (d == 0) {
          __hip_atomic_store(to, top, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
          __hip_atomic_store(to + 1, sum, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
      }
    }
    if (!whole) {
      // ---- the last workgroup of the row joins its parts, in order ----
      __asm__ volatile("s_waitcnt vmcnt(0)" ::: "memory");
      __syncthreads();
      if (tid == 0)
        lds_last = __hip_atomic_fetch_add(&a.counters[w_first], 1u, __ATOMIC_RELAXED,
                                          __HIP_MEMORY_SCOPE_AGENT) ==
                   (unsigned)(w_last - w_first);
      __syncthreads();
      if (lds_last) {
        const int parts = w_last - w_first + 1;
        auto part = [&](int i) {
          return a.partial + ((int64_t)(w_first + i) * 2 + (i == 0 ? 1 : 0)) * slot_floats;
        };
        for (int i = tid; i < heads * (DIM / 4); i += kThreads) {
          const int h = i / (DIM / 4), d = (i - h * (DIM / 4)) * 4;
          float top = -__builtin_inff();
          for (int n = 0; n < parts; ++n)
            top = fmaxf(top, __hip_atomic_load(part(n) + h * (DIM + 2), __ATOMIC_RELAXED,
                                               __HIP_MEMORY_SCOPE_AGENT));
          const float base = top == -__builtin_inff() ? 0.0f : top;
          f32x4 o = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
          float sum = 0.0f;
          for (int n = 0; n < parts; ++n) {
            const float* from = part(n) + h * (DIM + 2);
            float v[6];
#pragma unroll
            for (int k = 0; k < 6; ++k)
              v[k] = __hip_atomic_load(from + (k < 2 ? k : d + k), __ATOMIC_RELAXED,
                                       __HIP_MEMORY_SCOPE_AGENT);
            const float f = __builtin_amdgcn_exp2f(v[0] - base);
            sum += v[1] * f;
            o += (f32x4){v[2], v[3], v[4], v[5]} * f;
          }
          const int64_t row = (int64_t)r * a.kv_heads * a.group + head0 + h;
          const float inv = sum == 0.0f ? 0.0f : a.value_scale / sum;
          if (d < a.dim) {
            u32x2 w;
            w.x = pack2<DT>(o.x * inv, o.y * inv);
            w.y = pack2<DT>(o.z * inv, o.w * inv);
            *reinterpret_cast<u32x2*>(a.out + row * a.dim + d) = w;
          }
          if (a.lse && d == 0)
            a.lse[row] = sum == 0.0f ? -__builtin_inff()
                                     : (top - kShift + __builtin_amdgcn_logf(sum)) *
                                           0.6931471805599453f;
        }
        if (tid == 0)
          __hip_atomic_store(&a.counters[w_first], 0u, __ATOMIC_RELAXED,
                             __HIP_MEMORY_SCOPE_AGENT);
      }
    }
    __syncthreads();  // the next segment writes the same LDS

    // ---- on to the next row ----
    u += tile_end - tile;
    tile = 0;
    row_u = row_end;
    if (++hr == hr_count) {
      hr = 0;
      ++r;
      if (u < u_end) {
        if (r - piece == 64) {
          piece = r;
          len_lane = piece + lane < a.requests ? a.lengths[piece + lane] : 0;
        }
        sp = span_of(readlane(len_lane, r - piece), most, a.window);
      }
    }
  }
}

template <int DT, bool FP8, int DIM>
hipError_t launch(const PagedAttentionArgs& a, int workgroups, hipStream_t stream) {
  const int slot = (int)paged_attention_slot_floats(a.group, a.dim);
  if (a.page_size % 8 == 0)
    paged_attention_kernel<DT, FP8, DIM, true><<<workgroups, kThreads, 0, stream>>>(a, slot);
  else
    paged_attention_kernel<DT, FP8, DIM, false><<<workgroups, kThreads, 0, stream>>>(a, slot);
  return hipGetLastError();
}

int padded_dim(int dim) { return dim <= 64 ? 64 : dim <= 128 ? 128 : 256; }

template <int DT, bool FP8>
hipError_t launch_dim(const PagedAttentionArgs& a, int workgroups, hipStream_t stream) {
  switch (padded_dim(a.dim)) {
    case 64: return launch<DT, FP8, 64>(a, workgroups, stream);
    case 128: return launch<DT, FP8, 128>(a, workgroups, stream);
    default: return launch<DT, FP8, 256>(a, workgroups, stream);
  }
}

}  // namespace

int paged_attention_workgroups(int cus, int64_t units) {
  const int64_t most = 2 * (int64_t)cus;
  return (int)(units < most ? (units > 0 ? units : 1) : most);
}

size_t paged_attention_slot_floats(int group, int dim) {
  return (size_t)(group < 16 ? group : 16) * (padded_dim(dim) + 2);
}

hipError_t launch_paged_attention(const PagedAttentionArgs& a, int dtype, bool fp8, int workgroups,
                                  hipStream_t stream) {
  if (dtype == kBF16)
    return fp8 ? launch_dim<kBF16, true>(a, workgroups, stream)
               : launch_dim<kBF16, false>(a, workgroups, stream);
  return fp8 ? launch_dim<kF16, true>(a, workgroups, stream)
             : launch_dim<kF16, false>(a, workgroups, stream);
}

}  // namespace mt
