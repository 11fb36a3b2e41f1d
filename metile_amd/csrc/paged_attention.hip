// Decode attention over a paged key-value cache: one new token of each request.
//
//   s_t = scale * q . k_t      o = sum_t exp(s_t - m) v_t / sum_t exp(s_t - m)      m = max_t s_t
//
// in one pass over the pages with a running maximum and sum (in powers of two: the scale holds
// log2 e). A wave takes 32 tokens of one row (request, key-value head, up to 16 query heads that
// share it) at a time:
//  * keys: v_mfma_f32_16x16x32 with the keys as rows and the query heads as columns, so a lane
//    holds scores of one head, eight consecutive tokens of it in two tiles (row i of tile t is
//    token 8 (i / 4) + 4 t + i % 4);
//  * values: a lane loads DIM / 16 dimensions of eight consecutive tokens; eight byte permutes
//    a dimension pair turn them into operands with the dimensions as rows, and the lane's own
//    eight probabilities are the other operand as they stand: no exchange between lanes.
//    The result has the head in the lane again, so rescaling is local to the lane;
//  * pages: a lane a token looks up its entry, one unit ahead, and reckons the row's offset, which
//    the lanes that load the row ask for (pages of one token 10.4 us; with the look-ups and their
//    divisions in every loading lane 13.2; pages of 16 the same).
// Scores, maxima, sums and results are fp32. Probabilities go to the matrix cores as two 16-bit
// parts (their rounding and the rest of it): a probability p is off by 2^-18 p at most with bf16, by
// 2^-24 p or 2^-39 of its row's largest with f16, where the result's own rounding is 2^-9 and 2^-12
// of it. A third part would add half as many products of values again. (The second part is zero or
// negative as often as not, and an infinite value times it is no number: a segment with sums that
// are not finite is taken again, with values that are not finite times the first parts, which are
// positive, alone.)
//
// Split: all rows, laid end to end in units of 32 tokens with a few more for the fixed cost of a
// row, are dealt out in equal contiguous runs to a fixed number of waves (each finds its place from
// a scan over the lengths), so ragged batches balance by themselves. A row that lies within one
// wave's run is written by that wave, with no exchange at all. A wave's parts of other rows (the
// first and the last of its run) meet in LDS at the end, and the workgroup's parts of rows that go
// on in other workgroups are stored with their maximum and sum and joined, in order, by the last
// of those workgroups to arrive (8 parts at a time, up to 16 at once).
//
// Bound by the bytes of keys and values where there are enough of them: 2 requests of 131072 tokens
// with 8 key-value heads of 128 bf16 values (1.07 GB) take 183 us, 5.9 TB/s (of 1 GiB, reads alone
// reach 6.3 and a copy 5.2); 64 requests of 1 to 8192 tokens (224 MB) 47.5 us, 4.7 TB/s. The
// shortest calls take 4.7 us: the launch, then lengths, table entry and first rows, a memory round
// trip each after the other; a row that several workgroups share costs about 4 us more for its join.
#include "common.h"
#include "paged.h"

namespace mt {
namespace {

constexpr int kWaves = 4;
constexpr int kThreads = 64 * kWaves;
constexpr int kUnit = kAttentionUnit;
constexpr int kRowCost = kAttentionRowCost;

// Inclusive sum over the lanes: within rows of 16, then across them.
template <int CTRL, int ROWS>
__device__ __forceinline__ int dpp_add(int v) {
  return v + __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xF, false);
}
__device__ __forceinline__ int wave_scan(int v) {
  v = dpp_add<0x111, 0xF>(v);  // row_shr:1
  v = dpp_add<0x112, 0xF>(v);
  v = dpp_add<0x114, 0xF>(v);
  v = dpp_add<0x118, 0xF>(v);
  v = dpp_add<kDppRowBcast15, 0xA>(v);
  return dpp_add<kDppRowBcast31, 0xC>(v);
}

__device__ __forceinline__ int readlane(int v, int l) { return __builtin_amdgcn_readlane(v, l); }
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

// A request's tokens as they are read: its length, the first token of its window rounded down to a
// unit, and its units (one for an empty request, which writes its zeros).
struct Span {
  int len, first, base, units;
};
__device__ __forceinline__ Span span_of(int length, int most, int window) {
  Span s;
  s.len = length < 0 ? 0 : (length > most ? most : length);
  s.first = window > 0 && s.len > window ? s.len - window : 0;
  s.base = s.first & ~(kUnit - 1);
  const int n = (int)(((unsigned)(s.len - s.base) + kUnit - 1) / kUnit);
  s.units = n > 0 ? n : 1;
  return s;
}

template <int DT>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  if constexpr (DT == kBF16)
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2){a, b}, bf16x2));
  else
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2){a, b}, f16x2));
}

// 16-bit keys and values of whole lines are read with the hint that this happens once (2 x 131072
// tokens of 8 heads of 128: 190.5 us without it, 183 with), all others are kept in the caches: where
// a head's row of a token is no whole lines, others read the rest of one (heads of 80 8-bit values,
// 2 x 68389 tokens: 172 us with the hint, 122 without), and so do further tiles of query heads (48
// heads on one, 366 requests of up to 5496 tokens: 119, 95). (Heads of 256, 5 x 78518 tokens: 100,
// 91; 8 bits, 75 x 2086 tokens of 8 heads of 128: 77, 75.)
template <bool ONCE, typename T>
__device__ __forceinline__ T stream_load(const T* p) {
  if constexpr (ONCE) return __builtin_nontemporal_load(p);
  else return *p;
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

// Two 16-bit floats, 0 in place of infinities and NaN.
template <int DT>
__device__ __forceinline__ uint32_t finite_pair(uint32_t w) {
  constexpr uint32_t kExponent = DT == kBF16 ? 0x7f80u : 0x7c00u;
  if ((w & kExponent) == kExponent) w &= 0xffff0000u;
  if ((w >> 16 & kExponent) == kExponent) w &= 0x0000ffffu;
  return w;
}

// A probability for its first part in f16, beside values that are not finite: 0 in place of one below
// f16's range would make no number of an infinite value. The second part makes up for the difference.
__device__ __forceinline__ float not_zero(float p) { return p > 0.0f ? fmaxf(p, 0x1p-14f) : p; }

// Rows of up to so many units are not split over waves: a unit costs a wave that has its SIMD to
// itself about 0.8 us, the exchange of a split row 1.5 to 5. (60 drawn calls, against no such rule:
// 4 units 1% faster in the mean, 8 the same with both gains and losses up to 15%, 16 6% slower.)
constexpr int kWholeUnits = 4;

// Where a workgroup's partial sums of a row are kept: [heads][kPartHead + DIM] floats a slot, the
// maximum and the sum in front of a head's values.
constexpr int kPartHead = 4;
// Parts that one workgroup joins at a time; rows of more are joined in levels. A level costs two
// round trips to memory and eight parts a third one, so up to 16 parts are joined at once unless
// they are large: one workgroup reads about 50 KB a microsecond (2 requests of 3960 to 7057 tokens,
// 28 heads of 128 values on 4: 32 parts at a time 22.1 us, 8 17.0; 64 requests of 1 to 8192 tokens
// 8 always 48.9, up to 16 at once 47.9).
constexpr int kJoin = 8, kJoinAll = 16, kLargePart = 8192;
// The counters of four levels (8^4 parts) of twice so many fit the workspace's region of them.
constexpr int kMostWorkgroups = 2048;
static_assert(kMostWorkgroups * 2 * 4 * 4 <= 64 * 1024 && kMostWorkgroups <= 8 * 8 * 8 * 8,
              "counters of every level");

// Waves a SIMD (and so workgroups a CU) that the registers are allotted for.
constexpr int attention_waves(int padded_dim) {
  return padded_dim == 256 ? 1 : padded_dim == 64 ? 3 : 2;
}

// DIM: the head's values, or with PADDED that many or more (the rest count as zero). Heads in several
// tiles are such calls too, for the sake of its loads without the hint.
template <int DT, bool FP8, int DIM, bool PADDED>
__global__ __launch_bounds__(kThreads, attention_waves(DIM)) void paged_attention_kernel(
    PagedAttentionArgs a, int slot_bytes) {
  constexpr int kElt = FP8 ? 1 : 2;
  constexpr int kMfmas = DIM / 32;               // K depth of a score
  constexpr int kLaneDims = DIM / 16;            // value dimensions of a lane
  constexpr int kKeyLoads = kMfmas * kElt / 2;   // 16-byte loads of a key row a lane makes
  constexpr int kValueWords = kLaneDims * kElt / 4;
  constexpr int kRow = DIM + 4;                  // floats: heads start four banks apart
  constexpr int kVecs = DIM / 4;
  constexpr bool kOnce = !PADDED && !FP8 && DIM <= 128;
  const int dim = PADDED ? a.dim : DIM;
  // f16 probabilities are scaled up so that small ones, and the second parts, stay above its
  // smallest numbers; the sum carries the same factor.
  constexpr float kShift = DT == kF16 ? 14.0f : 0.0f;

  // Parts of rows that a wave shares with others: of the row it begins in, of the one it ends in.
  constexpr int kSlots = 2 * kWaves;
  __shared__ __attribute__((aligned(16))) float lds_acc[kSlots][16][kRow];
  __shared__ float lds_m[kSlots][16];
  __shared__ float lds_l[kSlots][16];
  __shared__ int lds_row[kSlots], lds_units[kSlots];
  __shared__ unsigned lds_data[kSlots];
  __shared__ int lds_last;

  const int tid = threadIdx.x;
  const int lane = tid & 63, wave = uniform(tid >> 6);
  const int c = lane & 15, g = lane >> 4;
  const int most = a.width * a.page_size;  // the host checks that it fits 31 bits
  const int hr_count = a.kv_heads * a.head_tiles;
  const __amdgpu_buffer_rsrc_t parts_rsrc =
      make_rsrc(a.partial, (uint32_t)gridDim.x * 2u * (uint32_t)slot_bytes);
  // Workgroups go to the XCDs in turn: each XCD takes neighbouring runs, whose rows share lines of
  // the cache where a head's row of a token is less than one, and all of it where they are query
  // heads of one key-value head.
  const int run = gridDim.x % 8 == 0 ? (blockIdx.x % 8) * (gridDim.x / 8) + blockIdx.x / 8
                                     : blockIdx.x;

  // ---- this wave's run of units ----
  const int chunk = (a.requests + 63) >> 6;
  int mine = 0, len_lane = 0;
  for (int i = 0; i < chunk; ++i) {
    const int r = lane * chunk + i;
    len_lane = r < a.requests ? a.lengths[r] : 0;
    if (r < a.requests) mine += span_of(len_lane, most, a.window).units + kRowCost;
  }
  const int inc = wave_scan(mine);
  // (far enough below 2^31, as the host checks; said to be the same in every lane)
  const unsigned units = (unsigned)readlane(inc, 63) * (unsigned)hr_count;
  const unsigned waves = gridDim.x * kWaves;
  const unsigned per_wave = max((unsigned)uniform((int)div_by(units + waves - 1, a.by_waves)),
                                (unsigned)(kAttentionLeast / kWaves));
  const unsigned per = per_wave * kWaves, wg_u = (unsigned)run * per;
  if (wg_u >= units) return;
  const unsigned wg_end = min(wg_u + per, units);
  const unsigned u = min(wg_u + (unsigned)wave * per_wave, wg_end);
  const unsigned u_end = min(u + per_wave, wg_end);
  int piece = 0, r = 0, hr = 0;
  unsigned row_u = 0;  // where the row begins; its units come behind its cost
  Span sp{};
  if (u < u_end) {
    const int target = uniform((int)div_by(u, a.by_rows));
    const int owner = __ffsll((unsigned long long)__ballot(inc > target)) - 1;
    int prefix = readlane(inc, owner) - readlane(mine, owner);  // units of the requests before r
    r = owner * chunk;
    if (chunk > 1) {  // the request is one of the lane's: 64 of them at a time, in len_lane
      for (piece = r;; piece += 64) {
        len_lane = piece + lane < a.requests ? a.lengths[piece + lane] : 0;
        const int t = piece + lane < a.requests
                          ? span_of(len_lane, most, a.window).units + kRowCost : 0;
        const int s = wave_scan(t) + prefix;
        const uint64_t hit = __ballot(s > target);
        if (hit) {
          const int at = __ffsll((unsigned long long)hit) - 1;
          r = piece + at;
          prefix = readlane(s, at) - readlane(t, at);
          break;
        }
        prefix = readlane(s, 63);
        if (piece + 64 >= a.requests) break;  // only if the lengths changed under the scan
      }
    }
    sp = span_of(readlane(len_lane, (r - piece) & 63), most, a.window);
    const unsigned off = u - (unsigned)prefix * (unsigned)hr_count;
    const unsigned row = (unsigned)(sp.units + kRowCost);
    hr = min(uniform((int)(off / row)), hr_count - 1);
    row_u = u - (off - (unsigned)hr * row);
  }
  if (lane < 2) lds_row[2 * wave + lane] = -1;
  const int page_size = a.page_size;

  // A row's first query head, and how many of its 16 columns are heads.
  auto first_head = [&](int hr) {
    const int kv = a.head_tiles == 1 ? hr : uniform(hr / a.head_tiles);
    return kv * a.group + (hr - kv * a.head_tiles) * 16;
  };
  auto head_count = [&](int hr) {
    const int kv = a.head_tiles == 1 ? hr : uniform(hr / a.head_tiles);
    return min(a.group - (hr - kv * a.head_tiles) * 16, 16);
  };
  auto lse_of = [&](float top, float sum) {
    return sum == 0.0f ? -__builtin_inff()
                       : (top - kShift + __builtin_amdgcn_logf(sum)) * 0.6931471805599453f;
  };

  auto next_row = [&]() {
    row_u += (unsigned)(sp.units + kRowCost);
    if (++hr == hr_count) {
      hr = 0;
      ++r;
      if (row_u < u_end && r < a.requests) {
        if (r - piece == 64) {
          piece = r;
          len_lane = piece + lane < a.requests ? a.lengths[piece + lane] : 0;
        }
        sp = span_of(readlane(len_lane, r - piece), most, a.window);
      }
    }
  };
  // Short rows are not split: they are whole the wave's whose run their first unit is in.
  if (u < u_end && sp.units <= kWholeUnits && row_u + kRowCost < u) next_row();

  while (u < u_end && r < a.requests) {
    const unsigned data_u = row_u + kRowCost;
    if (data_u >= u_end) break;
    const bool split = sp.units > kWholeUnits;
    const int unit = split && u > data_u ? (int)(u - data_u) : 0;  // this wave's units of the row
    const int unit_end = split ? (int)(min(u_end, data_u + (unsigned)sp.units) - data_u) : sp.units;
    const int kv = a.head_tiles == 1 ? hr : uniform(hr / a.head_tiles);
    const int head0 = first_head(hr), heads = head_count(hr);
    const int32_t* table = a.tables + (int64_t)r * a.table_stride;
    const unsigned char* kbase = a.key + (int64_t)kv * a.k_head;
    const unsigned char* vbase = a.value + (int64_t)kv * a.v_head;
    const int len = sp.len, first = sp.first, last = len - 1;

    float m = -__builtin_inff(), l = 0.0f;
    f32x4 acc[kLaneDims];
#pragma unroll
    for (int e = 0; e < kLaneDims; ++e) acc[e] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};

    u32x4 kf[2][kKeyLoads];
    uint32_t vf[8][kValueWords];

    // Where a unit's tokens are: the page of token lane % 32, and the place in it. Tokens past the end
    // stand for the last one; tokens of a page that is none of the cache's for page 0. Both are
    // masked.
    struct Place {
      int page, slot;
    };
    auto look_up = [&](int tok0, Place& p) {
      const int token = min(tok0 + (lane & 31), last);
      const int col = (int)div_by((uint32_t)token, a.by_page);
      p.page = table[col];
      p.slot = token - col * page_size;
    };
    // Its row is reckoned once, by that lane; those that load it ask for the offset.
    auto offset_of = [&](const Place& p, uint32_t page_stride, uint32_t slot_stride) {
      const uint32_t page = (uint32_t)p.page < (uint32_t)a.pages ? (uint32_t)p.page : 0u;
      return (uint64_t)page * page_stride + (uint64_t)(uint32_t)p.slot * slot_stride;
    };
    auto of_token = [&](uint64_t offset, int i) {
      const uint32_t lo = (uint32_t)__builtin_amdgcn_ds_bpermute(4 * i, (int)(uint32_t)offset);
      const uint32_t hi = (uint32_t)__builtin_amdgcn_ds_bpermute(4 * i, (int)(offset >> 32));
      return (uint64_t)hi << 32 | lo;
    };
    auto load_keys = [&](const Place& p) {
      const uint64_t offset = offset_of(p, a.k_page, a.k_slot);
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const unsigned char* row = kbase + of_token(offset, 8 * (c >> 2) + 4 * t + (c & 3));
#pragma unroll
        for (int k = 0; k < kKeyLoads; ++k) {
          const int d = FP8 ? 64 * k + 16 * g : 32 * k + 8 * g;
          kf[t][k] = stream_load<kOnce>(
              reinterpret_cast<const u32x4*>(row + (d < dim ? d * kElt : 0)));
        }
      }
    };
    auto load_values = [&](const Place& p) {
      const uint64_t offset = offset_of(p, a.v_page, a.v_slot);
      const int d = kLaneDims * c;
      const unsigned char* lane_base = vbase + (d < dim ? d * kElt : 0);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const unsigned char* row = lane_base + of_token(offset, 8 * g + j);
        if constexpr (kValueWords >= 4) {
#pragma unroll
          for (int w = 0; w < kValueWords; w += 4) {
            const u32x4 v =
                stream_load<kOnce>(reinterpret_cast<const u32x4*>(row + 4 * w));
            vf[j][w] = v.x, vf[j][w + 1] = v.y, vf[j][w + 2] = v.z, vf[j][w + 3] = v.w;
          }
        } else if constexpr (kValueWords == 2) {
          const u32x2 v = stream_load<kOnce>(reinterpret_cast<const u32x2*>(row));
          vf[j][0] = v.x, vf[j][1] = v.y;
        } else {
          vf[j][0] = stream_load<kOnce>(reinterpret_cast<const uint32_t*>(row));
        }
      }
    };

    auto start_of = [&](int t) { return sp.base + t * kUnit; };
    // Table entries are looked up one unit further ahead than rows, so that no row waits for one.
    Place now, ahead;
    u32x4 q[kMfmas];
    bool all_finite = true;
    int tok0;
    bool live;
  again:
    // (given values here so that none of an earlier row's is kept through the join of its parts)
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int k = 0; k < kKeyLoads; ++k) kf[t][k] = (u32x4){0, 0, 0, 0};
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
      for (int w = 0; w < kValueWords; ++w) vf[j][w] = 0;
#pragma unroll
    for (int k = 0; k < kMfmas; ++k) q[k] = (u32x4){0, 0, 0, 0};
    now = ahead = Place{};
    int t = unit;
    tok0 = start_of(t);
    live = t < unit_end && tok0 < len;
    if (live) {
      look_up(tok0, now);
      // the query heads, as columns: dimensions in the order of the key loads
      const bool has = c < heads;
      const uint16_t* row = a.query + (int64_t)r * a.q_row_stride +
                            (int64_t)(head0 + (has ? c : 0)) * a.q_head_stride;
#pragma unroll
      for (int k = 0; k < kMfmas; ++k) {
        const int d = FP8 ? 64 * (k >> 1) + 16 * g + 8 * (k & 1) : 32 * k + 8 * g;
        q[k] = *reinterpret_cast<const u32x4*>(row + (d < dim ? d : 0));
        if (!has || d >= dim) q[k] = (u32x4){0, 0, 0, 0};
      }
      load_keys(now);
      load_values(now);
      if (t + 1 < unit_end) look_up(start_of(t + 1), ahead);
    }
    while (live) {
      const int next = start_of(t + 1);
      const bool more = t + 1 < unit_end;
      // which of the unit's tokens are attended to: past the ends of the window and the request, and
      // on pages that are none, they are not
      const int token = tok0 + (lane & 31);
      const uint32_t here = (uint32_t)__ballot((uint32_t)now.page < (uint32_t)a.pages &&
                                               token >= first && token < len);
      const bool all = here == 0xffffffffu;
      const uint32_t ok = here >> (8 * g);

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
          if (PADDED) {  // dimensions that the cache does not have
            const int d = FP8 ? 64 * (k >> 1) + 16 * g + 8 * (k & 1) : 32 * k + 8 * g;
            if (d >= dim) key = (u32x4){0, 0, 0, 0};
          }
          s[h] = mfma16<DT>(key, q[k], s[h]);
        }
      }
      if (more) {
        load_keys(ahead);
        now = ahead;
        if (t + 2 < unit_end) look_up(start_of(t + 2), ahead);
      }

      // ---- running maximum and sum ----
      float x[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = s[j >> 2][j & 3] * a.scale_log2;
      if (!all) {
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = (ok >> j) & 1 ? x[j] : -__builtin_inff();
      }
      float top = fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])),
                        fmaxf(fmaxf(x[4], x[5]), fmaxf(x[6], x[7])));
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
      float sum[2] = {0.0f, 0.0f};
#pragma unroll
      for (int j = 0; j < 8; j += 2) {
        const float p0 = __builtin_amdgcn_exp2f(x[j] - zero_at);
        const float p1 = __builtin_amdgcn_exp2f(x[j + 1] - zero_at);
        sum[0] += p0;
        sum[1] += p1;
        const uint32_t hi = pack2<DT>(p0, p1);
        p_hi[j >> 1] = hi;
        p_lo[j >> 1] = pack2<DT>(p0 - lo16<DT>(hi), p1 - hi16<DT>(hi));
      }
      l += sum[0] + sum[1];
      if (!FP8 && DT == kF16 && !all_finite) {
#pragma unroll
        for (int j = 0; j < 8; j += 2) {
          const float p0 = __builtin_amdgcn_exp2f(x[j] - zero_at);
          const float p1 = __builtin_amdgcn_exp2f(x[j + 1] - zero_at);
          const uint32_t hi = pack2<DT>(not_zero(p0), not_zero(p1));
          p_hi[j >> 1] = hi;
          p_lo[j >> 1] = pack2<DT>(p0 - lo16<DT>(hi), p1 - hi16<DT>(hi));
        }
      }

      // ---- values ----
      if (!all) {  // what masked rows hold must not reach the sums, not even times zero
#pragma unroll
        for (int j = 0; j < 8; ++j)
#pragma unroll
          for (int w = 0; w < kValueWords; ++w) vf[j][w] = (ok >> j) & 1 ? vf[j][w] : 0u;
      }
      u32x4 v[kLaneDims];  // dimension e of the lane's eight tokens
      if constexpr (!FP8) {
#pragma unroll
        for (int e = 0; e < kLaneDims; ++e)
#pragma unroll
          for (int j = 0; j < 8; j += 2)
            v[e][j >> 1] = __builtin_amdgcn_perm(vf[j + 1][e >> 1], vf[j][e >> 1],
                                                 (e & 1) ? 0x07060302u : 0x05040100u);
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
          for (int e = 0; e < 4; ++e) v[4 * w + e] = fp8_eight<DT>(d[0][e], d[1][e]);
        }
      }
#pragma unroll
      for (int e = 0; e < kLaneDims; ++e) acc[e] = mfma16<DT>(v[e], p_hi, acc[e]);
      if (!all_finite) {
#pragma unroll
        for (int e = 0; e < kLaneDims; ++e)
#pragma unroll
          for (int j = 0; j < 4; ++j) v[e][j] = finite_pair<DT>(v[e][j]);
      }
#pragma unroll
      for (int e = 0; e < kLaneDims; ++e) acc[e] = mfma16<DT>(v[e], p_lo, acc[e]);
      if (more) load_values(now);
      tok0 = next;
      live = more;
      ++t;
    }
    float finite = 0.0f;
#pragma unroll
    for (int e = 0; e < kLaneDims; ++e)
#pragma unroll
      for (int i = 0; i < 4; ++i) finite = fmaf(acc[e][i], 0.0f, finite);
    if (all_finite && __any(finite != 0.0f)) {
      all_finite = false;
      m = -__builtin_inff();
      l = 0.0f;
#pragma unroll
      for (int e = 0; e < kLaneDims; ++e) acc[e] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
      goto again;
    }
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);

    if (unit == 0 && unit_end == sp.units) {
      // the whole row: a lane has 4 kLaneDims consecutive values of its head
      const int64_t row = (int64_t)r * a.kv_heads * a.group + head0 + c;
      const float inv = l == 0.0f ? 0.0f : a.value_scale / l;
      if (c < heads) {
        uint32_t w[2 * kLaneDims];
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int e = 0; e < kLaneDims; e += 2)
            w[(i * kLaneDims + e) / 2] = pack2<DT>(acc[e][i] * inv, acc[e + 1][i] * inv);
#pragma unroll
        for (int k = 0; k < 2 * kLaneDims; k += 4) {
          const int d = 4 * kLaneDims * g + 2 * k;
          if (d < dim)
            *reinterpret_cast<u32x4*>(a.out + row * dim + d) =
                (u32x4){w[k], w[k + 1], w[k + 2], w[k + 3]};
        }
        if (a.lse && g == 0) a.lse[row] = lse_of(m, l);
      }
    } else {
      const int s = 2 * wave + (unit == 0 ? 1 : 0);
      if (c < heads) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int e = 0; e < kLaneDims; e += 4)
            *reinterpret_cast<f32x4*>(&lds_acc[s][c][kLaneDims * (4 * g + i) + e]) =
                (f32x4){acc[e][i], acc[e + 1][i], acc[e + 2][i], acc[e + 3][i]};
        if (g == 0) {
          lds_m[s][c] = m;
          lds_l[s][c] = l;
        }
      }
      if (lane == 0) {
        lds_row[s] = r * hr_count + hr;
        lds_units[s] = sp.units;
        lds_data[s] = data_u;
      }
    }

    next_row();
  }
  __syncthreads();

  // ---- rows that waves of this workgroup share ----
  // A head's four values of a row: the result, or a part of it.
  auto write_row = [&](int row, int h, int d, f32x4 o, float top, float sum) {
    const int rr = row / hr_count;
    const int64_t at = (int64_t)rr * a.kv_heads * a.group + first_head(row - rr * hr_count) + h;
    const float inv = sum == 0.0f ? 0.0f : a.value_scale / sum;
    if (d < dim)
      *reinterpret_cast<u32x2*>(a.out + at * dim + d) =
          (u32x2){pack2<DT>(o.x * inv, o.y * inv), pack2<DT>(o.z * inv, o.w * inv)};
    if (a.lse && d == 0) a.lse[at] = lse_of(top, sum);
  };
  // Byte offset of part n of a row that begins in workgroup w_first.
  auto slot_of = [&](int w_first, int n) {
    return ((uint32_t)(w_first + n) * 2u + (n == 0 ? 1u : 0u)) * (uint32_t)slot_bytes;
  };
  auto write_part = [&](uint32_t slot, int h, int d, f32x4 o, float top, float sum) {
    const uint32_t at = slot + (uint32_t)(h * (kPartHead + DIM)) * 4u;
    __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, o), parts_rsrc,
                                           at + (uint32_t)(kPartHead + d) * 4u, 0, kDeviceScope);
    if (d == 0)
      __builtin_amdgcn_raw_buffer_store_b64(
          (u32x2){__float_as_uint(top), __float_as_uint(sum)}, parts_rsrc, at, 0, kDeviceScope);
  };
  // The rows that go on in other workgroups: the one this one begins in (0), the one it ends in.
  int open_row[2] = {-1, -1}, open_first[2] = {0, 0}, open_parts[2] = {0, 0};
  const int row_lane = lane < kSlots ? lds_row[lane] : -1;
  const int units_lane = lane < kSlots ? lds_units[lane] : 0;
  const int data_lane = lane < kSlots ? (int)lds_data[lane] : 0;
  uint64_t slots = __ballot(row_lane >= 0);
#pragma unroll 1
  while (slots) {
    const int s = __ffsll((unsigned long long)slots) - 1;
    const int row = readlane(row_lane, s);
    const uint64_t same = __ballot(row_lane == row);  // the row's slots: one wave after another
    slots &= ~same;
    const unsigned data_u = (unsigned)readlane(data_lane, s);
    const unsigned row_end = data_u + (unsigned)readlane(units_lane, s);
    const bool whole = data_u >= wg_u && row_end <= wg_end;
    const int w_first = whole ? run : uniform((int)(data_u / per));
    uint32_t slot = 0;
    if (!whole) {
      const int k = w_first == run ? 1 : 0;
      open_row[k] = row;
      open_first[k] = w_first;
      open_parts[k] = uniform((int)((row_end - 1) / per)) - w_first + 1;
      slot = slot_of(w_first, run - w_first);
    }
    const int heads = head_count(uniform(row % hr_count));
#pragma unroll 1
    for (int i = tid; i < heads * kVecs; i += kThreads) {
      const int h = i / kVecs, d = (i - h * kVecs) * 4;
      float top = -__builtin_inff(), sum = 0.0f;
      f32x4 o = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
      for (uint64_t rest = same; rest; rest &= rest - 1) {
        const int k = __ffsll((unsigned long long)rest) - 1;
        const float m = lds_m[k][h], l = lds_l[k][h];
        const f32x4 v = *reinterpret_cast<const f32x4*>(&lds_acc[k][h][d]);
        const float t = fmaxf(top, m), base = t == -__builtin_inff() ? 0.0f : t;
        const float old = __builtin_amdgcn_exp2f(top - base);
        const float now = __builtin_amdgcn_exp2f(m - base);
        sum = sum * old + l * now;
        o = o * old + v * now;
        top = t;
      }
      if (whole) write_row(row, h, d, o, top, sum);
      else write_part(slot, h, d, o, top, sum);
    }
  }
  if (open_row[0] < 0 && open_row[1] < 0) return;

  // ---- rows that workgroups share: the last to arrive joins their parts, in order ----
  // Every store of the workgroup has arrived, then one count: true in the last of `of` to come.
  auto arrived_last = [&](uint32_t* counter, int of) {
    __asm__ volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (tid == 0) {
      const bool is_last = __hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED,
                                                  __HIP_MEMORY_SCOPE_AGENT) == (unsigned)(of - 1);
      if (is_last) __hip_atomic_store(counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      lds_last = is_last;
    }
    __syncthreads();
    return lds_last != 0;
  };
  // Parts are joined `fan` at a time (level 0), then the results of `fan` such joins (level 1), and
  // so on. The counter of a join whose first part is n0 belongs to that part's workgroup, two to a
  // level: a workgroup can hold the first part of one row and a later part of another, no more.
  const int items = head_count(0) * kVecs;  // the most of a row
#pragma unroll 1
  for (int k = 0; k < 2; ++k) {
    const int row = k ? open_row[1] : open_row[0];
    if (row < 0) continue;
    const int w_first = k ? open_first[1] : open_first[0];
    const int parts = k ? open_parts[1] : open_parts[0];
    const int heads = head_count(uniform(row % hr_count));
    const int fan = parts <= kJoinAll && slot_bytes <= kLargePart ? kJoinAll : kJoin;
    int part = run - w_first, step = 1;
    uint32_t* counters = a.counters;
#pragma unroll 1
    for (;;) {
      const int span = step * fan;  // parts under one join of this level
      const int n0 = part / span * span, n_end = min(parts, n0 + span);
      const int arrivals = (n_end - n0 + step - 1) / step;
      if (!arrived_last(counters + (n0 ? gridDim.x : 0) + w_first + n0, arrivals)) break;
      // parts n0, n0 + step, ... below n_end, in that order, eight requested at a time
      const bool final = n_end - n0 == parts;
      constexpr int kItems = DIM == 256 ? 4 : 1;  // of a thread at a time
#pragma unroll 1
      for (int first = tid; first < items; first += kItems * kThreads) {
        float top[kItems], sum[kItems];
        f32x4 o[kItems];
#pragma unroll
        for (int i = 0; i < kItems; ++i) {
          top[i] = -__builtin_inff();
          sum[i] = 0.0f;
          o[i] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
        }
#pragma unroll 1
        for (int n = n0; n < n_end; n += 8 * step) {
          u32x4 v[kItems][8];
          u32x2 ml[kItems][8];
#pragma unroll
          for (int i = 0; i < kItems; ++i) {
            const int item = first + i * kThreads, h = item / kVecs, d = (item - h * kVecs) * 4;
#pragma unroll
            for (int q = 0; q < 8; ++q) {
              // (what is not there is not read)
              const uint32_t at = oob_unless(item < items && n + q * step < n_end,
                                             slot_of(w_first, n + q * step) +
                                                 (uint32_t)(h * (kPartHead + DIM)) * 4u);
              ml[i][q] = __builtin_amdgcn_raw_buffer_load_b64(parts_rsrc, at, 0, kDeviceScope);
              v[i][q] = load16_device(parts_rsrc, at + (uint32_t)(kPartHead + d) * 4u);
            }
          }
#pragma unroll
          for (int i = 0; i < kItems; ++i) {
            float t = top[i];
#pragma unroll
            for (int q = 0; q < 8; ++q) {
              const uint32_t x = ml[i][q].x;
              if (n + q * step < n_end) t = fmaxf(t, __uint_as_float(x));
            }
            const float base = t == -__builtin_inff() ? 0.0f : t;
            const float fix = __builtin_amdgcn_exp2f(top[i] - base);
            o[i] *= fix;
            sum[i] *= fix;
            top[i] = t;
#pragma unroll
            for (int q = 0; q < 8; ++q) {
              const uint32_t x = ml[i][q].x, y = ml[i][q].y;
              if (n + q * step < n_end) {
                const float f = __builtin_amdgcn_exp2f(__uint_as_float(x) - base);
                sum[i] += __uint_as_float(y) * f;
                o[i] += __builtin_bit_cast(f32x4, v[i][q]) * f;
              }
            }
          }
        }
#pragma unroll
        for (int i = 0; i < kItems; ++i) {
          const int item = first + i * kThreads, h = item / kVecs, d = (item - h * kVecs) * 4;
          if (h >= heads) continue;
          if (final) write_row(row, h, d, o[i], top[i], sum[i]);
          else write_part(slot_of(w_first, n0), h, d, o[i], top[i], sum[i]);
        }
      }
      if (final) break;
      part = n0;
      step = span;
      counters += 2 * gridDim.x;
    }
    __syncthreads();  // lds_last
  }
}

template <int DT, bool FP8, int DIM>
hipError_t launch(const PagedAttentionArgs& a, int workgroups, hipStream_t stream) {
  const int slot = (int)paged_attention_slot_floats(a.group, a.dim) * 4;
  if (a.dim == DIM && (FP8 || DIM > 128 || a.head_tiles == 1))
    paged_attention_kernel<DT, FP8, DIM, false><<<workgroups, kThreads, 0, stream>>>(a, slot);
  else
    paged_attention_kernel<DT, FP8, DIM, true><<<workgroups, kThreads, 0, stream>>>(a, slot);
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

int paged_attention_workgroups(int cus, int dim, int64_t units) {
  const int64_t most = attention_waves(padded_dim(dim)) * (int64_t)cus;
  const int64_t runs = (units + kAttentionLeast - 1) / kAttentionLeast;
  const int64_t n = runs < most ? (runs > 0 ? runs : 1) : most;
  return (int)(n < kMostWorkgroups ? n : kMostWorkgroups);
}

size_t paged_attention_slot_floats(int group, int dim) {
  return (size_t)(group < 16 ? group : 16) * (padded_dim(dim) + kPartHead);
}

hipError_t launch_paged_attention(const PagedAttentionArgs& args, int dtype, bool fp8,
                                  int workgroups, hipStream_t stream) {
  PagedAttentionArgs a = args;
  a.by_page = div_magic((uint32_t)a.page_size);
  a.by_waves = div_magic((uint32_t)workgroups * kWaves);
  a.by_rows = div_magic((uint32_t)(a.kv_heads * a.head_tiles));
  if (dtype == kBF16)
    return fp8 ? launch_dim<kBF16, true>(a, workgroups, stream)
               : launch_dim<kBF16, false>(a, workgroups, stream);
  return fp8 ? launch_dim<kF16, true>(a, workgroups, stream)
             : launch_dim<kF16, false>(a, workgroups, stream);
}

}  // namespace mt
