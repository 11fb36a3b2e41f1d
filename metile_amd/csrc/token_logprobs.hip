// Log probabilities of given tokens, entropies of their distributions and the likeliest alternatives.
//
//   log p_i = (x_i - m) / T - log S      S = sum_j exp((x_j - m) / T)      m = max_j x_j
//   H = log S - (sum_j exp((x_j - m) / T) (x_j - m) / T) / S
//   rank of a token: how many logits are larger, or as large and before it
//
// in one pass over the logits: a thread keeps a running maximum, sum and weighted sum of its own, a
// batch of 32 values at a time. For the alternatives it also keeps each batch's maximum. The k-th
// largest of those, t, is a lower bound of the k-th largest logit, so all that is larger than t lies in
// the fewer than k groups of 32 whose maximum is: they alone are read again. What is left to k are the
// first logits that equal t. Order is by value, then by index, and no sum goes by the order in which
// threads arrive.
//
// A workgroup takes a row, or with few rows a part of one; the parts are joined by a second launch.
#include <algorithm>

#include "common.h"
#include "token_logprobs.h"

namespace mt {
namespace {

constexpr int kThreads = 256, kWaves = kThreads / 64;
constexpr int kUnits = 4;                        // runs of 8 values of a thread in a batch
constexpr int kRun = kThreads * 8;               // values of a unit, next to each other
constexpr int kBatch = kRun * kUnits;            // values of a batch
constexpr int kMostBatches = 32;                 // of a part: their maxima fit LDS
constexpr int kMostTop = kLogprobsMostTop;
constexpr int kF32 = 2;
constexpr float kLowest = -3.402823466e38f;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

// Order of values as unsigned numbers: -0 and +0 alike, NaN below all others.
__device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t u = __float_as_uint(x + 0.0f);
  return x != x ? 0u : (u >> 31) ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t key) {
  return __uint_as_float(key >> 31 ? key & 0x7fffffffu : ~key);
}

struct Sums {
  float m, s, w;  // maximum; sum of exp((x - m) / T), and of that times x - m
};
// A weighted sum w beside a sum s once its maximum is |d| smaller than the new one, f = exp(d / T). A sum
// that does not count any more adds nothing, whatever its distance; sums that are no numbers stay so.
__device__ __forceinline__ float moved(float w, float s, float d, float f) {
  return f > 0.0f ? f * (w + s * d) : s * 0.0f;
}
__device__ __forceinline__ Sums join(Sums a, Sums b, float scale) {
  Sums r;
  r.m = fmaxf(a.m, b.m);
  const float at = r.m == -__builtin_inff() ? 0.0f : r.m;
  const float da = fmaxf(a.m - at, kLowest), db = fmaxf(b.m - at, kLowest);
  const float fa = __builtin_amdgcn_exp2f(da * scale), fb = __builtin_amdgcn_exp2f(db * scale);
  r.s = a.s * fa + b.s * fb;
  r.w = moved(a.w, a.s, da, fa) + moved(b.w, b.s, db, fb);
  return r;
}

// What a part of a row hands on: 16 bytes, then its alternatives as (key, index), largest first.
struct Part {
  Sums sums;
  int32_t larger;
};

template <int DT>
__device__ __forceinline__ void load8(const unsigned char* p, float (&x)[8]) {
  if constexpr (DT == kF32) {
    __builtin_memcpy(x, p, 32);
  } else {
    u32x4 v;
    __builtin_memcpy(&v, p, 16);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t w = v[j];
      x[2 * j] = lo16<DT>(w);
      x[2 * j + 1] = hi16<DT>(w);
    }
  }
}
template <int DT>
__device__ __forceinline__ float load1(const unsigned char* row, int i) {
  if constexpr (DT == kF32) return reinterpret_cast<const float*>(row)[i];
  else return act_to_f32<DT>(reinterpret_cast<const uint16_t*>(row)[i]);
}
// Eight values from i on, -inf behind `end`.
template <int DT>
__device__ __forceinline__ void load8_to(const unsigned char* row, int i, int end, float (&x)[8]) {
  if (i + 8 <= end) {
    load8<DT>(row + (int64_t)i * (DT == kF32 ? 4 : 2), x);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = i + j < end ? load1<DT>(row, i + j) : -__builtin_inff();
  }
}

__device__ __forceinline__ uint64_t wave_max64(uint64_t v) {
  for (int d = 32; d; d /= 2) {
    const uint64_t o = (uint64_t)__shfl_xor((unsigned long long)v, d);
    v = o > v ? o : v;
  }
  return v;
}

// Sum over the workgroup, in every thread. `lds` holds kWaves words; two barriers.
__device__ __forceinline__ int block_sum(int v, int* lds) {
  for (int d = 32; d; d /= 2) v += __shfl_xor(v, d);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  v = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) v += lds[w];
  return v;
}

// The n (at most kMostTop) largest of `count` different numbers in LDS, put in order into best[].
__device__ __forceinline__ void put_in_order(const uint64_t* from, int count, int n, uint64_t* best) {
  for (int i = threadIdx.x; i < count; i += kThreads) {
    const uint64_t v = from[i];
    int rank = 0;
    for (int j = 0; j < count && rank < n; ++j) rank += from[j] > v;
    if (rank < n) best[rank] = v;
  }
}

__device__ __forceinline__ void write_row(const LogprobsArgs& a, int row, Sums sums, float given,
                                          bool in_vocab, int larger, const uint64_t* best) {
  const float log_s = __builtin_amdgcn_logf(sums.s) * kLn2;  // -inf for a row of -inf alone
  auto logprob = [&](float x) {
    if (sums.s == 0.0f) return -__builtin_inff();
    return (x - sums.m) * a.inv_temperature - log_s;
  };
  if (threadIdx.x == 0) {
    a.entropies[row] = sums.s == 0.0f ? 0.0f : log_s - a.inv_temperature * sums.w / sums.s;
    if (a.tokens) {
      a.logprobs[row] = in_vocab ? logprob(given) : -__builtin_inff();
      a.ranks[row] = in_vocab ? larger : -1;
    }
  }
  for (int i = threadIdx.x; i < a.top; i += kThreads) {
    const uint32_t key = (uint32_t)(best[i] >> 32);
    a.top_logprobs[(int64_t)row * a.top + i] =
        key ? logprob(value_of(key)) : __builtin_nanf("");
    a.top_tokens[(int64_t)row * a.top + i] = key ? (int64_t)(~(uint32_t)best[i]) : -1;
  }
}

template <int DT>
__global__ __launch_bounds__(kThreads) void logprobs_kernel(LogprobsArgs a) {
  extern __shared__ uint32_t group_keys[];  // [batches][kThreads], with alternatives
  __shared__ uint64_t larger_than[32 * kMostTop];
  __shared__ uint64_t best[kMostTop];
  __shared__ Sums wave_sums[kWaves];
  __shared__ int wave_count[kWaves], counts[2], groups[kMostTop];
  __shared__ uint64_t flagged;

  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int row = blockIdx.x / (unsigned)a.num_parts, part = blockIdx.x % (unsigned)a.num_parts;
  const unsigned char* x_row = static_cast<const unsigned char*>(a.logits) +
                               (int64_t)row * a.row_stride * (DT == kF32 ? 4 : 2);
  const int64_t part_size = (int64_t)a.part_batches * kBatch;
  const int begin = (int)(part * part_size);
  const int end = (int)min((int64_t)a.vocab, begin + part_size);
  const int batches = (end - begin + kBatch - 1) / kBatch;
  const float scale = a.inv_temperature * kLog2e;

  int token = -1;
  float given = 0.0f;
  bool in_vocab = false;
  if (a.tokens) {
    const int64_t t = a.tokens[row];
    in_vocab = t >= 0 && t < a.vocab;
    token = in_vocab ? (int)t : 0;
    given = load1<DT>(x_row, token);
  }

  // ---- sums, and each group's maximum ----
  Sums own = {-__builtin_inff(), 0.0f, 0.0f};
  int larger = 0;  // of the wave
  for (int b = 0; b < batches; ++b) {
    const int at = begin + b * kBatch;
    float x[kUnits][8];
#pragma unroll
    for (int u = 0; u < kUnits; ++u) load8_to<DT>(x_row, at + u * kRun + tid * 8, end, x[u]);
    float top = x[0][0];
#pragma unroll
    for (int u = 0; u < kUnits; ++u)
#pragma unroll
      for (int j = 0; j < 8; ++j) top = fmaxf(top, x[u][j]);
    if (a.top) group_keys[b * kThreads + tid] = key_of(top);
    const float m = fmaxf(own.m, top), zero_at = m == -__builtin_inff() ? 0.0f : m;
    const float step = fmaxf(own.m - zero_at, kLowest);
    const float fix = __builtin_amdgcn_exp2f(step * scale);
    float w = moved(own.w, own.s, step, fix), s = own.s * fix;
    own.m = m;
#pragma unroll
    for (int u = 0; u < kUnits; ++u)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float t = x[u][j] - zero_at;
        const float e = __builtin_amdgcn_exp2f(t * scale);
        s += e;
        w = fmaf(e, fmaxf(t, kLowest), w);  // (0 times -inf is none)
      }
    own.s = s;
    own.w = w;
    if (a.tokens) {
#pragma unroll
      for (int u = 0; u < kUnits; ++u) {
        const int from = at + u * kRun;
        if (token >= from + kRun) {  // those before the token count if they are as large
#pragma unroll
          for (int j = 0; j < 8; ++j) larger += __popcll(__ballot(x[u][j] >= given));
        } else if (token < from) {
#pragma unroll
          for (int j = 0; j < 8; ++j) larger += __popcll(__ballot(x[u][j] > given));
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j)
            larger += __popcll(__ballot(x[u][j] > given ||
                                        (x[u][j] == given && from + tid * 8 + j < token)));
        }
      }
    }
  }
  for (int d = 32; d; d /= 2) {
    Sums other;
    other.m = __shfl_xor(own.m, d);
    other.s = __shfl_xor(own.s, d);
    other.w = __shfl_xor(own.w, d);
    own = (lane & d) ? join(other, own, scale) : join(own, other, scale);
  }
  if (lane == 0) {
    wave_sums[wave] = own;
    wave_count[wave] = larger;
  }
  if (tid < kMostTop) best[tid] = 0;
  if (tid == 0) counts[0] = counts[1] = 0, flagged = 0;
  __syncthreads();
  Sums sums = wave_sums[0];
  larger = wave_count[0];
#pragma unroll
  for (int w = 1; w < kWaves; ++w) {
    sums = join(sums, wave_sums[w], scale);
    larger += wave_count[w];
  }

  // ---- alternatives ----
  if (a.top) {
    const int k = a.top;
    // the k-th largest of the groups' maxima: the largest key that k of them reach (0: fewer do)
    uint32_t bound = 0;
    constexpr int kLowBit = DT == kF32 ? 0 : DT == kBF16 ? 16 : 13;  // 16-bit values have no others
    for (int bit = 31; bit >= kLowBit; --bit) {
      const uint32_t middle = bound | 1u << bit;
      int n = 0;
      for (int b = 0; b < batches; ++b) n += group_keys[b * kThreads + tid] >= middle;
      if (block_sum(n, wave_count) >= k) bound = middle;
    }
    // negative values of 16 bits have ones below: the key itself, not its first bits
    if (kLowBit && !(bound >> 31)) bound = bound ? bound | ((1u << kLowBit) - 1) : 0;
    // (fewer than k) groups with larger values, and the batches that have values of the bound
    for (int b = 0; b < batches; ++b) {
      const uint32_t key = group_keys[b * kThreads + tid];
      if (key > bound) groups[atomicAdd(&counts[0], 1)] = b * kThreads + tid;
      if (key >= bound && bound) atomicOr((unsigned long long*)&flagged, 1ull << b);
    }
    __syncthreads();
    const int num_groups = counts[0];
    {
      const int g = tid / 8, u = tid % 8 / 2, j0 = tid % 2 * 4;
      if (g < num_groups) {
        const int group = groups[g];
        const int at = begin + group / kThreads * kBatch + u * kRun + group % kThreads * 8 + j0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t key = at + j < end ? key_of(load1<DT>(x_row, at + j)) : 0;
          if (key > bound)
            larger_than[atomicAdd(&counts[1], 1)] = (uint64_t)key << 32 | ~(uint32_t)(at + j);
        }
      }
    }
    __syncthreads();
    const int found = counts[1];
    put_in_order(larger_than, found, k, best);
    int have = min(found, k);
    // the first values that equal the bound, unit by unit
    for (uint64_t rest = flagged; rest && have < k; rest &= rest - 1) {
      const int b = __ffsll((unsigned long long)rest) - 1;
      for (int u = 0; u < kUnits && have < k; ++u) {
        const int at = begin + b * kBatch + u * kRun + tid * 8;
        float x[8];
        load8_to<DT>(x_row, at, end, x);
        int n = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) n += at + j < end && key_of(x[j]) == bound;
        // those of the threads before
        int before = n;
        for (int d = 1; d < 64; d *= 2) {
          const int o = __shfl_up(before, d);
          if (lane >= d) before += o;
        }
        __syncthreads();
        if (lane == 63) wave_count[wave] = before;
        __syncthreads();
        int all = 0;
        before -= n;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
          if (w < wave) before += wave_count[w];
          all += wave_count[w];
        }
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (at + j < end && key_of(x[j]) == bound) {
            if (have + before < k)
              best[have + before] = (uint64_t)bound << 32 | ~(uint32_t)(at + j);
            ++before;
          }
        have = min(k, have + all);
      }
    }
    __syncthreads();
  }

  if (a.num_parts == 1) {
    write_row(a, row, sums, given, in_vocab, larger, best);
    return;
  }
  unsigned char* to = a.parts + (int64_t)blockIdx.x * (sizeof(Part) + a.top * 8);
  if (tid == 0) *reinterpret_cast<Part*>(to) = Part{sums, larger};
  if (tid < a.top) reinterpret_cast<uint64_t*>(to + sizeof(Part))[tid] = best[tid];
}

template <int DT>
__global__ __launch_bounds__(kThreads) void join_kernel(LogprobsArgs a) {
  extern __shared__ uint64_t candidates[];  // [num_parts * top]
  __shared__ uint64_t best[kMostTop];
  __shared__ int count;
  __shared__ uint64_t wave_least[kWaves];
  const int tid = threadIdx.x, row = blockIdx.x;
  const int step = (int)sizeof(Part) + a.top * 8;
  const unsigned char* from = a.parts + (int64_t)row * a.num_parts * step;
  const float scale = a.inv_temperature * kLog2e;
  const unsigned char* x_row = static_cast<const unsigned char*>(a.logits) +
                               (int64_t)row * a.row_stride * (DT == kF32 ? 4 : 2);
  float given = 0.0f;
  bool in_vocab = false;
  if (a.tokens) {
    const int64_t t = a.tokens[row];
    in_vocab = t >= 0 && t < a.vocab;
    given = load1<DT>(x_row, in_vocab ? (int)t : 0);
  }
  Sums sums = {-__builtin_inff(), 0.0f, 0.0f};
  int larger = 0;
  for (int p = 0; p < a.num_parts; ++p) {
    const Part part = *reinterpret_cast<const Part*>(from + (int64_t)p * step);
    sums = join(sums, part.sums, scale);
    larger += part.larger;
  }
  if (tid < kMostTop) best[tid] = 0;
  if (tid == 0) count = 0;
  if (a.top) {
    auto entry = [&](int p, int i) {
      return reinterpret_cast<const uint64_t*>(from + (int64_t)p * step + sizeof(Part))[i];
    };
    // nothing below a part's last is among the first of all
    uint64_t least = 0;
    for (int p = tid; p < a.num_parts; p += kThreads) least = max(least, entry(p, a.top - 1));
    least = wave_max64(least);
    if ((tid & 63) == 0) wave_least[tid >> 6] = least;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWaves; ++w) least = max(least, wave_least[w]);
    for (int n = tid; n < a.num_parts * a.top; n += kThreads) {
      const uint64_t v = entry(n / a.top, n % a.top);
      if (v && v >= least) candidates[atomicAdd(&count, 1)] = v;
    }
    __syncthreads();
    put_in_order(candidates, count, a.top, best);
    __syncthreads();
  }
  write_row(a, row, sums, given, in_vocab, larger, best);
}

template <int DT>
hipError_t launch(const LogprobsArgs& args, hipStream_t stream) {
  const int keys = args.top ? std::min(args.part_batches, (args.vocab + kBatch - 1) / kBatch) * kThreads * 4 : 0;
  // rows of a launch, so that its threads are counted in 32 bits; the parts of one are joined before
  // those of the next are made
  const int most = std::max(1, (1 << 22) / args.num_parts);
  for (int64_t row = 0; row < args.rows; row += most) {
    LogprobsArgs a = args;
    a.logits = static_cast<const unsigned char*>(a.logits) +
               row * a.row_stride * (DT == kF32 ? 4 : 2);
    a.entropies += row;
    if (a.tokens) a.tokens += row, a.logprobs += row, a.ranks += row;
    if (a.top) a.top_logprobs += row * a.top, a.top_tokens += row * a.top;
    const int rows = (int)std::min<int64_t>(most, args.rows - row);
    logprobs_kernel<DT><<<(unsigned)rows * (unsigned)a.num_parts, kThreads, keys, stream>>>(a);
    if (a.num_parts > 1) join_kernel<DT><<<rows, kThreads, a.num_parts * a.top * 8, stream>>>(a);
    if (const hipError_t e = hipGetLastError()) return e;
  }
  return hipSuccess;
}

}  // namespace

// A workgroup a row, unless that leaves CUs without one: then parts of whole batches, so many that
// there are four workgroups a CU, at most 64.
LogprobsPlan plan_token_logprobs(int rows, int vocab, int cus) {
  const int batches = std::max(1, (int)(((int64_t)vocab + kBatch - 1) / kBatch));
  int parts = (int)std::min<int64_t>(batches, std::max<int64_t>(1, 4ll * cus / std::max(rows, 1)));
  parts = std::min(parts, 64);
  const int per = std::min(kMostBatches, (batches + parts - 1) / parts);
  return {per, (batches + per - 1) / per};
}

size_t logprobs_part_bytes(int top) { return sizeof(Part) + (size_t)top * 8; }

hipError_t launch_token_logprobs(const LogprobsArgs& a, int dtype, hipStream_t stream) {
  if (dtype == kBF16) return launch<kBF16>(a, stream);
  if (dtype == kF16) return launch<kF16>(a, stream);
  return launch<kF32>(a, stream);
}

}  // namespace mt
