// Log probabilities of given tokens, entropies of their distributions and the likeliest alternatives.
//
//   log p_i = (y_i - log2 S) ln 2      y_j = c x_j - R      c = log2 e / T      S = sum_j 2^(y_j)
//   H = (log2 S - (sum_j 2^(y_j) y_j) / S) ln 2
//   rank of a token: how many logits are larger, or as large and before it
//
// in one pass over the logits. R is any whole number near c times the largest logit: exact in fp32, so
// that y has one rounding, and kept until a logit passes it by four powers of two, so that the sums
// are hardly ever rescaled. For the alternatives a thread keeps the maximum of each group of 32 values.
// The k-th largest of the threads' maxima, t, is a lower bound of the k-th largest logit, so all of the k
// lie in groups whose maximum reaches t: they alone are read again (as many of them as there are
// alternatives, or a few more; where there are many, for equal logits or a long run of large ones, those
// above the k-th largest maximum, and then the first logits that equal it). Order is by value, then by
// index, and no sum goes by the order in which threads arrive.
//
// A workgroup takes a row, or with few rows a part of one; the parts are joined by a second launch.
//
// What bounds it: vector instructions, 9.1 a value, which issue for 86% of the time: 2048 rows of 152064 bf16
// values take 129 us, 4.8 TB/s of the 6.3 that reads alone reach; of fp32 values 218, 5.7 TB/s. A row of 32000
// takes 11 us of round trips.
#include <algorithm>

#include "common.h"
#include "token_logprobs.h"

namespace mt {
namespace {

// Threads of a workgroup. With as many rows as CUs or fewer and more than 16384 values in each, 16 waves
// take a row with fewer parts to join (us with 4 waves -> 16, top 20 of 152064 values: 1 row 23.2 -> 21.7,
// 64 rows 25.7 -> 23.7, 256 rows 34.7 -> 26.1); below that 4 have less to exchange (1 row of 1000 values
// 8.0, with 16 waves 11.0).
constexpr int kFew = 1024, kMany = 256;
constexpr int kUnits = 4;                        // runs of 8 values of a thread in a batch
constexpr int kMostKept = 8192;                  // groups of a part: their maxima fit LDS
constexpr int kBounds = 256;                     // maxima that the bound is found from
constexpr int kMostGroups = 64;                  // that are read again
constexpr int kMostTop = kLogprobsMostTop;
constexpr int kF32 = 2;
constexpr float kLowest = -3.402823466e38f;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kNothing = -0x1p100f;  // the reference before any logit
constexpr double kNone = -1e300;       // and of a sum of nothing, below that of every logit
constexpr float kRoom = 4.0f;

// Order of values as unsigned numbers: -0 and +0 alike, NaN below all others.
__device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t u = __float_as_uint(x + 0.0f);
  return x != x ? 0u : (u >> 31) ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t key) {
  return __uint_as_float(key >> 31 ? key & 0x7fffffffu : ~key);
}

// (In 64 bits: beside the sum of a likely token the others' are small, and round alike.)
struct Sums {
  double ref;   // R
  double s, w;  // sums of 2^y and 2^y y
};
// A weighted sum w beside a sum s once its reference is d (below 0) from the new one, f = 2^d. A sum
// that does not count any more adds nothing, whatever its distance; sums that are no numbers stay so.
template <typename F>
__device__ __forceinline__ F moved(F w, F s, F d, F f) {
  return f > 0 ? f * (w + s * d) : s * 0;
}
__device__ __forceinline__ Sums join(Sums a, Sums b) {
  Sums r;
  r.ref = a.ref > b.ref ? a.ref : b.ref;
  const double da = a.ref - r.ref, db = b.ref - r.ref;
  const double fa = __builtin_amdgcn_exp2f((float)da), fb = __builtin_amdgcn_exp2f((float)db);
  r.s = a.s * fa + b.s * fb;
  r.w = moved(a.w, a.s, da, fa) + moved(b.w, b.s, db, fb);
  return r;
}

// What a part of a row hands on, and behind it its alternatives as (key, index), largest first.
struct Part {
  Sums sums;
  int64_t larger;
};

// The largest of three, without the instructions that would quiet NaN first.
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  __asm__("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
}

// Eight values as they lie in memory.
template <int DT>
struct Raw {
  u32x4 v[DT == kF32 ? 2 : 1];
};
template <int DT>
__device__ __forceinline__ float load1(const unsigned char* row, int i) {
  if constexpr (DT == kF32) return reinterpret_cast<const float*>(row)[i];
  else return act_to_f32<DT>(reinterpret_cast<const uint16_t*>(row)[i]);
}
// Addresses need the alignment of a value only.
template <int DT>
__device__ __forceinline__ Raw<DT> load8(const unsigned char* p) {
  Raw<DT> r;
  __builtin_memcpy(&r, p, sizeof r);
  return r;
}
template <int DT>
__device__ __forceinline__ void values8(const Raw<DT>& r, float (&x)[8]) {
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const uint32_t w = DT == kF32 ? r.v[j / 4][j % 4] : r.v[0][j / 2];
    if constexpr (DT == kF32) x[j] = __uint_as_float(w);
    else x[j] = j % 2 ? hi16<DT>(w) : lo16<DT>(w);
  }
}
// The eight values from i on, -inf behind `end`.
template <int DT>
__device__ __forceinline__ void tail8(const unsigned char* row, int i, int end, float (&x)[8]) {
  if (i + 8 <= end) {
    values8<DT>(load8<DT>(row + (int64_t)i * (DT == kF32 ? 4 : 2)), x);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = -__builtin_inff();
#pragma unroll 1
    for (int j = 0; i + j < end; ++j) {
      const float v = load1<DT>(row, i + j);
#pragma unroll
      for (int k = 0; k < 8; ++k) x[k] = j == k ? v : x[k];
    }
  }
}

__device__ __forceinline__ uint64_t wave_max64(uint64_t v) {
  for (int d = 32; d; d /= 2) {
    const uint64_t o = (uint64_t)__shfl_xor((unsigned long long)v, d);
    v = o > v ? o : v;
  }
  return v;
}

// Sum over the workgroup of its waves' counts, in every thread. `turn` alternates the LDS used, so that
// one barrier is enough.
template <int kWaves>
__device__ __forceinline__ int block_sum(int of_wave, int (&lds)[2][kWaves], int& turn) {
  if ((threadIdx.x & 63) == 0) lds[turn][threadIdx.x >> 6] = of_wave;
  __syncthreads();
  int v = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) v += lds[turn][w];
  turn ^= 1;
  return v;
}

// The n (at most kMostTop) largest of `count` different numbers in LDS, put in order into best[].
__device__ __forceinline__ void put_in_order(const uint64_t* from, int count, int n, uint64_t* best) {
  for (int i = threadIdx.x; i < count; i += blockDim.x) {
    const uint64_t v = from[i];
    int rank = 0;
    for (int j = 0; j < count && rank < n; ++j) rank += from[j] > v;
    if (rank < n) best[rank] = v;
  }
}

__device__ __forceinline__ void write_row(const LogprobsArgs& a, int row, Sums sums, float given,
                                          bool in_vocab, int larger, const uint64_t* best) {
  const float scale = a.inv_temperature * kLog2e;
  const float log_s = __builtin_amdgcn_logf((float)sums.s);
  auto logprob = [&](float x) {
    if (sums.s == 0.0) return -__builtin_inff();  // a row of -inf alone
    const float l = (float)(((double)x * (double)scale - sums.ref - (double)log_s) * 0.6931471805599453);
    return l > 0.0f ? 0.0f : l;
  };
  if (threadIdx.x == 0) {
    const float h = sums.s == 0.0 ? 0.0f : (log_s - (float)(sums.w / sums.s)) * kLn2;
    a.entropies[row] = h < 0.0f ? 0.0f : h;
    if (a.tokens) {
      a.logprobs[row] = in_vocab ? logprob(given) : -__builtin_inff();
      a.ranks[row] = in_vocab ? larger : -1;
    }
  }
  for (int i = threadIdx.x; i < a.top; i += blockDim.x) {
    const uint32_t key = (uint32_t)(best[i] >> 32);
    a.top_logprobs[(int64_t)row * a.top + i] =
        key ? logprob(value_of(key)) : __builtin_nanf("");
    a.top_tokens[(int64_t)row * a.top + i] = key ? (int64_t)(~(uint32_t)best[i]) : -1;
  }
}

template <int DT, int kThreads>
__global__ __launch_bounds__(kThreads) void logprobs_kernel(LogprobsArgs a) {
  constexpr int kWaves = kThreads / 64;
  constexpr int kRun = kThreads * 8, kBatch = kRun * kUnits;  // values of a unit, next to each other
  // each group's maximum, [batches][kThreads]; later the candidates, kMostGroups * 32 of them
  extern __shared__ __attribute__((aligned(16))) uint32_t group_keys[];
  __shared__ uint64_t best[kMostTop], flagged;
  __shared__ Sums wave_sums[kWaves];
  __shared__ uint32_t thread_keys[kBounds];
  __shared__ int wave_count[2][kWaves], counts[2], groups[kMostGroups];

  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int row = blockIdx.x / (unsigned)a.num_parts, part = blockIdx.x % (unsigned)a.num_parts;
  const unsigned char* x_row = static_cast<const unsigned char*>(a.logits) +
                               (int64_t)row * a.row_stride * (DT == kF32 ? 4 : 2);
  const int64_t part_size = (int64_t)a.part_batches * kBatch;
  const int begin = (int)(part * part_size);
  const int end = (int)min((int64_t)a.vocab, begin + part_size);
  const int batches = (end - begin + kBatch - 1) / kBatch;
  const float scale = a.inv_temperature * kLog2e;

  // ---- sums, and each group's maximum ----
  constexpr uint32_t kSize = DT == kF32 ? 4 : 2;
  Raw<DT> next[kUnits];
  auto request = [&](int b) {  // a batch that is whole
    const unsigned char* p = x_row + (int64_t)(begin + b * kBatch) * kSize;
#pragma unroll
    for (int u = 0; u < kUnits; ++u) next[u] = load8<DT>(p + (u * kRun + (uint32_t)tid * 8) * kSize);
  };
  const int whole = (end - begin) / kBatch;
  if (whole) request(0);
  int token = -1;
  float given = 0.0f;
  bool in_vocab = false;
  if (a.tokens) {
    const int64_t t = a.tokens[row];
    in_vocab = t >= 0 && t < a.vocab;
    token = in_vocab ? (int)t : 0;
    given = load1<DT>(x_row, token);
  }
  auto tail = [&](int b, float (&x)[kUnits][8]) {
#pragma unroll
    for (int u = 0; u < kUnits; ++u)
      tail8<DT>(x_row, begin + b * kBatch + u * kRun + tid * 8, end, x[u]);
  };
  // Sums of 2 d lanes, in each of them.
  auto of_lanes = [&](Sums own, int d) {
    for (; d; d /= 2) {
      Sums other;
      other.ref = __shfl_xor(own.ref, d);
      other.s = __shfl_xor(own.s, d);
      other.w = __shfl_xor(own.w, d);
      own = (lane & d) ? join(other, own) : join(own, other);
    }
    return own;
  };
  auto of_waves = [&](Sums own) {
    if (lane == 0) wave_sums[wave] = own;
    __syncthreads();
    return of_lanes(wave_sums[lane % kWaves], kWaves / 2);
  };
  float ref = kNothing, s = 0.0f, w = 0.0f, own_top = -__builtin_inff();  // ref is the wave's
  int larger = 0;                                                        // of the wave
  bool masked = false;  // the wave has met -inf
  // Values as large as the token's count if they are before it: those larger than the next value below.
  const uint32_t bits = __float_as_uint(given);
  const float below = __uint_as_float(given == 0.0f ? 0x80000001u : bits >> 31 ? bits + 1 : bits - 1);
  auto take = [&](int b, const float (&x)[kUnits][8]) {
    const int at = begin + b * kBatch + tid * 8;
    float tops[kUnits];
#pragma unroll
    for (int u = 0; u < kUnits; ++u) tops[u] = max3(x[u][0], x[u][1], x[u][2]);
#pragma unroll
    for (int u = 0; u < kUnits; ++u) tops[u] = max3(tops[u], x[u][3], x[u][4]);
#pragma unroll
    for (int u = 0; u < kUnits; ++u) tops[u] = max3(tops[u], x[u][5], x[u][6]);
    float top = max3(tops[0], x[0][7], x[1][7]);
    top = max3(top, max3(tops[1], x[2][7], x[3][7]), max3(tops[2], tops[2], tops[3]));
    if (a.top) {
      group_keys[b * kThreads + tid] = key_of(top);
      own_top = fmaxf(own_top, top);
    }
    if (__any(fmaf(top, scale, -ref) > kRoom)) {
      float most = top;
      for (int d = 32; d; d /= 2) most = fmaxf(most, __shfl_xor(most, d));
      const float to = rintf(most * scale), d = ref - to, f = __builtin_amdgcn_exp2f(d);
      w = moved(w, s, d, f);
      s *= f;
      ref = to;
    }
    // The sums of the batch. (2^y y is no number for y of -inf, which adds nothing: a wave that has met
    // one bounds y, an instruction more.)
    const float s0 = s, w0 = w;
    if (!masked) {
#pragma unroll
      for (int u = 0; u < kUnits; ++u)
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float y = fmaf(x[u][j], scale, -ref);
          const float e = __builtin_amdgcn_exp2f(y);
          s += e;
          w = fmaf(e, y, w);
        }
      masked = __any(w != w);
    }
    if (masked) {
      s = s0;
      w = w0;
      const float same = opaque(ref);  // (no exponential is to be kept for this)
#pragma unroll
      for (int u = 0; u < kUnits; ++u)
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float y = fmaf(x[u][j], scale, -same);
          const float e = __builtin_amdgcn_exp2f(y);
          s += e;
          w = fmaf(e, fmaxf(y, kLowest), w);
        }
    }
    if (a.tokens && __any(top >= given)) {
#pragma unroll
      for (int u = 0; u < kUnits; ++u) {
        const float bound = at + u * kRun + 8 <= token ? below : given;
#pragma unroll
        for (int j = 0; j < 8; ++j) larger += __popcll(__ballot(x[u][j] > bound));
      }
    }
  };
  for (int b = 0; b < whole; ++b) {
    float x[kUnits][8];
#pragma unroll
    for (int u = 0; u < kUnits; ++u) values8<DT>(next[u], x[u]);
    if (b + 1 < whole) request(b + 1);
    take(b, x);
  }
  if (whole < batches) {
    float x[kUnits][8];
    tail(whole, x);
    take(whole, x);
  }
  if (in_vocab && token >= begin && token < end && tid == 0)  // those of the token's own eight
    for (int i = token & ~7; i < token; ++i) larger += load1<DT>(x_row, i) == given;
  // The rank's count by the definition, of the wave.
  auto count_larger = [&]() {
    larger = 0;
    for (int i = begin + tid; i < end; i += kThreads) {
      const float x = load1<DT>(x_row, i);
      larger += __popcll(__ballot(x > given || (x == given && i < token)));
    }
  };
  if (in_vocab && given == -__builtin_inff()) count_larger();  // (nothing is below -inf)
  if (lane == 0) wave_count[0][wave] = larger;
  if (tid < kMostTop) best[tid] = 0;
  if (tid == 0) counts[0] = counts[1] = 0, flagged = 0;
  double wave_s = s, wave_w = w;
  for (int d = 32; d; d /= 2) wave_s += __shfl_xor(wave_s, d), wave_w += __shfl_xor(wave_w, d);
  Sums sums = of_waves({wave_s == 0.0 ? kNone : (double)ref, wave_s, wave_w});
  uint32_t own_key = key_of(own_top);
  if (!(sums.s > 0.0 && sums.s < (double)__builtin_inff())) {
    // NaN or infinities, logits too large for c times them, or none that is allowed: again, with
    // references in 64 bits and maxima by whole numbers, and the rank's count without maxima
    Sums own = {kNone, 0.0, 0.0};
    own_key = 0;
#pragma unroll 1
    for (int b = 0; b < batches; ++b) {
      float x[kUnits][8];
      tail(b, x);
      uint32_t key = 0;
#pragma unroll 1
      for (int u = 0; u < kUnits; ++u) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float v = u == 0 ? x[0][j] : u == 1 ? x[1][j] : u == 2 ? x[2][j] : x[3][j];
          key = max(key, key_of(v));
          if (v == -__builtin_inff()) continue;
          const Sums one = {(double)v * (double)scale, v - v == 0.0f ? 1.0 : (double)(v - v), 0.0};
          own = join(own, one);
        }
      }
      if (a.top) group_keys[b * kThreads + tid] = key;
      own_key = max(own_key, key);
    }
    if (in_vocab) {  // (maxima that a signalling NaN had part in may have hidden larger values)
      count_larger();
      if (lane == 0) wave_count[0][wave] = larger;
    }
    __syncthreads();
    sums = of_waves(of_lanes(own, 32));
  }
  larger = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) larger += wave_count[0][w];

  // ---- alternatives ----
  if (a.top) {
    const int k = a.top;
    constexpr int kLowBit = DT == kF32 ? 0 : DT == kBF16 ? 16 : 13;  // 16-bit values have no others
    auto exact = [&](uint32_t bound) {  // keys of negative values have ones there
      return kLowBit && bound && !(bound >> 31) ? bound | ((1u << kLowBit) - 1) : bound;
    };
    // the k-th largest of the threads' maxima (of 16 waves, the fours of threads'): the largest key
    // that k of them reach (0: fewer do)
    constexpr int kEach = kThreads / kBounds, kKeys = kBounds / 64;
    for (int d = 1; d < kEach; d *= 2) own_key = max(own_key, (uint32_t)__shfl_xor((int)own_key, d));
    if (tid % kEach == 0) thread_keys[tid / kEach] = own_key;
    __syncthreads();
    uint32_t bound = 0;
    {
      uint32_t keys[kKeys];
#pragma unroll
      for (int i = 0; i < kKeys; ++i) keys[i] = thread_keys[64 * i + lane];
      for (int bit = 31; bit >= kLowBit; --bit) {
        const uint32_t middle = bound | 1u << bit;
        int n = 0;
#pragma unroll
        for (int i = 0; i < kKeys; ++i) n += __popcll(__ballot(keys[i] >= middle));
        if (n >= k) bound = middle;
      }
      bound = exact(bound);
    }
    // groups that reach `least`
    auto collect = [&](uint32_t least) {
      for (int b = 0; b < batches; ++b)
        if (group_keys[b * kThreads + tid] >= least) {
          const int n = atomicAdd(&counts[0], 1);
          if (n < kMostGroups) groups[n] = b * kThreads + tid;
        }
      __syncthreads();
    };
    uint32_t least = max(bound, 1u);
    collect(least);
    const bool many = counts[0] > kMostGroups;
    if (many) {
      // Many equal values, or many large ones in one thread's groups: the k-th largest of all groups'
      // maxima, the fewer than k groups above it, and the batches that have values of it.
      int turn = 1;
      uint32_t of_groups = 0;
      for (int bit = 31; bit >= kLowBit; --bit) {
        const uint32_t middle = of_groups | 1u << bit;
        int n = 0;
        for (int b = 0; b < batches; ++b)
          n += __popcll(__ballot(group_keys[b * kThreads + tid] >= middle));
        if (block_sum(n, wave_count, turn) >= k) of_groups = middle;
      }
      bound = exact(of_groups);
      least = bound + 1;
      __syncthreads();
      if (tid == 0) counts[0] = 0;
      for (int b = 0; b < batches; ++b)
        if (bound && group_keys[b * kThreads + tid] >= bound)
          atomicOr((unsigned long long*)&flagged, 1ull << b);
      __syncthreads();
      collect(least);
    }
    const int num_groups = counts[0];
    uint64_t* candidates = reinterpret_cast<uint64_t*>(group_keys);
    for (int g = tid / 8; g < num_groups; g += kThreads / 8) {
      const int u = tid % 8 / 2, j0 = tid % 2 * 4, group = groups[g];
      const int at = begin + group / kThreads * kBatch + u * kRun + group % kThreads * 8 + j0;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t key = at + j < end ? key_of(load1<DT>(x_row, at + j)) : 0;
        if (key >= least)
          candidates[atomicAdd(&counts[1], 1)] = (uint64_t)key << 32 | ~(uint32_t)(at + j);
      }
    }
    __syncthreads();
    const int found = counts[1];
    put_in_order(candidates, found, k, best);
    int have = min(found, k), turn = 1;
    // with many, the first values that equal the bound, unit by unit
    for (uint64_t rest = many ? flagged : 0; rest && have < k; rest &= rest - 1) {
      const int b = __ffsll((unsigned long long)rest) - 1;
      for (int u = 0; u < kUnits && have < k; ++u) {
        const int at = begin + b * kBatch + u * kRun + tid * 8;
        float x[8];
        tail8<DT>(x_row, at, end, x);
        int n = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) n += at + j < end && key_of(x[j]) == bound;
        // those of the threads before
        int before = n;
        for (int d = 1; d < 64; d *= 2) {
          const int o = __shfl_up(before, d);
          if (lane >= d) before += o;
        }
        if (lane == 63) wave_count[turn][wave] = before;
        __syncthreads();
        int all = 0;
        before -= n;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
          if (w < wave) before += wave_count[turn][w];
          all += wave_count[turn][w];
        }
        turn ^= 1;
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
__global__ __launch_bounds__(kMany) void join_kernel(LogprobsArgs a) {
  constexpr int kThreads = kMany, kWaves = kThreads / 64;
  extern __shared__ uint64_t candidates[];  // [num_parts * top]
  __shared__ uint64_t best[kMostTop];
  __shared__ int count;
  __shared__ uint64_t wave_least[kWaves];
  const int tid = threadIdx.x, row = blockIdx.x;
  const int step = (int)sizeof(Part) + a.top * 8;
  const unsigned char* from = a.parts + (int64_t)row * a.num_parts * step;
  const unsigned char* x_row = static_cast<const unsigned char*>(a.logits) +
                               (int64_t)row * a.row_stride * (DT == kF32 ? 4 : 2);
  float given = 0.0f;
  bool in_vocab = false;
  if (a.tokens) {
    const int64_t t = a.tokens[row];
    in_vocab = t >= 0 && t < a.vocab;
    given = load1<DT>(x_row, in_vocab ? (int)t : 0);
  }
  Sums sums = {kNone, 0.0, 0.0};
  int larger = 0;
  for (int p = 0; p < a.num_parts; ++p) {
    const Part part = *reinterpret_cast<const Part*>(from + (int64_t)p * step);
    sums = join(sums, part.sums);
    larger += (int)part.larger;
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

template <int DT, int kThreads>
hipError_t launch_threads(const LogprobsArgs& args, hipStream_t stream) {
  constexpr int kBatch = kThreads * 8 * kUnits;
  const int batches = std::min(args.part_batches, (args.vocab + kBatch - 1) / kBatch);
  const int keys = args.top ? std::max(batches * kThreads * 4, kMostGroups * 32 * 8) : 0;
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
    logprobs_kernel<DT, kThreads>
        <<<(unsigned)rows * (unsigned)a.num_parts, kThreads, keys, stream>>>(a);
    if (a.num_parts > 1) join_kernel<DT><<<rows, kMany, a.num_parts * a.top * 8, stream>>>(a);
    if (const hipError_t e = hipGetLastError()) return e;
  }
  return hipSuccess;
}
template <int DT>
hipError_t launch(const LogprobsArgs& a, hipStream_t stream) {
  return a.threads == kFew ? launch_threads<DT, kFew>(a, stream) : launch_threads<DT, kMany>(a, stream);
}

}  // namespace

// A workgroup a row, unless that leaves CUs without one: then parts of four batches or more, so many
// that there are four workgroups a CU (one of 16 waves), at most 64.
LogprobsPlan plan_token_logprobs(int rows, int vocab, int cus) {
  const int threads = rows <= cus && vocab > 16384 ? kFew : kMany, batch = threads * 8 * kUnits;
  const int batches = std::max(1, (int)(((int64_t)vocab + batch - 1) / batch));
  const int64_t wanted = (threads == kFew ? 1ll : 4ll) * cus / std::max(rows, 1);
  const int parts = (int)std::min<int64_t>({(batches + 3) / 4, std::max<int64_t>(1, wanted), 64});
  const int per = std::min(kMostKept / threads, (batches + parts - 1) / parts);
  return {threads, per, (batches + per - 1) / per};
}

size_t logprobs_part_bytes(int top) { return sizeof(Part) + (size_t)top * 8; }

hipError_t launch_token_logprobs(const LogprobsArgs& a, int dtype, hipStream_t stream) {
  if (dtype == kBF16) return launch<kBF16>(a, stream);
  if (dtype == kF16) return launch<kF16>(a, stream);
  return launch<kF32>(a, stream);
}

}  // namespace mt
