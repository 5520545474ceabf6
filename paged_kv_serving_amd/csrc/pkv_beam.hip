// Beam search over a paged cache: the best continuations of a group's beams, and the beams' tables and last blocks moved
// to the beams that go on.
#include <float.h>
#include <math.h>

#include <algorithm>
#include <type_traits>

#include "pkv_common.h"

namespace pkv {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / kWave;
constexpr int kMergeThreads = 512;
constexpr int kMergeWaves = kMergeThreads / kWave;
constexpr int kCapacity = 256;  // of a workgroup's list of candidates, PKV_BEAM_MAX_COUNT or more
constexpr int kMaxLists = 4096;  // of a group: beams times chunks

typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
typedef u32x4 u32x4_at4 __attribute__((aligned(4)));  // rows of an odd length start anywhere
typedef u32x4 u32x4_at2 __attribute__((aligned(2)));


// ---------------------------------------------------------------------------------------------
// Selection. A row is cut into chunks, whose numbers a workgroup holds in registers: the logits are read once.
// ---------------------------------------------------------------------------------------------

// Numbers in their order as unsigned ones, 0 below all of them.
__device__ __forceinline__ uint32_t ordered(float x) {
  const uint32_t u = __float_as_uint(x);
  return u ^ (static_cast<uint32_t>(static_cast<int32_t>(u) >> 31) | 0x80000000u);
}
__device__ __forceinline__ float number_of(uint32_t order) {
  return __uint_as_float(order & 0x80000000u ? order ^ 0x80000000u : ~order);
}
__device__ __forceinline__ uint64_t ordered(double x) {
  const uint64_t u = static_cast<uint64_t>(__double_as_longlong(x));
  return u ^ (static_cast<uint64_t>(static_cast<int64_t>(u) >> 63) | (1ull << 63));
}
__device__ __forceinline__ double number_of(uint64_t order) {
  return __longlong_as_double(static_cast<long long>(order >> 63 ? order ^ (1ull << 63) : ~order));
}
// A candidate of a row: falling keys are falling logits, and of equal ones rising tokens. No two of a row are alike; 0 is none.
__device__ __forceinline__ uint64_t key_of(float x, uint32_t token) {
  return static_cast<uint64_t>(ordered(x + 0.f)) << 32 | static_cast<uint32_t>(~token);  // -0 and 0 are one logit
}
__device__ __forceinline__ double logit_of(uint64_t key) { return static_cast<double>(number_of(static_cast<uint32_t>(key >> 32))); }

// The larger of two, NaN where one is.
__device__ __forceinline__ float maximum(float a, float b) { return __builtin_elementwise_maximum(a, b); }

// e^x in double precision for x <= 690, from e^-690 on: 2^k p(x / ln 2 - k), k being the nearest whole number, which adding
// 1.5 * 2^52 leaves in the low bits. p is the interpolation of 2^r at the ten Chebyshev nodes of [-1/2, 1/2], within 2^-45 of it.
// Additions and products alone: conversions and ldexp run at a fraction of their rate. Differences come in, not their terms:
// a product of each with 1 / ln 2 would lose what a difference of large ones keeps.
__device__ __forceinline__ double exp_of(double x) {
  constexpr double kWhole = 6755399441055744.0, kLog2E = 1.4426950408889634;
  x = fmax(x, -690.0);
  const double shifted = __builtin_fma(kLog2E, x, kWhole);
  const double r = __builtin_fma(kLog2E, x, kWhole - shifted);
  double p = 1.0205905413765595e-07;
  p = __builtin_fma(p, r, 1.325964524488711e-06);
  p = __builtin_fma(p, r, 1.5252672924850737e-05);
  p = __builtin_fma(p, r, 0.0001540343375125101);
  p = __builtin_fma(p, r, 0.0013333558200794592);
  p = __builtin_fma(p, r, 0.009618129193934313);
  p = __builtin_fma(p, r, 0.05550410866465167);
  p = __builtin_fma(p, r, 0.2402265069564034);
  p = __builtin_fma(p, r, 0.6931471805599462);
  p = __builtin_fma(p, r, 1.0000000000000135);
  u32x2 bits = __builtin_bit_cast(u32x2, p);
  bits[1] += __builtin_bit_cast(u32x2, shifted)[0] << 20;
  return __builtin_bit_cast(double, bits);
}

// Lanes of the groups that a workgroup of `threads` makes of its wavefronts' lanes: `count` groups or more, none across wavefronts.
__device__ __forceinline__ int group_lanes(int threads, int count) {
  int size = kWave;
  while (threads / size < count) size /= 2;
  return size;
}

// Adjacent lanes, as many as there are for each of `found` candidates, that count the larger ones together.
__device__ __forceinline__ int shares_of(int threads, int found) {
  int shares = 1;
  while (shares < kWave && 2 * shares * found <= threads) shares *= 2;
  return shares;
}

struct Select {
  pkv_beam g;
  int32_t chunks;
  double* sums;     // [rows, chunks] of e^(logit - the chunk's largest)
  float* tops;      // [rows, chunks]
  uint64_t* keys;   // [rows, chunks, count], falling
};

// Whether a row's logits are looked at.
__device__ __forceinline__ bool looked_at(const pkv_beam& g, int64_t row) {
  return fabsf(g.scores[row]) < INFINITY && !(g.finished && g.finished[row]);
}

// A chunk of a row: its largest logit, the sum of exponentials, its `count` best in order. The lanes of all wavefronts that are
// alike modulo a power of two make `count` classes or more, so the smallest of the classes' largest logits is a number that at
// least `count` logits reach, and few more: 8192 of them and 8 classes list about 23. Classes of lanes rather than neighbours:
// a row's last chunk, which has numbers for the first threads alone, leaves no class empty. Each one's place is the number of
// larger ones. Where too many reach it (128 classes: about 700; equal logits), bisection finds a number that fewer do.
// 32 groups of 8 beams over 128256 float32 logits, 131 MB: about 38 us. Bound by the vector units: their instructions, two thirds of
// them the exponentials' 17 operations, take 20 us of issue, 81% of the cycles in which a CU has work, and overlap with the reads, 20 us,
// in part; the kernel takes 21 us without the exponentials. Half the bytes (bf16) take the same time. 7 wavefronts on a SIMD take
// 1.3 us less than the 5 of 88 registers.
template <typename T, int kPer>
__global__ __launch_bounds__(kThreads, 7) void chunk_kernel(const Select a) {
  constexpr int kVec = 16 / sizeof(T), kLoads = kPer / kVec, kAhead = kLoads < 3 ? kLoads : 3;
  __shared__ uint64_t s_list[kWaves][kCapacity];  // a wavefront's own, so that no place needs an atomic
  __shared__ float s_top[kWaves][kWave];
  __shared__ double s_sum[kWaves];
  __shared__ int32_t s_part[kWaves];
  const pkv_beam& g = a.g;
  const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = tid / kWave;
  const int64_t row = blockIdx.x / static_cast<uint32_t>(a.chunks);
  const uint32_t chunk = blockIdx.x % static_cast<uint32_t>(a.chunks);
  if (!looked_at(g, row)) return;
  const uint32_t vocab = static_cast<uint32_t>(g.vocab_size);
  const uint32_t first = chunk * (kThreads * kPer) + tid * kVec;  // this thread's: kVec numbers every kThreads * kVec
  const T* p = static_cast<const T*>(g.logits) + row * g.row_stride;
  using Vec = std::conditional_t<sizeof(T) == 4, u32x4_at4, u32x4_at2>;

  const auto token = [&](int i) { return first + i / kVec * (kThreads * kVec) + i % kVec; };

  // A thread asks for four loads at a time: with all eight, every workgroup's numbers arrive at about the same time, when the
  // vector units have waited long (32 x 8 beams, both kernels: 50 us, with two, four and five loads 46).
  // The exponentials are taken as the numbers arrive, against the largest of the thread's first ones: double precision holds those
  // of numbers 600 above and below it, and where a thread has others it starts again, against its largest.
  float x[kPer], top, base;
  double sum = 0.0;
  const auto add = [&](int i, double from) { sum += exp_of(static_cast<double>(x[i]) - from); };
  const auto take = [&](auto whole) {
    u32x4 v[kLoads];
    const auto ask = [&](int i) {
      if constexpr (whole) v[i] = __builtin_nontemporal_load(reinterpret_cast<const Vec*>(p + token(i * kVec)));
    };
#pragma unroll
    for (int i = 0; i < kAhead; ++i) ask(i);
    if constexpr (!whole) {
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        const T one = p[min(token(i), vocab - 1)];
        if constexpr (sizeof(T) == 4) x[i] = one;
        else x[i] = __uint_as_float(static_cast<uint32_t>(one) << 16);
        if (token(i) >= vocab) x[i] = -INFINITY;
      }
    }
#pragma unroll
    for (int j = 0; j < kLoads; ++j) {
      if (j + kAhead < kLoads) ask(j + kAhead);
      __builtin_amdgcn_sched_barrier(0);
      if constexpr (whole) {
#pragma unroll
        for (int e = 0; e < kVec; ++e) {
          if constexpr (sizeof(T) == 4) x[j * kVec + e] = __uint_as_float(v[j][e]);
          else x[j * kVec + e] = e % 2 == 0 ? bf16_lo(v[j][e / 2]) : bf16_hi(v[j][e / 2]);
        }
      }
#pragma unroll
      for (int i = j * kVec; i < (j + 1) * kVec; ++i) top = i == 0 ? x[0] : maximum(top, x[i]);
      if (j == 0) base = fabsf(top) < INFINITY ? top : 0.f;
      const double from = base;
#pragma unroll
      for (int i = j * kVec; i < (j + 1) * kVec; ++i) add(i, from);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  if ((chunk + 1) * (kThreads * kPer) <= vocab) take(std::true_type{});
  else take(std::false_type{});
  if (fabsf(top) < INFINITY && !(fabsf(top - base) < 600.f)) {
    base = top;
    sum = 0.0;
    const double from = base;
#pragma unroll
    for (int i = 0; i < kPer; ++i) add(i, from);
  }
  // Without a number above -inf (masked, or behind the row's end) a thread adds nothing: its exponentials of -inf are e^-690, and what
  // they would be multiplied by below, e^-(the chunk's largest), may be anything.
  const bool counts = top > -INFINITY;
  int classes = 1;
  while (classes < kWave && classes < g.count) classes *= 2;
  for (int m = kWave / 2; m >= classes; m /= 2) top = maximum(top, __shfl_xor(top, m));
  if (lane < classes) s_top[wave][lane] = top;
  __syncthreads();
  const int c = lane % classes;
  const float even = maximum(s_top[0][c], s_top[2][c]), odd = maximum(s_top[1][c], s_top[3][c]);
  top = maximum(even, odd);
  float reach = g.count > kWave ? fminf(even, odd) : top;
  for (int m = 1; m < classes; m *= 2) {
    top = maximum(top, __shfl_xor(top, m));
    reach = fminf(reach, __shfl_xor(reach, m));
  }
  reach = fmaxf(reach, -FLT_MAX);  // -inf is no candidate
  const int64_t index = row * a.chunks + chunk;
  uint64_t* out = a.keys + index * g.count;
  if (!(fabsf(top) < INFINITY)) {  // nothing, or a row without continuations
    if (tid == 0) a.sums[index] = 0.0, a.tops[index] = top;
    for (int32_t i = tid; i < g.count; i += kThreads) out[i] = 0;
    return;
  }

  // Of others `base` is their first largest, no more than `top`, or 0 and within 600 of their own: exp_of's range.
  sum = counts ? sum * exp_of(static_cast<double>(base) - static_cast<double>(top)) : 0.0;
  for (int m = kWave / 2; m > 0; m >>= 1) sum += __shfl_xor(sum, m);
  if (lane == 0) s_sum[wave] = sum;

  // Lists the numbers that a condition holds for; how many there are.
  const auto list = [&](auto holds) {
    int32_t n = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const bool one = holds(i);
      const uint64_t those = __ballot(one);
      if (those == 0) continue;
      const int32_t place = n + __builtin_amdgcn_mbcnt_hi(static_cast<uint32_t>(those >> 32), __builtin_amdgcn_mbcnt_lo(static_cast<uint32_t>(those), 0));
      if (one && place < kCapacity) s_list[wave][place] = key_of(x[i], token(i));
      n += __popcll(those);
    }
    if (lane == 0) s_part[wave] = n;
    __syncthreads();
    n = 0;
    for (int w = 0; w < kWaves; ++w) n += s_part[w];
    return n;
  };
  int32_t found = list([&](int i) { return x[i] >= reach; });
  if (tid == 0) {
    sum = 0.0;
    for (int w = 0; w < kWaves; ++w) sum += s_sum[w];
    a.sums[index] = sum;
    a.tops[index] = top;
  }
  if (found > kCapacity) {
    // How many of the chunk's numbers a condition holds for.
    const auto number = [&](auto holds) {
      int32_t n = 0;
#pragma unroll
      for (int i = 0; i < kPer; ++i) n += __popcll(__ballot(holds(i)));
      __syncthreads();
      if (lane == 0) s_part[wave] = n;
      __syncthreads();
      n = 0;
      for (int w = 0; w < kWaves; ++w) n += s_part[w];
      return n;
    };
    // More than the capacity reach `low`, fewer than `count` reach `high`.
    uint32_t low = ordered(reach), high = ordered(top) + 1;
    bool fits = false;
    while (high - low > 1) {
      const uint32_t middle = low + (high - low) / 2;
      const float at = number_of(middle);
      const int32_t n = number([&](int i) { return x[i] >= at; });
      fits = n >= g.count && n <= kCapacity;
      if (fits || n > kCapacity) low = middle;
      else high = middle;
      if (fits) break;
    }
    reach = number_of(low);
    // All that reach it, or all above it and of the equal ones the first tokens.
    uint32_t last = ~0u;
    if (!fits) {
      const int32_t rest = g.count - number([&](int i) { return x[i] > reach; });
      uint32_t under = chunk * (kThreads * kPer);  // `last` is enough, `under - 1` is not
      last = under + kThreads * kPer - 1;
      while (under < last) {
        const uint32_t middle = under + (last - under) / 2;
        if (number([&](int i) { return x[i] == reach && token(i) <= middle; }) >= rest) last = middle;
        else under = middle + 1;
      }
    }
    __syncthreads();
    found = list([&](int i) { return x[i] > reach || (x[i] == reach && token(i) <= last); });
  }
  if (tid < found) {
    int32_t of = 0, at = tid, place = 0;
    while (at >= s_part[of]) at -= s_part[of++];
    const uint64_t key = s_list[of][at];
    for (int w = 0; w < kWaves; ++w) {
      const int32_t n = s_part[w];
#pragma unroll 4
      for (int32_t j = 0; j < n; ++j) place += s_list[w][j] > key ? 1 : 0;
    }
    if (place < g.count) out[place] = key;
  }
  for (int32_t i = found + tid; i < g.count; i += kThreads) out[i] = 0;
}

// A group: the logarithms of its rows' sums, then the chunks' candidates by score, in the same way. The candidates are numbered
// through the lists' first ones, then their second ones and so on, and dealt out to the groups of lanes one by one, so that every
// group has some of the best. Bound by latency: 32 groups of 8 beams and 16 chunks take 8 us, 4.5 us of which are the launch and
// the reads; 1 group of 64 beams for 128 continuations 30 us.
__global__ __launch_bounds__(kMergeThreads) void merge_kernel(const Select a) {
  constexpr int kHeld = 4;  // candidates of a thread in registers, which give a number that `count` of them reach
  __shared__ double s_top_logit[PKV_BEAM_MAX], s_log[PKV_BEAM_MAX], s_score[PKV_BEAM_MAX];
  __shared__ uint8_t s_kind[PKV_BEAM_MAX];  // 0: no continuation, 1: its row's, 2: the end token
  __shared__ double s_scores[kCapacity];
  __shared__ uint64_t s_keys[kCapacity];
  __shared__ uint8_t s_beams[kCapacity];
  __shared__ double s_top[kMergeWaves], s_reach[kMergeWaves];
  __shared__ int32_t s_count, s_part[kMergeWaves];
  const pkv_beam& g = a.g;
  const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = tid / kWave;
  const int64_t group = blockIdx.x, row0 = group * g.num_beams;
  const uint32_t lists = static_cast<uint32_t>(g.num_beams) * a.chunks, total = lists * g.count;
  const uint64_t* keys = a.keys + row0 * a.chunks * g.count;
  const auto key_at = [&](uint32_t i) { return keys[static_cast<int64_t>(i % lists) * g.count + i / lists]; };

  const int size = group_lanes(kMergeThreads, g.count);
  const uint32_t groups = kMergeThreads / size, mine = tid / size + groups * (tid % size);  // and every kMergeThreads further on

  uint64_t held[kHeld];  // what a row that is not looked at has here is not used
#pragma unroll
  for (int j = 0; j < kHeld; ++j) {
    const uint32_t i = mine + j * kMergeThreads;
    held[j] = i < total ? key_at(i) : 0;
  }
  for (int32_t b = wave; b < g.num_beams; b += kMergeWaves) {
    const int64_t row = row0 + b;
    const float* tops = a.tops + row * a.chunks;
    const double* sums = a.sums + row * a.chunks;
    const float score = g.scores[row];
    const bool finished = g.finished && g.finished[row];
    const float top0 = lane < a.chunks ? tops[lane] : -INFINITY;
    const double sum0 = lane < a.chunks ? sums[lane] : 0.0;
    float top = top0;
    for (int32_t c = lane + kWave; c < a.chunks; c += kWave) top = maximum(top, tops[c]);
    for (int m = kWave / 2; m > 0; m >>= 1) top = maximum(top, __shfl_xor(top, m));
    double sum = 0.0;
    const auto add = [&](float one, double part) {
      if (part != 0.0) sum += part * exp_of(static_cast<double>(one) - static_cast<double>(top));
    };
    add(top0, sum0);
    for (int32_t c = lane + kWave; c < a.chunks; c += kWave) add(tops[c], sums[c]);
    for (int m = kWave / 2; m > 0; m >>= 1) sum += __shfl_xor(sum, m);
    if (lane == 0) {
      const bool usable = fabsf(score) < INFINITY, counts = usable && !finished && fabsf(top) < INFINITY;
      s_top_logit[b] = top;
      s_log[b] = counts ? log(sum) : 0.0;
      s_score[b] = score;
      s_kind[b] = counts ? 1 : usable && finished ? 2 : 0;
    }
  }
  if (tid == 0) s_count = 0;
  __syncthreads();

  const auto beam_of = [&](uint32_t i) { return i % lists / a.chunks; };
  // The score of candidate i, -inf if it is none; of a beam that has ended, its first one is the end token.
  const auto score_of = [&](uint32_t i, uint64_t key) {
    const uint32_t b = beam_of(i);
    const int32_t kind = s_kind[b];
    if (kind == 2) return i == b * a.chunks ? s_score[b] : -INFINITY;
    return kind == 1 && key != 0 ? s_score[b] + ((logit_of(key) - s_top_logit[b]) - s_log[b]) : -INFINITY;
  };
  double scores[kHeld];
#pragma unroll
  for (int j = 0; j < kHeld; ++j) {
    const uint32_t i = mine + j * kMergeThreads;
    scores[j] = i < total ? score_of(i, held[j]) : -INFINITY;
  }
  double top = -INFINITY;
#pragma unroll
  for (int j = 0; j < kHeld; ++j) top = fmax(top, scores[j]);
  for (int m = 1; m < size; m *= 2) top = fmax(top, __shfl_xor(top, m));
  double reach = top;
  for (int m = size; m < kWave; m *= 2) {
    top = fmax(top, __shfl_xor(top, m));
    reach = fmin(reach, __shfl_xor(reach, m));
  }
  if (lane == 0) s_top[wave] = top, s_reach[wave] = reach;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kMergeWaves; ++w) top = fmax(top, s_top[w]), reach = fmin(reach, s_reach[w]);

  // Bisection over the held candidates, where many reach it (one beam far above the others, or alone): `count` of them or
  // little more, as candidates that are not held will reach it too.
  const auto held_ones = [&](double at) {
    int32_t n = 0;
#pragma unroll
    for (int j = 0; j < kHeld; ++j) n += __popcll(__ballot(scores[j] > -INFINITY && scores[j] >= at));
    __syncthreads();
    if (lane == 0) s_part[wave] = n;
    __syncthreads();
    n = 0;
#pragma unroll
    for (int w = 0; w < kMergeWaves; ++w) n += s_part[w];
    return n;
  };
  const int32_t enough = total <= kHeld * kMergeThreads ? kCapacity : g.count + g.count / 2 + 8;
  if (held_ones(reach) > enough) {
    uint64_t low = ordered(reach), high = ordered(top) + 1;
    while (high - low > 1) {
      const uint64_t middle = low + (high - low) / 2;
      const int32_t n = held_ones(number_of(middle));
      if (n >= g.count) low = middle;
      else high = middle;
      if (n >= g.count && n <= enough) break;
    }
    reach = number_of(low);
  }

  // f(beam, key, score) for the candidates that reach it: the held ones, and of what is left of each list the first ones.
  const double least_score = reach;
  const auto each = [&](auto f) {
#pragma unroll
    for (int j = 0; j < kHeld; ++j) {
      if (scores[j] > -INFINITY && scores[j] >= least_score) f(beam_of(mine + j * kMergeThreads), held[j], scores[j]);
    }
    if (total <= kHeld * kMergeThreads) return;
    for (uint32_t l = tid; l < lists; l += kMergeThreads) {
      const uint32_t before = l < kHeld * kMergeThreads ? (kHeld * kMergeThreads - l + lists - 1) / lists : 0;
      for (uint32_t i = l + before * lists; i < total; i += lists) {
        const uint64_t key = key_at(i);
        const double score = score_of(i, key);
        if (!(score > -INFINITY && score >= least_score)) break;
        f(beam_of(i), key, score);
      }
    }
  };
  const auto list = [&](uint32_t b, uint64_t key, double score) {
    const int32_t place = atomicAdd(&s_count, 1);
    if (place < kCapacity) s_scores[place] = score, s_keys[place] = key, s_beams[place] = static_cast<uint8_t>(b);
  };
  each(list);
  __syncthreads();
  int32_t found = s_count;
  if (found > kCapacity) {
    const auto number = [&](auto holds) {
      int32_t n = 0;
      each([&](uint32_t b, uint64_t key, double score) { n += holds(b, key, score) ? 1 : 0; });
      for (int m = kWave / 2; m > 0; m >>= 1) n += __shfl_xor(n, m);
      __syncthreads();
      if (lane == 0) s_part[wave] = n;
      __syncthreads();
      n = 0;
      for (int w = 0; w < kMergeWaves; ++w) n += s_part[w];
      return n;
    };
    // More than the capacity reach `low`, fewer than `count` reach `high`.
    uint64_t low = ordered(reach), high = ordered(top) + 1;
    bool fits = false;
    while (high - low > 1) {
      const uint64_t middle = low + (high - low) / 2;
      const double at = number_of(middle);
      const int32_t n = number([&](uint32_t, uint64_t, double score) { return score >= at; });
      fits = n >= g.count && n <= kCapacity;
      if (fits || n > kCapacity) low = middle;
      else high = middle;
      if (fits) break;
    }
    reach = number_of(low);
    // All that reach it, or all above it and of the equal ones the first beams', of the last of those the largest keys.
    uint32_t last = PKV_BEAM_MAX;
    uint64_t least = 0;
    if (!fits) {
      const int32_t rest = g.count - number([&](uint32_t, uint64_t, double score) { return score > reach; });
      uint32_t under = 0;
      last = g.num_beams - 1;
      while (under < last) {
        const uint32_t middle = under + (last - under) / 2;
        if (number([&](uint32_t b, uint64_t, double score) { return score == reach && b <= middle; }) >= rest) last = middle;
        else under = middle + 1;
      }
      const int32_t own = rest - number([&](uint32_t b, uint64_t, double score) { return score == reach && b < last; });
      uint64_t over = ~0ull;  // `least` is low enough, `over + 1` is not
      while (least < over) {
        const uint64_t middle = over - (over - least) / 2;
        const auto holds = [&](uint32_t b, uint64_t key, double score) { return score == reach && b == last && key >= middle; };
        if (number(holds) >= own) least = middle;
        else over = middle - 1;
      }
    }
    __syncthreads();
    if (tid == 0) s_count = 0;
    __syncthreads();
    each([&](uint32_t b, uint64_t key, double score) {
      if (score > reach || (score == reach && (b < last || (b == last && key >= least)))) list(b, key, score);
    });
    __syncthreads();
    found = min(s_count, kCapacity);
  }
  // Places. Of equal scores the lower beam's is first, in a beam the larger key.
  const int64_t out = group * g.count;
  const int shares = shares_of(kMergeThreads, found), own = tid / shares;
  if (own < found) {
    const double score = s_scores[own];
    const uint64_t key = s_keys[own];
    const int32_t b = s_beams[own];
    int32_t place = 0, equal = 0;
#pragma unroll 4
    for (int32_t j = tid % shares; j < found; j += shares) {
      const double other = s_scores[j];
      place += other > score ? 1 : 0;
      equal += other == score ? 1 : 0;
    }
    for (int m = 1; m < shares; m *= 2) equal += __shfl_xor(equal, m);
    if (equal > 1) {  // as bfloat16 logits often are
#pragma unroll 4
      for (int32_t j = tid % shares; j < found; j += shares) {
        const int32_t beam = s_beams[j];
        const bool larger = s_keys[j] > key;
        place += (s_scores[j] == score) & ((beam < b) | ((beam == b) & larger)) ? 1 : 0;
      }
    }
    for (int m = 1; m < shares; m *= 2) place += __shfl_xor(place, m);
    if (tid % shares == 0 && place < g.count) {
      g.best_scores[out + place] = static_cast<float>(score);
      g.best_beams[out + place] = b;
      g.best_tokens[out + place] = s_kind[b] == 2 ? g.end_token : static_cast<int32_t>(~static_cast<uint32_t>(key));
    }
  }
  for (int32_t i = found + tid; i < g.count; i += kMergeThreads) {
    g.best_scores[out + i] = -INFINITY;
    g.best_beams[out + i] = 0;
    g.best_tokens[out + i] = g.end_token;
  }
}

// ---------------------------------------------------------------------------------------------
// Reordering. One workgroup for a child and a layer, of every state; a child that takes its parent's block over has nothing to
// copy. Every workgroup finds its group's moves by itself: the parents that earlier children named are a word of bits.
// Bound: HBM for large blocks, latency for small ones. 32 groups of 8 beams, 32 layers of 16 KB blocks and their scales, 252 MB read and
// written: 53 us, 4.8 TB/s.
// ---------------------------------------------------------------------------------------------
constexpr int kTogether = 4;  // units that a thread loads before it stores them
struct Reorder {
  pkv_reorder g;
  int32_t unit[PKV_BEAM_STATES];  // bytes that are moved together: 16, 4 or 1
  // Whether every state's block is one batch of a wavefront. The wavefronts then have a state each, and the states' latencies run
  // at the same time: 18 groups of 16 beams, 22 layers, 1 KB each of keys and values with their scales, 20 us, together 28.
  bool apart;
};

template <typename U, int kThreadsOf>
__device__ __forceinline__ void copy_units(void* to, const void* from, int64_t count, int first) {
  for (int64_t i = first; i < count; i += kThreadsOf * kTogether) {
    U x[kTogether];
#pragma unroll
    for (int j = 0; j < kTogether; ++j) {
      if (i + j * kThreadsOf < count) x[j] = static_cast<const U*>(from)[i + j * kThreadsOf];
    }
#pragma unroll
    for (int j = 0; j < kTogether; ++j) {
      if (i + j * kThreadsOf < count) static_cast<U*>(to)[i + j * kThreadsOf] = x[j];
    }
  }
}

__global__ __launch_bounds__(kThreads) void reorder_kernel(const Reorder a) {
  const pkv_reorder& g = a.g;
  const int tid = threadIdx.x, lane = tid & (kWave - 1);
  const int32_t beams = g.num_beams, child = static_cast<int32_t>(blockIdx.x % static_cast<uint32_t>(beams));
  const int64_t group = blockIdx.x / static_cast<uint32_t>(beams), row0 = group * beams;
  const int32_t layer = blockIdx.y;
  int32_t named = lane < beams ? g.parents[row0 + lane] : 0;
  if (named < 0 || named >= beams) named = lane;
  const int32_t context = min(static_cast<int64_t>(max(g.context_lens[group], 0)), static_cast<int64_t>(g.table_stride) * g.block_size);
  const int32_t full = context / g.block_size;
  const bool part = context % g.block_size != 0;
  uint64_t seen = 0, further = 0;  // parents that have a child, and children that are not their parent's first
  for (int32_t c = 0; c < beams; ++c) {
    const int32_t p = __builtin_amdgcn_readlane(named, c);
    further |= ((seen >> p) & 1) << c;
    seen |= 1ull << p;
  }
  const int32_t parent = __builtin_amdgcn_readlane(named, child);
  int32_t keeper = parent;  // the row whose last block this child has from now on
  if ((further >> child) & 1) {
    uint64_t idle = ~seen;  // rows without a child: as many as further children
    for (int n = __popcll(further & ((1ull << child) - 1)); n > 0; --n) idle &= idle - 1;
    keeper = __builtin_ctzll(idle);
  }
  const int32_t* tables = g.block_tables + row0 * g.table_stride;
  if (layer == 0) {
    int32_t* out = g.new_tables + (row0 + child) * g.table_stride;
    for (int32_t j = tid; j < g.table_stride; j += kThreads) {
      const int32_t from = j < full ? parent : j == full && part ? keeper : child;
      out[j] = tables[static_cast<int64_t>(from) * g.table_stride + j];
    }
  }
  if (!part || keeper == parent) return;
  const int32_t source = tables[static_cast<int64_t>(parent) * g.table_stride + full];
  const int32_t target = tables[static_cast<int64_t>(keeper) * g.table_stride + full];
  if (source < 0 || source >= g.num_blocks || target < 0 || target >= g.num_blocks || source == target) return;
  const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  for (int32_t s = a.apart ? wave : 0; s < g.num_states; s += a.apart ? kWaves : 1) {
    if (layer >= g.num_layers[s]) continue;
    char* base = static_cast<char*>(g.states[s]) + layer * g.layer_bytes[s];
    const int64_t bytes = g.block_bytes[s];
    char* to = base + target * bytes;
    const char* from = base + source * bytes;
    if (a.apart) {
      if (a.unit[s] == 16) copy_units<u32x4, kWave>(to, from, bytes / 16, lane);
      else if (a.unit[s] == 4) copy_units<uint32_t, kWave>(to, from, bytes / 4, lane);
      else copy_units<uint8_t, kWave>(to, from, bytes, lane);
    } else {
      if (a.unit[s] == 16) copy_units<u32x4, kThreads>(to, from, bytes / 16, tid);
      else if (a.unit[s] == 4) copy_units<uint32_t, kThreads>(to, from, bytes / 4, tid);
      else copy_units<uint8_t, kThreads>(to, from, bytes, tid);
    }
  }
}

// Numbers of a chunk per thread, 0 where no cut serves: a few rows are cut finer, so that they fill the GPU.
int per_thread(int64_t num_groups, int32_t num_beams, int64_t vocab_size) {
  if (num_groups < 0 || num_beams < 1 || num_beams > PKV_BEAM_MAX || vocab_size < 1 || vocab_size > (int64_t{1} << 25)) return 0;
  if (num_groups > (1 << 20) || num_groups * num_beams > (1 << 20)) return 0;
  const auto chunks = [&](int per) { return (vocab_size + kThreads * per - 1) / (kThreads * per); };
  if (num_groups * num_beams * chunks(32) < 512 && num_beams * chunks(8) <= kMaxLists) return 8;
  return num_beams * chunks(32) <= kMaxLists ? 32 : 0;
}

template <typename T>
int select(Select a, int per, hipStream_t stream) {
  const int64_t rows = a.g.num_groups * a.g.num_beams;
  const dim3 chunks(static_cast<uint32_t>(rows * a.chunks)), block(kThreads);
  if (per == 8) {
    hipLaunchKernelGGL((chunk_kernel<T, 8>), chunks, block, 0, stream, a);
  } else {
    hipLaunchKernelGGL((chunk_kernel<T, 32>), chunks, block, 0, stream, a);
  }
  hipLaunchKernelGGL(merge_kernel, dim3(static_cast<uint32_t>(a.g.num_groups)), dim3(kMergeThreads), 0, stream, a);
  return check_launch();
}

}  // namespace
}  // namespace pkv

extern "C" int64_t pkv_beam_workspace_bytes(int64_t num_groups, int32_t num_beams, int64_t vocab_size, int32_t count) {
  const int per = pkv::per_thread(num_groups, num_beams, vocab_size);
  if (per == 0 || count < 1 || count > PKV_BEAM_MAX_COUNT) return PKV_EINVAL;
  const int64_t chunks = (vocab_size + pkv::kThreads * per - 1) / (pkv::kThreads * per);
  return (num_groups * num_beams * chunks * (8 + 4 + 8 * static_cast<int64_t>(count)) + 15) / 16 * 16;
}

extern "C" int pkv_beam_select(const pkv_beam* args, int device, void* stream) {
  using namespace pkv;
  if (!args) return PKV_EINVAL;
  const pkv_beam& g = *args;
  if (g.num_groups < 0 || g.num_beams < 1 || g.vocab_size < 1 || g.count < 1) return PKV_EINVAL;
  if (g.dtype != PKV_F32 && g.dtype != PKV_BF16) return PKV_EINVAL;
  if (g.num_beams > PKV_BEAM_MAX || g.count > PKV_BEAM_MAX_COUNT) return PKV_EUNSUPPORTED;
  const int per = per_thread(g.num_groups, g.num_beams, g.vocab_size);
  if (per == 0) return PKV_EUNSUPPORTED;
  if (g.count > g.num_beams * g.vocab_size) return PKV_EINVAL;
  if (g.row_stride < g.vocab_size) return PKV_EINVAL;
  const int64_t rows = g.num_groups * g.num_beams, chunks = (g.vocab_size + kThreads * per - 1) / (kThreads * per);
  if (rows * chunks > 0x7fffffff / kThreads) return PKV_EUNSUPPORTED;
  if (g.num_groups == 0) return PKV_OK;
  if (!g.best_scores || !g.best_beams || !g.best_tokens || !g.logits || !g.scores) return PKV_EINVAL;
  // A group's scores are read before its own best ones are written, but other groups' may not be.
  const bool in_place = g.best_scores == g.scores && g.count == g.num_beams;
  if (!in_place && g.best_scores < g.scores + rows && g.scores < g.best_scores + g.num_groups * g.count) return PKV_EINVAL;
  const int64_t need = pkv_beam_workspace_bytes(g.num_groups, g.num_beams, g.vocab_size, g.count);
  if (!g.workspace || !aligned16(g.workspace) || g.workspace_bytes < need) return PKV_EINVAL;
  Select a{};
  a.g = g;
  a.chunks = static_cast<int32_t>(chunks);
  a.keys = static_cast<uint64_t*>(g.workspace);
  a.sums = reinterpret_cast<double*>(a.keys + rows * chunks * g.count);
  a.tops = reinterpret_cast<float*>(a.sums + rows * chunks);
  DeviceGuard guard(device);
  if (!guard.ok()) return PKV_EHIP;
  const auto s = static_cast<hipStream_t>(stream);
  return g.dtype == PKV_F32 ? select<float>(a, per, s) : select<uint16_t>(a, per, s);
}

extern "C" int pkv_beam_reorder(const pkv_reorder* args, int device, void* stream) {
  using namespace pkv;
  if (!args) return PKV_EINVAL;
  const pkv_reorder& g = *args;
  if (g.num_groups < 0 || g.num_blocks < 0 || g.num_beams < 1 || g.table_stride < 0 || g.block_size < 1 || g.num_states < 0) return PKV_EINVAL;
  if (g.num_beams > PKV_BEAM_MAX || g.num_states > PKV_BEAM_STATES) return PKV_EUNSUPPORTED;
  if (static_cast<int64_t>(g.table_stride) * g.block_size > 0x7fffffff) return PKV_EUNSUPPORTED;
  Reorder a{};
  a.g = g;
  a.apart = true;
  int32_t layers = 1;
  for (int s = 0; s < g.num_states; ++s) {
    if (g.num_layers[s] < 0 || g.block_bytes[s] < 0 || g.layer_bytes[s] < 0) return PKV_EINVAL;
    if (g.num_layers[s] > 0 && g.block_bytes[s] > 0 && g.num_blocks > 0 && !g.states[s]) return PKV_EINVAL;
    if (g.num_layers[s] > 65535) return PKV_EUNSUPPORTED;
    layers = std::max(layers, g.num_layers[s]);
    const uint64_t bits = reinterpret_cast<uintptr_t>(g.states[s]) | static_cast<uint64_t>(g.block_bytes[s]) | static_cast<uint64_t>(g.layer_bytes[s]);
    a.unit[s] = bits % 16 == 0 ? 16 : bits % 4 == 0 ? 4 : 1;
    a.apart = a.apart && g.block_bytes[s] / a.unit[s] <= kWave * kTogether;
  }
  if (g.num_groups > 0x7fffffff / (kThreads * PKV_BEAM_MAX)) return PKV_EUNSUPPORTED;
  if (g.num_groups == 0) return PKV_OK;
  if (!g.parents || !g.context_lens || (g.table_stride > 0 && (!g.new_tables || !g.block_tables))) return PKV_EINVAL;
  // Rows are read while others are written.
  const int64_t entries = g.num_groups * g.num_beams * g.table_stride;
  if (entries > 0 && g.new_tables < g.block_tables + entries && g.block_tables < g.new_tables + entries) return PKV_EINVAL;
  DeviceGuard guard(device);
  if (!guard.ok()) return PKV_EHIP;
  hipLaunchKernelGGL(reorder_kernel, dim3(static_cast<uint32_t>(g.num_groups * g.num_beams), static_cast<uint32_t>(layers)), dim3(kThreads), 0,
                     static_cast<hipStream_t>(stream), a);
  return check_launch();
}
