// Sampling from logits rows with temperature, top-k, min-p and top-p, from given uniform numbers.
//
// The four settings are all cuts of one order, the tokens by falling logit (equal ones by id): every
// kept set is a beginning of it, and the draw is a place in it. With exact sums of fixed-point weights
//     W[i] = round(2^46 exp((logit[i] - max) / T))
// each step is the same question, "which token is the first whose cumulative mass (or count) reaches
// X?": X = top_k in counts gives the mass M of the first cut; X = ceil(top_p * M) gives the kept mass
// S; X = floor(uniform * S) + 1 gives the token. A row is never sorted as a whole:
//   - Where top-k or min-p leave at most kFew tokens, those are listed and put in order in LDS.
//   - Otherwise a histogram of the masses over bins of 1/128 octave finds the bin that holds the answer,
//     and only that bin's tokens are compared with each other.
// Integer sums make the result independent of the order of the atomics.
//
// One workgroup of 1024 threads per row, so that nothing is joined outside LDS: a pass for the largest
// logit, then a pass for the list, or one for the histogram and one or two for the bins. Bound: at 256 rows of
// 128256, 131 MB a pass, the passes' reads (5.9 TB/s of caches) and, in the histogram, the issue of some 24
// vector instructions per token (23 us for a row by itself; reading all rows once takes 22): 44 us with top-k, 70 plain
// and with top-p. At few rows the workgroup's own latencies: 1 row of 32000 with top-p 17.2 us (the largest 2.7,
// histogram 6, sums 1.3, bins and tokens 5.5, a launch 1.7), 64 rows of 50257 with top-k 50 and top-p 12.6 us.
// Keeping a thread's first 16 to 64 values in registers for the later passes made 256 rows 3 to 8% faster and
// short rows 7 to 60% slower (longer code, fetched anew by every launch): not kept.
#include <math.h>

#include "pkv_common.h"

namespace pkv {
namespace {

constexpr int kThreads = 1024;
constexpr int kWaves = kThreads / kWave;
constexpr int kPerOctave = 128;                    // bins, and entries of the table of powers
constexpr int kBins = 48 * kPerOctave;             // 2^-47.5 * 2^46 < 1/2: later bins weigh nothing
constexpr int kBinsPerThread = kBins / kThreads;
constexpr int kList = 1024;                        // tokens of one bin that are compared with each other
constexpr int kFew = 512;                          // tokens that are put in order instead of counted in bins
constexpr int kCrowded = 960;                      // threads (of kThreads) that meet a token that the cuts may keep
constexpr int kKept = 4096;                        // tokens that are kept in LDS instead of read again

typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));

struct Args {
  int32_t* out;
  const void* logits;
  int64_t row_stride;
  int32_t vocab;
  const float* uniforms;
  const float* temperatures;
  const int32_t* top_ks;
  const float* top_ps;
  const float* min_ps;
  float temperature, top_p, min_p;
  int32_t top_k;
  double one;  // 2^(fractional bits)
};

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(uint16_t x) { return __uint_as_float(static_cast<uint32_t>(x) << 16); }

// Unsigned integers in the order of the floats; both zeros are one.
__device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t bits = __float_as_uint(x + 0.f);
  return bits ^ ((bits >> 31) ? 0xffffffffu : 0x80000000u);
}

__device__ __forceinline__ float float_of(uint32_t key) {
  return __uint_as_float(key ^ ((key >> 31) ? 0x80000000u : 0xffffffffu));
}

// f(value, index) for every element of a row with test(value), each by some thread of the workgroup: the
// 16-byte aligned body in vectors, kLoads of them in flight per thread, what lies before and after it one
// element per thread. Where tests are seldom true, a vector's are made together before any branch (a pass
// for the tokens of some bins over 1 row of 128256: 12.6 -> 7.2 us).
template <int kLoads, typename T, typename P, typename F>
__device__ __forceinline__ void for_each_if(const T* x, int32_t n, P test, F f) {
  constexpr int kVec = 16 / sizeof(T);
  const int32_t before = static_cast<int32_t>(((16 - (reinterpret_cast<uintptr_t>(x) & 15)) & 15) / sizeof(T));
  const int32_t head = before < n ? before : n;
  const u32x4* body = reinterpret_cast<const u32x4*>(x + head);
  const int32_t vectors = (n - head) / kVec;
  auto use = [&](const u32x4& raw, int32_t i) {
    float v[kVec];
    bool any = false;
#pragma unroll
    for (int e = 0; e < kVec; ++e) {
      v[e] = sizeof(T) == 4 ? __uint_as_float(raw[e * 4 / kVec]) : e % 2 == 0 ? bf16_lo(raw[e * 4 / kVec]) : bf16_hi(raw[e * 4 / kVec]);
      any |= test(v[e]);
    }
    if (!any) return;
#pragma unroll
    for (int e = 0; e < kVec; ++e) {
      if (test(v[e])) f(v[e], i + e);
    }
  };
  int32_t q = threadIdx.x;
  for (; q + (kLoads - 1) * kThreads < vectors; q += kLoads * kThreads) {
    u32x4 raw[kLoads];
#pragma unroll
    for (int u = 0; u < kLoads; ++u) raw[u] = body[q + u * kThreads];
#pragma unroll
    for (int u = 0; u < kLoads; ++u) use(raw[u], head + (q + u * kThreads) * kVec);
  }
  for (; q < vectors; q += kThreads) use(body[q], head + q * kVec);
  const int32_t tail = head + vectors * kVec;
  const int32_t t = threadIdx.x;
  if (t < head + (n - tail)) {
    const int32_t i = t < head ? t : tail + (t - head);
    if (test(to_float(x[i]))) f(to_float(x[i]), i);
  }
}

template <int kLoads, typename T, typename F>
__device__ __forceinline__ void for_each(const T* x, int32_t n, F f) {
  for_each_if<kLoads>(x, n, [](float) { return true; }, f);
}

// Where a row's tokens come from: the row, or (kept >= 0) the tokens kept in LDS.
template <typename T>
struct Source {
  const T* x;
  int32_t vocab;
  const uint64_t* list;
  int32_t kept;

  template <int kLoads, typename P, typename F>
  __device__ __forceinline__ void each_if(P test, F f) const {
    if (kept < 0) {
      for_each_if<kLoads>(x, vocab, test, f);
      return;
    }
#pragma unroll 1
    for (int32_t i = threadIdx.x; i < kept; i += kThreads) {
      const uint64_t token = list[i];
      const float v = float_of(static_cast<uint32_t>(token >> 32));
      if (test(v)) f(v, static_cast<int32_t>(0xffffffffu - static_cast<uint32_t>(token)));
    }
  }
};

struct Shared {
  __align__(16) uint64_t kept[kKept];       // tokens as order_of gives them: all that the cuts can keep
  uint64_t mass[kBins + 2];   // exclusive sums over the bins before, once summed up
  uint32_t count[kBins + 2];
  __align__(16) uint64_t list[kList];       // and those that are compared with each other
  __align__(16) uint64_t list_mass[kList];
  uint64_t before[kList];     // of each token of the list: the mass, and the number, that come before it
  uint32_t rank[kList];
  double power[kPerOctave];   // 2^(j / kPerOctave) * 2^(fractional bits)
  __align__(16) uint64_t sum[kWaves];
  __align__(16) float tops[kWaves];
  __align__(16) uint32_t waves[kWaves];
  uint64_t found_mass;
  uint32_t listed;
  int32_t found;
};

// What the weights of one row go by. Its largest logit is finite here.
struct Row {
  float top;
  double rate;      // bins per unit of logit: kPerOctave * log2(e) / T
  double step;      // and units of logit per bin, for the bins' bounds
  double least;     // min_p * 2^(fractional bits)
  const double* power;
  double series[4];  // of 2^(f / kPerOctave) - 1 in f, kept in registers
};

// a * b + c, not in place: the coefficients stay where they are.
__device__ __forceinline__ double fma_apart(double a, double b, double c) {
  double d;
  asm("v_fma_f64 %0, %1, %2, %3" : "=v"(d) : "v"(a), "v"(b), "v"(c));
  return d;
}

struct Weight {
  int32_t bin;
  uint64_t mass;
};

__device__ __forceinline__ uint64_t* mass_of_bin(uint64_t* masses, int32_t bin) {  // an index in one instruction
  return reinterpret_cast<uint64_t*>(reinterpret_cast<char*>(masses) + __mul24(-bin, -8));
}

// The bin and weight of a finite logit; what lies below the bins weighs 0. Its depth z below the top in bins is
// n + f with a whole number n <= 0 and |f| <= 1/2, and its weight is
//     2^(z / 128) = 2^(n >> 7) * power[n & 127] * 2^(f / 128),
// the last factor by its series (the first term left out is below 2^-49) and the first added to the
// exponent. Each step to n rounds monotonically: bins fall with the logit. Adding 2^52 * 1.5 or 2^52 leaves
// a number rounded to a whole one in the low bits.
template <bool kMin>
__device__ __forceinline__ Weight weigh(const Row& r, float x) {
  const double z = fmax((static_cast<double>(x) - static_cast<double>(r.top)) * r.rate, -(kBins + 1.0));
  const double whole = z + 0x1.8p52;
  const int32_t n = __double2loint(whole);
  const double f = z - (whole - 0x1.8p52);
  const double series = fma_apart(f, fma_apart(f, fma_apart(f, r.series[3], r.series[2]), r.series[1]), r.series[0]);
  const double base = r.power[n & (kPerOctave - 1)];
  const double close = base + base * f * series;
  const double w = __builtin_ldexp(close, n >> 7);
  const double in_place = w + 0x1p52;
  uint64_t mass = (static_cast<uint64_t>(__double2hiint(in_place) & 0xfffff) << 32) | static_cast<uint32_t>(__double2loint(in_place));
  if constexpr (kMin) mass = w >= r.least ? mass : 0;
  return {-n, mass};
}

// A logit that lies no higher than any of bin `bin`'s: what is below it need not be looked at. The
// margin covers the rounding of the product and of the difference to float32.
__device__ __forceinline__ float floor_of_bin(const Row& r, int32_t bin) {
  const double x = static_cast<double>(r.top) - (bin + 0.5) * r.step;
  const double low = x - (fabs(x) + fabs(static_cast<double>(r.top))) * 0x1p-22;
  return low >= -3.4028234663852886e38 ? static_cast<float>(low) : -3.4028234663852886e38f;
}
__device__ __forceinline__ float ceiling_of_bin(const Row& r, int32_t bin) {
  const double x = static_cast<double>(r.top) - (bin - 0.5) * r.step;
  const double high = x + (fabs(x) + fabs(static_cast<double>(r.top))) * 0x1p-22;
  return high <= 3.4028234663852886e38 ? static_cast<float>(high) : 3.4028234663852886e38f;
}

// Tokens as numbers whose larger one comes first.
__device__ __forceinline__ uint64_t order_of(uint32_t key, int32_t index) {
  return (static_cast<uint64_t>(key) << 32) | (0xffffffffu - static_cast<uint32_t>(index));
}

// v of the lane that DPP control kCtrl names, where it has one within the rows of kRows, else 0.
template <int kCtrl, int kRows>
__device__ __forceinline__ uint64_t dpp64(uint64_t v) {
  const uint32_t lo = __builtin_amdgcn_update_dpp(0, static_cast<int>(static_cast<uint32_t>(v)), kCtrl, kRows, 0xf, false);
  const uint32_t hi = __builtin_amdgcn_update_dpp(0, static_cast<int>(static_cast<uint32_t>(v >> 32)), kCtrl, kRows, 0xf, false);
  return (static_cast<uint64_t>(hi) << 32) | lo;
}

// The inclusive sum over the wavefront's lanes before and this one: within rows of 16 lanes, then the
// last lane of a row on to the next row, and of the second on to the third and fourth.
__device__ __forceinline__ uint64_t wave_scan(uint64_t v) {
  v += dpp64<0x111, 0xf>(v);
  v += dpp64<0x112, 0xf>(v);
  v += dpp64<0x114, 0xf>(v);
  v += dpp64<0x118, 0xf>(v);
  v += dpp64<0x142, 0xa>(v);
  v += dpp64<0x143, 0xc>(v);
  return v;
}

__device__ __forceinline__ void add64(uint64_t* to, uint64_t v) {
  atomicAdd(reinterpret_cast<unsigned long long*>(to), static_cast<unsigned long long>(v));
}

// The inclusive sum of v over the threads before and this one, and the sum over all.
struct Scan {
  uint64_t upto, all;
};
__device__ __forceinline__ Scan scan_threads(Shared& s, uint64_t v) {
  const int wave = threadIdx.x / kWave;
  Scan r{wave_scan(v), 0};
  __syncthreads();
  if ((threadIdx.x & (kWave - 1)) == kWave - 1) s.sum[wave] = r.upto;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    const uint64_t sum = s.sum[w];
    r.upto += w < wave ? sum : 0;
    r.all += sum;
  }
  return r;
}

__device__ __forceinline__ uint64_t block_sum(Shared& s, uint64_t v) { return scan_threads(s, v).all; }

// The largest v of all threads, or NaN where `odd` is true in any.
__device__ __forceinline__ float block_max(Shared& s, float v, bool odd) {
#pragma unroll
  for (int m = kWave / 2; m > 0; m >>= 1) v = fmaxf(v, __shfl_xor(v, m));
  if (__ballot(odd) != 0) v = __uint_as_float(0x7fc00000u);
  if ((threadIdx.x & (kWave - 1)) == 0) s.tops[threadIdx.x / kWave] = v;
  __syncthreads();
  bool any = false;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    const float top = s.tops[w];
    any = any || top != top;
    v = fmaxf(v, top);
  }
  return any ? __uint_as_float(0x7fc00000u) : v;
}

// Replaces values[0 .. kBins) by the exclusive sums of of(value, bin), values[kBins] by their total.
template <typename V, typename F>
__device__ __forceinline__ void scan_bins(Shared& s, V* values, F of) {
  V* at = values + threadIdx.x * kBinsPerThread;
  V own[kBinsPerThread];
  uint64_t sum = 0;
#pragma unroll
  for (int i = 0; i < kBinsPerThread; ++i) own[i] = at[i];
#pragma unroll
  for (int i = 0; i < kBinsPerThread; ++i) {
    own[i] = of(own[i], threadIdx.x * kBinsPerThread + i);
    sum += own[i];
  }
  const Scan scan = scan_threads(s, sum);
  uint64_t before = scan.upto - sum;
#pragma unroll
  for (int i = 0; i < kBinsPerThread; ++i) {
    at[i] = static_cast<V>(before);
    before += own[i];
  }
  if (threadIdx.x == 0) values[kBins] = static_cast<V>(scan.all);
  __syncthreads();
}

// The bin b with sums[b] < target <= sums[b + 1]: there is one. Every wavefront looks for it, 64 places at a time.
template <typename V>
__device__ __forceinline__ int32_t bin_reaching(const V* sums, uint64_t target) {
  constexpr int kFar = kBins / kWave | 1, kNear = (kFar + kWave - 1) / kWave;  // odd: each lane in a bank of its own
  static_assert(kFar * kWave >= kBins, "every bin");
  const int lane = threadIdx.x & (kWave - 1);
  const int32_t far = (__popcll(__ballot(sums[min(lane * kFar, kBins)] < target)) - 1) * kFar;
  int32_t at = far;
#pragma unroll
  for (int i = kNear - 1; i >= 0; --i) {
    const int32_t first = far + i * kWave, n = min(kWave, kFar - i * kWave);
    const int below = __popcll(__ballot(lane < n && sums[min(first + min(lane, n - 1), kBins)] < target));
    if (below > 0 && at == far) at = first + below - 1;
  }
  return __builtin_amdgcn_readfirstlane(at);
}

// For each of the `listed` tokens of `list` how many of them (kMass: what mass too) come before it:
// all pairs, the threads of a token sharing the others among them.
template <bool kMass>
__device__ __forceinline__ void rank_list(Shared& s, const uint64_t* list, uint32_t listed) {
  uint32_t slots = kWave;
  while (slots < listed) slots *= 2;
  const uint32_t mine = threadIdx.x & (slots - 1), part = threadIdx.x / slots, parts = kThreads / slots;
  const uint32_t each = ((listed + parts - 1) / parts + 3) / 4 * 4;
  if (threadIdx.x < listed) {
    s.rank[threadIdx.x] = 0;
    if constexpr (kMass) s.before[threadIdx.x] = 0;
  }
  __syncthreads();
  if (mine < listed) {
    const uint64_t own = list[mine];
    uint64_t mass = 0;
    uint32_t count = 0;
    const uint32_t end = min((part + 1) * each, listed);
    uint32_t j = part * each;
    for (; j + 4 <= end; j += 4) {
      uint64_t other[4], weight[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) other[e] = list[j + e];
      if constexpr (kMass) {
#pragma unroll
        for (int e = 0; e < 4; ++e) weight[e] = s.list_mass[j + e];
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        count += other[e] > own;
        if constexpr (kMass) mass += other[e] > own ? weight[e] : 0;
      }
    }
    for (; j < end; ++j) {
      count += list[j] > own;
      if constexpr (kMass) mass += list[j] > own ? s.list_mass[j] : 0;
    }
    if (count) atomicAdd(&s.rank[mine], count);
    if constexpr (kMass) {
      if (mass) atomicAdd(reinterpret_cast<unsigned long long*>(&s.before[mine]), static_cast<unsigned long long>(mass));
    }
  }
  __syncthreads();
}

// The `rank`-th token, from 0, of those with this key, along their ids (there is one).
template <typename T>
__device__ __forceinline__ int32_t nth_of_key(Shared& s, const T* x, int32_t vocab, uint32_t key, uint64_t rank) {
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
  __syncthreads();
  for (int64_t start = 0; start < vocab; start += kThreads) {
    const int64_t i = start + threadIdx.x;
    const bool match = i < vocab && key_of(to_float(x[i])) == key;
    const uint64_t ballot = __ballot(match);
    if (lane == 0) s.waves[wave] = __popcll(ballot);
    __syncthreads();
    uint32_t before = __popcll(ballot & ((1ull << lane) - 1)), all = 0;
    for (int w = 0; w < kWaves; ++w) {
      before += w < wave ? s.waves[w] : 0;
      all += s.waves[w];
    }
    if (match && before == rank) s.found = static_cast<int32_t>(i);
    __syncthreads();
    if (rank < all) break;
    rank -= all;
  }
  return s.found;
}

struct Place {
  uint64_t mass;  // cumulative, the token's own included
  int32_t index;
};

// The first token of the order whose cumulative count (by_count) or mass reaches `target`, which
// the row's totals reach. Every thread gets the answer.
template <typename T>
__device__ __forceinline__ Place locate(Shared& s, const Row& r, const Source<T>& source, bool by_count, uint64_t target) {
  __syncthreads();
  if (threadIdx.x == 0) s.listed = 0;
  __syncthreads();
  const int32_t bin = by_count ? bin_reaching(s.count, target) : bin_reaching(s.mass, target);
  uint64_t base_mass = s.mass[bin];
  uint32_t base_count = by_count ? s.count[bin] : 0;
  const float floor = floor_of_bin(r, bin), ceiling = ceiling_of_bin(r, bin);
  uint32_t low = 0, high = 0xffffffffu;  // keys still in question
  // f(value, index, key, weight) for the bin's tokens with keys of [from, to].
  auto tokens = [&](uint32_t from, uint32_t to, auto f) {
    source.template each_if<4>([&](float v) { return (v >= floor) & (v <= ceiling); }, [&](float v, int32_t i) {
      const Weight w = weigh<true>(r, v);
      const uint32_t key = key_of(v);
      if (w.bin == bin && key >= from && key <= to && w.mass != 0) f(i, key, w.mass);
    });
  };
  auto collect = [&]() {
    tokens(low, high, [&](int32_t i, uint32_t key, uint64_t w) {
      const uint32_t at = atomicAdd(&s.listed, 1u);
      if (at < kList) {
        s.list[at] = order_of(key, i);
        s.list_mass[at] = w;
      }
    });
    __syncthreads();
  };
  collect();
  uint32_t listed = s.listed;
  if (listed > kList) {
    // A bin with more tokens than the list holds: halve the range of keys that holds the answer.
    while (listed > kList && low < high) {
      const uint32_t mid = low + (high - low) / 2 + 1;
      uint64_t mass = 0, count = 0;
      tokens(mid, high, [&](int32_t, uint32_t, uint64_t w) {
        mass += w;
        ++count;
      });
      mass = block_sum(s, mass);
      count = block_sum(s, count);
      if ((by_count ? base_count + count : base_mass + mass) >= target) {
        low = mid;
        listed = static_cast<uint32_t>(count);
      } else {
        base_mass += mass;
        base_count += static_cast<uint32_t>(count);
        high = mid - 1;
        listed -= static_cast<uint32_t>(count);
      }
    }
    if (listed > kList) {  // equal logits: the one that far along their ids
      const uint64_t w = weigh<true>(r, float_of(low)).mass;
      const uint64_t rank = by_count ? target - base_count - 1 : (target - base_mass - 1) / w;
      return {base_mass + (rank + 1) * w, nth_of_key(s, source.x, source.vocab, low, rank)};
    }
    if (threadIdx.x == 0) s.listed = 0;
    __syncthreads();
    collect();
    listed = s.listed;
  }
  rank_list<true>(s, s.list, listed);
  if (threadIdx.x < listed) {
    const uint64_t before = base_mass + s.before[threadIdx.x];
    const uint64_t upto = before + s.list_mass[threadIdx.x];
    if (by_count ? base_count + s.rank[threadIdx.x] + 1 == target : before < target && target <= upto) {
      s.found = static_cast<int32_t>(0xffffffffu - static_cast<uint32_t>(s.list[threadIdx.x]));
      s.found_mass = upto;
    }
  }
  __syncthreads();
  return {s.found_mass, s.found};
}

// The mass that top_p keeps of `mass` is the cumulative one of the first token to reach this.
__device__ __forceinline__ uint64_t nucleus(float top_p, uint64_t mass) {
  const double want = top_p > 0.f ? ceil(static_cast<double>(top_p) * static_cast<double>(mass)) : 1.0;
  const uint64_t target = static_cast<uint64_t>(want);
  return target < 1 ? 1 : target < mass ? target : mass;
}

// The token is the first whose cumulative mass reaches this.
__device__ __forceinline__ uint64_t place_of(float u, uint64_t mass) {
  const uint64_t at = u > 0.f ? static_cast<uint64_t>(static_cast<double>(u) * static_cast<double>(mass)) : 0;
  return at < mass ? at + 1 : mass;
}

// The end of top-p and the draw from one pass over the tokens; -1 where they do not fit the list. `mass` is
// what top-k leaves. The nucleus ends in bin `edge`, with a mass between `target` and `most`, and so the draw
// falls into one of the bins [first, last] (one or two as a rule), none of them behind the edge's. One pass
// less: 256 rows of 128256 tokens with top_p 93 -> 77 us, 2 rows of 1000 11.2 -> 10.2.
template <typename T>
__device__ __forceinline__ int32_t nucleus_and_draw(Shared& s, const Row& r, const Source<T>& source, uint64_t target, uint64_t mass,
                                                    float u) {
  __syncthreads();
  if (threadIdx.x == 0) s.listed = 0;
  __syncthreads();
  const int32_t edge = bin_reaching(s.mass, target);
  const uint64_t most = min(s.mass[edge + 1], mass);
  const int32_t first = bin_reaching(s.mass, place_of(u, target)), last = bin_reaching(s.mass, place_of(u, most));
  // No token weighs less than 2^(-1 / 256) of its bin's middle, so masses say how many they are at most.
  const auto tokens_of = [&](int32_t from, int32_t to) {
    return static_cast<float>(s.mass[to + 1] - s.mass[from]) * exp2f((to + 0.5f) * (1.f / kPerOctave)) / static_cast<float>(r.power[0]);
  };
  if (tokens_of(first, last) + (edge > last ? tokens_of(edge, edge) : 0.f) > kList) return -1;
  const float floor = floor_of_bin(r, edge), ceiling = ceiling_of_bin(r, edge);
  const float draw_floor = floor_of_bin(r, last), draw_ceiling = ceiling_of_bin(r, first);
  const auto near = [&](float v) { return (v >= floor) & (v <= ceiling) | (v >= draw_floor) & (v <= draw_ceiling); };
  source.template each_if<4>(near, [&](float v, int32_t i) {
    const uint32_t at = atomicAdd(&s.listed, 1u);
    if (at < kList) s.list[at] = order_of(key_of(v), i);
  });
  __syncthreads();
  const uint32_t listed = s.listed;
  if (listed > kList) return -1;
  // Between a bin's bounds lie some tokens of the bins beside it: these turn into one behind all others.
  Weight own{-1, 0};
  if (threadIdx.x < listed) {
    own = weigh<true>(r, float_of(static_cast<uint32_t>(s.list[threadIdx.x] >> 32)));
    if (own.bin != edge && (own.bin < first || own.bin > last)) own.mass = 0;
    if (own.mass == 0) s.list[threadIdx.x] = 0;
    s.list_mass[threadIdx.x] = own.mass;
  }
  __syncthreads();
  rank_list<true>(s, s.list, listed);
  // Cumulative masses: of what is not in the list, the bins before the first come before the draw's tokens,
  // those between them and the edge's before the edge's too.
  uint64_t before = 0;
  if (own.mass != 0) {
    before = s.before[threadIdx.x] + s.mass[first];
    if (own.bin > last) before += s.mass[edge] - s.mass[last + 1];
    if (before < target && target <= before + own.mass) s.found_mass = before + own.mass;
  }
  __syncthreads();
  const uint64_t place = place_of(u, s.found_mass);
  if (before < place && place <= before + own.mass) s.found = static_cast<int32_t>(0xffffffffu - static_cast<uint32_t>(s.list[threadIdx.x]));
  __syncthreads();
  return s.found;
}

// The whole row's answer from the `listed` <= kFew tokens of its list, which hold every token that the
// cuts can keep: put in order by counting, then summed up along the order, a token per thread.
__device__ __forceinline__ int32_t from_list(Shared& s, const Row& r, uint32_t listed, int32_t top_k, float top_p, float u) {
  rank_list<false>(s, s.kept, listed);
  if (threadIdx.x < listed) s.before[s.rank[threadIdx.x]] = s.kept[threadIdx.x];
  __syncthreads();
  const bool kept = threadIdx.x < listed && (top_k <= 0 || threadIdx.x < static_cast<uint32_t>(top_k));
  const uint64_t token = kept ? s.before[threadIdx.x] : 0;
  const uint64_t own = kept ? weigh<true>(r, float_of(static_cast<uint32_t>(token >> 32))).mass : 0;
  const Scan scan = scan_threads(s, own);
  const uint64_t upto = scan.upto;
  uint64_t mass = scan.all;
  if (!(top_p >= 1.f)) {
    const uint64_t target = nucleus(top_p, mass);
    if (own != 0 && upto - own < target && target <= upto) s.found_mass = upto;
    __syncthreads();
    mass = s.found_mass;
  }
  const uint64_t target = place_of(u, mass);
  if (own != 0 && upto - own < target && target <= upto) s.found = static_cast<int32_t>(0xffffffffu - static_cast<uint32_t>(token));
  __syncthreads();
  return s.found;
}

// The answer by a histogram of the masses (and counts) of the tokens from `floor` on.
template <typename T>
__device__ __forceinline__ int32_t from_bins(Shared& s, const Row& r, const Source<T>& source, float floor, int32_t top_k, float top_p,
                                             float u) {
  const bool counting = top_k > 0;
  const auto every = [](float) { return true; };  // most tokens lie above the floor: tests together cost 5% here
  if (counting || r.least > 0.0) {
    source.template each_if<2>(every, [&](float v, int32_t) {
      if (!(v >= floor)) return;
      const Weight w = weigh<true>(r, v);
      if (w.mass == 0) return;
      add64(mass_of_bin(s.mass, w.bin), w.mass);
      if (counting) atomicAdd(&s.count[w.bin], 1u);
    });
  } else {
    source.template each_if<2>(every, [&](float v, int32_t) {
      if (!(v >= floor)) return;
      const Weight w = weigh<false>(r, v);
      add64(mass_of_bin(s.mass, w.bin), w.mass);
    });
  }
  __syncthreads();
  scan_bins(s, s.mass, [](uint64_t mass, int) { return mass; });
  if (counting) scan_bins(s, s.count, [](uint32_t count, int) { return count; });

  // The end of top-k, then that of top-p and the draw: together, or where that fails one after the other.
  uint64_t mass = s.mass[kBins];
  const bool cut = counting && s.count[kBins] > static_cast<uint32_t>(top_k), nuclear = !(top_p >= 1.f);
  int32_t token = -1;
  for (int step = 0; step < 3; ++step) {
    if ((step == 0 && !cut) || (step == 1 && !nuclear)) continue;
    const uint64_t target = step == 0 ? static_cast<uint64_t>(top_k) : step == 1 ? nucleus(top_p, mass) : place_of(u, mass);
    if (step == 1) {
      token = nucleus_and_draw(s, r, source, target, mass, u);
      if (token >= 0) break;
    }
    const Place place = locate(s, r, source, step == 0, target);
    mass = place.mass;
    token = place.index;
  }
  return token;
}

// One workgroup per row.
template <typename T>
__global__ __launch_bounds__(kThreads) void sample_kernel(const Args a) {
  __shared__ Shared s;
  const int64_t row = blockIdx.x;
  const T* x = static_cast<const T*>(a.logits) + row * a.row_stride;
  const float temperature = a.temperatures ? a.temperatures[row] : a.temperature;
  const int32_t top_k = a.top_ks ? a.top_ks[row] : a.top_k;
  const float top_p = a.top_ps ? a.top_ps[row] : a.top_p;
  const float min_p = a.min_ps ? a.min_ps[row] : a.min_p;
  const float u = a.uniforms[row];

  // LDS is made ready while the row arrives.
  if (threadIdx.x < kPerOctave) s.power[threadIdx.x] = exp2(threadIdx.x * (1.0 / kPerOctave)) * a.one;
  for (int i = threadIdx.x; i < kBins + 2; i += kThreads) {
    s.mass[i] = 0;
    s.count[i] = 0;
  }
  if (threadIdx.x == 0) s.listed = 0;

  float most = -INFINITY;
  bool odd = false;
  for_each<8>(x, a.vocab, [&](float v, int32_t) {
    most = fmaxf(most, v);
    odd = odd || v != v;
  });
  const float top = block_max(s, most, odd);
  const bool any_odd = top != top;
  if (any_odd || top == -INFINITY || !(temperature > 0.f)) {  // the greedy token: the first NaN, else the first of the largest
    if (threadIdx.x == 0) s.found = a.vocab;
    __syncthreads();
    int32_t first = a.vocab;
    for_each<4>(x, a.vocab, [&](float v, int32_t i) {
      if (any_odd ? v != v : v == top) first = min(first, i);
    });
    if (first < a.vocab) atomicMin(&s.found, first);
    __syncthreads();
    if (threadIdx.x == 0) a.out[row] = s.found;
    return;
  }
  if (top == INFINITY) {  // equal weights for the tokens of +inf, nothing for others
    uint64_t count = 0;
    for_each<4>(x, a.vocab, [&](float v, int32_t) { count += v == top; });
    count = block_sum(s, count);
    if (top_k > 0) count = min(count, static_cast<uint64_t>(top_k));
    if (!(top_p >= 1.f)) count = nucleus(top_p, count);
    const int32_t token = nth_of_key(s, x, a.vocab, key_of(top), place_of(u, count) - 1);
    if (threadIdx.x == 0) a.out[row] = token;
    return;
  }

  Row r;
  r.top = top;
  r.rate = fmax(kPerOctave * 1.44269504088896340736 / static_cast<double>(temperature), 1e-300);  // T may be infinite
  r.step = 1.0 / r.rate;
  r.least = min_p > 0.f ? fmin(static_cast<double>(min_p), 1.0) * a.one : 0.0;
  r.power = s.power;
  constexpr double kStep = 0.69314718055994530942 / kPerOctave;
  r.series[0] = kStep;
  r.series[1] = kStep * kStep / 2;
  r.series[2] = kStep * kStep * kStep / 6;
  r.series[3] = kStep * kStep * kStep * kStep / 24;
#pragma unroll
  for (double& c : r.series) asm volatile("" : "+v"(c));

  // The bins that the kept tokens lie in, where the settings bound them beforehand: min-p by its weight;
  // top-k by the threads' largest tokens, of which there are top_k in the bins up to the pivot's.
  const float lowest = floor_of_bin(r, kBins - 1);
  int32_t last = kBins - 1;
  if (min_p > 0.f) {
    const double deep = ceil(-log2(fmin(static_cast<double>(min_p), 1.0)) * kPerOctave) + 1.0;
    last = deep < last ? static_cast<int32_t>(deep) : last;
  }
  if (top_k > 0 && top_k <= kThreads) {
    if (most >= lowest) {
      const int32_t bin = weigh<false>(r, most).bin;
      if (bin < kBins) atomicAdd(&s.count[bin], 1u);
    }
    __syncthreads();
    scan_bins(s, s.count, [](uint32_t count, int) { return count; });
    if (s.count[kBins] >= static_cast<uint32_t>(top_k)) last = min(last, bin_reaching(s.count, top_k));
    __syncthreads();
    for (int i = threadIdx.x; i < kBins + 2; i += kThreads) s.count[i] = 0;
  }
  const float floor = floor_of_bin(r, last);
  Source<T> source{x, a.vocab, s.kept, -1};
  // Were m of the 1024 threads to meet a token from the floor on, some -1024 ln(1 - m / 1024) tokens lie there:
  // 2840 for kCrowded threads, so that the list seldom overflows.
  if (a.vocab <= kFew || (last < kBins - 1 && __syncthreads_count(most >= floor) <= kCrowded)) {
    for_each_if<8>(x, a.vocab, [&](float v) { return v >= floor; }, [&](float v, int32_t i) {
      const uint32_t slot = atomicAdd(&s.listed, 1u);
      if (slot < kKept) s.kept[slot] = order_of(key_of(v), i);
    });
    __syncthreads();
    const uint32_t kept = s.listed;
    if (kept <= kFew) {
      const int32_t token = from_list(s, r, kept, top_k, top_p, u);
      if (threadIdx.x == 0) a.out[row] = token;
      return;
    }
    if (kept <= kKept) source.kept = kept;
  }
  __syncthreads();
  const int32_t token = from_bins(s, r, source, floor, top_k, top_p, u);
  if (threadIdx.x == 0) a.out[row] = token;
}

}  // namespace
}  // namespace pkv

extern "C" int pkv_sample_tokens(const pkv_sample* args, int device, void* stream) {
  using namespace pkv;
  if (!args) return PKV_EINVAL;
  const pkv_sample& g = *args;
  if (g.num_rows < 0 || g.vocab_size < 1 || g.vocab_size > 0x7fffffff || g.row_stride < g.vocab_size) return PKV_EINVAL;
  if (g.dtype != PKV_F32 && g.dtype != PKV_BF16) return PKV_EINVAL;
  if (g.num_rows == 0) return PKV_OK;
  if (!g.token_ids || !g.logits || !g.uniforms) return PKV_EINVAL;
  if (g.num_rows > 0xffffffffll / kThreads) return PKV_EUNSUPPORTED;  // a launch's threads are counted in 32 bits
  Args a{};
  a.out = g.token_ids;
  a.logits = g.logits;
  a.row_stride = g.row_stride;
  a.vocab = static_cast<int32_t>(g.vocab_size);
  a.uniforms = g.uniforms;
  a.temperatures = g.temperatures;
  a.top_ks = g.top_ks;
  a.top_ps = g.top_ps;
  a.min_ps = g.min_ps;
  a.temperature = g.temperature;
  a.top_k = g.top_k;
  a.top_p = g.top_p;
  a.min_p = g.min_p;
  int bits = 0;  // vocab tokens of weight 1 must not overflow 63 bits
  while ((g.vocab_size >> bits) > 0) ++bits;
  a.one = static_cast<double>(1ull << (bits <= 63 - PKV_SAMPLE_BITS ? PKV_SAMPLE_BITS : 63 - bits));
  DeviceGuard guard(device);
  if (!guard.ok()) return PKV_EHIP;
  const dim3 grid(static_cast<uint32_t>(g.num_rows));
  auto st = static_cast<hipStream_t>(stream);
  if (g.dtype == PKV_F32) {
    hipLaunchKernelGGL(sample_kernel<float>, grid, dim3(kThreads), 0, st, a);
  } else {
    hipLaunchKernelGGL(sample_kernel<uint16_t>, grid, dim3(kThreads), 0, st, a);
  }
  return check_launch();
}
