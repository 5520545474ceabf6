// Sampling from logits rows with temperature, top-k, min-p and top-p, from given uniform numbers.
//
// The four settings are all cuts of one order, the tokens by falling logit (equal ones by id): every
// kept set is a beginning of it, and the draw is a place in it. With exact sums of fixed-point weights
//     W[i] = round(2^46 exp((logit[i] - max) / T))
// each step is the same question, "which token is the first whose cumulative mass (or count) reaches
// X?": X = top_k in counts gives the mass M of the first cut; X = ceil(top_p * M) gives the kept mass
// S; X = floor(uniform * S) + 1 gives the token. Nothing is sorted: a histogram of the masses over
// bins that fall with the logit finds the token's bin, and only that bin's tokens are compared with
// each other. Integer sums make the result independent of the order of the atomics.
#include <math.h>

#include "pkv_common.h"

namespace pkv {
namespace {

constexpr int kThreads = 1024;
constexpr int kWaves = kThreads / kWave;
constexpr int kBins = 4096;
constexpr int kBinsPerThread = kBins / kThreads;
constexpr int kList = 2048;      // tokens of one bin that are compared in LDS
constexpr float kReach = 33.f;   // exp(-33) * 2^46 < 1/2: a token this many temperatures down weighs 0
constexpr uint32_t kNoBin = 0xffffffffu;

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

// f(value, index) for every element of a row, each by some thread of the workgroup: the 16-byte
// aligned body in vectors, what lies before and after it one element per thread.
template <typename T, typename F>
__device__ __forceinline__ void for_each(const T* x, int32_t n, F f) {
  constexpr int kVec = 16 / sizeof(T);
  const int32_t before = static_cast<int32_t>(((16 - (reinterpret_cast<uintptr_t>(x) & 15)) & 15) / sizeof(T));
  const int32_t head = before < n ? before : n;
  const u32x4* body = reinterpret_cast<const u32x4*>(x + head);
  const int32_t vectors = (n - head) / kVec;
  for (int32_t q = threadIdx.x; q < vectors; q += kThreads) {
    const u32x4 raw = body[q];
    const int32_t i = head + q * kVec;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      if constexpr (sizeof(T) == 4) {
        f(__uint_as_float(raw[w]), i + w);
      } else {
        f(bf16_lo(raw[w]), i + 2 * w);
        f(bf16_hi(raw[w]), i + 2 * w + 1);
      }
    }
  }
  const int32_t tail = head + vectors * kVec;
  const int32_t t = threadIdx.x;
  if (t < head + (n - tail)) {
    const int32_t i = t < head ? t : tail + (t - head);
    f(to_float(x[i]), i);
  }
}

// What the weights of one row go by.
struct Row {
  float top;     // the largest logit
  float scale;   // bins per unit of logit
  double inv_t;
  double one;
  double min_p;
};

__device__ __forceinline__ uint32_t bin_of(const Row& r, float x) {
  if (x == r.top) return 0;
  const float at = (r.top - x) * r.scale;  // falls with x: each step rounds monotonically
  return at < static_cast<float>(kBins - 1) ? static_cast<uint32_t>(at) : kBins - 1;
}

__device__ __forceinline__ uint64_t weight_of(const Row& r, float x) {
  const double d = x == r.top ? 0.0 : static_cast<double>(x) - static_cast<double>(r.top);
  if (!(d > -INFINITY)) return 0;
  const double w = exp(d * r.inv_t);
  return w >= r.min_p ? static_cast<uint64_t>(__double2ull_rn(w * r.one)) : 0;
}

struct Shared {
  uint64_t mass[kBins + 1];   // exclusive sums over the bins before, once summed up
  uint32_t count[kBins + 1];
  uint64_t list_mass[kList];
  uint32_t list_key[kList];
  int32_t list_index[kList];
  uint64_t sum[kWaves];
  uint32_t waves[kWaves];
  uint64_t base_mass, found_mass;
  uint32_t base_count, bin, listed;
  int32_t found;
};

__device__ __forceinline__ uint64_t shfl_xor64(uint64_t v, int mask) {
  const uint32_t lo = __shfl_xor(static_cast<uint32_t>(v), mask);
  const uint32_t hi = __shfl_xor(static_cast<uint32_t>(v >> 32), mask);
  return (static_cast<uint64_t>(hi) << 32) | lo;
}

__device__ __forceinline__ uint64_t shfl_up64(uint64_t v, int delta) {
  const uint32_t lo = __shfl_up(static_cast<uint32_t>(v), delta);
  const uint32_t hi = __shfl_up(static_cast<uint32_t>(v >> 32), delta);
  return (static_cast<uint64_t>(hi) << 32) | lo;
}

__device__ uint64_t block_sum(Shared& s, uint64_t v) {
  for (int m = kWave / 2; m > 0; m >>= 1) v += shfl_xor64(v, m);
  __syncthreads();
  if ((threadIdx.x & (kWave - 1)) == 0) s.sum[threadIdx.x / kWave] = v;
  __syncthreads();
  uint64_t total = 0;
  for (int w = 0; w < kWaves; ++w) total += s.sum[w];
  return total;
}

// Replaces values[0 .. kBins) by their exclusive sums, values[kBins] by the total.
template <typename V>
__device__ void scan_bins(Shared& s, V* values) {
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
  V own[kBinsPerThread];
  V sum = 0;
#pragma unroll
  for (int i = 0; i < kBinsPerThread; ++i) {
    own[i] = values[threadIdx.x * kBinsPerThread + i];
    sum += own[i];
  }
  uint64_t upto = sum;
  for (int d = 1; d < kWave; d <<= 1) {
    const uint64_t other = shfl_up64(upto, d);
    if (lane >= d) upto += other;
  }
  __syncthreads();
  if (lane == kWave - 1) s.sum[wave] = upto;
  __syncthreads();
  uint64_t before = upto - sum;
  for (int w = 0; w < wave; ++w) before += s.sum[w];
#pragma unroll
  for (int i = 0; i < kBinsPerThread; ++i) {
    values[threadIdx.x * kBinsPerThread + i] = static_cast<V>(before);
    before += own[i];
  }
  if (threadIdx.x == kThreads - 1) values[kBins] = static_cast<V>(before);
  __syncthreads();
}

struct Place {
  uint64_t mass;  // cumulative, the token's own included
  int32_t index;
};

// The first token of the order whose cumulative count (by_count) or mass reaches `target`, which
// the row's totals reach. Every thread gets the answer.
template <typename T>
__device__ Place locate(Shared& s, const Row& r, const T* x, int32_t vocab, bool by_count, uint64_t target) {
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kBinsPerThread; ++i) {
    const int b = threadIdx.x * kBinsPerThread + i;
    const uint64_t lo = by_count ? s.count[b] : s.mass[b];
    const uint64_t hi = by_count ? s.count[b + 1] : s.mass[b + 1];
    if (lo < target && target <= hi) {
      s.bin = b;
      s.base_mass = s.mass[b];
      s.base_count = s.count[b];
    }
  }
  if (threadIdx.x == 0) s.listed = 0;
  __syncthreads();
  const uint32_t bin = s.bin;
  uint64_t base_mass = s.base_mass;
  uint32_t base_count = s.base_count;
  uint32_t low = 0, high = 0xffffffffu;  // keys still in question
  auto collect = [&]() {
    for_each(x, vocab, [&](float v, int32_t i) {
      if (bin_of(r, v) != bin) return;
      const uint32_t key = key_of(v);
      if (key < low || key > high) return;
      const uint64_t w = weight_of(r, v);
      if (w == 0) return;
      const uint32_t at = atomicAdd(&s.listed, 1u);
      if (at < kList) {
        s.list_key[at] = key;
        s.list_index[at] = i;
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
      for_each(x, vocab, [&](float v, int32_t) {
        if (bin_of(r, v) != bin) return;
        const uint32_t key = key_of(v);
        if (key < mid || key > high) return;
        const uint64_t w = weight_of(r, v);
        mass += w;
        count += w != 0;
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
      const uint64_t w = weight_of(r, float_of(low));
      uint64_t rank = by_count ? target - base_count - 1 : (target - base_mass - 1) / w;
      const uint64_t mass = base_mass + (rank + 1) * w;
      const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
      for (int64_t start = 0; start < vocab; start += kThreads) {
        const int64_t i = start + threadIdx.x;
        const bool match = i < vocab && key_of(to_float(x[i])) == low;
        const uint64_t ballot = __ballot(match);
        if (lane == 0) s.waves[wave] = __popcll(ballot);
        __syncthreads();
        uint32_t before = __popcll(ballot & ((1ull << lane) - 1)), all = 0;
        for (int w2 = 0; w2 < kWaves; ++w2) {
          before += w2 < wave ? s.waves[w2] : 0;
          all += s.waves[w2];
        }
        if (match && before == rank) s.found = static_cast<int32_t>(i);
        __syncthreads();
        if (rank < all) break;
        rank -= all;
      }
      return {mass, s.found};
    }
    if (threadIdx.x == 0) s.listed = 0;
    __syncthreads();
    collect();
    listed = s.listed;
  }
  for (uint32_t i = threadIdx.x; i < listed; i += kThreads) {
    const uint32_t key = s.list_key[i];
    const int32_t index = s.list_index[i];
    uint64_t mass = base_mass, count = base_count;
    for (uint32_t j = 0; j < listed; ++j) {
      const uint32_t other = s.list_key[j];
      if (other > key || (other == key && s.list_index[j] < index)) {
        mass += s.list_mass[j];
        ++count;
      }
    }
    const uint64_t upto = mass + s.list_mass[i];
    if (by_count ? count + 1 == target : mass < target && target <= upto) {
      s.found = index;
      s.found_mass = upto;
    }
  }
  __syncthreads();
  return {s.found_mass, s.found};
}

// One workgroup per row.
template <typename T>
__global__ __launch_bounds__(kThreads) void sample_kernel(const Args a) {
  __shared__ Shared s;
  const int64_t row = blockIdx.x;
  const T* x = static_cast<const T*>(a.logits) + row * a.row_stride;
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
  const float temperature = a.temperatures ? a.temperatures[row] : a.temperature;
  const int32_t top_k = a.top_ks ? a.top_ks[row] : a.top_k;
  const float top_p = a.top_ps ? a.top_ps[row] : a.top_p;
  const float min_p = a.min_ps ? a.min_ps[row] : a.min_p;

  // The greedy token (the first NaN, else the first of the largest), and the smallest finite logit.
  // A NaN counts as the largest key.
  uint64_t best = 0;  // key, then the complement of the index
  float least = INFINITY;
  for_each(x, a.vocab, [&](float v, int32_t i) {
    const uint32_t key = isnan(v) ? 0xffffffffu : key_of(v);
    const uint64_t mine = (static_cast<uint64_t>(key) << 32) | (0xffffffffu - static_cast<uint32_t>(i));
    best = mine > best ? mine : best;
    if (v > -INFINITY && v < least) least = v;
  });
  for (int m = kWave / 2; m > 0; m >>= 1) {
    const uint64_t other = shfl_xor64(best, m);
    best = other > best ? other : best;
    least = fminf(least, __shfl_xor(least, m));
  }
  if (lane == 0) {
    s.sum[wave] = best;
    s.waves[wave] = __float_as_uint(least);
  }
  __syncthreads();
  for (int w = 0; w < kWaves; ++w) {
    best = s.sum[w] > best ? s.sum[w] : best;
    least = fminf(least, __uint_as_float(s.waves[w]));
  }
  const uint32_t top_key = static_cast<uint32_t>(best >> 32);
  const int32_t greedy = static_cast<int32_t>(0xffffffffu - static_cast<uint32_t>(best));
  const bool drawn = temperature > 0.f && top_key != 0xffffffffu && top_key > key_of(-INFINITY);
  if (!drawn) {
    if (threadIdx.x == 0) a.out[row] = greedy;
    return;
  }

  Row r;
  r.top = float_of(top_key);
  r.inv_t = 1.0 / static_cast<double>(temperature);
  r.one = a.one;
  r.min_p = min_p > 0.f ? fmin(static_cast<double>(min_p), 1.0) : 0.0;
  const float range = fminf(r.top - least, kReach * temperature);
  r.scale = range > 0.f ? fminf(kBins / range, 1e30f) : 0.f;

  const bool counting = top_k > 0;
  for (int i = threadIdx.x; i <= kBins; i += kThreads) {
    s.mass[i] = 0;
    s.count[i] = 0;
  }
  __syncthreads();
  for_each(x, a.vocab, [&](float v, int32_t) {
    const uint64_t w = weight_of(r, v);
    if (w == 0) return;
    const uint32_t b = bin_of(r, v);
    atomicAdd(reinterpret_cast<unsigned long long*>(&s.mass[b]), static_cast<unsigned long long>(w));
    if (counting) atomicAdd(&s.count[b], 1u);
  });
  __syncthreads();
  scan_bins(s, s.mass);
  if (counting) scan_bins(s, s.count);

  uint64_t mass = s.mass[kBins];
  if (counting && s.count[kBins] > static_cast<uint32_t>(top_k)) mass = locate(s, r, x, a.vocab, true, top_k).mass;
  if (!(top_p >= 1.f)) {
    const double want = top_p > 0.f ? ceil(static_cast<double>(top_p) * static_cast<double>(mass)) : 1.0;
    uint64_t target = static_cast<uint64_t>(want);
    target = target < 1 ? 1 : target;
    mass = locate(s, r, x, a.vocab, false, target < mass ? target : mass).mass;
  }
  const float u = a.uniforms[row];
  uint64_t at = u > 0.f ? static_cast<uint64_t>(static_cast<double>(u) * static_cast<double>(mass)) : 0;
  at = at < mass ? at : mass - 1;
  const Place place = locate(s, r, x, a.vocab, false, at + 1);
  if (threadIdx.x == 0) a.out[row] = place.index;
}

}  // namespace
}  // namespace pkv

extern "C" int64_t pkv_sample_workspace_bytes(int64_t num_rows, int64_t vocab_size) {
  if (num_rows < 0 || vocab_size < 1) return PKV_EINVAL;
  return 0;
}

extern "C" int pkv_sample_tokens(const pkv_sample* args, int device, void* stream) {
  using namespace pkv;
  if (!args) return PKV_EINVAL;
  const pkv_sample& g = *args;
  if (g.num_rows < 0 || g.vocab_size < 1 || g.vocab_size > 0x7fffffff || g.row_stride < g.vocab_size) return PKV_EINVAL;
  if (g.dtype != PKV_F32 && g.dtype != PKV_BF16) return PKV_EINVAL;
  if (g.num_rows == 0) return PKV_OK;
  if (!g.token_ids || !g.logits || !g.uniforms) return PKV_EINVAL;
  if (g.num_rows > 0x7fffffff) return PKV_EUNSUPPORTED;
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
