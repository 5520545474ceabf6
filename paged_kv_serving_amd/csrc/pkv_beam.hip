// Beam search over a paged cache: the best continuations of a group's beams, and the beams' tables and last blocks moved
// to the beams that go on.
#include <math.h>

#include <algorithm>

#include "pkv_common.h"

namespace pkv {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / kWave;
constexpr int kCapacity = 1024;  // of a workgroup's list of candidates
constexpr int kMaxLists = 4096;  // of a group: beams times chunks
constexpr int kStagedKeys = 8192;  // of a group, kept in LDS

typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

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
// A candidate of a row: falling keys are falling logits, and of equal ones rising tokens. No two of a row are alike; 0 is none.
__device__ __forceinline__ uint64_t key_of(float x, uint32_t token) {
  return x == -INFINITY ? 0 : static_cast<uint64_t>(ordered(x)) << 32 | static_cast<uint32_t>(~token);
}

// e^x for x <= 0 in double precision: 2^k e^r with |r| <= ln 2 / 2 and e^r's series up to r^10 / 10!, which leaves out 2^-42.
__device__ __forceinline__ double exp_of(double x) {
  x = x < -1000.0 ? -1000.0 : x;  // 0 from there on; a NaN stays one
  const double k = __builtin_rint(x * 1.4426950408889634);
  const double r = __builtin_fma(k, -0.6931471805599453, x);
  double p = 1.0 / 3628800.0;
  p = __builtin_fma(p, r, 1.0 / 362880.0);
  p = __builtin_fma(p, r, 1.0 / 40320.0);
  p = __builtin_fma(p, r, 1.0 / 5040.0);
  p = __builtin_fma(p, r, 1.0 / 720.0);
  p = __builtin_fma(p, r, 1.0 / 120.0);
  p = __builtin_fma(p, r, 1.0 / 24.0);
  p = __builtin_fma(p, r, 1.0 / 6.0);
  p = __builtin_fma(p, r, 0.5);
  p = __builtin_fma(p, r, 1.0);
  p = __builtin_fma(p, r, 1.0);
  return ldexp(p, static_cast<int>(fmax(k, -2000.0)));
}

// The largest / smallest over aligned groups of lanes, `size` of them (a power of two), in each lane.
__device__ __forceinline__ uint64_t group_max(uint64_t x, int size) {
  for (int m = 1; m < size; m *= 2) x = max(x, static_cast<uint64_t>(__shfl_xor(static_cast<unsigned long long>(x), m)));
  return x;
}
__device__ __forceinline__ uint64_t group_min(uint64_t x, int from, int size) {
  for (int m = from; m < size; m *= 2) x = min(x, static_cast<uint64_t>(__shfl_xor(static_cast<unsigned long long>(x), m)));
  return x;
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

// A chunk of a row: its largest logit, the sum of exponentials, its `count` best in order. A thread's largest keys give a
// number that at least `count` keys reach: the lanes of a wavefront make `count` groups or more, and the smallest of the
// groups' largest keys is one. The keys that reach it, a few times `count`, are listed, and each one's place is the number of
// larger ones.
template <typename T, int kPer>
__global__ __launch_bounds__(kThreads) void chunk_kernel(const Select a) {
  constexpr int kVec = 16 / sizeof(T), kLoads = kPer / kVec;
  __shared__ uint64_t s_list[kCapacity], s_reach[kWaves];
  __shared__ float s_top[kWaves];
  __shared__ double s_sum[kWaves];
  __shared__ int32_t s_count;
  const pkv_beam& g = a.g;
  const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = tid / kWave;
  const int64_t row = blockIdx.x / static_cast<uint32_t>(a.chunks);
  const uint32_t chunk = blockIdx.x % static_cast<uint32_t>(a.chunks);
  if (!looked_at(g, row)) return;
  const uint32_t vocab = static_cast<uint32_t>(g.vocab_size);
  const uint32_t first = chunk * (kThreads * kPer) + tid * kVec;  // this thread's: kVec numbers every kThreads * kVec
  const T* p = static_cast<const T*>(g.logits) + row * g.row_stride;
  const bool aligned = (reinterpret_cast<uintptr_t>(p) & 15u) == 0;

  float x[kPer];
#pragma unroll
  for (int i = 0; i < kLoads; ++i) {
    const uint32_t at = first + i * (kThreads * kVec);
    if (aligned && at + kVec <= vocab) {
      if constexpr (sizeof(T) == 4) {
        const f32x4 v = __builtin_nontemporal_load(reinterpret_cast<const f32x4*>(p + at));
#pragma unroll
        for (int e = 0; e < 4; ++e) x[i * kVec + e] = v[e];
      } else {
        const u32x4 v = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(p + at));
#pragma unroll
        for (int e = 0; e < 4; ++e) x[i * kVec + 2 * e] = bf16_lo(v[e]), x[i * kVec + 2 * e + 1] = bf16_hi(v[e]);
      }
    } else {
#pragma unroll
      for (int e = 0; e < kVec; ++e) {
        x[i * kVec + e] = -INFINITY;
        if (at + e < vocab) {
          if constexpr (sizeof(T) == 4) x[i * kVec + e] = p[at + e];
          else x[i * kVec + e] = __uint_as_float(static_cast<uint32_t>(p[at + e]) << 16);
        }
      }
    }
  }
  const auto token = [&](int i) { return first + i / kVec * (kThreads * kVec) + i % kVec; };

  // This thread's largest, of its even and its odd places apart: the lowest token of equal ones.
  float best[2] = {-INFINITY, -INFINITY};
  int at[2] = {0, 0};
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    x[i] += 0.f;  // -0 and 0 are one logit
    const int side = i % 2;
    if (x[i] > best[side]) best[side] = x[i], at[side] = i;
  }
  uint64_t half[2];
#pragma unroll
  for (int s = 0; s < 2; ++s) half[s] = key_of(best[s], token(at[s]));
  uint64_t reach;
  if (g.count > kWave) {
    reach = group_min(min(half[0], half[1]), 1, kWave);
  } else {
    int size = kWave;  // lanes of a group
    while (kWave / size < g.count) size /= 2;
    reach = group_min(group_max(max(half[0], half[1]), size), size, kWave);
  }
  float top = fmaxf(best[0], best[1]);
  for (int m = kWave / 2; m > 0; m >>= 1) top = fmaxf(top, __shfl_xor(top, m));
  if (lane == 0) s_top[wave] = top, s_reach[wave] = reach;
  if (tid == 0) s_count = 0;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWaves; ++w) top = fmaxf(top, s_top[w]), reach = max(reach, s_reach[w]);

  // A NaN or +inf makes the sum NaN.
  double sum = 0.0;
  const double from = top == -INFINITY ? 0.0 : static_cast<double>(top);
#pragma unroll
  for (int i = 0; i < kPer; ++i) sum += exp_of(static_cast<double>(x[i]) - from);
  for (int m = kWave / 2; m > 0; m >>= 1) sum += __shfl_xor(sum, m);
  if (lane == 0) s_sum[wave] = sum;

#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const uint64_t key = key_of(x[i], token(i));
    if (key != 0 && key >= reach) {
      const int32_t place = atomicAdd(&s_count, 1);
      if (place < kCapacity) s_list[place] = key;
    }
  }
  __syncthreads();
  const int64_t index = row * a.chunks + chunk;
  uint64_t* out = a.keys + index * g.count;
  if (tid == 0) {
    sum = 0.0;
    for (int w = 0; w < kWaves; ++w) sum += s_sum[w];
    a.sums[index] = sum;
    a.tops[index] = top;
  }
  const int32_t found = s_count;
  if (found <= kCapacity) {
    for (int32_t i = tid; i < found; i += kThreads) {
      const uint64_t mine = s_list[i];
      int32_t place = 0;
      for (int32_t j = 0; j < found; ++j) place += s_list[j] > mine ? 1 : 0;
      if (place < g.count) out[place] = mine;
    }
    for (int32_t i = found + tid; i < g.count; i += kThreads) out[i] = 0;
    return;
  }
  // Too many reach it (rows of which most logits are -inf in certain places): one after the other.
  uint64_t last = ~0ull;
  for (int32_t n = 0; n < g.count; ++n) {
    uint64_t most = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const uint64_t key = key_of(x[i], token(i));
      if (key < last) most = max(most, key);
    }
    most = group_max(most, kWave);
    __syncthreads();
    if (lane == 0) s_reach[wave] = most;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWaves; ++w) most = max(most, s_reach[w]);
    if (tid == 0) out[n] = most;
    last = most;
  }
}

// A group's chunks: the logarithms of its rows' sums, then one wavefront takes the best of the lists' first candidates `count`
// times. Lists are a row's chunks, each with falling keys.
__global__ __launch_bounds__(kThreads) void merge_kernel(const Select a) {
  extern __shared__ __align__(16) uint64_t s_keys[];  // the lists, where they fit
  __shared__ double s_norm[PKV_BEAM_MAX], s_score[PKV_BEAM_MAX];
  __shared__ uint8_t s_kind[PKV_BEAM_MAX];  // 0: no continuation, 1: its row's, 2: the end token
  __shared__ uint8_t s_at[kMaxLists];
  const pkv_beam& g = a.g;
  const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = tid / kWave;
  const int64_t group = blockIdx.x, row0 = group * g.num_beams;
  const int32_t lists = g.num_beams * a.chunks;
  const bool staged = static_cast<int64_t>(lists) * g.count <= kStagedKeys;
  const uint64_t* keys = a.keys + row0 * a.chunks * g.count;
  for (int32_t l = tid; l < lists; l += kThreads) s_at[l] = 0;
  if (staged) {
    for (int32_t i = tid; i < lists * g.count; i += kThreads) {
      if (looked_at(g, row0 + i / (a.chunks * g.count))) s_keys[i] = keys[i];
    }
  }
  for (int32_t b = wave; b < g.num_beams; b += kWaves) {
    const int64_t row = row0 + b;
    const bool look = looked_at(g, row);
    double sum = 0.0;
    float top = -INFINITY;
    if (look) {
      for (int32_t c = lane; c < a.chunks; c += kWave) top = fmaxf(top, a.tops[row * a.chunks + c]);
      for (int m = kWave / 2; m > 0; m >>= 1) top = fmaxf(top, __shfl_xor(top, m));
      for (int32_t c = lane; c < a.chunks; c += kWave) {
        const float one = a.tops[row * a.chunks + c];
        const double part = a.sums[row * a.chunks + c];
        if (part != 0.0) sum += part * exp_of(static_cast<double>(one) - static_cast<double>(top));
      }
      for (int m = kWave / 2; m > 0; m >>= 1) sum += __shfl_xor(sum, m);
    }
    if (lane == 0) {
      const bool counts = look && sum > 0.0 && sum < INFINITY && fabsf(top) < INFINITY;
      const float score = g.scores[row];
      s_norm[b] = counts ? static_cast<double>(top) + log(sum) : 0.0;
      s_score[b] = score;
      s_kind[b] = counts ? 1 : (fabsf(score) < INFINITY && g.finished && g.finished[row]) ? 2 : 0;
    }
  }
  __syncthreads();
  if (wave != 0) return;

  // The first candidate of list l that is left: its key (0: none) and its score.
  const auto head = [&](int32_t l, uint64_t& key, uint64_t& score) {
    const int32_t b = l / a.chunks, at = s_at[l], kind = s_kind[b];
    key = 0;
    score = 0;
    if (kind == 2 && l == b * a.chunks && at == 0) {
      key = 1;
      score = ordered(s_score[b]);
    } else if (kind == 1 && at < g.count) {
      key = staged ? s_keys[l * g.count + at] : keys[static_cast<int64_t>(l) * g.count + at];
      if (key != 0) score = ordered(s_score[b] + (static_cast<double>(number_of(static_cast<uint32_t>(key >> 32))) - s_norm[b]));
    }
  };
  // The best of this lane's lists. Of equal scores the lower beam's, and in a beam the larger key.
  int32_t mine = -1;
  uint64_t key = 0, score = 0;
  const auto look = [&]() {
    mine = -1;
    key = score = 0;
    for (int32_t l = lane; l < lists; l += kWave) {
      uint64_t k, s;
      head(l, k, s);
      if (k == 0) continue;
      const bool same = s == score && mine >= 0;
      if (mine < 0 || s > score || (same && l / a.chunks == mine / a.chunks && k > key)) mine = l, key = k, score = s;
    }
  };
  look();
  for (int32_t n = 0; n < g.count; ++n) {
    const int64_t out = group * g.count + n;
    const uint64_t most = group_max(score, kWave);
    uint64_t winners = __ballot(mine >= 0 && score == most);
    if (winners == 0) {  // nothing is left
      if (lane == 0) g.best_scores[out] = -INFINITY, g.best_beams[out] = 0, g.best_tokens[out] = g.end_token;
      continue;
    }
    if (winners & (winners - 1)) {  // equal scores
      const uint64_t inside = (winners >> lane) & 1 ? ~0ull : 0;
      // The lower beam, whose lists lower numbers have; then the larger key.
      const uint64_t beam = group_max(inside & static_cast<uint64_t>(PKV_BEAM_MAX - mine / a.chunks), kWave);
      const bool there = inside && static_cast<uint64_t>(PKV_BEAM_MAX - mine / a.chunks) == beam;
      const uint64_t largest = group_max(there ? key : 0, kWave);
      winners = __ballot(there && key == largest);
    }
    if (lane == __builtin_ctzll(winners)) {
      const int32_t b = mine / a.chunks;
      const bool ended = s_kind[b] == 2;
      const double at = ended ? s_score[b] : s_score[b] + (static_cast<double>(number_of(static_cast<uint32_t>(key >> 32))) - s_norm[b]);
      g.best_scores[out] = static_cast<float>(at);
      g.best_beams[out] = b;
      g.best_tokens[out] = ended ? g.end_token : static_cast<int32_t>(~static_cast<uint32_t>(key));
      s_at[mine] += 1;
      look();
    }
  }
}

// ---------------------------------------------------------------------------------------------
// Reordering. One workgroup for a child and a layer, of every state; a child that takes its parent's block over has nothing to
// copy. Every workgroup finds its group's moves by itself: the parents that earlier children named are a word of bits.
// Bound: HBM.
// ---------------------------------------------------------------------------------------------
struct Reorder {
  pkv_reorder g;
  int32_t unit[PKV_BEAM_STATES];  // bytes that are moved together: 16, 4 or 1
};

template <typename U>
__device__ __forceinline__ void copy_units(void* to, const void* from, int64_t count) {
  constexpr int kTogether = 4;
  for (int64_t i = threadIdx.x; i < count; i += kThreads * kTogether) {
    U x[kTogether];
#pragma unroll
    for (int j = 0; j < kTogether; ++j) {
      if (i + j * kThreads < count) x[j] = static_cast<const U*>(from)[i + j * kThreads];
    }
#pragma unroll
    for (int j = 0; j < kTogether; ++j) {
      if (i + j * kThreads < count) static_cast<U*>(to)[i + j * kThreads] = x[j];
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
  for (int32_t s = 0; s < g.num_states; ++s) {
    if (layer >= g.num_layers[s]) continue;
    char* base = static_cast<char*>(g.states[s]) + layer * g.layer_bytes[s];
    const int64_t bytes = g.block_bytes[s];
    char* to = base + target * bytes;
    const char* from = base + source * bytes;
    if (a.unit[s] == 16) copy_units<u32x4>(to, from, bytes / 16);
    else if (a.unit[s] == 4) copy_units<uint32_t>(to, from, bytes / 4);
    else copy_units<uint8_t>(to, from, bytes);
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
  const int64_t keys = static_cast<int64_t>(a.g.num_beams) * a.chunks * a.g.count;
  const uint32_t lds = keys <= kStagedKeys ? static_cast<uint32_t>(keys * sizeof(uint64_t)) : 0;
  hipLaunchKernelGGL(merge_kernel, dim3(static_cast<uint32_t>(a.g.num_groups)), block, lds, stream, a);
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
  int32_t layers = 1;
  for (int s = 0; s < g.num_states; ++s) {
    if (g.num_layers[s] < 0 || g.block_bytes[s] < 0 || g.layer_bytes[s] < 0) return PKV_EINVAL;
    if (g.num_layers[s] > 0 && g.block_bytes[s] > 0 && g.num_blocks > 0 && !g.states[s]) return PKV_EINVAL;
    if (g.num_layers[s] > 65535) return PKV_EUNSUPPORTED;
    layers = std::max(layers, g.num_layers[s]);
    const uint64_t bits = reinterpret_cast<uintptr_t>(g.states[s]) | static_cast<uint64_t>(g.block_bytes[s]) | static_cast<uint64_t>(g.layer_bytes[s]);
    a.unit[s] = bits % 16 == 0 ? 16 : bits % 4 == 0 ? 4 : 1;
  }
  if (g.num_groups > 0x7fffffff / (kThreads * PKV_BEAM_MAX)) return PKV_EUNSUPPORTED;
  if (g.num_groups == 0) return PKV_OK;
  if (!g.parents || !g.context_lens || (g.table_stride > 0 && (!g.new_tables || !g.block_tables))) return PKV_EINVAL;
  if (g.table_stride > 0 && g.new_tables == g.block_tables) return PKV_EINVAL;
  DeviceGuard guard(device);
  if (!guard.ok()) return PKV_EHIP;
  hipLaunchKernelGGL(reorder_kernel, dim3(static_cast<uint32_t>(g.num_groups * g.num_beams), static_cast<uint32_t>(layers)), dim3(kThreads), 0,
                     static_cast<hipStream_t>(stream), a);
  return check_launch();
}
