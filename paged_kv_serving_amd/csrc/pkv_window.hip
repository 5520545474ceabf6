// Paged causal attention with a sliding window and sinks, for grouped heads.
//
// A query row at position p of a sequence with context length c sees the keys j < min(c, p + 1) with
// j > p - window or j < sinks:
//     out = sum_j exp(s_j) v_j / sum_j exp(s_j),  s_j = scale * q . k_j
// with an online softmax (running maximum and sum), everything in float32 and one rounding to the
// output's type, but for the weights that a bfloat16 tile multiplies its values by (16 bits, at tile_kernel).
#include <math.h>

#include <algorithm>

#include "pkv_common.h"

namespace pkv {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / kWave;
constexpr int kTileQueries = 128;  // (row, head) pairs of a tile
constexpr int kMinRun = PKV_WINDOW_MIN_RUN;
constexpr float kLazyLog2 = 8.f;

typedef unsigned __int128 uint128;
typedef float floatx2 __attribute__((ext_vector_type(2)));
typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef float floatx16 __attribute__((ext_vector_type(16)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

struct Window {
  void* out;
  const void* queries;
  int64_t query_stride;
  const int32_t* positions;
  const int32_t* seqs;
  int64_t num_queries;
  const void* keys;
  const void* values;
  int64_t num_blocks;
  const int32_t* tables;
  const int32_t* contexts;
  float* workspace;
  int32_t block_size, table_stride, num_seqs, num_heads, num_kv_heads, group;
  int32_t window, sinks, max_context, splits;
  int32_t subgroups;       // of up to 16 query heads of a group
  int32_t tile_rows;       // rows of a tile: the aligned blocks of rows that runs lie in
  uint32_t tile_items;     // workgroups with tiles; the others have rows
  int32_t tiled;           // whether the tile pass computes the runs
  int32_t min_run;         // rows of one sequence next to each other that a tile takes
  int32_t* list;           // the rows that no tile takes (list_kernel); NULL without tiles
  float scale_log2;  // scale * log2(e): scores are kept in base 2
  float given_scale;  // the same before the next two
  // A negative scale of bfloat16 queries turns their signs instead, so that the largest product is the
  // largest score; a zero one clears them, so that a hidden key's -inf stays what it is.
  uint32_t keep, flip;
};

__device__ __forceinline__ float load_one(const float* p) { return *p; }
__device__ __forceinline__ float load_one(const uint16_t* p) { return __uint_as_float(static_cast<uint32_t>(*p) << 16); }
__device__ __forceinline__ void store_one(float* p, float v) { *p = v; }
__device__ __forceinline__ void store_one(uint16_t* p, float v) { *p = static_cast<uint16_t>(f32_to_bf16_bits(v)); }

// N adjacent values of an output row.
template <typename T, int N>
__device__ __forceinline__ void store_row(T* p, const float (&v)[N]) {
  if constexpr (sizeof(T) == 4 && N % 4 == 0) {
#pragma unroll
    for (int i = 0; i < N; i += 4) *reinterpret_cast<f32x4*>(p + i) = f32x4{v[i], v[i + 1], v[i + 2], v[i + 3]};
  } else if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < N; ++i) p[i] = v[i];
  } else {
    uint32_t w[N / 2];
#pragma unroll
    for (int i = 0; i < N / 2; ++i) w[i] = f32_to_bf16_bits(v[2 * i]) | (f32_to_bf16_bits(v[2 * i + 1]) << 16);
    if constexpr (N == 8) {
      *reinterpret_cast<u32x4*>(p) = u32x4{w[0], w[1], w[2], w[3]};
    } else if constexpr (N == 4) {
      *reinterpret_cast<u32x2*>(p) = u32x2{w[0], w[1]};
    } else {
      *reinterpret_cast<uint32_t*>(p) = w[0];
    }
  }
}

// Bits low .. high - 1 of a word, as far as it has them.
__device__ __forceinline__ uint32_t bits_between(int32_t low, int32_t high) {
  low = max(low, 0);
  high = min(high, 32);
  return low < high ? (0xffffffffu >> (32 - (high - low))) << low : 0u;
}

// The keys a row sees: [0, sinks) and [begin, end), or nothing.
struct Span {
  int32_t sinks, begin, end;
  __device__ __forceinline__ int32_t count() const { return sinks + end - begin; }
  __device__ __forceinline__ int32_t key(int32_t i) const { return i < sinks ? i : begin + (i - sinks); }
  // Which of items at .. at + 31 of a span of more rows this row sees.
  __device__ __forceinline__ uint32_t seen_of(const Span& all, int32_t at) const {
    const int32_t first = all.begin - all.sinks + at;  // the key of item `at`, were it past the sinks
    const uint32_t window = bits_between(begin - first, end - first) | bits_between(-first, sinks - first);
    if (at >= all.sinks) return window;
    const uint32_t early = bits_between(begin - at, end - at) | bits_between(-at, sinks - at);
    const uint32_t which = bits_between(0, all.sinks - at);
    return (early & which) | (window & ~which);
  }
  __device__ __forceinline__ bool sees(int32_t key) const { return key < end && (key >= begin || key < sinks); }
};

__device__ __forceinline__ Span span_of(const Window& a, int32_t seq, int32_t pos) {
  const int32_t context = min(a.contexts[seq], a.max_context);
  Span s;
  s.end = pos < 0 ? 0 : (pos < context ? pos + 1 : max(context, 0));
  s.begin = pos >= a.window ? pos - a.window + 1 : 0;
  s.begin = min(s.begin, s.end);
  s.sinks = min(a.sinks, s.begin);
  return s;
}

// Slot (block * block_size + offset) of a key; -1 in a block outside the pool.
__device__ __forceinline__ int32_t slot_of(const Window& a, const int32_t* table, int32_t key) {
  const uint32_t page = static_cast<uint32_t>(key) / static_cast<uint32_t>(a.block_size);
  const int32_t block = table[page];
  if (block < 0 || block >= a.num_blocks) return -1;
  return block * a.block_size + (key - static_cast<int32_t>(page) * a.block_size);
}

// Element offset of a slot's row of one head in the pools.
__device__ __forceinline__ int64_t row_of(const Window& a, int32_t slot, int32_t kv_head, int d) {
  return (static_cast<int64_t>(slot) * a.num_kv_heads + kv_head) * d;
}

// A row's split results in the workspace: maxima, sums, then the unnormalised outputs.
__device__ __forceinline__ int64_t split_index(const Window& a, int64_t t, int32_t head, int32_t split) {
  return (t * a.num_heads + head) * a.splits + split;
}
__device__ __forceinline__ float* split_acc(const Window& a, int64_t index, int d) {
  return a.workspace + (2 * a.num_queries * a.num_heads * a.splits + 3) / 4 * 4 + index * d;  // 16-byte aligned
}
__device__ __forceinline__ void store_split_sums(const Window& a, int64_t index, float top, float sum) {
  a.workspace[index] = top;
  a.workspace[a.num_queries * a.num_heads * a.splits + index] = sum;
}

// The maximum / sum over the four lanes {n, n + 16, n + 32, n + 48}, in each of them.
__device__ __forceinline__ float column_max(float x) {
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float column_sum(float x) {
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// Three bfloat16 pieces of pairs of floats, each the next 8 significant bits rounded to nearest:
// their sum is the float. What is not finite is its first piece alone.
__device__ __forceinline__ uint32_t take_piece(float& x0, float& x1) {
  const uint32_t pair = __builtin_bit_cast(uint32_t, __builtin_convertvector((floatx2{x0, x1}), bf16x2));
  const float h0 = bf16_lo(pair), h1 = bf16_hi(pair);
  x0 = fabsf(h0) < INFINITY ? x0 - h0 : 0.f;
  x1 = fabsf(h1) < INFINITY ? x1 - h1 : 0.f;
  return pair;
}

// Pieces without the guard: what is not finite turns into NaN, which its user looks for at the end.
__device__ __forceinline__ uint32_t cut_piece(float& x0, float& x1) {
  const uint32_t pair = __builtin_bit_cast(uint32_t, __builtin_convertvector((floatx2{x0, x1}), bf16x2));
  x0 -= bf16_lo(pair);
  x1 -= bf16_hi(pair);
  return pair;
}

// ---------------------------------------------------------------------------------------------
// One (row, head) over items [first, last) of a span, by the definition: a wavefront, 64 keys at a
// time; a lane scores one key, then owns dimensions. For rows that the matrix products cannot
// serve: an infinity or NaN does not survive being cut into pieces, and 0 * inf is not 0.
// ---------------------------------------------------------------------------------------------
template <typename QT, typename KVT, int D>
__device__ __forceinline__ void exact_row(const Window& a, int64_t t, int32_t head, int32_t seq, Span own, Span keys,
                                                    int32_t first, int32_t last, int32_t split) {
  constexpr int kOwn = (D + kWave - 1) / kWave;
  const int lane = threadIdx.x & (kWave - 1);
  const int32_t kv_head = head / a.group;
  const int32_t* table = a.tables + static_cast<int64_t>(seq) * a.table_stride;
  const QT* q = static_cast<const QT*>(a.queries) + t * a.query_stride + static_cast<int64_t>(head) * D;
  float top = -INFINITY, sum = 0.f, acc[kOwn] = {};
  for (int32_t at = first; at < last; at += kWave) {
    const int32_t key = at + lane < last ? keys.key(at + lane) : -1;
    const int32_t slot = key >= 0 && own.sees(key) ? slot_of(a, table, key) : -1;
    float score = -INFINITY;
    if (slot >= 0) {
      const KVT* k = static_cast<const KVT*>(a.keys) + row_of(a, slot, kv_head, D);
      score = 0.f;
      for (int d = 0; d < D; ++d) score += load_one(q + d) * load_one(k + d);
      score *= a.given_scale;
    }
    const uint64_t seen = __ballot(slot >= 0);
    if (seen == 0) continue;
    // The maximum leaves a NaN out; a visible NaN score makes the row NaN by its weight.
    float next = score;
    for (int m = kWave / 2; m > 0; m >>= 1) next = fmaxf(next, __shfl_xor(next, m));
    next = fmaxf(top, next);
    const float from = next == -INFINITY ? 0.f : next;
    const float keep = exp2f(top - from);
    const float p = slot >= 0 ? exp2f(score - from) : 0.f;
    float all = p;
    for (int m = kWave / 2; m > 0; m >>= 1) all += __shfl_xor(all, m);
    sum = sum * keep + all;
    top = next;
    for (int e = 0; e < kOwn; ++e) acc[e] *= keep;
    for (int j = 0; j < kWave; ++j) {
      if (!((seen >> j) & 1)) continue;
      const float pj = __shfl(p, j);
      const KVT* v = static_cast<const KVT*>(a.values) + row_of(a, __shfl(slot, j), kv_head, D);
      for (int e = 0; e < kOwn; ++e) {
        const int d = e * kWave + lane;
        if (d < D) acc[e] += pj * load_one(v + d);
      }
    }
  }
  if (a.splits == 1) {
    QT* out = static_cast<QT*>(a.out) + (t * a.num_heads + head) * D;
    for (int e = 0; e < kOwn; ++e) {
      const int d = e * kWave + lane;
      if (d < D) store_one(out + d, sum == 0.f ? 0.f : acc[e] / sum);
    }
    return;
  }
  const int64_t index = split_index(a, t, head, split);
  if (lane == 0) store_split_sums(a, index, top, sum);
  for (int e = 0; e < kOwn; ++e) {
    const int d = e * kWave + lane;
    if (d < D) split_acc(a, index, D)[d] = acc[e];
  }
}

// ---------------------------------------------------------------------------------------------
// Rows by themselves (decode): one workgroup per (row, key head, split) and up to 16 of the query
// heads that share the key head. The row's keys are handed to the wavefronts, four or eight, kKeys at a time.
// With lane l = (c = l / 16, n = l % 16):
//
//   S^T = K Q^T    16 keys x 16 heads per product, K straight from the pool as the left operand: lane
//                  (c, n) loads 16 bytes of key n's row. bfloat16 keys: v_mfma_f32_16x16x32_bf16, the
//                  lane's 8 dimensions are its 8 terms (float32 queries in three pieces); float32 keys:
//                  v_mfma_f32_16x16x4_f32, its 4 dimensions are 4 steps. Register r of the result is
//                  the score of key 4c + r for head n.
//   O^T = V^T P^T  V comes straight from the pool too: lane (c, i) loads kVWidth adjacent values of keys 4c + r
//                  and uses each in a product of its own. float32: v_mfma_f32_16x16x4_f32, step r taking keys
//                  4c + r of the lane groups c, P being the lane's own register r. bfloat16:
//                  v_mfma_f32_16x16x32_bf16 with the lane's eight keys of two blocks as its terms, P cut into three
//                  pieces, which hold all its bits: 3/16 of the float32 steps' time, which one row felt (2 key
//                  heads x 64, 516 keys: 10.4 -> 9.5 us). Two pieces leave out 2^-17 of a weight and took 8.8 us there
//                  and the same elsewhere (64 rows of up to 4100 keys, 32/8 heads x 128: 181 us with either).
//
// So nothing is staged: every key and value row goes from the pool to the registers that multiply it,
// and all heads of a group share one read of it. The loads of the next keys are
// issued before the present ones are used (a second set of registers for the values, so that they too
// are a whole round ahead, measured 3 to 5% slower).
//
// Bound: HBM. 64 rows with contexts of 2048 to 16384 and a window of 4096, 32 heads on 8 x 128, bfloat16, 1.1 GB:
// 180 us, 6.0 TB/s; contexts of 512 to 4096 and a window of 1024, 32 x 128 heads in float32, 2.2 GB: 345 us, 6.3
// TB/s (only reading one head's rows at a time in that pattern: 5.4).
// One row of 2 key heads x 64 and 516 keys: 9.5 us, the latency of a few dependent loads.
// ---------------------------------------------------------------------------------------------
template <typename QT, typename KVT, int D>
struct RowShape {
  static constexpr bool kBf16 = sizeof(KVT) == 2;
  static constexpr int kPieces = kBf16 ? (sizeof(QT) == 4 ? 3 : 1) : 1;
  static constexpr int kPPieces = 3;                         // of the weights, over bfloat16 values
  static constexpr int kBlocks = kBf16 && D <= 128 ? 2 : 1;  // 16-key blocks per round
  static constexpr int kKeys = 16 * kBlocks;
  static constexpr int kKLoads = kBf16 ? D / 32 : D / 16;    // 16-byte loads of a key row per lane
  static constexpr int kPerLane = D / 16;                    // values of a value row per lane
  static constexpr int kVWidth = kPerLane < 16 / int(sizeof(KVT)) ? kPerLane : 16 / int(sizeof(KVT));
  static constexpr int kVLoads = kPerLane / kVWidth;
  static constexpr int kVWords = kVWidth * int(sizeof(KVT)) / 4;
  static constexpr int kQRegs = kBf16 ? 4 * kKLoads * kPieces : D / 4;
};

template <int N>
struct Words {
  uint32_t w[N];
};

template <int N>
__device__ __forceinline__ Words<N> load_words(const void* p) {
  Words<N> x;
  if constexpr (N == 4) {
    const u32x4 v = __builtin_nontemporal_load(static_cast<const u32x4*>(p));
    x.w[0] = v.x, x.w[1] = v.y, x.w[2] = v.z, x.w[3] = v.w;
  } else if constexpr (N == 2) {
    const u32x2 v = __builtin_nontemporal_load(static_cast<const u32x2*>(p));
    x.w[0] = v.x, x.w[1] = v.y;
  } else {
    x.w[0] = __builtin_nontemporal_load(static_cast<const uint32_t*>(p));
  }
  return x;
}

// The rows that no tile computes, in any order: list[0] is their number. A tile takes the runs of a.min_run
// rows or more of one sequence next to each other inside an aligned block of a.tile_rows rows; rows
// outside every sequence are left out. One workgroup of independent wavefronts, 5.0 us for 4096 rows (with
// barriers for an order 6.3): a workgroup per possible row that finds out for itself took 48 us of a
// prefill of 8 x 512 rows.
constexpr int kListThreads = 1024;
__global__ __launch_bounds__(kListThreads) void list_kernel(const Window a) {
  __shared__ int32_t s_found;
  if (threadIdx.x == 0) s_found = 0;
  __syncthreads();
  const int lane = threadIdx.x & (kWave - 1);
  for (int64_t start = threadIdx.x - lane; start < a.num_queries; start += kListThreads) {
    const int64_t t = min(start + lane, a.num_queries - 1);
    const int32_t seq = a.seqs[t];
    const int64_t begin = t / a.tile_rows * a.tile_rows;
    const int64_t end = min(begin + a.tile_rows, a.num_queries);
    int32_t before[kMinRun - 1], after[kMinRun - 1];
#pragma unroll
    for (int i = 1; i < kMinRun; ++i) {
      before[i - 1] = a.seqs[max(t - i, begin)];
      after[i - 1] = a.seqs[min(t + i, end - 1)];
    }
    bool left = true, right = true;
    int32_t length = 1;
#pragma unroll
    for (int i = 1; i < kMinRun; ++i) {
      left = left && t - i >= begin && before[i - 1] == seq;
      right = right && t + i < end && after[i - 1] == seq;
      length += (left ? 1 : 0) + (right ? 1 : 0);
    }
    const bool listed = start + lane < a.num_queries && seq >= 0 && seq < a.num_seqs && length < a.min_run;
    const uint64_t ballot = __ballot(listed);
    int32_t at = 0;
    if (lane == 0 && ballot != 0) at = atomicAdd(&s_found, static_cast<int32_t>(__popcll(ballot)));
    at = __builtin_amdgcn_readfirstlane(at) + __popcll(ballot & ((1ull << lane) - 1));
    if (listed) a.list[1 + at] = static_cast<int32_t>(t);
  }
  __syncthreads();
  if (threadIdx.x == 0) a.list[0] = s_found;
}

// What a workgroup of the row pass keeps in LDS.
template <int D, int kRowWaves, int kPair>
struct RowScratch {
  float acc[kPair][kRowWaves / 2][D / 16 * 4 * kWave];
  float top[kPair][kRowWaves][kWave], sum[kPair][kRowWaves][kWave];
  int redo[kPair];
};

// The items of workgroup `block` of `blocks`.
template <typename QT, typename KVT, int D, int kRowWaves, int kPair>
__device__ __forceinline__ void row_pass(const Window& a, RowScratch<D, kRowWaves, kPair>& shared, uint32_t block, uint32_t blocks) {
  using S = RowShape<QT, KVT, D>;
  constexpr int kTiles = D / 16;  // output tiles of 16 dimensions
  auto& s_acc = shared.acc;
  auto& s_top = shared.top;
  auto& s_sum = shared.sum;
  auto& s_redo = shared.redo;
  const int lane = threadIdx.x & (kWave - 1), c = lane / 16, n = lane % 16;
  const int side = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave % kPair);  // which key head of the pair
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave / kPair);
  const uint32_t head_groups = a.num_kv_heads / kPair;
  // Items: heads fastest, so that one XCD has its share of the heads of every row.
  const int64_t rows = a.tiled ? a.list[0] : a.num_queries;
  const int64_t items = rows * a.splits * a.subgroups * head_groups;
  for (int64_t next = block; next < items; next += blocks) {
    uint32_t item = static_cast<uint32_t>(next);
    const int32_t kv_head = item % head_groups * kPair + side;
    item /= head_groups;
    const int32_t sub = item % static_cast<uint32_t>(a.subgroups);
    item /= static_cast<uint32_t>(a.subgroups);
    const int32_t split = item % static_cast<uint32_t>(a.splits);
    item /= static_cast<uint32_t>(a.splits);
    const int64_t t = a.tiled ? a.list[1 + item] : static_cast<int64_t>(item);
    const int32_t heads = min(16, a.group - sub * 16);
    const int32_t head0 = kv_head * a.group + sub * 16;
    const auto* keys = static_cast<const char*>(a.keys);
    const auto* values = static_cast<const char*>(a.values);
    const int64_t row_bytes = static_cast<int64_t>(a.num_kv_heads) * D * sizeof(KVT);
    const int64_t k_at = (static_cast<int64_t>(kv_head) * D + (S::kBf16 ? 8 : 4) * c) * sizeof(KVT);
    const int64_t v_at = (static_cast<int64_t>(kv_head) * D + S::kVWidth * n) * sizeof(KVT);
    const int32_t seq = a.seqs[t];
    if (seq < 0 || seq >= a.num_seqs) continue;
    const int32_t* table = a.tables + static_cast<int64_t>(seq) * a.table_stride;
    const Span span = span_of(a, seq, a.positions[t]);
    const int32_t count = span.count();
    const int32_t rounds = (count + S::kKeys - 1) / S::kKeys;
    const int32_t first = static_cast<int32_t>(static_cast<int64_t>(rounds) * split / a.splits);
    const int32_t last = static_cast<int32_t>(static_cast<int64_t>(rounds) * (split + 1) / a.splits);

    // The queries, the right operand of S^T: lane (c, n) holds its c's dimensions of head n.
    uint32_t qr[S::kQRegs];
    {
      const QT* q = static_cast<const QT*>(a.queries) + t * a.query_stride + static_cast<int64_t>(head0 + min(n, heads - 1)) * D;
      if constexpr (S::kBf16 && sizeof(QT) == 2) {
#pragma unroll
        for (int u = 0; u < S::kKLoads; ++u) {
          const u32x4 x = *reinterpret_cast<const u32x4*>(q + 32 * u + 8 * c);
#pragma unroll
          for (int e = 0; e < 4; ++e) qr[4 * u + e] = (x[e] & a.keep) ^ a.flip;
        }
      } else if constexpr (S::kBf16) {
#pragma unroll
        for (int u = 0; u < S::kKLoads; ++u) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float x0 = q[32 * u + 8 * c + 2 * e] * a.scale_log2, x1 = q[32 * u + 8 * c + 2 * e + 1] * a.scale_log2;
#pragma unroll
            for (int p = 0; p < 3; ++p) qr[4 * (p * S::kKLoads + u) + e] = take_piece(x0, x1);
          }
        }
      } else {
#pragma unroll
        for (int u = 0; u < S::kKLoads; ++u) {
          const f32x4 x = *reinterpret_cast<const f32x4*>(q + 16 * u + 4 * c);
#pragma unroll
          for (int e = 0; e < 4; ++e) qr[4 * u + e] = __float_as_uint(x[e] * a.scale_log2);
        }
      }
    }

    floatx4 o[kTiles];
#pragma unroll
    for (int b = 0; b < kTiles; ++b) o[b] = floatx4{0.f, 0.f, 0.f, 0.f};
    float top = -INFINITY, sum = 0.f;

    // Slot of the key that this lane looks up for a round (lanes past kKeys repeat).
    auto look_up = [&](int32_t round) {
      const int32_t i = round * S::kKeys + lane % S::kKeys;
      return round < last && i < count ? slot_of(a, table, span.key(i)) : -1;
    };
    Words<4> kx[S::kBlocks][S::kKLoads];
    Words<S::kVWords> vx[S::kBlocks][4][S::kVLoads];
    auto load_keys = [&](int32_t slot) {
#pragma unroll
      for (int j = 0; j < S::kBlocks; ++j) {
        const char* p = keys + max(__shfl(slot, 16 * j + n), 0) * row_bytes + k_at;
#pragma unroll
        for (int u = 0; u < S::kKLoads; ++u) kx[j][u] = load_words<4>(p + u * 64);
      }
    };
    auto load_values = [&](int32_t slot) {
#pragma unroll
      for (int j = 0; j < S::kBlocks; ++j) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const char* p = values + max(__shfl(slot, 16 * j + 4 * c + r), 0) * row_bytes + v_at;
#pragma unroll
          for (int g = 0; g < S::kVLoads; ++g) vx[j][r][g] = load_words<S::kVWords>(p + g * 16 * S::kVWidth * int(sizeof(KVT)));
        }
      }
    };

    constexpr uint64_t kAll = S::kKeys == 32 ? 0xffffffffull : 0xffffull;
    int32_t round = first + wave;
    int32_t slot = look_up(round);
    uint32_t live = static_cast<uint32_t>(__ballot(slot >= 0) & kAll);  // the round's keys that count
    if (live != 0) {
      load_keys(slot);
      load_values(slot);
    }
    int32_t slot_next = look_up(round + kRowWaves);
    for (; round < last; round += kRowWaves) {
      const uint32_t live_next = static_cast<uint32_t>(__ballot(slot_next >= 0) & kAll);
      floatx4 st[S::kBlocks];
      if (live != 0) {
#pragma unroll
        for (int j = 0; j < S::kBlocks; ++j) {
          st[j] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int u = 0; u < S::kKLoads; ++u) {
            if constexpr (S::kBf16) {
#pragma unroll
              for (int p = S::kPieces - 1; p >= 0; --p) {  // the smallest pieces first
                const uint32_t* q = qr + 4 * (p * S::kKLoads + u);
                st[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, kx[j][u]),
                                                                __builtin_bit_cast(bf16x8, (u32x4{q[0], q[1], q[2], q[3]})), st[j], 0, 0, 0);
              }
            } else {
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                st[j] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(kx[j][u].w[e]), __uint_as_float(qr[4 * u + e]), st[j], 0, 0, 0);
              }
            }
          }
        }
      }
      if (live_next != 0) load_keys(slot_next);
      if (live != 0) {
        float most = -INFINITY;
#pragma unroll
        for (int j = 0; j < S::kBlocks; ++j) {
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            if constexpr (sizeof(QT) == 2) st[j][r] *= a.scale_log2;
            st[j][r] = (live >> (16 * j + 4 * c + r)) & 1 ? st[j][r] : -INFINITY;
            most = fmaxf(most, st[j][r]);
          }
        }
        most = column_max(most);
        if (__ballot(most > top) != 0) {
          const float next = fmaxf(top, most);
          const float keep = next == -INFINITY ? 1.f : fast_exp2(top - next);
          sum *= keep;
#pragma unroll
          for (int b = 0; b < kTiles; ++b) o[b] *= keep;
          top = next;
        }
        const float from = top == -INFINITY ? 0.f : top;
#pragma unroll
        for (int j = 0; j < S::kBlocks; ++j) {
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            st[j][r] = fast_exp2(st[j][r] - from);
            sum += st[j][r];
          }
        }
#pragma unroll
        for (int j = 0; j < S::kBlocks; ++j) {
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            if (live != kAll && !((live >> (16 * j + 4 * c + r)) & 1)) {  // 0 * inf is not 0
#pragma unroll
              for (int g = 0; g < S::kVLoads; ++g) {
#pragma unroll
                for (int w = 0; w < S::kVWords; ++w) vx[j][r][g].w[w] = 0;
              }
            }
            if constexpr (!S::kBf16) {
#pragma unroll
              for (int g = 0; g < S::kVLoads; ++g) {
#pragma unroll
                for (int e = 0; e < S::kVWidth; ++e) {
                  o[g * S::kVWidth + e] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(vx[j][r][g].w[e]), st[j][r],
                                                                               o[g * S::kVWidth + e], 0, 0, 0);
                }
              }
            }
          }
        }
        if constexpr (S::kBf16) {
          // Term 4j + r of a lane's eight is key 16j + 4c + r: of the weights its own registers, of a dimension
          // the eight values of it that it has loaded.
          u32x4 pr[S::kPPieces] = {};
#pragma unroll
          for (int j = 0; j < S::kBlocks; ++j) {
#pragma unroll
            for (int r = 0; r < 4; r += 2) {
              float x0 = st[j][r], x1 = st[j][r + 1];
#pragma unroll
              for (int p = 0; p < S::kPPieces; ++p) pr[p][2 * j + r / 2] = cut_piece(x0, x1);
            }
          }
#pragma unroll
          for (int g = 0; g < S::kVLoads; ++g) {
#pragma unroll
            for (int e = 0; e < S::kVWidth; ++e) {
              u32x4 v = {};
#pragma unroll
              for (int j = 0; j < S::kBlocks; ++j) {
#pragma unroll
                for (int r = 0; r < 4; r += 2) {
                  v[2 * j + r / 2] = __builtin_amdgcn_perm(vx[j][r + 1][g].w[e / 2], vx[j][r][g].w[e / 2], e % 2 ? 0x07060302 : 0x05040100);
                }
              }
#pragma unroll
              for (int p = S::kPPieces - 1; p >= 0; --p) {
                o[g * S::kVWidth + e] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                    __builtin_bit_cast(bf16x8, v), __builtin_bit_cast(bf16x8, pr[p]), o[g * S::kVWidth + e], 0, 0, 0);
              }
            }
          }
        }
      }
      if (live_next != 0) load_values(slot_next);
      live = live_next;
      slot_next = look_up(round + 2 * kRowWaves);
    }
    sum = column_sum(sum);

    // The wavefronts' results, lane by lane: every wavefront holds the same places.
    __syncthreads();  // the row before has been read
    s_top[side][wave][lane] = top;
    s_sum[side][wave][lane] = sum;
    __syncthreads();
    float all = -INFINITY;
#pragma unroll
    for (int w = 0; w < kRowWaves; ++w) all = fmaxf(all, s_top[side][w][lane]);
    const float base = all == -INFINITY ? 0.f : all;
    const float mine = fast_exp2(top - base);
#pragma unroll
    for (int b = 0; b < kTiles; ++b) o[b] *= mine;
    sum = 0.f;
#pragma unroll
    for (int w = 0; w < kRowWaves; ++w) sum += s_sum[side][w][lane] * fast_exp2(s_top[side][w][lane] - base);
#pragma unroll
    for (int half = kRowWaves / 2; half > 0; half /= 2) {
      if (wave >= half && wave < 2 * half) {
#pragma unroll
        for (int b = 0; b < kTiles; ++b) {
#pragma unroll
          for (int r = 0; r < 4; ++r) s_acc[side][wave - half][(b * 4 + r) * kWave + lane] = o[b][r];
        }
      }
      __syncthreads();
      if (wave < half) {
#pragma unroll
        for (int b = 0; b < kTiles; ++b) {
#pragma unroll
          for (int r = 0; r < 4; ++r) o[b][r] += s_acc[side][wave][(b * 4 + r) * kWave + lane];
        }
      }
      __syncthreads();
    }
    if constexpr (S::kBf16) {  // what is not finite is computed again from whole numbers
      if (wave == 0) {
        bool bad = false;
#pragma unroll
        for (int b = 0; b < kTiles; ++b) {
#pragma unroll
          for (int r = 0; r < 4; ++r) bad = bad || !(fabsf(o[b][r]) < INFINITY);
        }
        const uint64_t any = __ballot((bad || !(fabsf(sum) < INFINITY)) && n < heads);
        if (lane == 0) s_redo[side] = any != 0;
      }
      __syncthreads();
      if (s_redo[side]) {
        for (int g = wave; g < heads; g += kRowWaves) {
          exact_row<QT, KVT, D>(a, t, head0 + g, seq, span, span, min(first * S::kKeys, count), min(last * S::kKeys, count), split);
        }
        continue;
      }
    }
    if (wave != 0 || n >= heads) continue;
    // Register r of output tile (g, e) is dimension 16 kVWidth g + kVWidth (4c + r) + e of head n.
    const int64_t out_row = t * a.num_heads + head0 + n;
    if (a.splits == 1) {
      const float scale = sum == 0.f ? 0.f : 1.f / sum;
      QT* out = static_cast<QT*>(a.out) + out_row * D;
#pragma unroll
      for (int g = 0; g < S::kVLoads; ++g) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          float x[S::kVWidth];
#pragma unroll
          for (int e = 0; e < S::kVWidth; ++e) x[e] = sum == 0.f ? 0.f : o[g * S::kVWidth + e][r] * scale;
          store_row<QT, S::kVWidth>(out + 16 * S::kVWidth * g + S::kVWidth * (4 * c + r), x);
        }
      }
    } else {
      const int64_t index = split_index(a, t, head0 + n, split);
      if (c == 0) store_split_sums(a, index, all, sum);
      if (sum == 0.f) continue;
#pragma unroll
      for (int g = 0; g < S::kVLoads; ++g) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          float x[S::kVWidth];
#pragma unroll
          for (int e = 0; e < S::kVWidth; ++e) x[e] = o[g * S::kVWidth + e][r];
          store_row<float, S::kVWidth>(split_acc(a, index, D) + 16 * S::kVWidth * g + S::kVWidth * (4 * c + r), x);
        }
      }
    }
  }
}

template <typename QT, typename KVT, int D, int kRowWaves, int kPair>
__global__ __launch_bounds__(kRowWaves * kPair * kWave) void row_kernel(const Window a) {
  __shared__ RowScratch<D, kRowWaves, kPair> shared;
  row_pass<QT, KVT, D, kRowWaves, kPair>(a, shared, blockIdx.x, gridDim.x);
}

// ---------------------------------------------------------------------------------------------
// Runs of rows (prompt chunks): one workgroup per (aligned block of rows, key head, split), whose
// kTileQueries = 128 queries are the block's rows times the heads that share the key head, 32 to a
// wavefront. Packing the heads keeps the rows of a tile close together, so a tile reads little more
// than one row's window, and serves every head of the group from one copy of the keys.
//
// With lane l = (c = l / 32, n = l % 32) and v_mfma_f32_32x32x16_bf16:
//   S^T = K Q^T    32 keys x 32 queries per product chain; K from LDS, 16 bytes of key n's row per lane,
//                  Q from registers. Register r holds the score of key 8 (r / 4) + 4c + r % 4.
//   O^T = V^T P^T  step s takes 16 keys, element e of lane group c being key 16 s + 8 (e / 4) + 4 c + e % 4:
//                  the P operand is the lane's own registers 8 s + e, rounded to pieces, and V is read
//                  transposed (ds_read_b64_tr_b16), four keys of one dimension at a time.
// Float32 operands are cut into three bfloat16 pieces, whose products (the 3 or 6 largest of them) add
// up to the float32 product within one float32 rounding. bfloat16 queries and keys are one piece; their
// weights P are two, 16 bits, off by 2^-17 of a weight: 2^-8 of the output's own rounding, which one piece
// would double. Three pieces would keep every bit and cost 16% (8 x 512 rows: 126 -> 147 us, 14% x 64, 13% x 256).
// Their sum is taken of the float32 weights.
//
// Keys and values are staged kKeys at a time in two LDS buffers: while one is used, the next tile's rows
// are in flight (bfloat16 pools: straight to LDS; float32 pools: to registers, cut on their way to LDS) and
// the slots of the one after are looked up.
//
// Bound: latency. 8 x 512 rows behind up to 2048 others, window 1024, bfloat16, 32 heads on 8 x 128: 126 us, 5 of
// them the list's, 550 TFLOP/s of visible products (1390 in a large library product); x 64 91 us, 16 on 4 x 256 167.
// Of the first's 304,000 cycles the matrix units are busy in 29%, vector instructions issue in 38% and LDS works in 21%,
// at two wavefronts per SIMD: a step's values are waited for before its products. Float32 queries over bfloat16
// 234 us (three products for one), over float32 438 (six, at one wavefront per SIMD). One piece of P instead of two was
// 9% faster.
// ---------------------------------------------------------------------------------------------
// float32 queries of head_dim 256 have no tiles (their pieces do not fit the registers, nor float32 pools' LDS): their
// rows go by themselves.
constexpr bool tiles_of(int q_size, int head_dim) { return q_size == 2 || head_dim <= 128; }

template <typename QT, typename KVT, int D>
struct TileShape {
  static constexpr int kQPieces = sizeof(QT) == 4 ? 3 : 1;
  static constexpr int kKvPieces = sizeof(KVT) == 4 ? 3 : 1;
  static constexpr int kPPieces = sizeof(QT) == 4 ? 3 : 2;
  static constexpr int kKeys = (sizeof(KVT) == 2 && D <= 128) || D == 32 ? 64 : 32;
  static constexpr int kChunks = D / 8;                                // 16-byte chunks of a bfloat16 row
  static constexpr int kPlane = kKeys * D;                             // elements of one piece of a staged tile
  static constexpr int kStaged = kKeys * kChunks / kThreads;           // chunks of a tile per thread, K and V each
  static constexpr int kLds = 2 * 2 * kKvPieces * kPlane * 2;          // bytes: two buffers of K and V
  static constexpr int kWaves = kLds <= 81920 && sizeof(QT) == 2 && D <= 128 ? 2 : 1;  // per SIMD
  static constexpr bool kFits = tiles_of(sizeof(QT), D);
  static_assert(!kFits || kLds <= 160 * 1024 - 2048, "a tile's buffers, slots and live bits fit LDS");
};

// The products of pieces i of one operand and j of the other that are computed: i + j <= 2.
__device__ __forceinline__ constexpr bool counted(int i, int j) { return i + j <= 2; }

__device__ __forceinline__ floatx16 mfma32(const u32x4& a, const u32x4& b, const floatx16& c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// Chunks of a staged row are permuted so that the lanes of a read lie in different banks: the key
// operand reads one chunk of 32 rows, the value operand two neighbouring ones of four rows.
template <int D>
__device__ __forceinline__ int key_chunk(int row, int chunk) {
  return D >= 64 ? chunk ^ (row & 7) : chunk ^ ((row >> 1) & 3);
}
template <int D>
__device__ __forceinline__ int value_chunk(int row, int chunk) {
  return D >= 64 ? chunk ^ (2 * (row & 3)) : chunk;
}

// The value operands of one step for `N` output tiles: of each, four keys of a lane's dimension from `lo` and
// four from 8 rows on. The reads of a step are issued together and waited for once, in one block: as separate
// ones the compiler waits for each, and for the next tile's rows on their way to LDS besides, which it takes
// for the same memory. Output tiles b and b + 2 lie 128 bytes apart; even and odd ones have their own address.
template <int N, int kRowBytes>
__device__ __forceinline__ void read_values(uint32_t even, uint32_t odd, u32x4 (&v)[N]) {
  u32x2 lo[N], hi[N];
  if constexpr (N == 1) {
    asm volatile(
        "ds_read_b64_tr_b16 %0, %2\n\tds_read_b64_tr_b16 %1, %2 offset:%3\n\ts_waitcnt lgkmcnt(0)"
        : "=&v"(lo[0]), "=&v"(hi[0])
        : "v"(even), "i"(8 * kRowBytes)
        : "memory");
  } else if constexpr (N == 2) {
    asm volatile(
        "ds_read_b64_tr_b16 %0, %4\n\tds_read_b64_tr_b16 %1, %4 offset:%6\n\t"
        "ds_read_b64_tr_b16 %2, %5\n\tds_read_b64_tr_b16 %3, %5 offset:%6\n\ts_waitcnt lgkmcnt(0)"
        : "=&v"(lo[0]), "=&v"(hi[0]), "=&v"(lo[1]), "=&v"(hi[1])
        : "v"(even), "v"(odd), "i"(8 * kRowBytes)
        : "memory");
  } else {
    static_assert(N == 4, "one, two or four output tiles at a time");
    asm volatile(
        "ds_read_b64_tr_b16 %0, %8\n\tds_read_b64_tr_b16 %1, %8 offset:%10\n\t"
        "ds_read_b64_tr_b16 %2, %9\n\tds_read_b64_tr_b16 %3, %9 offset:%10\n\t"
        "ds_read_b64_tr_b16 %4, %8 offset:128\n\tds_read_b64_tr_b16 %5, %8 offset:%11\n\t"
        "ds_read_b64_tr_b16 %6, %9 offset:128\n\tds_read_b64_tr_b16 %7, %9 offset:%11\n\ts_waitcnt lgkmcnt(0)"
        : "=&v"(lo[0]), "=&v"(hi[0]), "=&v"(lo[1]), "=&v"(hi[1]), "=&v"(lo[2]), "=&v"(hi[2]), "=&v"(lo[3]), "=&v"(hi[3])
        : "v"(even), "v"(odd), "i"(8 * kRowBytes), "i"(8 * kRowBytes + 128)
        : "memory");
  }
#pragma unroll
  for (int b = 0; b < N; ++b) v[b] = u32x4{lo[b].x, lo[b].y, hi[b].x, hi[b].y};
}

// What a tile's rows in no block of the pool are read from.
__device__ const u32x4 kZeros = {0, 0, 0, 0};

__device__ __forceinline__ uint32_t lds_address(const uint16_t* p) {
  return static_cast<uint32_t>(reinterpret_cast<uintptr_t>((const __attribute__((address_space(3))) uint16_t*)(p)));
}

// 16 bytes per lane from global memory to LDS: `to`, the same in every lane, is the first lane's place.
__device__ __forceinline__ void load_to_lds(const void* from, uint16_t* to) {
  typedef const __attribute__((address_space(1))) void* global_ptr;
  typedef __attribute__((address_space(3))) void* lds_ptr;
  __builtin_amdgcn_global_load_lds((global_ptr)(from), (lds_ptr)(to), 16, 0, 0);
}

__device__ __forceinline__ int32_t wave_min(int32_t x) {
  for (int m = kWave / 2; m > 0; m >>= 1) x = min(x, __shfl_xor(x, m));
  return __builtin_amdgcn_readfirstlane(x);
}
__device__ __forceinline__ int32_t wave_max(int32_t x) {
  for (int m = kWave / 2; m > 0; m >>= 1) x = max(x, __shfl_xor(x, m));
  return __builtin_amdgcn_readfirstlane(x);
}

template <typename QT, typename KVT, int D>
__global__ __launch_bounds__(kThreads, (TileShape<QT, KVT, D>::kWaves)) void tile_kernel(const Window a) {
  using S = TileShape<QT, KVT, D>;
  constexpr int kBlocks = D / 32;       // output tiles of 32 dimensions
  constexpr int kSteps = D / 16;        // steps of a score product
  constexpr int kSub = S::kKeys / 32;   // 32-key blocks of a staged tile
  // Steps whose keys are read together: one at a time the compiler waits for each read before its product
  // (8 sequences of 512 tokens in bfloat16: 141 us, and 137 by fours).
  constexpr int kAhead = S::kKvPieces > 1 || kSteps < 4 ? 2 : 4;
  constexpr int kTogether = kBlocks < 4 ? kBlocks : 4;  // output tiles whose values are read together
  extern __shared__ __align__(16) uint16_t s_kv[];  // [buffer][K, V][piece][key][D]
  __shared__ int32_t s_slot[3][S::kKeys];
  __shared__ uint64_t s_live[3];
  const int tid = threadIdx.x, lane = tid & (kWave - 1), c = lane / 32, n = lane % 32;
  const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  // The rows outside the runs in the same launch, before bfloat16's tiles and behind float32's, which take
  // longer (24 rows beside 2 x 301, window 500, 16 heads x 64, float32 over bfloat16: 44 us, before the tiles 49; 64 rows of
  // up to 4096 keys beside 512, 32/8 heads x 128, bfloat16: 225 us, behind the tiles 247). In a launch of their own after
  // the tiles the first took 35% longer, the second 4%.
  constexpr bool kRowsFirst = sizeof(QT) == 2;
  const uint32_t row_blocks = gridDim.x - a.tile_items, before = kRowsFirst ? row_blocks : a.tile_items;
  if ((blockIdx.x < before) == kRowsFirst) {
    row_pass<QT, KVT, D, kWaves, 1>(a, *reinterpret_cast<RowScratch<D, kWaves, 1>*>(s_kv), blockIdx.x - (kRowsFirst ? 0 : before), row_blocks);
    return;
  }
  uint32_t item = blockIdx.x - (kRowsFirst ? before : 0);
  const int32_t kv_head = item % static_cast<uint32_t>(a.num_kv_heads);
  item /= static_cast<uint32_t>(a.num_kv_heads);
  const int32_t split = item % static_cast<uint32_t>(a.splits);
  const int64_t block0 = static_cast<int64_t>(item / static_cast<uint32_t>(a.splits)) * a.tile_rows;
  const int64_t block1 = min(block0 + a.tile_rows, a.num_queries);
  const KVT* keys = static_cast<const KVT*>(a.keys);
  const KVT* values = static_cast<const KVT*>(a.values);
  const void* zeros = &kZeros;
  auto plane = [&](int buffer, int which, int piece) {
    return s_kv + ((buffer * 2 + which) * S::kKvPieces + piece) * S::kPlane;
  };

  // The runs: rows that begin a stretch of one sequence (all 128 rows' bits at once; row after row, the look
  // alone took 15 us of a chunk of 128), and of these the ones whose stretch is long enough.
  uint128 starts, runs;
  {
    uint64_t same[2], known[2], inside[2];
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      const int64_t t = block0 + w * kWave + lane;
      const int32_t seq = a.seqs[min(t, block1 - 1)], last = a.seqs[max(min(t, block1) - 1, block0)];
      inside[w] = __ballot(t < block1);
      same[w] = __ballot(t < block1 && t > block0 && seq == last);
      known[w] = __ballot(t < block1 && seq >= 0 && seq < a.num_seqs);
    }
    const uint128 alike = static_cast<uint128>(same[1]) << 64 | same[0];
    starts = (static_cast<uint128>(inside[1]) << 64 | inside[0]) & ~alike;
    runs = starts & (static_cast<uint128>(known[1]) << 64 | known[0]);
    for (int i = 1; i < a.min_run; ++i) runs &= alike >> i;
  }
  const auto first_of = [](uint128 bits) {
    const uint64_t low = static_cast<uint64_t>(bits);
    return low != 0 ? __builtin_ctzll(low) : 64 + __builtin_ctzll(static_cast<uint64_t>(bits >> 64));
  };
  for (; runs != 0; runs &= runs - 1) {
    const int at = first_of(runs);
    const uint128 behind = starts & ~((static_cast<uint128>(2) << at) - 1);
    const int64_t run0 = block0 + at, run1 = behind != 0 ? block0 + first_of(behind) : block1;
    const int32_t seq = a.seqs[run0];
    const int32_t* table = a.tables + static_cast<int64_t>(seq) * a.table_stride;
    const int32_t rows = static_cast<int32_t>(run1 - run0);

    // The keys that any row sees: the sinks, then [begin, end).
    Span all{0, INT32_MAX, 0};
    for (int32_t i = lane; i < rows; i += kWave) {
      const Span one = span_of(a, seq, a.positions[run0 + i]);
      if (one.count() > 0) all.begin = min(all.begin, one.begin), all.end = max(all.end, one.end);
    }
    all.begin = wave_min(all.begin);
    all.end = wave_max(all.end);
    all.begin = min(all.begin, all.end);  // no row sees any: nothing
    all.sinks = min(a.sinks, all.begin);
    const int32_t count = all.count();
    const int32_t tiles = (count + S::kKeys - 1) / S::kKeys;
    const int32_t first = static_cast<int32_t>(static_cast<int64_t>(tiles) * split / a.splits);
    const int32_t last = static_cast<int32_t>(static_cast<int64_t>(tiles) * (split + 1) / a.splits);

    // This lane's query: column n of its wavefront.
    const int32_t m = wave * 32 + n;
    const int32_t local = m / a.group;
    const bool active = local < rows;
    const int64_t t = run0 + min(local, rows - 1);
    const int32_t head = kv_head * a.group + (m - local * a.group);
    const Span own = span_of(a, seq, a.positions[t]);
    // Keys [wave_begin, wave_end) and sinks are all that this wavefront's rows see; every one of them
    // sees [full_begin, full_end).
    const bool sees = active && own.count() > 0;
    const int32_t wave_begin = wave_min(sees ? own.begin : INT32_MAX);
    const int32_t wave_end = wave_max(sees ? own.end : 0);
    const int32_t wave_sinks = wave_max(sees ? own.sinks : 0);
    const int32_t full_begin = wave_max(!active ? 0 : sees ? own.begin : INT32_MAX);
    const int32_t full_end = wave_min(!active ? INT32_MAX : own.end);

    // The queries, the right operand of S^T: lane (c, n) holds dimensions 16 s + 8 c of query n.
    u32x4 qr[S::kQPieces][kSteps];
    {
      const QT* q = static_cast<const QT*>(a.queries) + t * a.query_stride + static_cast<int64_t>(head) * D + 8 * c;
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
        if constexpr (sizeof(QT) == 2) {
          qr[0][s] = (*reinterpret_cast<const u32x4*>(q + 16 * s) & a.keep) ^ a.flip;
        } else {
          f32x4 x[2] = {*reinterpret_cast<const f32x4*>(q + 16 * s), *reinterpret_cast<const f32x4*>(q + 16 * s + 4)};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float x0 = x[e / 2][e % 2 * 2] * a.scale_log2, x1 = x[e / 2][e % 2 * 2 + 1] * a.scale_log2;
#pragma unroll
            for (int p = 0; p < S::kQPieces; ++p) qr[p][s][e] = cut_piece(x0, x1);
          }
        }
      }
    }

    floatx16 o[kBlocks];
#pragma unroll
    for (int b = 0; b < kBlocks; ++b) {
#pragma unroll
      for (int r = 0; r < 16; ++r) o[b][r] = 0.f;
    }
    float top = -INFINITY, sum = 0.f;

    // Staging. Slots of a tile by the first wavefront, rows by all. A tile's table entries are loaded long
    // before they are used, and before the rows that are loaded in between: loads arrive in order.
    struct Entry {
      int32_t key, block;
    };
    auto look_up = [&](int32_t tile) {
      const int32_t i = tile * S::kKeys + tid;
      Entry e{-1, -1};
      if (tid < S::kKeys && tile < last && i < count) {
        e.key = all.key(i);
        e.block = table[static_cast<uint32_t>(e.key) / static_cast<uint32_t>(a.block_size)];
      }
      return e;
    };
    auto keep_slots = [&](int32_t tile, const Entry& e) {
      if (wave == 0) {
        const int32_t slot = e.block < 0 || e.block >= a.num_blocks
                                 ? -1
                                 : e.block * a.block_size + static_cast<int32_t>(static_cast<uint32_t>(e.key) % static_cast<uint32_t>(a.block_size));
        const uint64_t live = __ballot(slot >= 0);
        if (tid < S::kKeys) s_slot[tile % 3][tid] = slot;
        if (tid == 0) s_live[tile % 3] = live;
      }
    };
    constexpr int kWide = sizeof(KVT) / 2;  // 16-byte loads of a chunk
    u32x4 kx[S::kStaged][kWide], vx[S::kStaged][kWide];
    auto load = [&](int32_t tile, int buffer) {
#pragma unroll
      for (int i = 0; i < S::kStaged; ++i) {
        const int at = tid + i * kThreads, row = at / S::kChunks, chunk = at % S::kChunks;
        const int32_t slot = s_slot[tile % 3][row];
        const int64_t from = row_of(a, slot, kv_head, D);
        if constexpr (kWide == 1) {
          // Straight to LDS, where a wavefront's 64 chunks lie one after the other: the permutation is made
          // by which chunk of the row a lane fetches (it is its own inverse).
          const void* k = slot >= 0 ? static_cast<const void*>(keys + from + 8 * key_chunk<D>(row, chunk)) : zeros;
          const void* v = slot >= 0 ? static_cast<const void*>(values + from + 8 * value_chunk<D>(row, chunk)) : zeros;
          load_to_lds(k, plane(buffer, 0, 0) + 8 * (wave * kWave + i * kThreads));
          load_to_lds(v, plane(buffer, 1, 0) + 8 * (wave * kWave + i * kThreads));
        } else {
#pragma unroll
          for (int w = 0; w < kWide; ++w) {
            kx[i][w] = slot >= 0 ? *reinterpret_cast<const u32x4*>(keys + from + chunk * 8 + w * 4) : u32x4{0, 0, 0, 0};
            vx[i][w] = slot >= 0 ? *reinterpret_cast<const u32x4*>(values + from + chunk * 8 + w * 4) : u32x4{0, 0, 0, 0};
          }
        }
      }
    };
    auto put = [&](int buffer, int which, int i, const u32x4 (&x)[kWide]) {
      const int at = tid + i * kThreads, row = at / S::kChunks, chunk = at % S::kChunks;
      const int to = row * D + 8 * (which == 0 ? key_chunk<D>(row, chunk) : value_chunk<D>(row, chunk));
      u32x4 piece[3];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float x0 = __uint_as_float(x[e / 2][e % 2 * 2]), x1 = __uint_as_float(x[e / 2][e % 2 * 2 + 1]);
#pragma unroll
        for (int p = 0; p < 3; ++p) piece[p][e] = cut_piece(x0, x1);
      }
#pragma unroll
      for (int p = 0; p < 3; ++p) *reinterpret_cast<u32x4*>(plane(buffer, which, p) + to) = piece[p];
    };
    auto stage = [&](int buffer) {
      if constexpr (kWide == 1) {
        __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0): this wavefront's loads to LDS have arrived
      } else {
#pragma unroll
        for (int i = 0; i < S::kStaged; ++i) {
          put(buffer, 0, i, kx[i]);
          put(buffer, 1, i, vx[i]);
        }
      }
    };

    __syncthreads();  // the run before is done with LDS
    keep_slots(first, look_up(first));
    keep_slots(first + 1, look_up(first + 1));
    __syncthreads();
    if (first < last) {
      load(first, 0);
      stage(0);
    }
    __syncthreads();
    for (int32_t tile = first; tile < last; ++tile) {
      const int buffer = (tile - first) & 1;
      const Entry ahead = look_up(tile + 2);
      if (tile + 1 < last) load(tile + 1, buffer ^ 1);
      const uint64_t tile_live = s_live[tile % 3];
      // The tile's 32-key blocks one after the other through the scores, together through the softmax.
      floatx16 st[kSub];
      bool any = false;
#pragma unroll
      for (int j = 0; j < kSub; ++j) {
        const int32_t at = tile * S::kKeys + 32 * j;  // the block's first item of the span
        const int32_t key0 = all.key(at), key1 = all.key(min(at + 31, count - 1));
        const bool needed = at < count && key0 < wave_end && (key0 < wave_sinks || key1 >= wave_begin);
        const uint32_t live = static_cast<uint32_t>(tile_live >> (32 * j));
        any = any || needed;
#pragma unroll
        for (int r = 0; r < 16; ++r) st[j][r] = needed ? 0.f : -INFINITY;
        if (needed) {
          const uint16_t* kp = plane(buffer, 0, 0) + (32 * j + n) * D;
#pragma unroll
          for (int s0 = 0; s0 < kSteps; s0 += kAhead) {
            u32x4 k[kAhead][S::kKvPieces];
#pragma unroll
            for (int s = 0; s < kAhead; ++s) {
#pragma unroll
              for (int p = 0; p < S::kKvPieces; ++p) {
                k[s][p] = *reinterpret_cast<const u32x4*>(kp + p * S::kPlane + 8 * key_chunk<D>(32 * j + n, 2 * (s0 + s) + c));
              }
            }
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int s = 0; s < kAhead; ++s) {
#pragma unroll
              for (int p = S::kKvPieces - 1; p >= 0; --p) {
#pragma unroll
                for (int q = S::kQPieces - 1; q >= 0; --q) {
                  if (counted(p, q)) st[j] = mfma32(k[s][p], qr[q][s0 + s], st[j]);
                }
              }
            }
          }
          if (!(key0 >= full_begin && key1 < full_end && key0 >= all.sinks && live == 0xffffffffu)) {
            const uint32_t seen = (own.seen_of(all, at) & live) >> (4 * c);
#pragma unroll
            for (int r = 0; r < 16; ++r) st[j][r] = (seen >> (8 * (r / 4) + r % 4)) & 1 ? st[j][r] : -INFINITY;
          }
        }
      }
      if (any) {
        // Scores are kept as they are, times scale (bfloat16) or already scaled (float32).
        const float scale = sizeof(QT) == 2 ? a.scale_log2 : 1.f;
        float most = -INFINITY;
#pragma unroll
        for (int j = 0; j < kSub; ++j) {
#pragma unroll
          for (int r = 0; r < 16; ++r) most = fmaxf(most, st[j][r]);
        }
        {
          const auto both = __builtin_amdgcn_permlane32_swap(__float_as_uint(most), __float_as_uint(most), false, false);
          most = fmaxf(__uint_as_float(both[0]), __uint_as_float(both[1])) * scale;
        }
        // The reference of the exponentials is raised only when a score passes it by 2^8: weights then
        // stay below 2^8, and the outputs are seldom rescaled.
        if (__ballot(most > top + kLazyLog2) != 0) {
          const float next = fmaxf(top, most);
          const float keep = next == -INFINITY ? 1.f : fast_exp2(top - next);
          sum *= keep;
#pragma unroll
          for (int b = 0; b < kBlocks; ++b) o[b] *= keep;
          top = next;
        }
        const float from = top == -INFINITY ? 0.f : top;
#pragma unroll
        for (int j = 0; j < kSub; ++j) {
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            st[j][r] = fast_exp2(__builtin_fmaf(st[j][r], scale, -from));
            sum += st[j][r];
          }
#pragma unroll
          for (int s = 0; s < 2; ++s) {
            u32x4 pr[S::kPPieces];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              float x0 = st[j][8 * s + 2 * e], x1 = st[j][8 * s + 2 * e + 1];
#pragma unroll
              for (int p = 0; p < S::kPPieces; ++p) pr[p][e] = cut_piece(x0, x1);
            }
            // Keys 16 s + 4 c .. + 3 and 8 more on; this lane reads row i / 4 of its 16 lanes' block.
            const int row = 32 * j + 16 * s + 4 * c + (lane % 16) / 4;
            const int part = (lane / 16 % 2) * 16 + lane % 4 * 4;  // its dimension within 32
#pragma unroll
            for (int b0 = 0; b0 < kBlocks; b0 += kTogether) {
              u32x4 v[S::kKvPieces][kTogether];
#pragma unroll
              for (int p = 0; p < S::kKvPieces; ++p) {
                const auto at = [&](int b) {
                  return lds_address(plane(buffer, 1, p) + row * D + 8 * value_chunk<D>(row, 4 * b + part / 8) + part % 8);
                };
                read_values<kTogether, 2 * D>(at(b0), kTogether > 1 ? at(b0 + 1) : 0, v[p]);
              }
#pragma unroll
              for (int b = 0; b < kTogether; ++b) {
#pragma unroll
                for (int p = S::kKvPieces - 1; p >= 0; --p) {
#pragma unroll
                  for (int q = S::kPPieces - 1; q >= 0; --q) {
                    if (counted(p, q)) o[b0 + b] = mfma32(v[p][b], pr[q], o[b0 + b]);
                  }
                }
              }
            }
          }
        }
      }
      if (tile + 1 < last) stage(buffer ^ 1);
      keep_slots(tile + 2, ahead);
      __syncthreads();
    }
    {
      const auto both = __builtin_amdgcn_permlane32_swap(__float_as_uint(sum), __float_as_uint(sum), false, false);
      sum = __uint_as_float(both[0]) + __uint_as_float(both[1]);
    }

    bool bad = !(fabsf(sum) < INFINITY);
#pragma unroll
    for (int b = 0; b < kBlocks; ++b) {
#pragma unroll
      for (int r = 0; r < 16; ++r) bad = bad || !(fabsf(o[b][r]) < INFINITY);
    }
    const uint64_t wrong = __ballot(bad && active);
    const uint32_t again = static_cast<uint32_t>(wrong) | static_cast<uint32_t>(wrong >> 32);
    if (active && !((again >> n) & 1)) {
      // Register r of output tile b is dimension 32 b + 8 (r / 4) + 4 c + r % 4 of query n.
      const int64_t out_row = t * a.num_heads + head;
      const int64_t index = split_index(a, t, head, split);
      if (a.splits > 1 && c == 0) store_split_sums(a, index, top, sum);
      const float divide = sum == 0.f ? 0.f : 1.f / sum;
      if (a.splits == 1 || sum != 0.f) {
#pragma unroll
        for (int b = 0; b < kBlocks; ++b) {
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            float x[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = a.splits == 1 ? o[b][4 * g + e] * divide : o[b][4 * g + e];
            const int d = 32 * b + 8 * g + 4 * c;
            if (a.splits == 1) {
              store_row<QT, 4>(static_cast<QT*>(a.out) + out_row * D + d, x);
            } else {
              store_row<float, 4>(split_acc(a, index, D) + d, x);
            }
          }
        }
      }
    }
    for (uint32_t left = again; left != 0; left &= left - 1) {
      const int col = __builtin_ctz(left);
      Span one;
      one.sinks = __shfl(own.sinks, col);
      one.begin = __shfl(own.begin, col);
      one.end = __shfl(own.end, col);
      const int32_t which = wave * 32 + col, row = which / a.group;
      exact_row<QT, KVT, D>(a, run0 + row, kv_head * a.group + (which - row * a.group), seq, one, all, min(first * S::kKeys, count),
                            min(last * S::kKeys, count), split);
    }
  }
}

// ---------------------------------------------------------------------------------------------
// Joins the splits of every row and head: D / 4 threads each, four dimensions a thread. Bound: latency; four splits are
// loaded together, their outputs before it is known whether they count (one after the other took 1 row of 8 splits
// of 512 keys, 32 heads x 128, from 15.4 us to 19.3).
// ---------------------------------------------------------------------------------------------
template <typename QT, int D>
__global__ __launch_bounds__(kThreads) void join_kernel(const Window a) {
  constexpr int kPer = D / 4, kTogether = 4;  // splits that are loaded together
  const uint32_t item = (blockIdx.x * static_cast<uint32_t>(kThreads) + threadIdx.x) / kPer;  // launch: below 2^28
  const int d = threadIdx.x % kPer * 4;
  const uint32_t t = item / static_cast<uint32_t>(a.num_heads);
  if (t >= a.num_queries) return;
  const int32_t seq = a.seqs[t];
  const int64_t index = static_cast<int64_t>(item) * a.splits;
  const float* tops = a.workspace + index;
  const float* sums = a.workspace + a.num_queries * a.num_heads * a.splits + index;
  float top = -INFINITY, sum = 0.f;
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  for (int first = 0; first < a.splits; first += kTogether) {
    float tp[kTogether], part[kTogether], most = top;
    f32x4 out[kTogether];
#pragma unroll
    for (int i = 0; i < kTogether; ++i) {
      const int p = min(first + i, a.splits - 1);
      tp[i] = tops[p];
      part[i] = first + i < a.splits ? sums[p] : 0.f;
      out[i] = *reinterpret_cast<const f32x4*>(split_acc(a, index + p, D) + d);
    }
#pragma unroll
    for (int i = 0; i < kTogether; ++i) most = fmaxf(most, tp[i]);
    const float from = most == -INFINITY ? 0.f : most, keep = exp2f(top - from);
    sum *= keep;
    acc *= keep;
#pragma unroll
    for (int i = 0; i < kTogether; ++i) {
      if (part[i] == 0.f) continue;  // no key in this split: its output may hold anything
      const float weight = exp2f(tp[i] - from);
      sum += part[i] * weight;
      acc += out[i] * weight;
    }
    top = most;
  }
  if (seq < 0 || seq >= a.num_seqs) return;
  float x[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) x[e] = sum == 0.f ? 0.f : acc[e] / sum;
  store_row<QT, 4>(static_cast<QT*>(a.out) + static_cast<int64_t>(item) * D + d, x);  // up to 2^33 elements
}

template <typename QT, typename KVT, int D>
int launch(Window a, hipStream_t stream) {
  using S = TileShape<QT, KVT, D>;
  a.subgroups = (a.group + 15) / 16;
  a.tile_rows = kTileQueries / a.group;
  a.min_run = std::min(kMinRun, a.tile_rows);
  a.tiled = S::kFits && a.list;  // no list without tiles
  const int64_t items = a.num_queries * a.num_kv_heads * a.subgroups * a.splits;
  // Beside tiles the number of rows is known on the device only: two workgroups for every CU share them.
  const int64_t groups = a.tiled ? std::min<int64_t>(items, 512) : items;
  const int64_t tiles = (a.num_queries + a.tile_rows - 1) / a.tile_rows * a.num_kv_heads * a.splits;
  const int64_t joins = (a.num_queries * a.num_heads * (D / 4) + kThreads - 1) / kThreads;
  constexpr int64_t kMost = 0xffffffffll / (2 * kThreads);  // workgroups whose threads, up to 512 each, 32 bits count
  if (groups > kMost || joins > kMost || tiles > kMost - 512 || items > 0x7fffffff) return PKV_EUNSUPPORTED;
  const auto join = [&]() {
    if (a.splits > 1) hipLaunchKernelGGL((join_kernel<QT, D>), dim3(static_cast<uint32_t>(joins)), dim3(kThreads), 0, stream, a);
  };
  if constexpr (S::kFits) {
    if (a.tiled) {
      static_assert(sizeof(RowScratch<D, kWaves, 1>) <= S::kLds, "the row pass's part fits");
      if (hipFuncSetAttribute(reinterpret_cast<const void*>(tile_kernel<QT, KVT, D>), hipFuncAttributeMaxDynamicSharedMemorySize,
                              S::kLds) != hipSuccess) {
        return PKV_EHIP;
      }
      a.tile_items = static_cast<uint32_t>(tiles);
      hipLaunchKernelGGL(list_kernel, dim3(1), dim3(kListThreads), 0, stream, a);
      hipLaunchKernelGGL((tile_kernel<QT, KVT, D>), dim3(static_cast<uint32_t>(tiles + groups)), dim3(kThreads), S::kLds, stream, a);
      join();
      return check_launch();
    }
  }
  // Few workgroups are of eight wavefronts (24 rows of 1024 keys, 8 x 64, float32: 34 -> 27 us; 1 row, 2 key heads x 64,
  // 516 keys, bfloat16: 9.4 and 9.5; 64 rows of 4100 keys 203 -> 208). head_dim 256 needs the registers of four, and so do
  // float32 queries of head_dim 128 over bfloat16 keys (8 rows of 1024 keys, 32/8 heads: 20.4 us, 21.9 with eight). Where
  // there are many and a key row is short, one of eight serves two neighbouring key heads, and so reads twice as much next
  // to each other.
  constexpr bool kShort = D * sizeof(KVT) <= 256;
  constexpr bool kWide = D < 128 || (D == 128 && sizeof(QT) == sizeof(KVT));
  const bool wide = kWide && groups <= 256;
  const bool pair = kShort && groups >= 512 && a.num_kv_heads % 2 == 0;
  const auto start = [&](auto kernel, int64_t count, int waves) {
    hipLaunchKernelGGL(kernel, dim3(static_cast<uint32_t>(count)), dim3(waves * kWave), 0, stream, a);
  };
  if constexpr (kWide) {
    if (wide) start(row_kernel<QT, KVT, D, 8, 1>, groups, 8);
  }
  if constexpr (kShort) {
    if (pair) start(row_kernel<QT, KVT, D, 4, 2>, groups / 2, 8);
  }
  if (!wide && !pair) start(row_kernel<QT, KVT, D, 4, 1>, groups, 4);
  join();
  return check_launch();
}

template <typename QT, typename KVT>
int dispatch(const Window& a, int32_t head_dim, hipStream_t stream) {
  switch (head_dim) {
    case 32: return launch<QT, KVT, 32>(a, stream);
    case 64: return launch<QT, KVT, 64>(a, stream);
    case 128: return launch<QT, KVT, 128>(a, stream);
    case 256: return launch<QT, KVT, 256>(a, stream);
    default: return PKV_EUNSUPPORTED;
  }
}

}  // namespace
}  // namespace pkv

namespace pkv {
namespace {
// Whether a call has tiles, and so a list of the rows outside them at the end of its workspace (kept
// for every call that may have them: the workspace's size does not go by the heads' grouping).
bool has_runs(int32_t max_query_len, int32_t group) { return max_query_len >= std::min(kMinRun, kTileQueries / group); }
int64_t list_bytes(int64_t num_queries) { return (num_queries + 4) / 4 * 16; }

int32_t choose_splits(int64_t num_queries, int32_t num_heads, int32_t num_kv_heads, int32_t window, int32_t sinks,
                      int32_t max_context_len, int32_t max_query_len, bool tiles) {
  if (num_queries < 0 || num_kv_heads < 1 || num_heads < num_kv_heads || num_heads % num_kv_heads != 0 || window < 1 ||
      sinks < 0 || max_context_len < 0 || max_query_len < 0) {
    return PKV_EINVAL;
  }
  const int64_t longest = std::min<int64_t>(max_context_len, static_cast<int64_t>(window) + sinks);
  const int32_t group = num_heads / num_kv_heads;
  if (group > PKV_WINDOW_MAX_GROUP) return PKV_EINVAL;
  const bool runs = tiles && has_runs(max_query_len, group);
  const int64_t rows = runs ? kTileQueries / group : 1;
  const int64_t groups = (num_queries + rows - 1) / rows * num_kv_heads * (runs ? 1 : (group + 15) / 16);
  // Tiles: two workgroups for every CU, 128 keys to a split at least. Rows: one workgroup of eight wavefronts for
  // every CU, 256 keys to a split, and one split below 1024 keys, which saves a launch. 8 key heads x 128, bfloat16,
  // with 1, 2, 4, 8, 16 splits: 1 row of 4096 keys 63, 38, 24, 18, 16 us, 4 rows 73, 44, 28, 21, 22, 16 rows 85, 56,
  // 51, 57, 69; 8 rows of 1024 keys 24, 18, 15, 15, 23; 1 row of 512 keys 12.4, 12.2, 11.3, 11.2, 12.3.
  // Rows without tiles have long key rows and four wavefronts: 128 keys to a split. Float32, 2 key heads x 256, with 1, 2, 4,
  // 8, 16 splits: 5 rows of 2000 keys 116, 61, 36, 25, 20, of 300 keys 23.2, 19.6, 16.1, 13.9, 14.5, 512 rows of some 1450
  // keys 265, 314, 397, 561, 858 (11 splits, as of tiles: 695; over bfloat16 168 and 600).
  const int64_t fewest = runs || !tiles ? 128 : longest < 1024 ? 1024 : 256;
  const int64_t most = std::max<int64_t>(1, std::min<int64_t>(PKV_WINDOW_MAX_SPLITS, longest / fewest));
  int64_t want = runs ? (512 + groups - 1) / std::max<int64_t>(1, groups) : 256 / std::max<int64_t>(1, groups);
  // More workgroups than CUs, which would leave many of them idle at the end: up to four splits of 1024 keys (8 key heads x
  // 128, 4100 keys, one split and four: 36 rows 171 and 134 us, in float32 295 and 214; 68 rows 298 and 232, 479 and
  // 376; 56 rows, seven eighths of two rounds, 191 and 190, with 2050 keys x 64 61 and 67).
  const int64_t round = (groups + 255) / 256 * 256;
  if (!runs && groups > 256 && groups * 20 < round * 17) want = std::min<int64_t>(4, longest / 1024);
  return static_cast<int32_t>(std::max<int64_t>(1, std::min(most, want)));
}
}  // namespace
}  // namespace pkv

extern "C" int32_t pkv_window_splits(int64_t num_queries, int32_t num_heads, int32_t num_kv_heads, int32_t window,
                                     int32_t sinks, int32_t max_context_len, int32_t max_query_len) {
  return pkv::choose_splits(num_queries, num_heads, num_kv_heads, window, sinks, max_context_len, max_query_len, true);
}

extern "C" int64_t pkv_window_workspace_bytes(int64_t num_queries, int32_t num_heads, int32_t head_dim, int32_t max_query_len,
                                              int32_t num_splits) {
  if (num_queries < 0 || num_heads < 1 || head_dim < 1 || max_query_len < 0 || num_splits < 1 || num_splits > PKV_WINDOW_MAX_SPLITS) {
    return PKV_EINVAL;
  }
  const int64_t parts = num_splits == 1 ? 0 : num_queries * num_heads * num_splits * (head_dim + 2) * static_cast<int64_t>(sizeof(float));
  return (parts + 15) / 16 * 16 + (max_query_len > 1 ? pkv::list_bytes(num_queries) : 0);
}

extern "C" int32_t pkv_window_sizes(int64_t num_queries, int32_t num_heads, int32_t num_kv_heads, int32_t head_dim,
                                    int32_t q_dtype, int32_t window, int32_t sinks, int32_t max_context_len,
                                    int32_t max_query_len, int32_t num_splits, int64_t* workspace_bytes) {
  const int size = pkv::dtype_size(static_cast<pkv_dtype>(q_dtype));
  if (size == 0 || !workspace_bytes || num_splits < 0) return PKV_EINVAL;
  const bool tiles = pkv::tiles_of(size, head_dim);
  const int32_t splits = num_splits > 0 ? num_splits
                                        : pkv::choose_splits(num_queries, num_heads, num_kv_heads, window, sinks, max_context_len,
                                                             max_query_len, tiles);
  if (splits < 1) return PKV_EINVAL;
  // Without tiles there is no list of the rows outside them.
  const int64_t need = pkv_window_workspace_bytes(num_queries, num_heads, head_dim, tiles ? max_query_len : 0, splits);
  if (need < 0) return PKV_EINVAL;
  *workspace_bytes = need;
  return splits;
}

extern "C" int pkv_window_attention(const pkv_window* args, int device, void* stream) {
  using namespace pkv;
  if (!args) return PKV_EINVAL;
  const pkv_window& g = *args;
  if (g.num_queries < 0 || g.num_heads < 1 || g.num_kv_heads < 1 || g.num_heads % g.num_kv_heads != 0 || g.num_seqs < 0 ||
      g.num_blocks < 0 || g.block_size < 1 || g.block_table_stride < 0 || g.window < 1 || g.sinks < 0 ||
      g.max_context_len < 0 || g.max_query_len < 0 || g.num_splits < 0 || g.num_splits > PKV_WINDOW_MAX_SPLITS) {
    return PKV_EINVAL;
  }
  if (static_cast<int64_t>(g.block_table_stride) * g.block_size < g.max_context_len) return PKV_EINVAL;
  if ((g.q_dtype != PKV_F32 && g.q_dtype != PKV_BF16) || (g.kv_dtype != PKV_F32 && g.kv_dtype != PKV_BF16)) return PKV_EINVAL;
  if (g.q_dtype == PKV_BF16 && g.kv_dtype == PKV_F32) return PKV_EUNSUPPORTED;
  if (g.head_dim != 32 && g.head_dim != 64 && g.head_dim != 128 && g.head_dim != 256) return PKV_EUNSUPPORTED;
  if (g.num_heads / g.num_kv_heads > PKV_WINDOW_MAX_GROUP) return PKV_EUNSUPPORTED;
  // Slots, and a span's items some tiles past its end, are 32-bit.
  if (g.num_blocks > 0x7fffffff / g.block_size || g.max_context_len > PKV_WINDOW_MAX_CONTEXT) return PKV_EUNSUPPORTED;
  if (g.num_queries == 0) return PKV_OK;
  if (!g.out || !g.queries || !g.query_positions || !g.query_seq || !g.key_cache || !g.value_cache || !g.block_tables ||
      !g.context_lens) {
    return PKV_EINVAL;
  }
  const int64_t row = static_cast<int64_t>(g.num_heads) * g.head_dim;
  const int64_t elems = 16 / dtype_size(static_cast<pkv_dtype>(g.q_dtype));
  if (g.query_token_stride < row || g.query_token_stride % elems != 0 || !aligned16(g.out) || !aligned16(g.queries) ||
      !aligned16(g.key_cache) || !aligned16(g.value_cache)) {
    return PKV_EINVAL;
  }
  const bool tiles = tiles_of(dtype_size(static_cast<pkv_dtype>(g.q_dtype)), g.head_dim);
  const bool runs = tiles && has_runs(g.max_query_len, g.num_heads / g.num_kv_heads);
  int64_t need = 0;
  const int32_t splits = pkv_window_sizes(g.num_queries, g.num_heads, g.num_kv_heads, g.head_dim, g.q_dtype, g.window, g.sinks,
                                          g.max_context_len, g.max_query_len, g.num_splits, &need);
  if (splits < 1) return PKV_EINVAL;
  if (need > 0 && (!g.workspace || !aligned16(g.workspace) || g.workspace_bytes < need)) return PKV_EINVAL;
  Window a{};
  a.out = g.out;
  a.queries = g.queries;
  a.query_stride = g.query_token_stride;
  a.positions = g.query_positions;
  a.seqs = g.query_seq;
  a.num_queries = g.num_queries;
  a.keys = g.key_cache;
  a.values = g.value_cache;
  a.num_blocks = g.num_blocks;
  a.tables = g.block_tables;
  a.contexts = g.context_lens;
  a.workspace = g.workspace;
  a.block_size = g.block_size;
  a.table_stride = g.block_table_stride;
  a.num_seqs = g.num_seqs;
  a.num_heads = g.num_heads;
  a.num_kv_heads = g.num_kv_heads;
  a.group = g.num_heads / g.num_kv_heads;
  a.window = g.window;
  a.sinks = g.sinks;
  a.max_context = g.max_context_len;
  a.splits = splits;
  a.scale_log2 = g.scale * 1.44269504088896340736f;
  a.given_scale = a.scale_log2;
  if (runs) a.list = reinterpret_cast<int32_t*>(reinterpret_cast<char*>(g.workspace) + need - list_bytes(g.num_queries));
  DeviceGuard guard(device);
  if (!guard.ok()) return PKV_EHIP;
  auto s = static_cast<hipStream_t>(stream);
  if (g.q_dtype == PKV_BF16) {
    a.flip = a.scale_log2 < 0.f ? 0x80008000u : 0u;
    a.keep = a.scale_log2 == 0.f ? 0u : 0xffffffffu;
    a.scale_log2 = a.scale_log2 == 0.f ? 1.f : std::fabs(a.scale_log2);
    return dispatch<uint16_t, uint16_t>(a, g.head_dim, s);
  }
  return g.kv_dtype == PKV_F32 ? dispatch<float, float>(a, g.head_dim, s)
                               : dispatch<float, uint16_t>(a, g.head_dim, s);
}
