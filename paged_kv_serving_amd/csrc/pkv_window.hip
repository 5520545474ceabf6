// Paged causal attention with a sliding window and sinks, for grouped heads.
//
// A query row at position p of a sequence with context length c sees the keys j < min(c, p + 1) with
// j > p - window or j < sinks:
//     out = sum_j exp(s_j) v_j / sum_j exp(s_j),  s_j = scale * q . k_j
// with an online softmax (running maximum and sum), everything in float32 and one rounding to the
// output's type, but for the weights that a bfloat16 tile multiplies its values by (16 bits, at tile_kernel).
//
// A cache may hold e4m3 codes with a power of two as the scale of each block and head. A code times such a scale is a
// bfloat16 number, so codes are widened on their way into the bfloat16 products, the scale being the conversion
// instruction's own operand, and all else is as over a bfloat16 cache.
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

struct Stream;

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
  uint32_t run_shares;     // of codes: workgroups that share a tile's runs
  int32_t tiled;           // whether the tile pass computes the runs
  int32_t min_run;         // rows of one sequence next to each other that a tile takes
  int32_t* list;           // the rows that no tile takes (list_kernel); NULL without tiles
  float scale_log2;  // scale * log2(e): scores are kept in base 2
  float given_scale;  // the same before the next two
  // A negative scale of bfloat16 queries turns their signs instead, so that the largest product is the
  // largest score; a zero one clears them, so that a hidden key's -inf stays what it is.
  uint32_t keep, flip;
  const float* key_scales;  // of e4m3 codes, [num_blocks, num_kv_heads]; else NULL
  const float* value_scales;
  int32_t page_groups;   // 16-key groups of a block, for page_kernel
  uint32_t page_magic;   // ceil(2^32 / page_groups)
  Stream* stream;        // for stream_kernel; NULL where a call has splits
  int32_t stream_groups; // shares
  int32_t stream_least;  // rounds of a share
  int64_t stream_places; // of parts in the workspace, two for each share and head
  int32_t* order;        // of the aligned blocks of rows, the longest first; NULL: as they come
};

__device__ __forceinline__ float load_one(const float* p) { return *p; }
__device__ __forceinline__ float load_one(const uint16_t* p) { return __uint_as_float(static_cast<uint32_t>(*p) << 16); }
__device__ __forceinline__ float load_one(const uint8_t* p) { return __builtin_amdgcn_cvt_f32_fp8(*p, 0); }
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
    if constexpr (N % 8 == 0) {
#pragma unroll
      for (int i = 0; i < N / 2; i += 4) *reinterpret_cast<u32x4*>(p + 2 * i) = u32x4{w[i], w[i + 1], w[i + 2], w[i + 3]};
    } else if constexpr (N == 4) {
      *reinterpret_cast<u32x2*>(p) = u32x2{w[0], w[1]};
    } else {
      static_assert(N == 2, "two, four, or groups of eight");
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

// Where the scale of a slot's block of one head lies.
__device__ __forceinline__ int64_t scale_of(const Window& a, int32_t slot, int32_t kv_head) {
  return static_cast<int64_t>(static_cast<uint32_t>(slot) / static_cast<uint32_t>(a.block_size)) * a.num_kv_heads + kv_head;
}

// Codes 0 and 1 of a word, or 2 and 3, as bfloat16 numbers times a power of two.
template <int kHalf>
__device__ __forceinline__ uint32_t widen(uint32_t codes, float scale) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes, scale, kHalf != 0));
}

// The power of two that a scale stands for, as the conversion takes it (its exponent; NaN where that is no number's): code 0x38 is 1.
__device__ __forceinline__ float power_of(float scale) { return bf16_lo(widen<0>(0x38, scale)); }

// Element offset of a slot's row of one head in the pools.
__device__ __forceinline__ int64_t row_of(const Window& a, int32_t slot, int32_t kv_head, int d) {
  return (static_cast<int64_t>(slot) * a.num_kv_heads + kv_head) * d;
}

// A row's split results in the workspace: maxima, sums, then the unnormalised outputs.
__device__ __forceinline__ int64_t split_index(const Window& a, int64_t t, int32_t head, int32_t split) {
  return (t * a.num_heads + head) * a.splits + split;
}

// Where a row's result for `heads` heads from `head0` on goes: to the output, or, unnormalised, to the workspace.
struct Place {
  bool direct;
  int64_t index;  // of head0's maximum and sum in the workspace, and of its output
  int64_t step;   // to the next head's
  int64_t total;  // of such results, where sums begin
};
__device__ __forceinline__ Place split_place(const Window& a, int64_t t, int32_t head0, int32_t split) {
  return Place{a.splits == 1, split_index(a, t, head0, split), a.splits, a.num_queries * a.num_heads * a.splits};
}
__device__ __forceinline__ void store_sums(const Window& a, const Place& to, int64_t index, float top, float sum) {
  a.workspace[index] = top;
  a.workspace[to.total + index] = sum;
}
__device__ __forceinline__ float* acc_of(const Window& a, const Place& to, int64_t index, int d) {
  return a.workspace + (2 * to.total + 3) / 4 * 4 + index * d;  // 16-byte aligned
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
                                                    int32_t first, int32_t last, const Place& to, int32_t place) {
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
      if constexpr (sizeof(KVT) == 1) {
        // A query times a code may pass float32's range where the key does not: a scale below 1 comes first, one above it last. How far
        // these loops are unrolled moves the tiles' registers: by four and one 8 x 512 bfloat16 rows of 128 take 170 us and 8 rows by
        // themselves that see a NaN 290, by eight and one 174 and 265, by two each 172 and 355.
        float by = power_of(a.key_scales[scale_of(a, slot, kv_head)]);
        if (by < 1.f) {
#pragma unroll 4
          for (int d = 0; d < D; ++d) score += load_one(q + d) * (load_one(k + d) * by);
          by = 1.f;
        } else {
#pragma unroll 1
          for (int d = 0; d < D; ++d) score += load_one(q + d) * load_one(k + d);
        }
        score *= a.given_scale;
        score *= by;
      } else {
        for (int d = 0; d < D; ++d) score += load_one(q + d) * load_one(k + d);
        score *= a.given_scale;
      }
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
      float pj = __shfl(p, j);
      const int32_t from_slot = __shfl(slot, j);
      const KVT* v = static_cast<const KVT*>(a.values) + row_of(a, from_slot, kv_head, D);
      if constexpr (sizeof(KVT) == 1) pj *= power_of(a.value_scales[scale_of(a, from_slot, kv_head)]);
      for (int e = 0; e < kOwn; ++e) {
        const int d = e * kWave + lane;
        if (d < D) acc[e] += pj * load_one(v + d);
      }
    }
  }
  if (to.direct) {
    QT* out = static_cast<QT*>(a.out) + (t * a.num_heads + head) * D;
    for (int e = 0; e < kOwn; ++e) {
      const int d = e * kWave + lane;
      if (d < D) store_one(out + d, sum == 0.f ? 0.f : acc[e] / sum);
    }
    return;
  }
  const int64_t index = to.index + place * to.step;
  if (lane == 0) store_sums(a, to, index, top, sum);
  for (int e = 0; e < kOwn; ++e) {
    const int d = e * kWave + lane;
    if (d < D) acc_of(a, to, index, D)[d] = acc[e];
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
  static constexpr bool kCodes = sizeof(KVT) == 1;  // e4m3, widened to bfloat16
  static constexpr bool kBf16 = sizeof(KVT) <= 2;   // the products
  static constexpr int kPieces = kBf16 ? (sizeof(QT) == 4 ? 3 : 1) : 1;
  static constexpr int kPPieces = 3;                         // of the weights, over bfloat16 values
  static constexpr int kBlocks = kBf16 && D <= 128 ? 2 : 1;  // 16-key blocks per round
  static constexpr int kKeys = 16 * kBlocks;
  static constexpr int kKSteps = D / 32;                     // products of 32 dimensions
  static constexpr int kKWidth = kCodes && D == 32 ? 8 : 16;  // bytes of a load of a key row per lane
  static constexpr int kKLoads = D * int(sizeof(KVT)) / (4 * kKWidth);
  static constexpr int kPerLane = D / 16;                    // values of a value row per lane
  static constexpr int kVWidth = kPerLane < 16 / int(sizeof(KVT)) ? kPerLane : 16 / int(sizeof(KVT));
  static constexpr int kVLoads = kPerLane / kVWidth;
  static constexpr int kVWords = (kVWidth * int(sizeof(KVT)) + 3) / 4;
  static constexpr int kQRegs = kBf16 ? 4 * kKSteps * kPieces : D / 4;
  // The first of the 8 dimensions that lane group c has of step u.
  __device__ static constexpr int dims(int u, int c) { return kCodes && D > 32 ? 64 * (u / 2) + 16 * c + 8 * (u % 2) : 32 * u + 8 * c; }
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
//
// kOrder: also the aligned blocks in the order of the keys that their rows see (three rows of a block speak for it), the most first, for
// as many blocks as the workgroup has threads. The tiles' workgroups then end together: 8 x 512 rows behind up to 2048 others,
// 32/8 heads x 128 over e4m3 codes, 248 -> 201 us.
constexpr int kListThreads = 1024;  // the order's keys hold a block's number in ten bits
template <bool kOrder>
__global__ __launch_bounds__(kListThreads) void list_kernel(const Window a) {
  __shared__ int32_t s_found;
  if constexpr (kOrder) {
    __shared__ __align__(16) uint32_t s_keys[kListThreads];  // keys, then the block's number from behind: no two alike
    const int32_t blocks = static_cast<int32_t>((a.num_queries + a.tile_rows - 1) / a.tile_rows), b = threadIdx.x;
    int32_t keys = 0;
    if (b < blocks) {
      const int64_t begin = static_cast<int64_t>(b) * a.tile_rows, end = min(begin + a.tile_rows, a.num_queries);
      const int64_t at[3] = {begin, (begin + end) / 2, end - 1};
#pragma unroll
      for (int i = 0; i < 3; ++i) {
        const int32_t seq = a.seqs[at[i]];
        if (seq >= 0 && seq < a.num_seqs) keys = max(keys, span_of(a, seq, a.positions[at[i]]).count());
      }
    }
    const uint32_t mine = b < blocks ? static_cast<uint32_t>(min(keys, (1 << 22) - 1)) << 10 | (kListThreads - 1 - b) : 0;
    s_keys[b] = mine;
    if (threadIdx.x == 0) s_found = 0;
    __syncthreads();
    if (b < blocks) {  // the other wavefronts go on
      int32_t place = 0;
#pragma unroll 4
      for (int32_t j = 0; j < blocks; j += 4) {
        const u32x4 four = *reinterpret_cast<const u32x4*>(s_keys + j);
#pragma unroll
        for (int e = 0; e < 4; ++e) place += four[e] > mine ? 1 : 0;
      }
      a.order[place] = b;
    }
  } else {
    if (threadIdx.x == 0) s_found = 0;
    __syncthreads();
  }
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

// The end of a row's pass: the wavefronts' maxima, sums and outputs `o` joined, and the row's result or its part's stored.
template <typename QT, typename KVT, int D, int kRowWaves, int kPair>
__device__ __forceinline__ void finish_row(const Window& a, RowScratch<D, kRowWaves, kPair>& shared, floatx4 (&o)[D / 16], float top, float sum,
                                           int64_t t, int32_t head0, int32_t heads, int32_t seq, const Span& span, int32_t first_item,
                                           int32_t last_item, const Place& to) {
  using S = RowShape<QT, KVT, D>;
  constexpr int kTiles = D / 16;  // output tiles of 16 dimensions
  auto& s_acc = shared.acc;
  auto& s_top = shared.top;
  auto& s_sum = shared.sum;
  auto& s_redo = shared.redo;
  const int lane = threadIdx.x & (kWave - 1), c = lane / 16, n = lane % 16;
  const int side = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave % kPair);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave / kPair);
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
        exact_row<QT, KVT, D>(a, t, head0 + g, seq, span, span, first_item, last_item, to, g);
      }
      return;
    }
  }
  if (wave != 0 || n >= heads) return;
  // Register r of output tile (g, e) is dimension 16 kVWidth g + kVWidth (4c + r) + e of head n.
  const int64_t out_row = t * a.num_heads + head0 + n;
  if (to.direct) {
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
    const int64_t index = to.index + n * to.step;
    if (c == 0) store_sums(a, to, index, all, sum);
    if (sum == 0.f) return;
#pragma unroll
    for (int g = 0; g < S::kVLoads; ++g) {
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        float x[S::kVWidth];
#pragma unroll
        for (int e = 0; e < S::kVWidth; ++e) x[e] = o[g * S::kVWidth + e][r];
        store_row<float, S::kVWidth>(acc_of(a, to, index, D) + 16 * S::kVWidth * g + S::kVWidth * (4 * c + r), x);
      }
    }
  }
}

// The items of workgroup `block` of `blocks`.
template <typename QT, typename KVT, int D, int kRowWaves, int kPair>
__device__ __forceinline__ void row_pass(const Window& a, RowScratch<D, kRowWaves, kPair>& shared, uint32_t block, uint32_t blocks) {
  using S = RowShape<QT, KVT, D>;
  constexpr int kTiles = D / 16;  // output tiles of 16 dimensions
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
    const int64_t k_at = (static_cast<int64_t>(kv_head) * D + S::kKWidth / int(sizeof(KVT)) * c) * sizeof(KVT);
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
        for (int u = 0; u < S::kKSteps; ++u) {
          const u32x4 x = *reinterpret_cast<const u32x4*>(q + S::dims(u, c));
#pragma unroll
          for (int e = 0; e < 4; ++e) qr[4 * u + e] = (x[e] & a.keep) ^ a.flip;
        }
      } else if constexpr (S::kBf16) {
#pragma unroll
        for (int u = 0; u < S::kKSteps; ++u) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float x0 = q[S::dims(u, c) + 2 * e] * a.scale_log2, x1 = q[S::dims(u, c) + 2 * e + 1] * a.scale_log2;
#pragma unroll
            for (int p = 0; p < 3; ++p) qr[4 * (p * S::kKSteps + u) + e] = take_piece(x0, x1);
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
    // Of codes also the scales of that key's block, for its key and its value.
    float key_scale = 1.f, value_scale = 1.f;  // of the round whose rows are loaded
    auto look_up_scales = [&](int32_t slot) {
      if constexpr (S::kCodes) {
        const bool known = slot >= 0;  // elsewhere 1: code 0 times a NaN is not 0
        const int64_t at = known ? scale_of(a, slot, kv_head) : 0;
        key_scale = known ? a.key_scales[at] : 1.f;
        value_scale = known ? a.value_scales[at] : 1.f;
      }
    };
    Words<S::kKWidth / 4> kx[S::kBlocks][S::kKLoads];
    Words<S::kVWords> vx[S::kBlocks][4][S::kVLoads];
    auto load_keys = [&](int32_t slot) {
#pragma unroll
      for (int j = 0; j < S::kBlocks; ++j) {
        const char* p = keys + max(__shfl(slot, 16 * j + n), 0) * row_bytes + k_at;
#pragma unroll
        for (int u = 0; u < S::kKLoads; ++u) kx[j][u] = load_words<S::kKWidth / 4>(p + u * 4 * S::kKWidth);
      }
    };
    auto load_values = [&](int32_t slot) {
#pragma unroll
      for (int j = 0; j < S::kBlocks; ++j) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const char* p = values + max(__shfl(slot, 16 * j + 4 * c + r), 0) * row_bytes + v_at;
#pragma unroll
          for (int g = 0; g < S::kVLoads; ++g) {
            if constexpr (S::kVWidth * sizeof(KVT) == 2) {
              vx[j][r][g].w[0] = __builtin_nontemporal_load(reinterpret_cast<const uint16_t*>(p));
            } else {
              vx[j][r][g] = load_words<S::kVWords>(p + g * 16 * S::kVWidth * int(sizeof(KVT)));
            }
          }
        }
      }
    };

    constexpr uint64_t kAll = S::kKeys == 32 ? 0xffffffffull : 0xffffull;
    int32_t round = first + wave;
    int32_t slot = look_up(round);
    uint32_t live = static_cast<uint32_t>(__ballot(slot >= 0) & kAll);  // the round's keys that count
    if (live != 0) {
      look_up_scales(slot);
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
          if constexpr (S::kBf16) {
            const float scale = S::kCodes ? __shfl(key_scale, 16 * j + n) : 1.f;  // of this lane's key
#pragma unroll
            for (int u = 0; u < S::kKSteps; ++u) {
              u32x4 k;
              if constexpr (S::kCodes) {
                const uint32_t* w = kx[j][D == 32 ? 0 : u / 2].w + (D == 32 ? 0 : u % 2 * 2);
                k = u32x4{widen<0>(w[0], scale), widen<1>(w[0], scale), widen<0>(w[1], scale), widen<1>(w[1], scale)};
              } else {
                k = __builtin_bit_cast(u32x4, kx[j][u]);
              }
#pragma unroll
              for (int p = S::kPieces - 1; p >= 0; --p) {  // the smallest pieces first
                const uint32_t* q = qr + 4 * (p * S::kKSteps + u);
                st[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, k),
                                                                __builtin_bit_cast(bf16x8, (u32x4{q[0], q[1], q[2], q[3]})), st[j], 0, 0, 0);
              }
            }
          } else {
#pragma unroll
            for (int u = 0; u < S::kKLoads; ++u) {
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                st[j] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(kx[j][u].w[e]), __uint_as_float(qr[4 * u + e]), st[j], 0, 0, 0);
              }
            }
          }
        }
      }
      const float values_by = value_scale;  // the present round's, before the next one's are looked up
      if (live_next != 0) {
        look_up_scales(slot_next);
        load_keys(slot_next);
      }
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
          // Pairs of a key's values in bfloat16.
          constexpr int kPairs = S::kVWidth / 2;
          uint32_t wide[S::kBlocks][4][S::kVLoads][kPairs];
#pragma unroll
          for (int j = 0; j < S::kBlocks; ++j) {
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              const float scale = S::kCodes ? __shfl(values_by, 16 * j + 4 * c + r) : 1.f;
#pragma unroll
              for (int g = 0; g < S::kVLoads; ++g) {
#pragma unroll
                for (int w = 0; w < kPairs; ++w) {
                  if constexpr (!S::kCodes) {
                    wide[j][r][g][w] = vx[j][r][g].w[w];
                  } else {
                    const uint32_t codes = vx[j][r][g].w[w / 2];
                    wide[j][r][g][w] = w % 2 ? widen<1>(codes, scale) : widen<0>(codes, scale);
                  }
                }
              }
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
                  v[2 * j + r / 2] = __builtin_amdgcn_perm(wide[j][r + 1][g][e / 2], wide[j][r][g][e / 2], e % 2 ? 0x07060302 : 0x05040100);
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
    finish_row<QT, KVT, D, kRowWaves, kPair>(a, shared, o, top, sum, t, head0, heads, seq, span, min(first * S::kKeys, count),
                                             min(last * S::kKeys, count), split_place(a, t, head0, split));
  }
}

template <typename QT, typename KVT, int D, int kRowWaves, int kPair>
__global__ __launch_bounds__(kRowWaves * kPair * kWave) void row_kernel(const Window a) {
  __shared__ RowScratch<D, kRowWaves, kPair> shared;
  row_pass<QT, KVT, D, kRowWaves, kPair>(a, shared, blockIdx.x, gridDim.x);
}

// ---------------------------------------------------------------------------------------------
// Rows by themselves over e4m3 codes without a window, where a block's tokens are a multiple of 16: the row pass above with
// every 16 keys of a product in one block. Their place and scales are the same for the whole wavefront, so addresses and
// scales are scalars (a wavefront looks 64 groups' up at once), and nothing is exchanged between lanes but the maximum.
// The codes of two neighbouring keys are interleaved before they are widened, which gives the value operand's pairs at
// once. The next round's keys are asked for as soon as the present one's are scores, its values when the present ones are used.
//
// Bound: HBM. 64 rows of 16384 keys, 32/8 heads x 128, bfloat16 queries, 2.15 GB: 361 us, 6.0 TB/s (reads of these bytes
// by the same pieces alone: 6.7; by the general row pass above, which exchanges slots and scales between lanes, 477).
// ---------------------------------------------------------------------------------------------
template <typename QT, int D>
struct PageShape {
  static constexpr int kBlocks = D <= 128 ? 2 : 1;  // 16-key groups of a round
  static constexpr int kBatch = kWave / kBlocks;    // rounds whose groups are looked up at once
};

// Rounds [first, last) of row t's `count` visible keys.
template <typename QT, int D, int kRowWaves, int kPair>
__device__ __forceinline__ void page_piece(const Window& a, RowScratch<D, kRowWaves, kPair>& shared, int64_t t, int32_t seq, int32_t count,
                                           int32_t first, int32_t last, int32_t kv_head, int32_t head0, int32_t heads, const Place& to) {
  using S = RowShape<QT, uint8_t, D>;
  using P = PageShape<QT, D>;
  constexpr int kTiles = D / 16, kKeys = 16 * P::kBlocks, kWords = S::kVWords;
  const int lane = threadIdx.x & (kWave - 1), c = lane / 16, n = lane % 16;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave / kPair);
  const int32_t* table = a.tables + static_cast<int64_t>(seq) * a.table_stride;
  const int32_t mine = (last - first - wave + kRowWaves - 1) / kRowWaves;  // this wavefront's rounds (0 or less: none)

  // The queries, the right operand of S^T: lane (c, n) holds its c's dimensions of head n.
  uint32_t qr[S::kQRegs];
  {
    const QT* q = static_cast<const QT*>(a.queries) + t * a.query_stride + static_cast<int64_t>(head0 + min(n, heads - 1)) * D;
#pragma unroll
    for (int u = 0; u < S::kKSteps; ++u) {
      if constexpr (sizeof(QT) == 2) {
        const u32x4 x = *reinterpret_cast<const u32x4*>(q + S::dims(u, c));
#pragma unroll
        for (int e = 0; e < 4; ++e) qr[4 * u + e] = (x[e] & a.keep) ^ a.flip;
      } else {
        const f32x4 x[2] = {*reinterpret_cast<const f32x4*>(q + S::dims(u, c)), *reinterpret_cast<const f32x4*>(q + S::dims(u, c) + 4)};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float x0 = x[e / 2][e % 2 * 2] * a.scale_log2, x1 = x[e / 2][e % 2 * 2 + 1] * a.scale_log2;
#pragma unroll
          for (int p = 0; p < 3; ++p) qr[4 * (p * S::kKSteps + u) + e] = take_piece(x0, x1);
        }
      }
    }
  }

  // Byte offsets of this lane from a group's first row: of its key, and of the first of its four values' keys.
  const uint32_t row_bytes = static_cast<uint32_t>(a.num_kv_heads) * D;
  const uint32_t k_at = static_cast<uint32_t>(kv_head) * D + n * row_bytes + S::kKWidth * c;
  const uint32_t v_at = static_cast<uint32_t>(kv_head) * D + 4 * c * row_bytes + S::kVWidth * n;
  const char* keys = static_cast<const char*>(a.keys);
  const char* values = static_cast<const char*>(a.values);

  // A batch: lane l has the slot (-1: in no block) and the scales of group l % kBlocks of this wavefront's l / kBlocks-th round.
  int32_t slots = -1, looked = -1;
  float key_scales = 1.f, value_scales = 1.f;
  const auto look_up = [&](int32_t from) {
    const int32_t round = first + wave + kRowWaves * (from + lane / P::kBlocks);
    const uint32_t group = static_cast<uint32_t>(round) * P::kBlocks + lane % P::kBlocks;
    slots = -1;
    key_scales = value_scales = 1.f;  // code 0 times a NaN is not 0
    if (round < last && static_cast<int32_t>(group * 16) < count) {
      const uint32_t page = a.page_groups == 1 ? group : __umulhi(group, a.page_magic);
      const int32_t block = table[page];
      if (block >= 0 && block < a.num_blocks) {
        slots = block * a.block_size + static_cast<int32_t>(group - page * a.page_groups) * 16;
        const int64_t at = static_cast<int64_t>(block) * a.num_kv_heads + kv_head;
        key_scales = a.key_scales[at];
        value_scales = a.value_scales[at];
      }
    }
  };

  struct Round {
    Words<S::kKWidth / 4> k[P::kBlocks][S::kKLoads];
    Words<kWords> v[P::kBlocks][4];
    float key_scale[P::kBlocks], value_scale[P::kBlocks];
    int32_t slot[P::kBlocks];
  };
  // Fetches behind the last round repeat it: without a branch around them, a wait for values leaves the keys that were
  // asked for after them in flight.
  const auto fetch_keys = [&](Round& x, int32_t k) {
    k = min(k, mine - 1);
    if (k % P::kBatch == 0 && k != looked) {
      looked = k;
      look_up(k);
      // Arrived before anything else is asked for.
      asm volatile("" : "+v"(slots), "+v"(key_scales), "+v"(value_scales));
    }
#pragma unroll
    for (int j = 0; j < P::kBlocks; ++j) {
      const int from = k % P::kBatch * P::kBlocks + j;
      x.slot[j] = __builtin_amdgcn_readlane(slots, from);
      x.key_scale[j] = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(key_scales), from));
      x.value_scale[j] = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(value_scales), from));
      const int64_t base = static_cast<int64_t>(max(x.slot[j], 0)) * row_bytes;
      const char* kp = keys + base;
#pragma unroll
      for (int u = 0; u < S::kKLoads; ++u) x.k[j][u] = load_words<S::kKWidth / 4>(kp + (k_at + u * 4 * S::kKWidth));
    }
    __builtin_amdgcn_sched_barrier(0);  // loads arrive in order: no value between the keys
  };
  const auto fetch_values = [&](Round& x) {
#pragma unroll
    for (int j = 0; j < P::kBlocks; ++j) {
      const char* vp = values + static_cast<int64_t>(max(x.slot[j], 0)) * row_bytes;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        if constexpr (S::kVWidth == 2) {
          x.v[j][r].w[0] = __builtin_nontemporal_load(reinterpret_cast<const uint16_t*>(vp + (v_at + r * row_bytes)));
        } else {
          x.v[j][r] = load_words<kWords>(vp + (v_at + r * row_bytes));
        }
      }
    }
  };

  floatx4 o[kTiles];
#pragma unroll
  for (int b = 0; b < kTiles; ++b) o[b] = floatx4{0.f, 0.f, 0.f, 0.f};
  float top = -INFINITY, sum = 0.f;
  const float scale = sizeof(QT) == 2 ? a.scale_log2 : 1.f;  // of the scores
  const auto use = [&](Round& x, int32_t k, int32_t ahead) {
    const int32_t key0 = (first + wave + kRowWaves * k) * kKeys;
    bool whole = key0 + kKeys <= count;
    floatx4 st[P::kBlocks];
#pragma unroll
    for (int j = 0; j < P::kBlocks; ++j) {
      whole = whole && x.slot[j] >= 0;
      st[j] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int u = 0; u < S::kKSteps; ++u) {
        const uint32_t* w = x.k[j][D == 32 ? 0 : u / 2].w + (D == 32 ? 0 : u % 2 * 2);
        const u32x4 key = {widen<0>(w[0], x.key_scale[j]), widen<1>(w[0], x.key_scale[j]), widen<0>(w[1], x.key_scale[j]),
                           widen<1>(w[1], x.key_scale[j])};
#pragma unroll
        for (int p = S::kPieces - 1; p >= 0; --p) {  // the smallest pieces first
          const uint32_t* q = qr + 4 * (p * S::kKSteps + u);
          st[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, key),
                                                          __builtin_bit_cast(bf16x8, (u32x4{q[0], q[1], q[2], q[3]})), st[j], 0, 0, 0);
        }
      }
    }
    int32_t slot_now[P::kBlocks];
    float value_scale_now[P::kBlocks];
#pragma unroll
    for (int j = 0; j < P::kBlocks; ++j) slot_now[j] = x.slot[j], value_scale_now[j] = x.value_scale[j];
    fetch_keys(x, ahead);
    if (!whole) {
#pragma unroll
      for (int j = 0; j < P::kBlocks; ++j) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const bool seen = slot_now[j] >= 0 && key0 + 16 * j + 4 * c + r < count;
          st[j][r] = seen ? st[j][r] : -INFINITY;
#pragma unroll
          for (int w = 0; w < kWords; ++w) x.v[j][r].w[w] = seen ? x.v[j][r].w[w] : 0;  // 0 * inf is not 0
        }
      }
    }
    float most = -INFINITY;
#pragma unroll
    for (int j = 0; j < P::kBlocks; ++j) {
#pragma unroll
      for (int r = 0; r < 4; ++r) most = fmaxf(most, st[j][r]);
    }
    most = column_max(most) * scale;
    if (__ballot(most > top) != 0) {
      const float next = fmaxf(top, most);
      const float keep = next == -INFINITY ? 1.f : fast_exp2(top - next);
      sum *= keep;
#pragma unroll
      for (int b = 0; b < kTiles; ++b) o[b] *= keep;
      top = next;
    }
    const float from = top == -INFINITY ? 0.f : top;
    // Term 4j + r of a lane's eight is key 16j + 4c + r.
    u32x4 pr[S::kPPieces] = {};
#pragma unroll
    for (int j = 0; j < P::kBlocks; ++j) {
#pragma unroll
      for (int r = 0; r < 4; r += 2) {
        float x0 = fast_exp2(__builtin_fmaf(st[j][r], scale, -from)), x1 = fast_exp2(__builtin_fmaf(st[j][r + 1], scale, -from));
        sum += x0 + x1;
#pragma unroll
        for (int p = 0; p < S::kPPieces; ++p) pr[p][2 * j + r / 2] = cut_piece(x0, x1);
      }
    }
#pragma unroll
    for (int e = 0; e < S::kVWidth; e += 2) {
      // Two dimensions of a word: pairs of codes of keys r and r + 1, first one dimension's, then the other's.
      u32x4 v[2] = {};
#pragma unroll
      for (int j = 0; j < P::kBlocks; ++j) {
#pragma unroll
        for (int r = 0; r < 4; r += 2) {
          const uint32_t pairs = __builtin_amdgcn_perm(x.v[j][r + 1].w[e / 4], x.v[j][r].w[e / 4], e % 4 ? 0x07030602 : 0x05010400);
          v[0][2 * j + r / 2] = widen<0>(pairs, value_scale_now[j]);
          v[1][2 * j + r / 2] = widen<1>(pairs, value_scale_now[j]);
        }
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int p = S::kPPieces - 1; p >= 0; --p) {
          o[e + h] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, v[h]), __builtin_bit_cast(bf16x8, pr[p]), o[e + h], 0, 0, 0);
        }
      }
    }
  };

  if (mine > 0) {
    Round x;
    fetch_keys(x, 0);
    fetch_values(x);
    for (int32_t k = 0; k < mine; ++k) {
      use(x, k, k + 1);
      fetch_values(x);
    }
  }
  finish_row<QT, uint8_t, D, kRowWaves, kPair>(a, shared, o, top, sum, t, head0, heads, seq, Span{0, 0, count}, min(first * kKeys, count),
                                               min(last * kKeys, count), to);
}

// The key head and the first of its query heads that a wavefront serves, of the workgroup's `group` of them.
struct Heads {
  int32_t kv_head, head0, count;
};
template <int kPair>
__device__ __forceinline__ Heads heads_of(const Window& a, uint32_t group) {
  const uint32_t head_groups = a.num_kv_heads / kPair;
  const int side = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave % kPair);
  const int32_t kv_head = group % head_groups * kPair + side, sub = group / head_groups;
  return Heads{kv_head, kv_head * a.group + sub * 16, min(16, a.group - sub * 16)};
}

// A row or one of its splits to a workgroup.
template <typename QT, int D, int kRowWaves, int kPair>
__global__ __launch_bounds__(kRowWaves * kPair * kWave) void page_kernel(const Window a) {
  constexpr int kKeys = 16 * PageShape<QT, D>::kBlocks;
  __shared__ RowScratch<D, kRowWaves, kPair> shared;
  const uint32_t groups = a.num_kv_heads / kPair * a.subgroups;
  const Heads h = heads_of<kPair>(a, blockIdx.x % groups);
  const uint32_t item = blockIdx.x / groups;
  const int32_t split = item % static_cast<uint32_t>(a.splits);
  const int64_t t = item / static_cast<uint32_t>(a.splits);
  const int32_t seq = a.seqs[t];
  if (seq < 0 || seq >= a.num_seqs) return;
  const int32_t count = span_of(a, seq, a.positions[t]).end;
  const int32_t rounds = (count + kKeys - 1) / kKeys;
  const int32_t first = static_cast<int32_t>(static_cast<int64_t>(rounds) * split / a.splits);
  const int32_t last = static_cast<int32_t>(static_cast<int64_t>(rounds) * (split + 1) / a.splits);
  page_piece<QT, D, kRowWaves, kPair>(a, shared, t, seq, count, first, last, h.kv_head, h.head0, h.count, split_place(a, t, h.head0, split));
}

// The listed rows of a call with tiles, item by item of workgroup `block` of `blocks`. 20 rows of 2481 to 2853 keys beside a run of 10,
// 32/8 heads x 128, bfloat16, blocks of 16: 38 us, of one token, which the general row pass takes, 49.
template <typename QT, int D>
__device__ __forceinline__ void page_pass(const Window& a, RowScratch<D, kWaves, 1>& shared, uint32_t block, uint32_t blocks) {
  constexpr int kKeys = 16 * PageShape<QT, D>::kBlocks;
  const uint32_t groups = a.num_kv_heads * a.subgroups;
  const int64_t items = static_cast<int64_t>(a.list[0]) * a.splits * groups;
  for (int64_t next = block; next < items; next += blocks) {
    const uint32_t item = static_cast<uint32_t>(next) / groups;
    const Heads h = heads_of<1>(a, static_cast<uint32_t>(next) % groups);
    const int32_t split = item % static_cast<uint32_t>(a.splits);
    const int64_t t = a.list[1 + item / static_cast<uint32_t>(a.splits)];
    const int32_t seq = a.seqs[t];
    const int32_t count = span_of(a, seq, a.positions[t]).end;
    const int32_t rounds = (count + kKeys - 1) / kKeys;
    const int32_t first = static_cast<int32_t>(static_cast<int64_t>(rounds) * split / a.splits);
    const int32_t last = static_cast<int32_t>(static_cast<int64_t>(rounds) * (split + 1) / a.splits);
    page_piece<QT, D, kWaves, 1>(a, shared, t, seq, count, first, last, h.kv_head, h.head0, h.count, split_place(a, t, h.head0, split));
  }
}

// ---------------------------------------------------------------------------------------------
// The same with equal shares of the whole call's rounds instead of splits of its rows, whose lengths only the device knows: every
// workgroup sums all rows' rounds, and takes the rounds from `share` times its number on, through as many rows as they
// are of. A row that lies in one share is finished there; of the others each share leaves a part in the workspace, at most
// two (its first row's and its last's), and stream_join_kernel joins them.
// 64 rows of 2048 to 32768 keys, 32/8 heads x 128, 2.29 GB: 379 us, 6.0 TB/s; in 16 splits of each row 437, in equal pieces of
// 1024 keys, which all begin and end at the same time, 530. Rows of one length gain nothing and pay for the sums and the join, some
// 10 us together: calls of up to kStreamKeys keys, and of more rows than LDS has room for the sums of, take splits (16 rows of up
// to 1024 keys: 16 us, in shares 19).
// ---------------------------------------------------------------------------------------------
constexpr int kStreamRows = 1024;
constexpr int64_t kStreamKeys = 32768;

struct Stream {
  int32_t share;                    // rounds of a workgroup
  int32_t before[kStreamRows + 1];  // rounds of the rows before
};

// The place of a share's part of a row for one head: of its first row, or of its last.
__device__ __forceinline__ int64_t part_index(const Window& a, int32_t share, bool first, int32_t head) {
  return (static_cast<int64_t>(share) * 2 + (first ? 0 : 1)) * a.num_heads + head;
}

template <typename QT, int D, int kRowWaves, int kPair>
__global__ __launch_bounds__(kRowWaves * kPair * kWave) void stream_kernel(const Window a) {
  constexpr int kKeys = 16 * PageShape<QT, D>::kBlocks, kCount = kRowWaves * kPair * kWave, kPer = kStreamRows / kCount;
  __shared__ RowScratch<D, kRowWaves, kPair> shared;
  __shared__ int32_t s_before[kStreamRows + 1], s_count[kStreamRows], s_seq[kStreamRows], s_wave[kCount / kWave];
  const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = tid / kWave;
  const int32_t rows = static_cast<int32_t>(a.num_queries);
  // The sums: kPer rows to a thread.
  int32_t rounds[kPer], all = 0;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int32_t t = tid * kPer + i;
    int32_t seq = t < rows ? a.seqs[t] : -1, count = 0;
    if (seq >= 0 && seq < a.num_seqs) count = span_of(a, seq, a.positions[t]).end;
    s_seq[t] = seq;
    s_count[t] = count;
    rounds[i] = (count + kKeys - 1) / kKeys;
    all += rounds[i];
  }
  int32_t sum = all;
#pragma unroll
  for (int m = 1; m < kWave; m *= 2) {
    const int32_t other = __shfl_up(sum, m);
    if (lane >= m) sum += other;
  }
  if (lane == kWave - 1) s_wave[wave] = sum;
  __syncthreads();
  int32_t before = sum - all, total = 0;
#pragma unroll
  for (int w = 0; w < kCount / kWave; ++w) {
    before += w < wave ? s_wave[w] : 0;
    total += s_wave[w];
  }
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    s_before[tid * kPer + i] = before;
    before += rounds[i];
  }
  if (tid == 0) s_before[kStreamRows] = total;
  total = __builtin_amdgcn_readfirstlane(total);
  const int32_t share = max((total + a.stream_groups - 1) / a.stream_groups, a.stream_least);
  __syncthreads();
  if (blockIdx.x == 0) {
    for (int i = tid; i <= rows; i += kCount) a.stream->before[i] = i < rows ? s_before[i] : total;
    if (tid == 0) a.stream->share = share;
  }
  const uint32_t groups = a.num_kv_heads / kPair * a.subgroups;
  const Heads h = heads_of<kPair>(a, blockIdx.x % groups);
  const int32_t mine = blockIdx.x / groups;
  const int32_t begin = min(static_cast<int64_t>(mine) * share, static_cast<int64_t>(total)), end = min(begin + share, total);
  if (begin >= end) return;
  int32_t low = 0, high = rows - 1;  // the last row that begins at or before `begin` and has rounds: the one that holds it
  while (low < high) {
    const int32_t middle = (low + high + 1) / 2;
    if (s_before[middle] <= begin) low = middle; else high = middle - 1;
  }
  // What comes from LDS is the same in every lane, and in scalars the loops' conditions are too.
  for (int32_t at = begin, t = __builtin_amdgcn_readfirstlane(low); at < end; ++t) {
    const int32_t row0 = __builtin_amdgcn_readfirstlane(s_before[t]), row1 = __builtin_amdgcn_readfirstlane(s_before[t + 1]);
    if (row1 <= at) continue;  // without rounds
    const int32_t until = min(row1, end);
    const Place to{row0 >= begin && row1 <= end, part_index(a, mine, row0 <= begin, h.head0), 1, a.stream_places};
    page_piece<QT, D, kRowWaves, kPair>(a, shared, t, __builtin_amdgcn_readfirstlane(s_seq[t]), __builtin_amdgcn_readfirstlane(s_count[t]), at - row0,
                                        until - row0, h.kv_head, h.head0, h.count, to);
    at = until;
  }
}

// Joins the parts of the rows that more than one share has, and clears the rows that see nothing: D / 4 threads for each row
// and head.
template <typename QT, int D>
__global__ __launch_bounds__(kThreads) void stream_join_kernel(const Window a) {
  constexpr int kPer = D / 4, kTogether = 4;
  const uint32_t item = (blockIdx.x * static_cast<uint32_t>(kThreads) + threadIdx.x) / kPer;
  const int d = threadIdx.x % kPer * 4;
  const uint32_t t = item / static_cast<uint32_t>(a.num_heads);
  if (t >= a.num_queries) return;
  const int32_t head = item % static_cast<uint32_t>(a.num_heads);
  const int32_t seq = a.seqs[t], share = a.stream->share, row0 = a.stream->before[t], row1 = a.stream->before[t + 1];
  if (seq < 0 || seq >= a.num_seqs) return;
  float x[4] = {0.f, 0.f, 0.f, 0.f};
  QT* out = static_cast<QT*>(a.out) + static_cast<int64_t>(item) * D + d;
  if (row0 == row1) {
    store_row<QT, 4>(out, x);
    return;
  }
  const int32_t from = row0 / share, until = (row1 - 1) / share;
  if (from == until) return;  // its share has finished it
  const Place place{false, 0, 1, a.stream_places};
  float top = -INFINITY, sum = 0.f;
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  for (int32_t first = from; first <= until; first += kTogether) {
    float tp[kTogether], part[kTogether], most = top;
    f32x4 its[kTogether];
#pragma unroll
    for (int i = 0; i < kTogether; ++i) {
      const int32_t p = min(first + i, until);
      const int64_t index = part_index(a, p, row0 <= p * share, head);
      tp[i] = a.workspace[index];
      part[i] = first + i <= until ? a.workspace[place.total + index] : 0.f;
      its[i] = *reinterpret_cast<const f32x4*>(acc_of(a, place, index, D) + d);
    }
#pragma unroll
    for (int i = 0; i < kTogether; ++i) most = fmaxf(most, part[i] == 0.f ? -INFINITY : tp[i]);
    const float base = most == -INFINITY ? 0.f : most, keep = exp2f(top - base);
    sum *= keep;
    acc *= keep;
#pragma unroll
    for (int i = 0; i < kTogether; ++i) {
      if (part[i] == 0.f) continue;  // no key in this part: its output may hold anything
      const float weight = exp2f(tp[i] - base);
      sum += part[i] * weight;
      acc += its[i] * weight;
    }
    top = most;
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) x[e] = sum == 0.f ? 0.f : acc[e] / sum;
  store_row<QT, 4>(out, x);
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
// Over e4m3 codes, without a window (86 GFLOP): 170 us, replayed back to back 201. The staged codes and scales take all 256
// registers and 11 more are spilled (48 bytes a lane); over bfloat16 244 do. The CUs have work in 73% of the cycles, and in these the
// matrix units are busy in 35%, vector instructions issue in 48% and LDS works in 39%. Float32 queries: 364 us, one wavefront per SIMD.
// ---------------------------------------------------------------------------------------------
// float32 queries of head_dim 256 have tiles over codes alone (float32 pools' pieces do not fit LDS): over pools their rows go by
// themselves (codes, 5 x 455 rows behind up to 2055 others, 8 heads: 254 us, by themselves 3277).
constexpr bool tiles_of(int q_size, int head_dim) { return q_size == 2 || head_dim <= 128; }

template <typename QT, typename KVT, int D>
struct TileShape {
  static constexpr int kQPieces = sizeof(QT) == 4 ? 3 : 1;
  static constexpr int kKvPieces = sizeof(KVT) == 4 ? 3 : 1;
  static constexpr int kPPieces = sizeof(QT) == 4 ? 3 : 2;
  static constexpr int kKeys = (sizeof(KVT) <= 2 && D <= 128) || D == 32 ? 64 : 32;
  static constexpr int kChunks = D / 8;                                // 16-byte chunks of a bfloat16 row
  static constexpr int kPlane = kKeys * D;                             // elements of one piece of a staged tile
  static constexpr int kStaged = kKeys * kChunks / kThreads;           // chunks of a tile per thread, K and V each
  static constexpr int kLds = 2 * 2 * kKvPieces * kPlane * 2;          // bytes: two buffers of K and V
  static constexpr int kWaves = kLds <= 81920 && sizeof(QT) == 2 && D <= 128 ? 2 : 1;  // per SIMD
  static constexpr bool kFits = tiles_of(sizeof(QT), D) || sizeof(KVT) == 1;
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

// Eight bytes from global memory: of a chosen pointer the compiler no longer knows that it is one into global memory.
__device__ __forceinline__ u32x2 load_global(const void* from) {
  return *(const __attribute__((address_space(1))) u32x2*)(from);
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
  __shared__ float s_scale[3][2][sizeof(KVT) == 1 ? S::kKeys : 1];  // of codes, for keys and values
  const int tid = threadIdx.x, lane = tid & (kWave - 1), c = lane / 32, n = lane % 32;
  const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  // The rows outside the runs in the same launch, before bfloat16's tiles and behind float32's, which take
  // longer (24 rows beside 2 x 301, window 500, 16 heads x 64, float32 over bfloat16: 44 us, before the tiles 49; 64 rows of
  // up to 4096 keys beside 512, 32/8 heads x 128, bfloat16: 225 us, behind the tiles 247). In a launch of their own after
  // the tiles the first took 35% longer, the second 4%.
  constexpr bool kRowsFirst = sizeof(QT) == 2;
  const uint32_t row_blocks = gridDim.x - a.tile_items, before = kRowsFirst ? row_blocks : a.tile_items;
  if ((blockIdx.x < before) == kRowsFirst) {
    auto& scratch = *reinterpret_cast<RowScratch<D, kWaves, 1>*>(s_kv);
    const uint32_t block = blockIdx.x - (kRowsFirst ? 0 : before);
    if constexpr (sizeof(KVT) == 1) {
      if (a.page_groups > 0) return page_pass<QT, D>(a, scratch, block, row_blocks);
    }
    row_pass<QT, KVT, D, kWaves, 1>(a, scratch, block, row_blocks);
    return;
  }
  uint32_t item = blockIdx.x - (kRowsFirst ? before : 0);
  const int32_t kv_head = item % static_cast<uint32_t>(a.num_kv_heads);
  item /= static_cast<uint32_t>(a.num_kv_heads);
  const int32_t split = item % static_cast<uint32_t>(a.splits);
  int64_t block0 = item / static_cast<uint32_t>(a.splits);
  uint32_t share = 0;
  if constexpr (sizeof(KVT) == 1) {
    share = static_cast<uint32_t>(block0) % a.run_shares;
    block0 = static_cast<uint32_t>(block0) / a.run_shares;
    if (a.order) block0 = a.order[block0];
  }
  block0 *= a.tile_rows;
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
  uint32_t nth = 0;
  for (; runs != 0; runs &= runs - 1) {
    if constexpr (sizeof(KVT) == 1) {
      if (nth++ % a.run_shares != share) continue;
    }
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
    // Scales of codes: asked for when a tile's table entries have arrived, one tile after these and one before the rows are put.
    constexpr bool kCodes = sizeof(KVT) == 1;
    struct Scales {
      float key, value;
    };
    auto look_up_scales = [&](const Entry& e) {
      Scales s{1.f, 1.f};  // in no block: code 0 times a NaN is not 0
      if (e.block >= 0 && e.block < a.num_blocks) {
        const int64_t at = static_cast<int64_t>(e.block) * a.num_kv_heads + kv_head;
        s = Scales{a.key_scales[at], a.value_scales[at]};
      }
      return s;
    };
    auto keep_scales = [&](int32_t tile, const Scales& s) {
      if (tid < S::kKeys) s_scale[tile % 3][0][tid] = s.key, s_scale[tile % 3][1][tid] = s.value;
    };
    constexpr int kWide = sizeof(KVT) / 2;  // 16-byte loads of a chunk
    u32x4 kx[S::kStaged][kWide ? kWide : 1], vx[S::kStaged][kWide ? kWide : 1];
    u32x2 kc[kCodes ? S::kStaged : 1], vc[kCodes ? S::kStaged : 1];  // eight codes each
    auto load = [&](int32_t tile, int buffer) {
#pragma unroll
      for (int i = 0; i < S::kStaged; ++i) {
        const int at = tid + i * kThreads, row = at / S::kChunks, chunk = at % S::kChunks;
        const int32_t slot = s_slot[tile % 3][row];
        const int64_t from = row_of(a, slot, kv_head, D);
        if constexpr (kCodes) {
          kc[i] = load_global(slot >= 0 ? static_cast<const void*>(keys + from + 8 * chunk) : zeros);
          vc[i] = load_global(slot >= 0 ? static_cast<const void*>(values + from + 8 * chunk) : zeros);
        } else if constexpr (kWide == 1) {
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
    auto place = [&](int which, int i) {  // of a staged chunk in its plane
      const int at = tid + i * kThreads, row = at / S::kChunks, chunk = at % S::kChunks;
      return row * D + 8 * (which == 0 ? key_chunk<D>(row, chunk) : value_chunk<D>(row, chunk));
    };
    auto put_codes = [&](int buffer, int which, int i, const u32x2& x, float scale) {
      *reinterpret_cast<u32x4*>(plane(buffer, which, 0) + place(which, i)) =
          u32x4{widen<0>(x.x, scale), widen<1>(x.x, scale), widen<0>(x.y, scale), widen<1>(x.y, scale)};
    };
    auto put = [&](int buffer, int which, int i, const u32x4 (&x)[kWide ? kWide : 1]) {
      const int to = place(which, i);
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
    auto stage = [&](int32_t tile, int buffer) {
      if constexpr (kWide == 1) {
        __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0): this wavefront's loads to LDS have arrived
      } else if constexpr (kCodes) {
#pragma unroll
        for (int i = 0; i < S::kStaged; ++i) {
          const int row = (tid + i * kThreads) / S::kChunks;
          put_codes(buffer, 0, i, kc[i], s_scale[tile % 3][0][row]);
          put_codes(buffer, 1, i, vc[i], s_scale[tile % 3][1][row]);
        }
      } else {
#pragma unroll
        for (int i = 0; i < S::kStaged; ++i) {
          put(buffer, 0, i, kx[i]);
          put(buffer, 1, i, vx[i]);
        }
      }
    };

    __syncthreads();  // the run before is done with LDS
    Entry waiting{-1, -1};  // of codes: the tile's after the next
    {
      const Entry one = look_up(first), two = look_up(first + 1);
      keep_slots(first, one);
      keep_slots(first + 1, two);
      if constexpr (kCodes) {
        waiting = look_up(first + 2);
        keep_scales(first, look_up_scales(one));
        keep_scales(first + 1, look_up_scales(two));
      }
    }
    __syncthreads();
    if (first < last) {
      load(first, 0);
      stage(first, 0);
    }
    __syncthreads();
    for (int32_t tile = first; tile < last; ++tile) {
      const int buffer = (tile - first) & 1;
      const Entry ahead = kCodes ? look_up(tile + 3) : look_up(tile + 2);
      const Scales scales = kCodes ? look_up_scales(waiting) : Scales{};
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
      if (tile + 1 < last) stage(tile + 1, buffer ^ 1);
      if constexpr (kCodes) {
        keep_slots(tile + 2, waiting);
        keep_scales(tile + 2, scales);
        waiting = ahead;
      } else {
        keep_slots(tile + 2, ahead);
      }
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
      const Place to = split_place(a, t, head, split);
      if (a.splits > 1 && c == 0) store_sums(a, to, to.index, top, sum);
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
              store_row<float, 4>(acc_of(a, to, to.index, D) + d, x);
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
      const int32_t its_head = kv_head * a.group + (which - row * a.group);
      exact_row<QT, KVT, D>(a, run0 + row, its_head, seq, one, all, min(first * S::kKeys, count), min(last * S::kKeys, count),
                            split_place(a, run0 + row, its_head, split), 0);
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
  const Place place = split_place(a, 0, 0, 0);
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
      out[i] = *reinterpret_cast<const f32x4*>(acc_of(a, place, index + p, D) + d);
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

// How stream_kernel serves a call: key heads of a workgroup, and its shares. Rows are read in pieces of D bytes a head, so
// neighbouring heads together where there is much to read (64 rows of 4096 keys, 8 key heads x 128, in even splits: 94 us with
// four heads to a workgroup, 103 with two, 123 with one; 1 row 17.0, 14.9, 12.6). One workgroup of eight wavefronts or
// two of four for every CU.
struct PageForm {
  int32_t pair, groups;
};
PageForm page_form(int64_t num_queries, int32_t num_kv_heads, int32_t subgroups, int32_t head_dim, int32_t max_context) {
  const bool much = head_dim <= 128 && num_queries * max_context > 32768;
  const int32_t pair = much && num_kv_heads % 4 == 0 ? 4 : much && num_kv_heads % 2 == 0 ? 2 : 1;
  const int64_t columns = static_cast<int64_t>(num_kv_heads) / pair * subgroups;
  return PageForm{pair, static_cast<int32_t>(std::max<int64_t>(1, (pair == 1 ? 512 : 256) / columns))};
}
int64_t stream_bytes(const PageForm& form, int32_t num_heads, int32_t head_dim) {
  const int64_t places = 2 * static_cast<int64_t>(form.groups) * num_heads;
  return ((2 * places + 3) / 4 * 4 + places * head_dim) * static_cast<int64_t>(sizeof(float)) + static_cast<int64_t>(sizeof(Stream) + 15) / 16 * 16;
}

template <typename QT, typename KVT, int D>
int launch(Window a, hipStream_t stream) {
  using S = TileShape<QT, KVT, D>;
  a.subgroups = (a.group + 15) / 16;
  a.tile_rows = kTileQueries / a.group;
  a.min_run = std::min(kMinRun, a.tile_rows);
  a.tiled = S::kFits && a.list;  // no list without tiles
  if (a.page_groups > 0) a.page_magic = static_cast<uint32_t>(((int64_t{1} << 32) + a.page_groups - 1) / a.page_groups);
  const int64_t items = a.num_queries * a.num_kv_heads * a.subgroups * a.splits;
  // Beside tiles the number of rows is known on the device only: two workgroups for every CU share them.
  const int64_t groups = a.tiled ? std::min<int64_t>(items, 512) : items;
  const int64_t tiles = (a.num_queries + a.tile_rows - 1) / a.tile_rows * a.num_kv_heads * a.splits * std::max(a.run_shares, 1u);
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
      if (a.order) {
        hipLaunchKernelGGL(list_kernel<true>, dim3(1), dim3(kListThreads), 0, stream, a);
      } else {
        hipLaunchKernelGGL(list_kernel<false>, dim3(1), dim3(kListThreads), 0, stream, a);
      }
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
  constexpr bool kShort = D * sizeof(KVT) <= 256 && D <= 128;
  constexpr bool kWide = D < 128 || (D == 128 && (sizeof(QT) == sizeof(KVT) || (sizeof(QT) == 2 && sizeof(KVT) == 1)));
  const bool wide = kWide && groups <= 256;
  const bool pair = kShort && groups >= 512 && a.num_kv_heads % 2 == 0;
  const auto start = [&](auto kernel, int64_t count, int waves) {
    hipLaunchKernelGGL(kernel, dim3(static_cast<uint32_t>(count)), dim3(waves * kWave), 0, stream, a);
  };
  if constexpr (sizeof(KVT) == 1) {
    if (a.page_groups > 0) {
      if (!a.stream) {
        // Where there are many rows, a workgroup serves four neighbouring key heads and so reads 4 D bytes next to each other
        // (128 rows of 256 keys, 8 key heads x 128: 17.0 us, a head to a workgroup 21.8; 16 rows 10.4 and 9.0).
        constexpr bool kFour = D <= 128;
        if (kFour && a.num_kv_heads % 4 == 0 && groups >= 1024) {
          if constexpr (kFour) start(page_kernel<QT, D, 2, 4>, groups / 4, 8);
        } else {
          start(page_kernel<QT, D, 4, 1>, groups, 4);
        }
        join();
        return check_launch();
      }
      const PageForm form = page_form(a.num_queries, a.num_kv_heads, a.subgroups, D, a.max_context);
      const int64_t shares = static_cast<int64_t>(a.stream_groups) * (a.num_kv_heads / form.pair) * a.subgroups;
      if constexpr (D <= 128) {
        if (form.pair == 4) start(stream_kernel<QT, D, 2, 4>, shares, 8);
        if (form.pair == 2) start(stream_kernel<QT, D, 4, 2>, shares, 8);
      }
      if (form.pair == 1) start(stream_kernel<QT, D, 4, 1>, shares, 4);
      hipLaunchKernelGGL((stream_join_kernel<QT, D>), dim3(static_cast<uint32_t>(joins)), dim3(kThreads), 0, stream, a);
      return check_launch();
    }
  }
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

namespace pkv {
namespace {
// How a call runs: its splits (below 1: refused), its bytes of workspace, and whether it has tiles beside its rows. Over codes:
// whether page_kernel's 16 keys to a block hold, and whether its rows are cut into equal shares instead of splits.
struct Plan {
  int32_t splits = 0;
  int64_t bytes = 0, order_bytes = 0;  // the order's are its last
  uint32_t run_shares = 1;
  bool runs = false, pages = false, stream = false;
  PageForm form{};
};

Plan window_plan(const pkv_window& g) {
  Plan p;
  p.runs = tiles_of(dtype_size(static_cast<pkv_dtype>(g.q_dtype)), g.head_dim) && has_runs(g.max_query_len, g.num_heads / g.num_kv_heads);
  p.splits = pkv_window_sizes(g.num_queries, g.num_heads, g.num_kv_heads, g.head_dim, g.q_dtype, g.window, g.sinks, g.max_context_len,
                              g.max_query_len, g.num_splits, &p.bytes);
  return p;
}

// The blocks of rows that list_kernel orders, 0 where they are too many.
int64_t ordered_blocks(int64_t num_queries, int32_t group) {
  const int64_t rows = kTileQueries / group, blocks = (num_queries + rows - 1) / rows;
  return blocks <= kListThreads ? blocks : 0;
}

Plan codes_plan(const pkv_window& g) {
  Plan p = window_plan(g);
  if (p.splits < 1) return p;
  const int32_t group = g.num_heads / g.num_kv_heads;
  // page_kernel's offsets within 16 rows are 32-bit, and its reciprocal holds for up to 64 groups to a block.
  p.pages = g.window == INT32_MAX && g.block_size % 16 == 0 && g.block_size <= 1024 && g.num_blocks > 0 && g.num_kv_heads <= (1 << 18);
  p.runs = has_runs(g.max_query_len, group);
  if (p.runs) {
    // Tiles of one split: one at least, as a workspace may be asked for without queries.
    const int64_t rows = kTileQueries / group, groups = std::max<int64_t>(1, (g.num_queries + rows - 1) / rows * g.num_kv_heads);
    p.bytes = pkv_window_workspace_bytes(g.num_queries, g.num_heads, g.head_dim, g.max_query_len, p.splits);
    if (g.num_splits == 0) {
      // Tiles of bfloat16 queries are two to a CU, of float32 ones one. Shares of 384 keys at least, of 128 where tiles are few: a part
      // more of every row is written and joined. 1 x 128 rows of up to 4128 keys, 32/8 heads x 128, float32, with 4, 8, 16 splits:
      // 46, 39, 53 us; 2 x 301 rows beside 24, 16 heads x 64, window 1000, with 1, 2, 3, 6: 58, 46, 54, 65; 1 x 32 rows of
      // 1032 keys, 16/2 heads x 64, bfloat16, with 2, 4, 8: 19, 15, 15; 3 x 339 rows of up to 610 keys, 8/1 heads x 64, float32 (64 tiles),
      // with 1, 2, 4, 8: 49, 39, 34, 34; 1 x 512 rows, 8 heads x 128, bfloat16 (32 tiles): 36, 30, 27, 27; 7 x 130 rows of 226 keys, 16/4
      // heads x 256 (116 tiles): 51, 51, 62, 94.
      const int64_t longest = std::min<int64_t>(g.max_context_len, static_cast<int64_t>(g.window) + g.sinks);
      const int64_t shares = groups <= 64 ? std::min(longest / 128, std::max<int64_t>(8, longest / 1024)) : longest / 384;
      const int64_t tiles = (g.q_dtype == PKV_F32 || (groups > 16 && groups <= 64) ? 256 : 512) / groups;
      // The rows by themselves, a sequence each at most, have the tiles' splits, and fill the GPU with fewer. 20 rows of 2481 to 2853 keys
      // beside a run of 10, 32/8 heads x 128, bfloat16, with 1, 3, 8, 22: 44, 39, 52, 81; 64 rows of 100 to 4000 beside 512, with 1, 3: 104,
      // 115; 61 of 64 beside a run of 6 with 1503, 16/8 heads x 64, float32, with 1, 3, 8: 65, 33, 48.
      const int64_t rows_fill = std::max(std::min<int64_t>(3, 256 / groups), 512 / std::max<int64_t>(1, static_cast<int64_t>(g.num_seqs) * g.num_kv_heads));
      p.splits = static_cast<int32_t>(std::max<int64_t>(1, std::min({int64_t{PKV_WINDOW_MAX_SPLITS}, shares, tiles, rows_fill})));
      p.bytes = pkv_window_workspace_bytes(g.num_queries, g.num_heads, g.head_dim, g.max_query_len, p.splits);
    }
    // A tile's runs one after the other cost their latencies; where tiles are few and runs surely shorter than they are, several
    // workgroups share them. 6 x 27 rows, 8 heads x 128, bfloat16: 17 us, in one workgroup each 52; 2 x 12 rows of up to 1191
    // keys, 8/2 heads x 128, float32: 24 us and 40.
    const int64_t parts = groups * p.splits, longest = g.max_query_len;
    // Of longer runs a tile may still hold the end of one and the start of the next: two workgroups for it, one of them mostly without
    // any, cost what their look does (7 x 211 rows, 16/8 heads x 32, float32: 25 us, with one 35; 2 x 465 rows beside 15, 8/1 heads x
    // 128, bfloat16, 240 workgroups: 42 and 34).
    const int64_t least = g.num_seqs > 1 && parts <= (g.q_dtype == PKV_F32 ? 256 : 192) ? 2 : 1;
    p.run_shares = static_cast<uint32_t>(std::max(least, std::min({int64_t{8}, 256 / parts, (2 * rows + longest - 1) / longest})));
    p.order_bytes = (ordered_blocks(g.num_queries, group) + 3) / 4 * 16;
    p.bytes += p.order_bytes;
    return p;
  }
  // A short row is one workgroup's, which saves the join's launch. Sums of rounds, of 16 keys at least, are 32-bit.
  p.stream = p.pages && g.num_splits == 0 && g.num_queries <= kStreamRows && g.num_queries * g.max_context_len > kStreamKeys &&
             g.num_queries * ((g.max_context_len + int64_t{15}) / 16) < (int64_t{1} << 30);
  if (p.stream) {
    const int32_t subgroups = (g.num_heads / g.num_kv_heads + 15) / 16;
    p.form = page_form(g.num_queries, g.num_kv_heads, subgroups, g.head_dim, g.max_context_len);
    p.splits = 1;
    p.bytes = stream_bytes(p.form, g.num_heads, g.head_dim);
  }
  return p;
}

// pkv_window_attention, and with scales pkv_attention_e4m3, whose pools hold codes (kv_dtype is not looked at then).
int attention(const pkv_window& g, const float* key_scales, const float* value_scales, bool codes, int device, void* stream) {
  if (g.num_queries < 0 || g.num_heads < 1 || g.num_kv_heads < 1 || g.num_heads % g.num_kv_heads != 0 || g.num_seqs < 0 ||
      g.num_blocks < 0 || g.block_size < 1 || g.block_table_stride < 0 || g.window < 1 || g.sinks < 0 ||
      g.max_context_len < 0 || g.max_query_len < 0 || g.num_splits < 0 || g.num_splits > PKV_WINDOW_MAX_SPLITS) {
    return PKV_EINVAL;
  }
  if (static_cast<int64_t>(g.block_table_stride) * g.block_size < g.max_context_len) return PKV_EINVAL;
  if (g.q_dtype != PKV_F32 && g.q_dtype != PKV_BF16) return PKV_EINVAL;
  if (!codes && g.kv_dtype != PKV_F32 && g.kv_dtype != PKV_BF16) return PKV_EINVAL;
  if (!codes && g.q_dtype == PKV_BF16 && g.kv_dtype == PKV_F32) return PKV_EUNSUPPORTED;
  if (g.head_dim != 32 && g.head_dim != 64 && g.head_dim != 128 && g.head_dim != 256) return PKV_EUNSUPPORTED;
  if (g.num_heads / g.num_kv_heads > PKV_WINDOW_MAX_GROUP) return PKV_EUNSUPPORTED;
  // Slots, and a span's items some tiles past its end, are 32-bit.
  if (g.num_blocks > 0x7fffffff / g.block_size || g.max_context_len > PKV_WINDOW_MAX_CONTEXT) return PKV_EUNSUPPORTED;
  if (g.num_queries == 0) return PKV_OK;
  if (!g.out || !g.queries || !g.query_positions || !g.query_seq || !g.key_cache || !g.value_cache || !g.block_tables ||
      !g.context_lens || (codes && (!key_scales || !value_scales))) {
    return PKV_EINVAL;
  }
  const int64_t row = static_cast<int64_t>(g.num_heads) * g.head_dim;
  const int64_t elems = 16 / dtype_size(static_cast<pkv_dtype>(g.q_dtype));
  if (g.query_token_stride < row || g.query_token_stride % elems != 0 || !aligned16(g.out) || !aligned16(g.queries) ||
      !aligned16(g.key_cache) || !aligned16(g.value_cache)) {
    return PKV_EINVAL;
  }
  const Plan plan = codes ? codes_plan(g) : window_plan(g);
  const int32_t splits = plan.splits;
  const int64_t need = plan.bytes;
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
  a.key_scales = key_scales;
  a.value_scales = value_scales;
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
  if (plan.runs) a.list = reinterpret_cast<int32_t*>(reinterpret_cast<char*>(g.workspace) + need - plan.order_bytes - list_bytes(g.num_queries));
  if (plan.order_bytes > 0) a.order = reinterpret_cast<int32_t*>(reinterpret_cast<char*>(g.workspace) + need - plan.order_bytes);
  a.run_shares = plan.run_shares;
  if (plan.pages) a.page_groups = g.block_size / 16;
  if (plan.stream) {
    a.stream_groups = plan.form.groups;
    a.stream_least = 8;
    a.stream_places = 2 * static_cast<int64_t>(a.stream_groups) * g.num_heads;
    a.stream = reinterpret_cast<Stream*>(reinterpret_cast<char*>(g.workspace) + need - (sizeof(Stream) + 15) / 16 * 16);
  }
  DeviceGuard guard(device);
  if (!guard.ok()) return PKV_EHIP;
  auto s = static_cast<hipStream_t>(stream);
  if (g.q_dtype == PKV_BF16) {
    a.flip = a.scale_log2 < 0.f ? 0x80008000u : 0u;
    a.keep = a.scale_log2 == 0.f ? 0u : 0xffffffffu;
    a.scale_log2 = a.scale_log2 == 0.f ? 1.f : std::fabs(a.scale_log2);
    return codes ? dispatch<uint16_t, uint8_t>(a, g.head_dim, s) : dispatch<uint16_t, uint16_t>(a, g.head_dim, s);
  }
  if (codes) return dispatch<float, uint8_t>(a, g.head_dim, s);
  return g.kv_dtype == PKV_F32 ? dispatch<float, float>(a, g.head_dim, s)
                               : dispatch<float, uint16_t>(a, g.head_dim, s);
}
}  // namespace
}  // namespace pkv

extern "C" int pkv_window_attention(const pkv_window* args, int device, void* stream) {
  return args ? pkv::attention(*args, nullptr, nullptr, false, device, stream) : PKV_EINVAL;
}

namespace pkv {
namespace {
pkv_window window_of(const pkv_e4m3_attention& g) {
  pkv_window w{};
  w.out = g.out;
  w.queries = g.queries;
  w.query_token_stride = g.query_token_stride;
  w.query_positions = g.query_positions;
  w.query_seq = g.query_seq;
  w.num_queries = g.num_queries;
  w.key_cache = g.key_cache;
  w.value_cache = g.value_cache;
  w.num_blocks = g.num_blocks;
  w.block_tables = g.block_tables;
  w.context_lens = g.context_lens;
  w.workspace = g.workspace;
  w.workspace_bytes = g.workspace_bytes;
  w.q_dtype = g.q_dtype;
  w.block_size = g.block_size;
  w.block_table_stride = g.block_table_stride;
  w.num_seqs = g.num_seqs;
  w.num_heads = g.num_heads;
  w.num_kv_heads = g.num_kv_heads;
  w.head_dim = g.head_dim;
  w.window = g.window;
  w.sinks = g.sinks;
  w.max_context_len = g.max_context_len;
  w.max_query_len = g.max_query_len;
  w.num_splits = g.num_splits;
  w.scale = g.scale;
  return w;
}
}  // namespace
}  // namespace pkv

extern "C" int64_t pkv_attention_e4m3_workspace_bytes(const pkv_e4m3_attention* args) {
  if (!args) return PKV_EINVAL;
  const pkv_e4m3_attention& g = *args;
  if (g.num_queries < 0 || g.num_heads < 1 || g.num_kv_heads < 1 || g.num_heads % g.num_kv_heads != 0 || g.head_dim < 1 || g.block_size < 1 ||
      g.window < 1 || g.sinks < 0 || g.max_context_len < 0 || g.max_query_len < 0 || g.num_splits < 0 || g.num_splits > PKV_WINDOW_MAX_SPLITS ||
      g.num_heads / g.num_kv_heads > PKV_WINDOW_MAX_GROUP) {
    return PKV_EINVAL;
  }
  const pkv::Plan plan = pkv::codes_plan(pkv::window_of(g));
  return plan.splits < 1 ? PKV_EINVAL : plan.bytes;
}

extern "C" int pkv_attention_e4m3(const pkv_e4m3_attention* args, int device, void* stream) {
  if (!args) return PKV_EINVAL;
  return pkv::attention(pkv::window_of(*args), args->key_scales, args->value_scales, true, device, stream);
}
