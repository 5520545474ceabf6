// Rotary embedding with several position axes fused with the append to a paged cache of grouped
// heads: one pass over a layer's fresh q, k, v rows that rotates q (to a caller buffer) and k (into
// the key pool at the token's slot) and copies v into the value pool.
//
// With R = 2 * half rotated dimensions of a head and frequency i < half turned by axis a(i):
//     c = cos[pos[a(i)]][i], s = sin[pos[a(i)]][i]
//     out[i] = x[i] * c - x[i + half] * s ;  out[i + half] = x[i + half] * c + x[i] * s
//     out[j] = x[j] for j >= R
// in float32, each product and sum rounded on its own, and one rounding to the output's type.
//
// Bound: HBM, every q, k, v element read once and written once; the tables come from the caches. Two
// heads per thread share their table entries and have four loads in flight, and what is read once goes past
// the caches. 4216 tokens of 32 + 2 * 32 heads x 128 in float32, 417 MB: 63 us, 6.6 TB/s, where the pools lie
// in the caches, 82 us, 5.1 TB/s, with other tensors each time (a copy of 4 GiB: 4.8 TB/s). 16384 tokens of
// 32 + 2 * 4 heads x 128 in bfloat16 with three axes, 345 MB: 67 us, 5.1 TB/s. 4 tokens: 4.0 us, a launch.
#include "pkv_common.h"

namespace pkv {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxAxes = 4;
constexpr int kHeads = 2;  // heads of one thread

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));

// kVec elements held as float32: 16 bytes of the input's type (4 or 8 elements), or one element.
template <typename T, int kVec>
__device__ __forceinline__ void load_vec(const T* p, float (&v)[kVec]) {
  if constexpr (kVec == 1) {
    if constexpr (sizeof(T) == 4) {
      v[0] = *p;
    } else {
      v[0] = __uint_as_float(static_cast<uint32_t>(*p) << 16);
    }
  } else if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < kVec; i += 4) {
      const f32x4 x = __builtin_nontemporal_load(reinterpret_cast<const f32x4*>(p + i));
#pragma unroll
      for (int e = 0; e < 4; ++e) v[i + e] = x[e];
    }
  } else {
    static_assert(kVec == 8, "16 bytes of bfloat16");
    const u32x4 x = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(p));
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      v[2 * e] = bf16_lo(x[e]);
      v[2 * e + 1] = bf16_hi(x[e]);
    }
  }
}

template <typename T, int kVec>
__device__ __forceinline__ void store_vec(T* p, const float (&v)[kVec]) {
  if constexpr (kVec == 1) {
    if constexpr (sizeof(T) == 4) {
      *p = v[0];
    } else {
      *p = static_cast<T>(f32_to_bf16_bits(v[0]));
    }
  } else if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < kVec; i += 4) {
      *reinterpret_cast<f32x4*>(p + i) = f32x4{v[i], v[i + 1], v[i + 2], v[i + 3]};
    }
  } else if constexpr (kVec == 8) {
    u32x4 x;
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = f32_to_bf16_bits(v[2 * e]) | (f32_to_bf16_bits(v[2 * e + 1]) << 16);
    *reinterpret_cast<u32x4*>(p) = x;
  } else {
    static_assert(kVec == 4, "8 bytes of bfloat16");
    *reinterpret_cast<uint2*>(p) = uint2{f32_to_bf16_bits(v[0]) | (f32_to_bf16_bits(v[1]) << 16),
                                         f32_to_bf16_bits(v[2]) | (f32_to_bf16_bits(v[3]) << 16)};
  }
}

// Table entries: read by every head of a token, so through the caches.
template <int kVec>
__device__ __forceinline__ void load_table(const float* p, float (&v)[kVec]) {
  if constexpr (kVec == 1) {
    v[0] = *p;
  } else {
#pragma unroll
    for (int i = 0; i < kVec; i += 4) {
      const f32x4 x = *reinterpret_cast<const f32x4*>(p + i);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[i + e] = x[e];
    }
  }
}

struct RopeAxes {
  void* rotated;
  const void* queries;
  const void* keys;
  const void* values;
  const int64_t* positions;
  const float* cos_table;
  const float* sin_table;
  void* key_pool;
  void* value_pool;
  const int64_t* slots;
  int64_t rotated_stride, q_stride, k_stride, v_stride;
  int64_t axis_stride, table_rows, num_slots, num_tokens;
  int32_t num_heads, num_kv_heads, head_dim, half;
  int32_t num_axes, interleaved;
  int32_t ends[kMaxAxes];  // frequencies of axes 0..a (their sections' running sum)
  int32_t sections[kMaxAxes];
  // A token's work: `chunks` pieces of a head (turned ones, kVec pairs each, then copied ones of kVec
  // elements) times `sets` sets of up to kHeads of the query, key and value heads.
  int32_t turned, chunks, sets;
};

// The axis that turns frequency i: contiguous sections, or one frequency of each axis in turn until
// an axis has its section's number (what is left over goes to axis 0).
__device__ __forceinline__ int axis_of(const RopeAxes& a, int i) {
  if (a.interleaved) {
    const int axis = i % a.num_axes;
    return i < a.num_axes * a.sections[axis] ? axis : 0;
  }
  int axis = 0;
#pragma unroll
  for (int n = 0; n < kMaxAxes - 1; ++n) axis += n + 1 < a.num_axes && i >= a.ends[n];
  return axis;
}

// One thread per (token, set of kHeads heads, piece of a head): the heads of a set share their table
// entries, and their loads are all in flight before the first is used. Heads of one set are a number of sets
// apart, so that the threads of a wavefront read neighbouring heads. The values' heads are copied by the
// threads of the same pieces.
template <typename IoT, typename PoolT, int kVec>
__global__ __launch_bounds__(kThreads) void rope_axes_kernel(const RopeAxes a) {
  const uint32_t item = blockIdx.x * static_cast<uint32_t>(kThreads) + threadIdx.x;
  const uint32_t rest = item / static_cast<uint32_t>(a.chunks);
  const int chunk = item - rest * a.chunks;
  const uint32_t token = rest / static_cast<uint32_t>(a.sets);
  const int set = rest - token * a.sets;
  if (token >= a.num_tokens) return;
  const int64_t t = token;
  const bool pair = chunk < a.turned;
  const int i = pair ? chunk * kVec : 2 * a.half + (chunk - a.turned) * kVec;  // dimension of the (lower) piece
  const int heads = a.num_heads + 2 * a.num_kv_heads;

  float lo[kHeads][kVec], hi[kHeads][kVec];
#pragma unroll
  for (int h = 0; h < kHeads; ++h) {
    const int head = set + h * a.sets;
    if (head >= heads) break;
    const int kv = head - a.num_heads;
    const IoT* src = kv < 0 ? static_cast<const IoT*>(a.queries) + t * a.q_stride + static_cast<int64_t>(head) * a.head_dim
                     : kv < a.num_kv_heads
                         ? static_cast<const IoT*>(a.keys) + t * a.k_stride + static_cast<int64_t>(kv) * a.head_dim
                         : static_cast<const IoT*>(a.values) + t * a.v_stride + static_cast<int64_t>(kv - a.num_kv_heads) * a.head_dim;
    load_vec<IoT, kVec>(src + i, lo[h]);
    if (pair) load_vec<IoT, kVec>(src + i + a.half, hi[h]);
  }

  int64_t pos[kMaxAxes];
  bool inside = true;
#pragma unroll
  for (int n = 0; n < kMaxAxes; ++n) {
    pos[n] = n < a.num_axes ? a.positions[n * a.axis_stride + t] : 0;
    inside = inside && pos[n] >= 0 && (n >= a.num_axes || pos[n] < a.table_rows);
  }
  const int64_t slot = a.slots[t];
  const bool stored = slot >= 0 && slot < a.num_slots;
  if (!inside) return;

  float c[kVec], s[kVec];
  if (pair) {
    auto row_of = [&](int n) { return n == 0 ? pos[0] : n == 1 ? pos[1] : n == 2 ? pos[2] : pos[3]; };
    const int axis = axis_of(a, i);
    if (a.num_axes == 1 || (!a.interleaved && axis == axis_of(a, i + kVec - 1))) {
      const int64_t row = row_of(axis) * a.half + i;
      load_table<kVec>(a.cos_table + row, c);
      load_table<kVec>(a.sin_table + row, s);
    } else {
#pragma unroll
      for (int e = 0; e < kVec; ++e) {
        const int64_t row = row_of(axis_of(a, i + e)) * a.half + i + e;
        c[e] = a.cos_table[row];
        s[e] = a.sin_table[row];
      }
    }
  }
  const int64_t pool_row = slot * a.num_kv_heads * static_cast<int64_t>(a.head_dim);
#pragma unroll
  for (int h = 0; h < kHeads; ++h) {
    const int head = set + h * a.sets;
    if (head >= heads) break;
    const int kv = head - a.num_heads;
    if (pair && kv < a.num_kv_heads) {
#pragma clang fp contract(off)
#pragma unroll
      for (int e = 0; e < kVec; ++e) {
        const float ac = lo[h][e] * c[e];
        const float bs = hi[h][e] * s[e];
        const float bc = hi[h][e] * c[e];
        const float as = lo[h][e] * s[e];
        lo[h][e] = ac - bs;
        hi[h][e] = bc + as;
      }
    }
    // The rotated queries may overwrite the queries in place: this thread has read its pieces of them.
    if (kv < 0) {
      IoT* to = static_cast<IoT*>(a.rotated) + t * a.rotated_stride + static_cast<int64_t>(head) * a.head_dim + i;
      store_vec<IoT, kVec>(to, lo[h]);
      if (pair) store_vec<IoT, kVec>(to + a.half, hi[h]);
    } else if (stored) {
      const bool key = kv < a.num_kv_heads;
      PoolT* to = static_cast<PoolT*>(key ? a.key_pool : a.value_pool) + pool_row +
                  static_cast<int64_t>(key ? kv : kv - a.num_kv_heads) * a.head_dim + i;
      store_vec<PoolT, kVec>(to, lo[h]);
      if (pair) store_vec<PoolT, kVec>(to + a.half, hi[h]);
    }
  }
}

template <typename IoT, typename PoolT, int kVec>
int launch(RopeAxes a, hipStream_t stream) {
  const int64_t heads = a.num_heads + 2 * static_cast<int64_t>(a.num_kv_heads);
  a.turned = a.half / kVec;
  a.chunks = a.turned + (a.head_dim - 2 * a.half) / kVec;
  a.sets = static_cast<int32_t>((heads + kHeads - 1) / kHeads);
  const int64_t items = a.num_tokens * a.chunks * a.sets;
  if (heads > 0x3fffffff || a.num_tokens > 0x7fffffff || items > 0xffff0000ll) return PKV_EUNSUPPORTED;
  hipLaunchKernelGGL((rope_axes_kernel<IoT, PoolT, kVec>), dim3(static_cast<uint32_t>((items + kThreads - 1) / kThreads)), dim3(kThreads),
                     0, stream, a);
  return check_launch();
}

// 16-byte accesses need every row start, the half and the rest of a head on vector bounds.
template <typename IoT, typename PoolT>
int dispatch_vec(const RopeAxes& a, hipStream_t stream) {
  constexpr int kVec = 16 / sizeof(IoT);
  const bool vectors = a.half % kVec == 0 && a.head_dim % kVec == 0 && a.rotated_stride % kVec == 0 &&
                       a.q_stride % kVec == 0 && a.k_stride % kVec == 0 && a.v_stride % kVec == 0 &&
                       aligned16(a.rotated) && aligned16(a.queries) && aligned16(a.keys) && aligned16(a.values) &&
                       aligned16(a.key_pool) && aligned16(a.value_pool) && aligned16(a.cos_table) &&
                       aligned16(a.sin_table);
  return vectors ? launch<IoT, PoolT, kVec>(a, stream) : launch<IoT, PoolT, 1>(a, stream);
}

}  // namespace
}  // namespace pkv

extern "C" int pkv_rope_append_axes(const pkv_rope_axes* args, int device, void* stream) {
  using namespace pkv;
  if (!args) return PKV_EINVAL;
  const pkv_rope_axes& g = *args;
  if (g.num_tokens < 0 || g.num_heads < 1 || g.num_kv_heads < 1 || g.head_dim < 2 || g.rotary_dim < 2 ||
      g.rotary_dim % 2 != 0 || g.rotary_dim > g.head_dim || g.num_slots < 0 || g.table_rows < 0) {
    return PKV_EINVAL;
  }
  if ((g.io_dtype != PKV_F32 && g.io_dtype != PKV_BF16) || (g.pool_dtype != PKV_F32 && g.pool_dtype != PKV_BF16)) {
    return PKV_EINVAL;
  }
  if (g.num_axes < 1 || g.num_axes > kMaxAxes) return PKV_EINVAL;
  RopeAxes a{};
  int64_t total = 0;
  for (int n = 0; n < g.num_axes; ++n) {
    if (g.sections[n] < 0 || g.sections[n] > g.rotary_dim) return PKV_EINVAL;
    total += g.sections[n];
    a.sections[n] = g.sections[n];
    a.ends[n] = static_cast<int32_t>(total);
  }
  if (total != g.rotary_dim / 2) return PKV_EINVAL;
  for (int n = 1; g.interleaved && n < g.num_axes; ++n) {  // the last frequency of axis n has to exist
    if (g.sections[n] > 0 && n + g.num_axes * static_cast<int64_t>(g.sections[n] - 1) >= total) return PKV_EINVAL;
  }
  if (g.num_tokens == 0) return PKV_OK;
  if (!g.rotated_queries || !g.queries || !g.keys || !g.values || !g.positions || !g.cos_table || !g.sin_table ||
      !g.key_pool || !g.value_pool || !g.slot_mapping) {
    return PKV_EINVAL;
  }
  const int64_t q_row = static_cast<int64_t>(g.num_heads) * g.head_dim;
  const int64_t kv_row = static_cast<int64_t>(g.num_kv_heads) * g.head_dim;
  if (g.query_token_stride < q_row || g.rotated_token_stride < q_row || g.key_token_stride < kv_row ||
      g.value_token_stride < kv_row || (g.num_axes > 1 && g.position_axis_stride < 0)) {
    return PKV_EINVAL;
  }
  if (g.rotated_queries == g.queries && g.rotated_token_stride != g.query_token_stride) return PKV_EINVAL;
  a.rotated = g.rotated_queries;
  a.queries = g.queries;
  a.keys = g.keys;
  a.values = g.values;
  a.positions = g.positions;
  a.cos_table = g.cos_table;
  a.sin_table = g.sin_table;
  a.key_pool = g.key_pool;
  a.value_pool = g.value_pool;
  a.slots = g.slot_mapping;
  a.rotated_stride = g.rotated_token_stride;
  a.q_stride = g.query_token_stride;
  a.k_stride = g.key_token_stride;
  a.v_stride = g.value_token_stride;
  a.axis_stride = g.position_axis_stride;
  a.table_rows = g.table_rows;
  a.num_slots = g.num_slots;
  a.num_tokens = g.num_tokens;
  a.num_heads = g.num_heads;
  a.num_kv_heads = g.num_kv_heads;
  a.head_dim = g.head_dim;
  a.half = g.rotary_dim / 2;
  a.num_axes = g.num_axes;
  a.interleaved = g.interleaved != 0;
  DeviceGuard guard(device);
  if (!guard.ok()) return PKV_EHIP;
  auto s = static_cast<hipStream_t>(stream);
  if (g.io_dtype == PKV_F32) {
    return g.pool_dtype == PKV_F32 ? dispatch_vec<float, float>(a, s) : dispatch_vec<float, uint16_t>(a, s);
  }
  return g.pool_dtype == PKV_F32 ? dispatch_vec<uint16_t, float>(a, s) : dispatch_vec<uint16_t, uint16_t>(a, s);
}
