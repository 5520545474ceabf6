// The append to a paged cache of 8-bit floats (e4m3: 4 exponent and 3 mantissa bits, up to 448) with a power of two as
// the scale of each block of tokens and head: a value is its code times its block's scale.
#include "pkv_common.h"

namespace pkv {
namespace {

constexpr int kThreads = 256;
constexpr int kHeld = 16;           // tokens whose values a wavefront holds between their maximum and their codes
constexpr int kLowExponent = -100;  // of a scale: far above where code times scale would leave bfloat16's normal numbers

typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

struct Append {
  uint8_t* pool[2];  // keys, values
  float* scales[2];
  const void* source[2];
  int64_t stride[2];
  int32_t aligned[2];  // 16-byte loads of the source rows
  const int64_t* slots;
  int64_t tokens;
  int32_t num_slots, block_size, kv_heads, window;
};

// Eight adjacent values of a source row.
struct Eight {
  float v[8];
};
__device__ __forceinline__ Eight load_eight(const float* p, bool aligned) {
  Eight x;
  if (aligned) {
    const f32x4 a = *reinterpret_cast<const f32x4*>(p), b = *reinterpret_cast<const f32x4*>(p + 4);
#pragma unroll
    for (int i = 0; i < 4; ++i) x.v[i] = a[i], x.v[4 + i] = b[i];
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) x.v[i] = p[i];
  }
  return x;
}
__device__ __forceinline__ Eight load_eight(const uint16_t* p, bool aligned) {
  Eight x;
  if (aligned) {
    const u32x4 a = *reinterpret_cast<const u32x4*>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) x.v[2 * i] = bf16_lo(a[i]), x.v[2 * i + 1] = bf16_hi(a[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) x.v[i] = __uint_as_float(static_cast<uint32_t>(p[i]) << 16);
  }
  return x;
}

// The same as they are stored, to be held in fewer registers.
template <typename T>
struct Stored {
  u32x4 w[sizeof(T) / 2];
};
template <typename T>
__device__ __forceinline__ Stored<T> load_stored(const T* p, bool aligned) {
  Stored<T> x;
  if (aligned) {
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T)) / 2; ++i) x.w[i] = reinterpret_cast<const u32x4*>(p)[i];
  } else {
#pragma unroll
    for (int i = 0; i < 2 * static_cast<int>(sizeof(T)); ++i) {
      if constexpr (sizeof(T) == 4) x.w[i / 4][i % 4] = __float_as_uint(p[i]);
      else x.w[0][i] = p[2 * i] | static_cast<uint32_t>(p[2 * i + 1]) << 16;
    }
  }
  return x;
}
__device__ __forceinline__ Eight eight_of(const Stored<float>& s) {
  Eight x;
#pragma unroll
  for (int i = 0; i < 8; ++i) x.v[i] = __uint_as_float(s.w[i / 4][i % 4]);
  return x;
}
__device__ __forceinline__ Eight eight_of(const Stored<uint16_t>& s) {
  Eight x;
#pragma unroll
  for (int i = 0; i < 4; ++i) x.v[2 * i] = bf16_lo(s.w[0][i]), x.v[2 * i + 1] = bf16_hi(s.w[0][i]);
  return x;
}

// The codes of eight values times a power of two, rounded to nearest, ties to even. What is not finite becomes NaN.
__device__ __forceinline__ u32x2 codes_of(const float (&v)[8], float times) {
  u32x2 w;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    int x = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * i] * times, v[4 * i + 1] * times, 0, false);
    w[i] = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * i + 2] * times, v[4 * i + 3] * times, x, true);
  }
  return w;
}

// The smallest power of two s of at least 2^kLowExponent with `most` <= 448 s = 1.75 * 2^8 s.
__device__ __forceinline__ float scale_for(float most) {
  const uint32_t bits = __float_as_uint(most);
  const int exponent = static_cast<int>(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
  return __uint_as_float(static_cast<uint32_t>(max(exponent, kLowExponent) + 127) << 23);
}

// The block of a slot, -1 outside the pool.
__device__ __forceinline__ int32_t block_of(const Append& a, int64_t slot) {
  return slot < 0 || slot >= a.num_slots ? -1 : static_cast<int32_t>(static_cast<uint32_t>(slot) / static_cast<uint32_t>(a.block_size));
}

// The codes of a block's first `rows` tokens times `ratio`, a power of two: exact but for codes that fall below 2^-6.
template <int D>
__device__ void scale_down(uint8_t* block, int64_t row_bytes, int32_t rows, float ratio) {
  constexpr int kLanes = D / 8, kRows = kWave / kLanes;
  const int lane = threadIdx.x & (kWave - 1), row = lane / kLanes, d = lane % kLanes * 8;
  for (int32_t r = row; r < rows; r += kRows) {
    u32x2* p = reinterpret_cast<u32x2*>(block + r * row_bytes + d);
    const u32x2 w = *p;
    float v[8];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      v[4 * i] = __builtin_amdgcn_cvt_f32_fp8(w[i], 0), v[4 * i + 1] = __builtin_amdgcn_cvt_f32_fp8(w[i], 1);
      v[4 * i + 2] = __builtin_amdgcn_cvt_f32_fp8(w[i], 2), v[4 * i + 3] = __builtin_amdgcn_cvt_f32_fp8(w[i], 3);
    }
    *p = codes_of(v, ratio);
  }
}

__device__ __forceinline__ float finite_size(float x) {
  const float size = fabsf(x);
  return size < INFINITY ? size : 0.f;
}

// ---------------------------------------------------------------------------------------------
// The tokens of one block that stand next to each other in the call (a run), of one head, keys or values: D / 8 lanes to a
// row. Their largest magnitude gives the scale; where the block has tokens before them and its scale has to grow, their
// codes are scaled down. No two wavefronts write the same block and head, so nothing waits for another. Here a run of more
// than kHeld tokens. Where blocks have more, kLong tokens (32 or 64) are held as they are stored, in registers that would cost a kernel of small
// blocks its wavefronts; longer runs are read twice, the second time from the caches. 16 x 512 tokens of 32 heads x 128,
// bfloat16, in blocks of 64: 50 us, read twice 66; 8 x 512, float32, in blocks of 32 with kLong 32 and 64: 33 and 53, of 64: 47
// and 38.
// ---------------------------------------------------------------------------------------------
template <typename T, int D, int kLong>
__device__ void append_run(const Append& a, int which, int32_t head, int64_t t0, int32_t block) {
  constexpr int kLanes = D / 8, kRows = kWave / kLanes, kSteps = kHeld / kRows;
  const int lane = threadIdx.x & (kWave - 1), row = lane / kLanes, d = lane % kLanes * 8;
  const bool aligned = a.aligned[which];
  const T* source = static_cast<const T*>(a.source[which]) + static_cast<int64_t>(head) * D + d;
  uint8_t* pool = a.pool[which] + static_cast<int64_t>(head) * D + d;
  const int64_t row_bytes = static_cast<int64_t>(a.kv_heads) * D;
  float* scale_at = a.scales[which] + static_cast<int64_t>(block) * a.kv_heads + head;
  const float held_scale = *scale_at;

  // The run, and the first place of the block that it writes.
  int64_t end = t0;
  int64_t low = INT64_MAX;
  for (;;) {
    const int64_t t = end + lane;
    const int64_t slot = t < a.tokens ? a.slots[t] : -1;
    const uint64_t other = ~__ballot(block_of(a, slot) == block);
    const int count = other == 0 ? kWave : __builtin_ctzll(other);
    if (lane < count) low = min(low, slot);
    end += count;
    if (count < kWave) break;
  }
  for (int m = kWave / 2; m > 0; m >>= 1) low = min(low, static_cast<int64_t>(__shfl_xor(static_cast<long long>(low), m)));
  const int64_t block0 = static_cast<int64_t>(block) * a.block_size;
  const int32_t before = static_cast<int32_t>(low - block0);  // tokens that the block keeps

  float most = 0.f;
  const auto look = [&](const Eight& one) {
#pragma unroll
    for (int e = 0; e < 8; ++e) most = fmaxf(most, finite_size(one.v[e]));
  };
  float times;
  const auto settle = [&]() {  // the scale, and the codes of the tokens before
    for (int m = kWave / 2; m > 0; m >>= 1) most = fmaxf(most, __shfl_xor(most, m));
    float scale = scale_for(most);
    if (before > 0) {
      scale = fmaxf(scale, held_scale);
      if (scale != held_scale) scale_down<D>(pool - d + block0 * row_bytes, row_bytes, before, held_scale / scale);
    }
    times = 1.f / scale;
    if (lane == 0) *scale_at = scale;
  };
  if constexpr (kLong > 0) {
    constexpr int kAll = kLong / kRows;
    if (end - t0 <= kAll * kRows) {
      Stored<T> held[kAll];
#pragma unroll
      for (int i = 0; i < kAll; ++i) held[i] = load_stored(source + min(t0 + i * kRows + row, end - 1) * a.stride[which], aligned);
#pragma unroll
      for (int i = 0; i < kAll; ++i) look(eight_of(held[i]));
      settle();
#pragma unroll
      for (int i = 0; i < kAll; ++i) {
        asm volatile("" : "+v"(held[i].w[0]));  // widened again, not kept widened
        const int64_t t = t0 + i * kRows + row;
        if (t < end) *reinterpret_cast<u32x2*>(pool + a.slots[t] * row_bytes) = codes_of(eight_of(held[i]).v, times);
      }
      return;
    }
  }
  Eight x[kSteps];
  const auto load = [&](int64_t from) {
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
      const int64_t t = min(from + i * kRows + row, end - 1);  // rows past the run repeat its last
      x[i] = load_eight(source + t * a.stride[which], aligned);
    }
  };
  for (int64_t from = t0; from < end; from += kHeld) {
    load(from);
#pragma unroll
    for (int i = 0; i < kSteps; ++i) look(x[i]);
  }
  settle();
  for (int64_t from = t0; from < end; from += kHeld) {
    load(from);
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
      const int64_t t = from + i * kRows + row;
      if (t < end) *reinterpret_cast<u32x2*>(pool + a.slots[t] * row_bytes) = codes_of(x[i].v, times);
    }
  }
}

// Runs within kHeld tokens from t0 on, all at once: lane j < kHeld speaks for token j. `slot` is the lane's (-1: none),
// `block` its block, `begins` the tokens that are not of the block of the one before, `count` the tokens, which end with a run.
template <typename T, int D>
__device__ __forceinline__ void append_runs(const Append& a, int which, int32_t head, int64_t t0, int32_t count, int64_t slot, int32_t block,
                                            uint32_t begins) {
  constexpr int kLanes = D / 8, kRows = kWave / kLanes, kSteps = kHeld / kRows;
  const int lane = threadIdx.x & (kWave - 1), row = lane / kLanes, d = lane % kLanes * 8;
  const bool aligned = a.aligned[which];
  const T* source = static_cast<const T*>(a.source[which]) + static_cast<int64_t>(head) * D + d;
  uint8_t* pool = a.pool[which] + static_cast<int64_t>(head) * D;
  const int64_t row_bytes = static_cast<int64_t>(a.kv_heads) * D;
  const bool speaks = lane < count && block >= 0;
  float* scale_at = a.scales[which] + static_cast<int64_t>(max(block, 0)) * a.kv_heads + head;
  const float held_scale = speaks ? *scale_at : 0.f;

  Eight x[kSteps];
#pragma unroll
  for (int i = 0; i < kSteps; ++i) x[i] = load_eight(source + (t0 + min(i * kRows + row, count - 1)) * a.stride[which], aligned);
  float most = 0.f;  // of this lane's token
#pragma unroll
  for (int i = 0; i < kSteps; ++i) {
    float its = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) its = fmaxf(its, finite_size(x[i].v[e]));
#pragma unroll
    for (int m = 1; m < kLanes; m *= 2) its = fmaxf(its, __shfl_xor(its, m));
    const float here = __shfl(its, lane % kRows * kLanes);
    most = lane / kRows == i ? here : most;
  }
  // The run's largest, and its first place in the block.
  const int32_t place = static_cast<int32_t>(slot - static_cast<int64_t>(block) * a.block_size);
  int32_t before = place;
  const uint32_t up_to = (2u << min(lane, kHeld - 1)) - 1;
  const int begin = 31 - __builtin_clz(begins & up_to), end = begins & ~up_to ? __builtin_ctz(begins & ~up_to) : count;
  const bool first = speaks && lane == begin;
#pragma unroll
  for (int m = 1; m < kHeld; m *= 2) {
    const float other = __shfl_up(most, m);
    const int32_t low = __shfl_up(before, m);
    if (lane - m >= begin) most = fmaxf(most, other), before = min(before, low);
  }
  most = __shfl(most, end - 1);
  before = __shfl(before, end - 1);
  float scale = scale_for(most);
  if (before > 0) scale = fmaxf(scale, held_scale);
  for (uint64_t grown = __ballot(first && before > 0 && scale != held_scale); grown != 0; grown &= grown - 1) {
    const int j = __builtin_ctzll(grown);
    const int64_t block0 = static_cast<int64_t>(__builtin_amdgcn_readfirstlane(__shfl(block, j))) * a.block_size;
    scale_down<D>(pool + block0 * row_bytes, row_bytes, __shfl(before, j), __shfl(held_scale / scale, j));
  }
  const float times = 1.f / scale;
#pragma unroll
  for (int i = 0; i < kSteps; ++i) {
    const int j = i * kRows + row;
    const int64_t to = __shfl(static_cast<long long>(speaks ? slot : -1), j);
    const float by = __shfl(times, j);
    if (to >= 0) *reinterpret_cast<u32x2*>(pool + to * row_bytes + d) = codes_of(x[i].v, by);
  }
  if (first) *scale_at = scale;
}

// A wavefront has the runs that begin in its window of kHeld tokens, of one head, keys or values. Short ones are taken together, as
// many as end within kHeld tokens: one after the other, the latency of each (2 us) counted.
// Bound: HBM for long prompts, latency for single tokens. 16 x 512 tokens of 32 heads x 128, bfloat16, in blocks of 16, 202 MB: 44 us,
// 4.6 TB/s; 64 single tokens of 8 heads x 128 5 us.
template <typename T, int D, int kLong>
__global__ __launch_bounds__(kThreads) void append_kernel(const Append a) {
  // Items: keys and values of a head, heads, then windows.
  const uint32_t item = __builtin_amdgcn_readfirstlane(blockIdx.x * (kThreads / kWave) + threadIdx.x / kWave);
  const uint32_t columns = 2 * static_cast<uint32_t>(a.kv_heads);
  const int which = item & 1;
  const int32_t head = static_cast<int32_t>(item % columns / 2);
  const int64_t window = static_cast<int64_t>(item / columns) * a.window, until = min(window + a.window, a.tokens);
  if (window >= a.tokens) return;
  const int lane = threadIdx.x & (kWave - 1);
  for (int64_t t0 = window; t0 < until;) {
    // Lane j: token t0 + j, its slot and block, and whether it begins a run or ends what stands before it.
    const int64_t t = t0 + lane;
    int64_t slot = t < a.tokens ? a.slots[t] : -1;
    const int64_t last_slot = t > 0 && t <= a.tokens ? a.slots[t - 1] : -1;
    const int32_t block = block_of(a, slot), last = block_of(a, last_slot);
    if (block < 0) slot = -1;
    const uint64_t changes = __ballot(block != last || lane == 0);  // t0 begins a run, or is its window's first token
    const uint64_t starts = __ballot(block >= 0 && block != last);
    // The first token in the window that begins a run.
    const uint64_t inside = until - t0 >= kWave ? ~0ull : (1ull << (until - t0)) - 1;
    if ((starts & inside) == 0) return;
    const int first = __builtin_ctzll(starts & inside);
    if (first > 0) {  // what is before it belongs to another wavefront, or to nobody
      t0 += first;
      continue;
    }
    // How many tokens from here on end with a run: up to the last change of at most kHeld tokens on (the call's end is one), and
    // to the first run that the next window's wavefront has.
    const uint64_t theirs = starts & ~inside;
    const int most = theirs == 0 ? kHeld : min(kHeld, __builtin_ctzll(theirs));
    const uint64_t ends = changes & ((2ull << most) - 2);
    if (ends == 0) {
      append_run<T, D, kLong>(a, which, head, t0, __builtin_amdgcn_readfirstlane(block));
      t0 += kHeld;  // the next run begins behind
      continue;
    }
    const int count = 63 - __builtin_clzll(ends);
    append_runs<T, D>(a, which, head, t0, count, slot, block, static_cast<uint32_t>(changes) & ((1u << count) - 1));
    t0 += count;
  }
}

int64_t groups_of(const Append& a) {
  const int64_t items = (a.tokens + a.window - 1) / a.window * 2 * a.kv_heads;
  return (items + kThreads / kWave - 1) / (kThreads / kWave);
}

template <typename T, int D>
void launch(const Append& a, hipStream_t stream) {
  const dim3 grid(static_cast<uint32_t>(groups_of(a))), block(kThreads);
  if (a.block_size <= kHeld) hipLaunchKernelGGL((append_kernel<T, D, 0>), grid, block, 0, stream, a);
  else if (a.block_size <= 32) hipLaunchKernelGGL((append_kernel<T, D, 32>), grid, block, 0, stream, a);
  else hipLaunchKernelGGL((append_kernel<T, D, 64>), grid, block, 0, stream, a);
}

template <typename T>
int dispatch(const Append& a, int32_t head_dim, hipStream_t stream) {
  switch (head_dim) {
    case 32: launch<T, 32>(a, stream); break;
    case 64: launch<T, 64>(a, stream); break;
    case 128: launch<T, 128>(a, stream); break;
    case 256: launch<T, 256>(a, stream); break;
    default: return PKV_EUNSUPPORTED;
  }
  return check_launch();
}

}  // namespace
}  // namespace pkv

extern "C" int pkv_append_e4m3(const pkv_e4m3_append* args, int device, void* stream) {
  using namespace pkv;
  if (!args) return PKV_EINVAL;
  const pkv_e4m3_append& g = *args;
  if (g.num_tokens < 0 || g.num_blocks < 0 || g.block_size < 1 || g.num_kv_heads < 1) return PKV_EINVAL;
  if (g.src_dtype != PKV_F32 && g.src_dtype != PKV_BF16) return PKV_EINVAL;
  if (g.head_dim != 32 && g.head_dim != 64 && g.head_dim != 128 && g.head_dim != 256) return PKV_EUNSUPPORTED;
  if (g.num_blocks > 0x7fffffff / g.block_size || g.num_kv_heads > (1 << 20) || g.num_tokens > 0x7fffffff) return PKV_EUNSUPPORTED;
  if (g.num_tokens == 0) return PKV_OK;
  if (!g.key_pool || !g.value_pool || !g.key_scales || !g.value_scales || !g.keys || !g.values || !g.slot_mapping) return PKV_EINVAL;
  const int64_t row = static_cast<int64_t>(g.num_kv_heads) * g.head_dim;
  if (g.key_token_stride < row || g.value_token_stride < row) return PKV_EINVAL;
  const int size = dtype_size(static_cast<pkv_dtype>(g.src_dtype));
  const auto aligned8 = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 7u) == 0; };
  if (!aligned8(g.key_pool) || !aligned8(g.value_pool)) return PKV_EINVAL;
  Append a{};
  a.pool[0] = static_cast<uint8_t*>(g.key_pool), a.pool[1] = static_cast<uint8_t*>(g.value_pool);
  a.scales[0] = g.key_scales, a.scales[1] = g.value_scales;
  a.source[0] = g.keys, a.source[1] = g.values;
  a.stride[0] = g.key_token_stride, a.stride[1] = g.value_token_stride;
  for (int i = 0; i < 2; ++i) a.aligned[i] = aligned16(a.source[i]) && a.stride[i] * size % 16 == 0;
  a.slots = g.slot_mapping;
  a.tokens = g.num_tokens;
  a.num_slots = static_cast<int32_t>(g.num_blocks * g.block_size);
  a.block_size = g.block_size;
  a.kv_heads = g.num_kv_heads;
  a.window = kHeld;
  if (groups_of(a) > 0x7fffffff / kThreads) return PKV_EUNSUPPORTED;
  DeviceGuard guard(device);
  if (!guard.ok()) return PKV_EHIP;
  const auto s = static_cast<hipStream_t>(stream);
  return g.src_dtype == PKV_F32 ? dispatch<float>(a, g.head_dim, s) : dispatch<uint16_t>(a, g.head_dim, s);
}
