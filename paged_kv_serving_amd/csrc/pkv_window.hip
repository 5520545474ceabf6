// Paged causal attention with a sliding window and sinks, for grouped heads.
//
// A query row at position p of a sequence with context length c sees the keys j < min(c, p + 1) with
// j > p - window or j < sinks:
//     out = sum_j exp(s_j) v_j / sum_j exp(s_j),  s_j = scale * q . k_j
// with an online softmax (running maximum and sum), everything in float32 and one rounding to the
// output's type.
#include <math.h>

#include "pkv_common.h"

namespace pkv {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / kWave;

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
  float scale_log2;  // scale * log2(e): scores are kept in base 2
};

__device__ __forceinline__ float load_one(const float* p) { return *p; }
__device__ __forceinline__ float load_one(const uint16_t* p) { return __uint_as_float(static_cast<uint32_t>(*p) << 16); }
__device__ __forceinline__ void store_one(float* p, float v) { *p = v; }
__device__ __forceinline__ void store_one(uint16_t* p, float v) { *p = static_cast<uint16_t>(f32_to_bf16_bits(v)); }

// The keys a row sees: [0, sinks) and [begin, end), or nothing.
struct Span {
  int32_t sinks, begin, end;
  __device__ __forceinline__ int32_t count() const { return sinks + end - begin; }
  __device__ __forceinline__ int32_t key(int32_t i) const { return i < sinks ? i : begin + (i - sinks); }
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

// Element offset of a key's row of one head in the pools; -1 in a block outside the pool.
__device__ __forceinline__ int64_t row_of(const Window& a, const int32_t* table, int32_t key, int32_t kv_head, int d) {
  const int32_t page = key / a.block_size;
  const int64_t block = table[page];
  if (block < 0 || block >= a.num_blocks) return -1;
  return ((block * a.block_size + (key - page * a.block_size)) * a.num_kv_heads + kv_head) * d;
}

// One wavefront per (row, head), 64 keys at a time: a lane scores one key, then owns dimensions.
template <typename QT, typename KVT, int D>
__global__ __launch_bounds__(kThreads) void plain_kernel(const Window a) {
  constexpr int kOwn = (D + kWave - 1) / kWave;
  const int lane = threadIdx.x & (kWave - 1);
  const int64_t item = static_cast<int64_t>(blockIdx.x) * kWaves + threadIdx.x / kWave;
  const int64_t t = item / a.num_heads;
  if (t >= a.num_queries) return;
  const int32_t head = static_cast<int32_t>(item - t * a.num_heads);
  const int32_t seq = a.seqs[t];
  if (seq < 0 || seq >= a.num_seqs) return;
  const int32_t kv_head = head / a.group;
  const int32_t* table = a.tables + static_cast<int64_t>(seq) * a.table_stride;
  const Span span = span_of(a, seq, a.positions[t]);
  const QT* q = static_cast<const QT*>(a.queries) + t * a.query_stride + static_cast<int64_t>(head) * D;
  float top = -INFINITY, sum = 0.f, acc[kOwn] = {};
  for (int32_t first = 0; first < span.count(); first += kWave) {
    const bool live = first + lane < span.count();
    const int64_t row = live ? row_of(a, table, span.key(first + lane), kv_head, D) : -1;
    float score = -INFINITY;
    if (row >= 0) {
      const KVT* k = static_cast<const KVT*>(a.keys) + row;
      score = 0.f;
      for (int d = 0; d < D; ++d) score += load_one(q + d) * load_one(k + d);
      score *= a.scale_log2;
    }
    float next = score;
    for (int m = kWave / 2; m > 0; m >>= 1) next = fmaxf(next, __shfl_xor(next, m));
    next = fmaxf(top, next);
    if (next == -INFINITY) continue;
    const float keep = exp2f(top - next);
    const float p = row >= 0 ? exp2f(score - next) : 0.f;
    float all = p;
    for (int m = kWave / 2; m > 0; m >>= 1) all += __shfl_xor(all, m);
    sum = sum * keep + all;
    top = next;
    for (int e = 0; e < kOwn; ++e) acc[e] *= keep;
    for (int j = 0; j < kWave; ++j) {
      const float pj = __shfl(p, j);
      const int64_t rj = __shfl(static_cast<long long>(row), j);
      if (rj < 0) continue;
      for (int e = 0; e < kOwn; ++e) {
        const int d = e * kWave + lane;
        if (d < D) acc[e] += pj * load_one(static_cast<const KVT*>(a.values) + rj + d);
      }
    }
  }
  QT* out = static_cast<QT*>(a.out) + (t * a.num_heads + head) * D;
  for (int e = 0; e < kOwn; ++e) {
    const int d = e * kWave + lane;
    if (d < D) store_one(out + d, sum == 0.f ? 0.f : acc[e] / sum);
  }
}

template <typename QT, typename KVT, int D>
int launch(const Window& a, hipStream_t stream) {
  const int64_t groups = (a.num_queries * a.num_heads + kWaves - 1) / kWaves;
  if (groups > 0x7fffffff) return PKV_EUNSUPPORTED;
  hipLaunchKernelGGL((plain_kernel<QT, KVT, D>), dim3(static_cast<uint32_t>(groups)), dim3(kThreads), 0, stream, a);
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

extern "C" int32_t pkv_window_splits(int64_t num_queries, int32_t num_heads, int32_t num_kv_heads, int32_t window,
                                     int32_t sinks, int32_t max_context_len, int32_t max_query_len) {
  if (num_queries < 0 || num_kv_heads < 1 || num_heads < num_kv_heads || num_heads % num_kv_heads != 0 || window < 1 ||
      sinks < 0 || max_context_len < 0 || max_query_len < 0) {
    return PKV_EINVAL;
  }
  return 1;
}

extern "C" int64_t pkv_window_workspace_bytes(int64_t num_queries, int32_t num_heads, int32_t head_dim, int32_t num_splits) {
  if (num_queries < 0 || num_heads < 1 || head_dim < 1 || num_splits < 1 || num_splits > PKV_WINDOW_MAX_SPLITS) {
    return PKV_EINVAL;
  }
  if (num_splits == 1) return 0;
  return num_queries * num_heads * num_splits * (head_dim + 2) * static_cast<int64_t>(sizeof(float));
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
  const int32_t splits = g.num_splits > 0 ? g.num_splits
                                          : pkv_window_splits(g.num_queries, g.num_heads, g.num_kv_heads, g.window, g.sinks,
                                                              g.max_context_len, g.max_query_len);
  const int64_t need = pkv_window_workspace_bytes(g.num_queries, g.num_heads, g.head_dim, splits);
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
  DeviceGuard guard(device);
  if (!guard.ok()) return PKV_EHIP;
  auto s = static_cast<hipStream_t>(stream);
  if (g.q_dtype == PKV_BF16) return dispatch<uint16_t, uint16_t>(a, g.head_dim, s);
  return g.kv_dtype == PKV_F32 ? dispatch<float, float>(a, g.head_dim, s) : dispatch<float, uint16_t>(a, g.head_dim, s);
}
