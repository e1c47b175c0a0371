// What the two attention operators share: how query rows are laid out over
// programs, which key tiles a program visits, and the kernel that joins the
// splits of a row.
//
// Rows. The queries of one KV head are one matrix of q_len * G rows (G query
// heads to a KV head), row r = query r / G of head r % G, so that all rows of
// a program share each key and value tile and a single token still fills G
// rows.
#pragma once
#include "common.h"

namespace newt_ops {

constexpr float kLog2e = 1.44269504088896341f;
constexpr float kInf = __builtin_inff();
constexpr int kTile = 64;  // keys of a tile

// A row's maximum may lag behind by this much (in powers of two) before sums
// and accumulators are rescaled: 2^8 more in a weight costs no precision in
// fp32 sums and stays far below fp16's largest number.
constexpr float kSlack = 8.0f;

// The keys that the rows of a program see: sinks [0, sinks) and [lo, hi).
struct Range {
  int64_t first, last;  // positions of the program's first and last query
  int64_t lo, hi, sinks;
  int64_t window;       // 0: none
  int64_t sink_tiles, lo_tile, tiles;

  __device__ __forceinline__ Range(int64_t first_, int64_t last_, int64_t keys, int64_t window_,
                                   int64_t sinks_)
      : first(first_), last(last_), sinks(sinks_), window(window_) {
    hi = last + 1 < keys ? last + 1 : keys;
    lo = window && first - window + 1 > 0 ? first - window + 1 : 0;
    if (hi < 0) hi = 0;
    if (sinks > hi) sinks = hi;
    lo_tile = lo / kTile;
    const int64_t hi_tile = (hi + kTile - 1) / kTile;
    sink_tiles = (sinks + kTile - 1) / kTile;
    if (sink_tiles > lo_tile) sink_tiles = lo_tile;
    tiles = sink_tiles + (hi_tile > lo_tile ? hi_tile - lo_tile : 0);
  }
  // first key of the i-th tile
  __device__ __forceinline__ int64_t tile(int64_t i) const {
    return (i < sink_tiles ? i : i - sink_tiles + lo_tile) * kTile;
  }
  // whether every row sees every key of the tile from `key` on
  __device__ __forceinline__ bool whole(int64_t key) const {
    return key + kTile <= hi && key + kTile - 1 <= first &&
           (!window || key > last - window || key + kTile <= sinks);
  }
  __device__ __forceinline__ bool sees(int64_t position, int64_t key) const {
    return key <= position && key < hi && (!window || position - key < window || key < sinks);
  }
  // whether any row sees the key
  __device__ __forceinline__ bool any(int64_t key) const {
    return key < hi && (key >= lo || key < sinks);
  }
};

// Where rows of queries and outputs lie.
struct Rows {
  int64_t stride_b, stride_h, stride_t;
  __device__ __forceinline__ int64_t at(int64_t b, int64_t head, int64_t i) const {
    return b * stride_b + head * stride_h + i * stride_t;
  }
};

// Partial results of `splits` programs for `rows` rows each: accumulators
// [unit, split, row, D], then maxima and sums [unit, split, row] each.
struct Parts {
  float* acc;
  float* m;
  float* l;
  __host__ __device__ Parts(void* workspace, int64_t units, int splits, int rows, int D) {
    const int64_t n = units * splits * rows;
    acc = (float*)workspace;
    m = acc + n * D;
    l = m + n;
  }
  static size_t bytes(int64_t units, int splits, int rows, int D) {
    return (size_t)units * splits * rows * (D + 2) * sizeof(float);
  }
};

// o = sum acc_s 2^(m_s - M) / sum l_s 2^(m_s - M); rows that saw nothing are 0.
// One wave a row.
template <typename T, int D>
__global__ void __launch_bounds__(256)
join_splits_kernel(const void* workspace, void* out, Rows o, int64_t units, int splits, int rows,
                   int64_t row_tiles, int64_t q_len, int kv_heads, int group) {
  const Parts parts((void*)workspace, units, splits, rows, D);
  const int lane = threadIdx.x & 63;
  const int64_t w = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (w >= units * rows) return;
  const int64_t unit = w / rows;
  const int row = (int)(w % rows);
  const int64_t r = unit % row_tiles * rows + row;
  const int64_t head = unit / row_tiles % kv_heads, b = unit / row_tiles / kv_heads;
  if (r >= q_len * group) return;
  constexpr int N = D / 64;
  float M = -kInf;
  for (int s = 0; s < splits; ++s)
    M = newt::Max::op(M, parts.m[(unit * splits + s) * rows + row]);
  const float ref = M == -kInf ? 0.0f : M;
  float l = 0.0f, acc[N] = {};
  for (int s = 0; s < splits; ++s) {
    const int64_t at = (unit * splits + s) * rows + row;
    const float f = __builtin_amdgcn_exp2f(parts.m[at] - ref);
    if (parts.m[at] == -kInf) {
      l += parts.l[at];  // 0, or NaN
      continue;
    }
    l += parts.l[at] * f;
    float a[N];
    newt::load_vec<float, N>(parts.acc + at * D + lane * N, a);
#pragma unroll
    for (int i = 0; i < N; ++i) acc[i] += a[i] * f;
  }
  T t[N];
#pragma unroll
  for (int i = 0; i < N; ++i) t[i] = (T)(l == 0.0f ? 0.0f : acc[i] / l);
  T* to = (T*)out + o.at(b, head * group + r % group, r / group) + lane * N;
  newt::store_vec<T, N>(to, t, newt::any_align());
}

template <typename T, int D>
int join_splits(const void* workspace, void* out, Rows o, int64_t units, int splits, int rows,
                int64_t row_tiles, int64_t q_len, int kv_heads, int group, hipStream_t stream) {
  const int64_t waves = units * rows;
  join_splits_kernel<T, D><<<dim3((unsigned)((waves + 3) / 4)), dim3(256), 0, stream>>>(
      workspace, out, o, units, splits, rows, row_tiles, q_len, kv_heads, group);
  return launched("join_splits");
}

}  // namespace newt_ops
