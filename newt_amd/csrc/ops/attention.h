// What the two attention operators share: how query rows are laid out over
// programs, which key tiles a program visits, and the kernel that joins the
// splits of a row.
//
// Rows. The queries of one KV head are one matrix of q_len * G rows (G query
// heads to a KV head), row r = query r / G of head r % G, so that all rows of
// a program share each key and value tile and a single token still fills G
// rows.
#pragma once
#include <utility>

#include "common.h"

namespace newt_ops {

constexpr float kLog2e = 1.44269504088896341f;
constexpr float kInf = __builtin_inff();
constexpr int kTile = 64;  // keys of a tile
constexpr int kLimit = 1 << 30;       // of lengths, positions and windows
constexpr int kNoWindow = 0x7fffffff; // sees all keys before it

// A row's maximum may lag behind by this much (in powers of two) before sums
// and accumulators are rescaled: 2^8 more in a weight costs no precision in
// fp32 sums and stays far below fp16's largest number.
constexpr float kSlack = 8.0f;

// Weights are 2^(score c - m) by one fma, where m is the largest score times c,
// rounded: by up to half a step, 2^-1 below this. A row whose m lies beyond it is
// done again with each score times c rounded first, so that the largest one's
// exponent is 0 whatever the scale.
constexpr float kExact = 8388608.0f;  // 2^23

__device__ __forceinline__ bool beyond_exact(float m) {
  return (__builtin_fabsf(m) > kExact) & (m != -kInf);
}

// The keys that the rows of a program see: sinks [0, sinks) and [lo, hi).
// Windows, sinks and `keys` stay below 2^30; positions need not, but fit an int
// with the tiles that a caller asks for behind the last one.
struct Range {
  int first, last;  // positions of the program's first and last query
  int lo, hi, sinks;
  int window;       // kNoWindow: none
  int sink_tiles, lo_tile, tiles;

  __device__ __forceinline__ Range(int first_, int last_, int keys, int window_, int sinks_)
      : first(first_), last(last_), sinks(sinks_), window(window_) {
    hi = last + 1 < keys ? last + 1 : keys;
    lo = first >= window ? first - window + 1 : 0;
    if (hi < 0) hi = 0;
    if (sinks > hi) sinks = hi;
    lo_tile = lo / kTile;
    const int hi_tile = (hi + kTile - 1) / kTile;
    sink_tiles = (sinks + kTile - 1) / kTile;
    if (sink_tiles > lo_tile) sink_tiles = lo_tile;
    tiles = sink_tiles + (hi_tile > lo_tile ? hi_tile - lo_tile : 0);
  }
  // first key of the i-th tile
  __device__ __forceinline__ int tile(int i) const {
    return (i < sink_tiles ? i : i - sink_tiles + lo_tile) * kTile;
  }
  // whether every row sees every key of the tile from `key` on
  __device__ __forceinline__ bool whole(int key) const {
    return key + kTile <= hi && key + kTile - 1 <= first &&
           ((u32)(last - key) < (u32)window || key + kTile <= sinks);
  }
  __device__ __forceinline__ bool sees(int position, int key) const {
    // position - key in [0, window), by one unsigned comparison, or a sink
    return (((u32)(position - key) < (u32)window) | ((key < sinks) & (key <= position))) & (key < hi);
  }
  // whether any row sees the key
  __device__ __forceinline__ bool any(int key) const {
    return (key < hi) & ((key >= lo) | (key < sinks));
  }
};

// Where rows of queries and outputs lie.
struct Rows {
  int64_t stride_b, stride_h, stride_t;
  __device__ __forceinline__ int64_t at(int b, int head, int i) const {
    return b * stride_b + head * stride_h + i * stride_t;
  }
};

// Workgroups go round the 8 dies of the chip, each with an L2 of its own; this
// gives each die a run of neighbouring programs, which share keys and values.
__device__ __forceinline__ int by_die(int i, int n) {
  const int die = i & 7, each = n >> 3, more = n & 7;
  return die * each + (die < more ? die : more) + (i >> 3);
}

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

constexpr int kMostSplits = 64;  // a lane of the joining wave for each

// o = sum acc_s 2^(m_s - M) / sum l_s 2^(m_s - M); rows that saw nothing are 0.
// One wave a row: lane s takes split s's maximum and sum, then every lane its
// dims of all accumulators, whose loads do not wait for each other.
template <typename T, int D>
__global__ void __launch_bounds__(256)
join_splits_kernel(const void* workspace, void* out, Rows o, int64_t units, int splits, int rows,
                   int row_tiles, int all_rows, int kv_heads, int group) {
  const Parts parts((void*)workspace, units, splits, rows, D);
  const int lane = threadIdx.x & 63;
  // rows that exist: row tiles are full but for a unit's last one
  const u32 w = blockIdx.x * 4 + wave_id();
  if (w >= (u32)units / row_tiles * all_rows) return;
  const u32 r = w % all_rows, sequence_head = w / all_rows;
  const int64_t unit = (int64_t)sequence_head * row_tiles + r / rows;
  const int64_t at = unit * splits * rows + r % rows;  // and `rows` further a split

  const float m = lane < splits ? parts.m[at + (int64_t)lane * rows] : -kInf;
  const float l = lane < splits ? parts.l[at + (int64_t)lane * rows] : 0.0f;
  const float M = newt::lane_reduce<newt::Max, 63>(m);
  // without a maximum a split has seen nothing, or NaN
  const float f = m == -kInf ? 0.0f : __builtin_amdgcn_exp2f(m - M);
  const float total = newt::lane_reduce<newt::Sum, 63>(m == -kInf ? l : l * f);
  // 16 bytes a lane: the wave reads SIDE splits at a time, AT_ONCE such pieces
  // without waiting in between
  constexpr int WIDE = D / 4, SIDE = 64 / WIDE, AT_ONCE = 8;
  const int side = lane / WIDE, d = lane % WIDE * 4;
  f32x4 acc = (f32x4)(0.0f);
  const float* from = parts.acc + at * D + d;
  for (int s = 0; s < splits; s += SIDE * AT_ONCE) {
    f32x4 a[AT_ONCE];
    float g[AT_ONCE];
#pragma unroll
    for (int j = 0; j < AT_ONCE; ++j) {
      const int split = s + j * SIDE + side;
      a[j] = *(const f32x4*)(from + (int64_t)(split < splits ? split : 0) * rows * D);
      g[j] = __shfl(f, split);
    }
#pragma unroll
    for (int j = 0; j < AT_ONCE; ++j)
      acc += s + j * SIDE + side < splits ? a[j] * g[j] : (f32x4)(0.0f);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (SIDE > 2) acc[i] = newt::lane_reduce<newt::Sum, 16>(acc[i]);
    if constexpr (SIDE > 1) acc[i] = newt::lane_reduce<newt::Sum, 32>(acc[i]);
  }
  if (side) return;
  T t[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) t[i] = (T)(total == 0.0f ? 0.0f : acc[i] / total);
  const u32 head = sequence_head % kv_heads, b = sequence_head / kv_heads;
  T* to = (T*)out + o.at(b, head * group + r % group, r / group) + d;
  newt::store_vec<T, 4>(to, t, newt::any_align());
}

// Whether rows of `dim` numbers in three dimensions share memory, which several
// programs would write at once: a dimension, from the smallest stride on, has to
// step over all that those before it reach. Slices, permutations and the like of
// a tensor without overlaps do.
inline bool rows_overlap(int dim, int64_t n0, int64_t s0, int64_t n1, int64_t s1, int64_t n2,
                         int64_t s2) {
  struct { int64_t n, stride; } d[3] = {{n0, s0}, {n1, s1}, {n2, s2}};
  for (auto& e : d) e.stride = e.stride < 0 ? -e.stride : e.stride;
  const auto order = [&](int i, int j) { if (d[j].stride < d[i].stride) std::swap(d[i], d[j]); };
  order(0, 1);
  order(1, 2);
  order(0, 1);
  double reach = dim;  // what strides of any size cannot exceed
  for (const auto& e : d) {
    if (e.n <= 1) continue;
    if ((double)e.stride < reach) return true;
    reach += (double)(e.n - 1) * (double)e.stride;
  }
  return false;
}

// What both operators refuse of their queries, outputs and scale; null: nothing.
template <typename P>
const char* queries_wrong(const P& p, int head_dim) {
  if (rows_overlap(head_dim, p.batch, p.o_stride_b, p.heads, p.o_stride_h, p.q_len, p.o_stride_t))
    return "rows of out overlap";
  // scores and their exponents stay finite for ordinary queries and keys
  if (!(__builtin_fabsf(p.scale) < 0x1p100f)) return "scale has to be finite, below 2^100";
  return nullptr;
}

// At most so many tiles can a program of `span` queries visit.
inline int64_t most_tiles(int64_t keys, int64_t window, int64_t sinks, int64_t span) {
  const int64_t all = (keys + kTile - 1) / kTile;
  if (!window) return all;
  const int64_t some = (window + span + 2 * kTile - 2) / kTile + (sinks + kTile - 1) / kTile;
  return some < all ? some : all;
}

// The programs of a launch: `rows` of a KV head's query rows each, and a row's
// tiles in `splits`. unit = (sequence * kv_heads + head) * row_tiles + row tile.
struct Plan {
  int row_tiles, rows, all_rows, splits;
  int64_t units;
  Plan(int64_t batch, int64_t q_len, int kv_heads, int group, int rows_)
      : rows(rows_), splits(1) {
    all_rows = (int)(q_len * group);
    row_tiles = (all_rows + rows - 1) / rows;
    units = batch * kv_heads * row_tiles;
  }
  // what no launch takes; q_len * heads below 2^31 is checked before
  bool too_large() const { return units * splits > 0x7fffffff || units * rows > 0x7fffffff; }
};

template <typename T, int D>
int join_splits(const void* workspace, void* out, Rows o, const Plan& r, int kv_heads, int group,
                hipStream_t stream) {
  const int64_t waves = r.units / r.row_tiles * r.all_rows;
  return run("newt_window_attention", join_splits_kernel<T, D>, (waves + 3) / 4, 256, 0, stream,
             workspace, out, o, r.units, r.splits, r.rows, r.row_tiles, r.all_rows, kv_heads, group);
}

}  // namespace newt_ops
