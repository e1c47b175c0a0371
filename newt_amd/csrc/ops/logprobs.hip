// Log probabilities of given tokens, entropy and the largest alternatives:
// with x = logits / T,  m = max x,  S = sum 2^d,  U = sum 2^d d,
// d = (x - m) log2(e):
//   logp = x[token] - m - ln S,  entropy = ln 2 (log2 S - U / S).
// One pass over the logits, which bound it. Each wave keeps m and its 64
// largest logits so far, sorted, an entry a lane, so the stream itself costs
// one comparison a chunk: only a chunk that holds something larger than the
// last entry that counts takes the slow path, which inserts it and, where the
// maximum grew, rescales S and U. The list begins with the sorted largest
// logits of each lane in the first four chunks; after that n logits in no order
// make about top * ln(n / 2048) insertions. Lists are joined by bitonic merges.
// bf16 2048 x 100003, two sets in turn: 89 us (4.6 TB/s) without alternatives,
// 96 with 5, 125 with 20; reading alone would take 58. 1 x 128000: 8 us without,
// 15 with 20, of them 5 in the second kernel.
#include "common.h"

namespace newt_ops {
namespace {

constexpr float kLog2e = 1.44269504088896341f;
constexpr float kLn2 = 0.693147180559945309f;
constexpr float kInf = __builtin_inff();
constexpr int kNone = 0x7fffffff;  // the id of an entry that is none: behind all others
constexpr int kMostSplits = 64;

__device__ __forceinline__ float uniform(float v, int lane) {
  return newt::bits_f32(__builtin_amdgcn_readlane(newt::f32_bits(v), lane));
}

// A list entry: larger logits first, then lower ids.
struct Entry {
  float value;
  int id;
  __device__ __forceinline__ bool before(const Entry& o) const {
    return (value > o.value) | ((value == o.value) & (id < o.id));
  }
};

// v of the lane that differs in bit M: rotations of 16 lanes, permlane swaps
// and quad permutations, on the VALU but for M = 4.
template <int M, typename V>
__device__ __forceinline__ V partner(V v, int lane) {
  if constexpr (M >= 16) {
    V lo, hi;
    newt::pair_lanes<M>(v, lo, hi);
    return (lane & M) ? lo : hi;
  } else if constexpr (M == 8) {
    return __builtin_bit_cast(
        V, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), 0x128, 0xF, 0xF, true));  // row_ror:8
  } else {
    return newt::xor_lane<M>(v);
  }
}

// v of the lane below; lane 0 keeps its own
template <typename V>
__device__ __forceinline__ V below(V v) {
  const int i = __builtin_bit_cast(int, v);
  return __builtin_bit_cast(V, __builtin_amdgcn_update_dpp(i, i, 0x138, 0xF, 0xF, false));  // wave_shr:1
}

// One step of a bitonic network over the lanes: of each pair of lanes that
// differ in bit M the one with that bit clear keeps the entry that comes first
// (where `down`, else last).
template <int M>
__device__ __forceinline__ void exchange(Entry& e, bool down, int lane) {
  const Entry o{partner<M>(e.value, lane), partner<M>(e.id, lane)};
  const bool keep_first = ((lane & M) == 0) == down;
  if (o.before(e) == keep_first) e = o;
}

// 64 entries that rise and then fall (or are a rotation of such) in order
__device__ __forceinline__ void merge_steps(Entry& e, int lane) {
  exchange<32>(e, true, lane);
  exchange<16>(e, true, lane);
  exchange<8>(e, true, lane);
  exchange<4>(e, true, lane);
  exchange<2>(e, true, lane);
  exchange<1>(e, true, lane);
}

__device__ __forceinline__ void sort(Entry& e, int lane) {
  exchange<1>(e, !(lane & 2), lane);
  exchange<2>(e, !(lane & 4), lane);
  exchange<1>(e, !(lane & 4), lane);
  exchange<4>(e, !(lane & 8), lane);
  exchange<2>(e, !(lane & 8), lane);
  exchange<1>(e, !(lane & 8), lane);
  exchange<8>(e, !(lane & 16), lane);
  exchange<4>(e, !(lane & 16), lane);
  exchange<2>(e, !(lane & 16), lane);
  exchange<1>(e, !(lane & 16), lane);
  exchange<16>(e, !(lane & 32), lane);
  exchange<8>(e, !(lane & 32), lane);
  exchange<4>(e, !(lane & 32), lane);
  exchange<2>(e, !(lane & 32), lane);
  exchange<1>(e, !(lane & 32), lane);
  merge_steps(e, lane);
}

// The 64 first of two sorted lists, the other one given in reverse.
__device__ __forceinline__ void merge(Entry& e, const Entry& reversed, int lane) {
  if (reversed.before(e)) e = reversed;
  merge_steps(e, lane);
}

// A candidate, the same in every lane, behind all entries that come before it.
__device__ __forceinline__ void insert(Entry& e, const Entry& c, int lane) {
  const int place = __popcll(__ballot(e.before(c)));
  const Entry left{below(e.value), below(e.id)};
  if (lane > place) e = left;
  if (lane == place) e = c;
}

// d = (x - m) c by one fma where the product m c is rounded by 2^-5 at most: by
// the same amount in all that is taken relative to this m, so that the rounding
// cancels in every result. Larger ones, whose rounding would drown the exponents
// (tiny temperatures, rows of the types' lowest numbers), take the longer way.
__device__ __forceinline__ bool near_zero(float m, float c) {
  return __builtin_fabsf(m * c) < 1048576.0f;  // 2^20
}
// What m c is rounded by in distances to m.
__device__ __forceinline__ float rounding(float m, float c) {
  return near_zero(m, c) ? __builtin_fmaf(m, c, -(m * c)) : 0.0f;
}
__device__ __forceinline__ float distance(float x, float m, float c) {
  return near_zero(m, c) ? __builtin_fmaf(x, c, -(m * c)) : (x - m) * c;
}

// The log probability but for the sum's share: the distance as a natural
// logarithm. Logits near the lowest number fp32 holds leave it on the way there.
__device__ __forceinline__ float natural(float x, float m, float c, float inv_temperature) {
  const float d = distance(x, m, c);
  if (d != -kInf) return d * kLn2;
  const float gap = x - m;
  return gap == -kInf && x > -kInf ? x * inv_temperature - m * inv_temperature
                                   : gap * inv_temperature;
}

// The sums over what a lane, a wave or a split has seen.
struct Sums {
  float m, S, U;

  // The same relative to the maximum `to` >= m.
  __device__ __forceinline__ void rescale(float to, float c) {
    if (!(to > m)) return;
    // S and U are relative to the rounded m c, what comes to the rounded `to` c
    const float d = (m - to) * c + (rounding(to, c) - rounding(m, c));
    const float f = __builtin_amdgcn_exp2f(d);
    if (f == 0.0f && S == S) {
      S = U = 0.0f;
    } else if (S != 0.0f) {
      U = f * (U + S * d);
      S *= f;
    }
    m = to;
  }

  // Those of all lanes, which may have different maxima, in every lane.
  __device__ __forceinline__ void join(float c) {
    rescale(newt::lane_reduce<newt::Max, 63>(m), c);
    S = newt::lane_reduce<newt::Sum, 63>(S);
    U = newt::lane_reduce<newt::Sum, 63>(U);
  }
};

// Results of a row.
template <typename T>
__device__ __forceinline__ void finish(const newt_logprobs_params& p, int64_t row, const Sums& s,
                                       const Entry& e, int lane) {
  const float c = kLog2e * p.inv_temperature;
  // every logit -inf: 0 / 0, as a softmax over them gives
  const float lse = s.S > 0.0f ? __builtin_logf(s.S) : __builtin_nanf("");
  if (lane == 0) {
    const int64_t token = ((const int64_t*)p.tokens)[row];
    float logp = __builtin_nanf("");
    if (token == -1) logp = 0.0f;
    else if (token >= 0 && token < p.vocab)
      logp = natural(newt::to_f32(((const T*)p.logits)[row * p.stride + token]), s.m, c,
                     p.inv_temperature) - lse;
    p.logp[row] = logp;
    p.entropy[row] = lse - kLn2 * (s.U / s.S);
  }
  if (lane < p.top) {
    const bool none = e.id == kNone;
    p.top_logp[row * p.top + lane] =
        none ? __builtin_nanf("") : natural(e.value, s.m, c, p.inv_temperature) - lse;
    p.top_ids[row * p.top + lane] = none ? -1 : e.id;
  }
}

template <typename T>
struct Chunk {
  static constexpr int V = 16 / (int)sizeof(T);
  static constexpr int STEP = 64 * V;  // logits of a wave's chunk
  u32x4 raw;

  // V logits at a 16-byte address; no other program reads them
  __device__ __forceinline__ void load(const T* x) {
    raw = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(x));
  }
  // `n` of V logits, -inf behind
  __device__ __forceinline__ void load(const T* x, int64_t n) {
    newt::vec_t<T, V> t;
#pragma unroll
    for (int i = 0; i < V; ++i) t.d[i] = i < n ? x[i] : (T)-kInf;
    raw = __builtin_bit_cast(u32x4, t);
  }
  __device__ __forceinline__ void get(float* f) const {
    const auto t = __builtin_bit_cast(newt::vec_t<T, V>, raw);
#pragma unroll
    for (int i = 0; i < V; ++i) f[i] = newt::to_f32(t.d[i]);
  }
};

// What a wave keeps of its part of a row.
template <typename T>
struct Wave {
  static constexpr int V = Chunk<T>::V;
  const int top, lane;
  const float c;
  int64_t hi;
  Sums s{-kInf, 0.0f, 0.0f};  // m is the wave's, S and U the lane's
  Entry e{-kInf, kNone};
  Entry last{-kInf, kNone};   // the last entry that counts
  int taken = kNone;          // the logit that the lane gave to the list in begin()

  __device__ __forceinline__ void find_last() {
    last = Entry{uniform(e.value, top - 1), __builtin_amdgcn_readlane(e.id, top - 1)};
  }

  // Each lane's first largest logit of the first `n` chunks begins the list:
  // with 64 sorted ones of up to 2048, few of the others come before the last.
  template <int N>
  __device__ __forceinline__ void begin(const Chunk<T> (&chunks)[N], int n, int64_t at,
                                        int64_t step) {
#pragma unroll
    for (int j = 0; j < N; ++j) {
      if (j >= n) break;
      float f[V];
      chunks[j].get(f);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const int64_t id = at + j * step + lane * V + i;
        const bool better = (f[i] > e.value) | ((e.id == kNone) & (f[i] == f[i]));  // never NaN
        if (better & (id < hi)) e = Entry{f[i], (int)id};
      }
    }
    taken = e.id;
    s.m = newt::lane_reduce<newt::Max, 63>(e.value);
    if (!top) {
      last.value = s.m;
      return;
    }
    sort(e, lane);
    find_last();
  }

  // Candidates of a chunk into the list, whose last entry that counts decides
  // which ones are.
  __device__ __forceinline__ void candidates(const float* f, int64_t at) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int id = (int)(at + lane * V + i);
      const Entry x{f[i], id};  // NaN comes before nothing
      u64 found = __ballot(x.before(last) & (id != taken) & (at + lane * V + i < hi));
      while (found) {
        const int from = __builtin_ctzll(found);
        insert(e, Entry{uniform(f[i], from), __builtin_amdgcn_readlane(id, from)}, lane);
        find_last();
        found &= found - 1;
        found &= __ballot(x.before(last));
      }
    }
  }

  // With EARLY, a chunk that ids of the list lie behind or among: an equal logit
  // may come before the last entry.
  template <bool EARLY>
  __device__ __forceinline__ void take(const Chunk<T>& chunk, int64_t at) {
    float f[V];
    chunk.get(f);
    float most = f[0];
#pragma unroll
    for (int i = 1; i < V; ++i) most = __builtin_fmaxf(most, f[i]);
    most = __builtin_fmaxf(most, -kInf);  // of NaN alone: nothing
    // entries missing (fewer logits than alternatives so far): anything may come in
    if (EARLY || __ballot(most > last.value) != 0 || (top && last.id == kNone)) {
      if (top) candidates(f, at);
      s.rescale(newt::lane_reduce<newt::Max, 63>(most), c);
      if (!top) last.value = s.m;
    }
    const float m = s.m == -kInf ? 0.0f : s.m;
    float d[V];
    if (near_zero(newt::bits_f32(__builtin_amdgcn_readfirstlane(newt::f32_bits(m))), c)) {
      const float mc = m * c;
#pragma unroll
      for (int i = 0; i < V; ++i) d[i] = __builtin_fmaf(f[i], c, -mc);
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) d[i] = (f[i] - m) * c;
    }
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float x = __builtin_amdgcn_exp2f(d[i]);  // NaN stays NaN
      s.S += x;
      // 2^-inf * -inf counts as 0; d is at most a rounding above 0 (med3: one
      // instruction where fmaxf first quiets a NaN)
      s.U += x * __builtin_amdgcn_fmed3f(d[i], -200.0f, 4.0f);
    }
  }
};

template <typename T, int WAVES>
__global__ void __launch_bounds__(64 * WAVES)
logprobs_kernel(newt_logprobs_params p, int splits, int64_t per_split) {
  constexpr int STEP = Chunk<T>::STEP, V = Chunk<T>::V;
  const int lane = threadIdx.x & 63, wave = wave_id();
  const int64_t row = blockIdx.x / splits;
  const int split = blockIdx.x % splits;
  const int64_t lo = split * per_split;
  const int64_t hi = lo + per_split < p.vocab ? lo + per_split : p.vocab;
  const T* x = (const T*)p.logits + row * p.stride;
  const int top = p.top;
  const float c = kLog2e * p.inv_temperature;

  // Rows of an odd length begin anywhere: the first wave takes what lies before
  // the first 16-byte address. From there on the waves' chunks lie side by
  // side; AHEAD of them are on their way while one is worked on, and none of
  // those asks for bounds.
  constexpr int AHEAD = 4;
  Wave<T> w{top, lane, c, hi};
  const int past = (int)((uintptr_t)(x + lo) % 16 / sizeof(T));
  int64_t start = past ? lo + V - past : lo;
  start = start < hi ? start : hi;
  const int64_t step = WAVES * STEP, first = start + wave * STEP;
  const int whole = first + STEP <= hi ? (int)((hi - STEP - first) / step) + 1 : 0;
  const int64_t behind = first + whole * step;  // the last chunk that is not whole, if any
  const T* from = x + first + lane * V;
  Chunk<T> next[AHEAD], end[1];
  if (whole) {
    // behind the last whole chunk that one is loaded again, to no use
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) next[i].load(from + (i < whole ? i : whole - 1) * step);
  }
  if (behind < hi) end[0].load(from + whole * step, hi - behind - lane * V);
  if (whole) w.begin(next, whole < AHEAD ? whole : AHEAD, first, step);
  else if (behind < hi) w.begin(end, 1, behind, 0);
  if (wave == 0 && start > lo) {
    Chunk<T> head;
    head.load(x + lo + lane * V, start - lo - lane * V);
    w.hi = start;
    w.template take<true>(head, lo);
    w.hi = hi;
  }
  for (int j = 0; j < whole; j += AHEAD) {
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      const Chunk<T> now = next[i];
      const int to = j + i + AHEAD;
      next[i].load(from + (to < whole ? to : whole - 1) * step);
      if (j + i >= whole) continue;
      if (j == 0) w.template take<true>(now, first + i * step);
      else w.template take<false>(now, first + (j + i) * step);
    }
  }
  if (behind < hi) w.template take<true>(end[0], behind);

  Sums s = w.s;
  Entry e = w.e;
  s.join(c);
  __shared__ Sums sums[WAVES];
  __shared__ Entry entries[WAVES][64];
  if (lane == 0) sums[wave] = s;
  entries[wave][lane] = e;
  __syncthreads();
  if (wave != 0) return;
  s = lane < WAVES ? sums[lane] : Sums{-kInf, 0.0f, 0.0f};
  s.join(c);
  if (top)
    for (int i = 1; i < WAVES; ++i) merge(e, entries[i][63 - lane], lane);
  if (splits == 1) {
    finish<T>(p, row, s, e, lane);
    return;
  }
  // the split's sums, then its entries
  float* sums_at = (float*)p.workspace + (row * splits + split) * 4;
  Entry* to = (Entry*)((float*)p.workspace + p.rows * splits * 4) + (row * splits + split) * top;
  if (lane == 0) {
    sums_at[0] = s.m;
    sums_at[1] = s.S;
    sums_at[2] = s.U;
  }
  if (lane < top) to[lane] = e;
}

// One workgroup a row joins its splits: four lists by each wave, then four of
// theirs by each of the first waves, then the rest by the first.
template <typename T>
__global__ void __launch_bounds__(1024) logprobs_join_kernel(newt_logprobs_params p, int splits) {
  constexpr int WAVES = kMostSplits / 4;
  const int lane = threadIdx.x & 63, wave = wave_id();
  const int64_t row = blockIdx.x;
  const int top = p.top;
  const float c = kLog2e * p.inv_temperature;
  const float* sums = (const float*)p.workspace + (row * splits + lane) * 4;
  Sums s{-kInf, 0.0f, 0.0f};
  if (wave == 0 && lane < splits) s = Sums{sums[0], sums[1], sums[2]};
  const Entry* from = (const Entry*)((const float*)p.workspace + p.rows * splits * 4) +
                      row * splits * top;
  const Entry none{-kInf, kNone};
  Entry e = none;
  if (top) {
    __shared__ Entry entries[WAVES][64];
    Entry list[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int at = i == 0 ? lane : 63 - lane, split = wave + i * WAVES;
      list[i] = at < top && split < splits ? from[split * top + at] : none;
    }
    e = list[0];
#pragma unroll
    for (int i = 1; i < 4; ++i)
      if (wave + i * WAVES < splits) merge(e, list[i], lane);
    int lists = WAVES;  // of which the first min(lists, splits) hold anything
#pragma unroll
    for (; lists > 1; lists /= 4) {
      if (wave < lists) entries[wave][lane] = e;
      __syncthreads();
      if (wave < lists / 4)
#pragma unroll
        for (int i = 1; i < 4; ++i)
          if (wave + i * (lists / 4) < splits) merge(e, entries[wave + i * (lists / 4)][63 - lane], lane);
      __syncthreads();
    }
  }
  if (wave != 0) return;
  s.join(c);
  finish<T>(p, row, s, e, lane);
}

// How rows are shared out: to 16 waves for each CU, as the list that each wave
// begins, and joins with the others', costs it as much as 10000 logits do. Few
// rows go to several workgroups each, with at least 8192 logits.
struct Plan {
  int waves, splits;
  int64_t per_split;
  Plan(int64_t rows, int64_t vocab) {
    waves = rows >= 4096 ? 1 : rows >= 2048 ? 2 : 4;
    int64_t n = rows ? (512 + rows - 1) / rows : 1;
    const int64_t most = (vocab + 8191) / 8192;
    n = n < most ? n : most;
    n = n < 1 ? 1 : n < kMostSplits ? n : kMostSplits;
    per_split = ((vocab + n - 1) / n + 7) / 8 * 8;
    splits = (int)((vocab + per_split - 1) / per_split);
  }
};

template <typename T, int WAVES>
int start(const newt_logprobs_params& p, const Plan& r, hipStream_t stream) {
  return run("newt_token_logprobs", logprobs_kernel<T, WAVES>, p.rows * r.splits, 64 * WAVES, 0,
             stream, p, r.splits, r.per_split);
}

template <typename T>
int launch(const newt_logprobs_params& p, hipStream_t stream) {
  const Plan r(p.rows, p.vocab);
  if (r.splits > 1 && !p.workspace)
    return fail(NEWT_ERR_INVALID, "newt_token_logprobs: null workspace");
  if (p.rows * r.splits > 0x7fffffff)
    return fail(NEWT_ERR_INVALID, "newt_token_logprobs: too many rows");
  const int status = r.waves == 1   ? start<T, 1>(p, r, stream)
                     : r.waves == 2 ? start<T, 2>(p, r, stream)
                                    : start<T, 4>(p, r, stream);
  if (status != NEWT_OK || r.splits == 1) return status;
  return run("newt_token_logprobs", logprobs_join_kernel<T>, p.rows, 1024, 0, stream, p, r.splits);
}

}  // namespace
}  // namespace newt_ops

extern "C" size_t newt_token_logprobs_workspace(int64_t rows, int64_t vocab, int32_t top, int32_t) {
  if (rows <= 0 || vocab <= 0) return 0;
  const newt_ops::Plan r(rows, vocab);
  return r.splits > 1 ? (size_t)rows * r.splits * (2 * top + 4) * sizeof(float) : 0;
}

extern "C" int newt_token_logprobs(const newt_logprobs_params* params, void* stream) {
  using namespace newt_ops;
  if (!params) return fail(NEWT_ERR_INVALID, "newt_token_logprobs: null params");
  const newt_logprobs_params& p = *params;
  if (p.rows == 0) return NEWT_OK;
  if (!p.logits || !p.tokens || !p.logp || !p.entropy || (p.top && (!p.top_logp || !p.top_ids)))
    return fail(NEWT_ERR_INVALID, "newt_token_logprobs: null tensor");
  if (p.rows < 0 || p.vocab <= 0 || p.vocab > 0x7fffffff)
    return fail(NEWT_ERR_INVALID, "newt_token_logprobs: %lld rows of %lld logits",
                (long long)p.rows, (long long)p.vocab);
  if (p.top < 0 || p.top > 64 || p.top > p.vocab)
    return fail(NEWT_ERR_INVALID, "newt_token_logprobs: no %d alternatives of %lld (at most 64)",
                p.top, (long long)p.vocab);
  if (!(p.inv_temperature > 0.0f))
    return fail(NEWT_ERR_INVALID, "newt_token_logprobs: temperature has to be positive");
  hipStream_t s = static_cast<hipStream_t>(stream);
  switch (p.dtype) {
    case NEWT_F32: return launch<float>(p, s);
    case NEWT_F16: return launch<f16>(p, s);
    case NEWT_BF16: return launch<bf16>(p, s);
    default: return fail(NEWT_ERR_INVALID, "newt_token_logprobs: unknown dtype %d", p.dtype);
  }
}
