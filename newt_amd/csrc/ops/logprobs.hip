// Log probabilities of given tokens, entropy and the largest alternatives:
// with x = logits / T,  m = max x,  S = sum 2^d,  U = sum 2^d d,
// d = (x - m) log2(e):
//   logp = x[token] - m - ln S,  entropy = ln 2 (log2 S - U / S).
// One pass over the logits, which bound it. Each wave keeps m and its 64
// largest logits so far, sorted, an entry a lane, so the stream itself costs
// one comparison a chunk: only a chunk that holds something larger than the
// last entry that counts takes the slow path, which inserts it and, where the
// maximum grew, rescales S and U. The list begins with the sorted largest
// logits of each lane in the first chunk; after that n logits in no order make
// about top * ln(n / 512) insertions. Lists are joined by bitonic merges.
#include "common.h"

namespace newt_ops {
namespace {

constexpr float kLog2e = 1.44269504088896341f;
constexpr float kLn2 = 0.693147180559945309f;
constexpr float kInf = __builtin_inff();
constexpr int kNone = 0x7fffffff;  // the id of an entry that is none: behind all others
constexpr int kWaves = 4;
constexpr int kMostSplits = 64;

__device__ __forceinline__ float uniform(float v, int lane) {
  return newt::bits_f32(__builtin_amdgcn_readlane(newt::f32_bits(v), lane));
}

// A list entry: larger logits first, then lower ids.
struct Entry {
  float value;
  int id;
  __device__ __forceinline__ bool before(const Entry& o) const {
    return value > o.value || (value == o.value && id < o.id);
  }
};

// One step of a bitonic network over the lanes: of each pair of lanes that
// differ in bit M the one with that bit clear keeps the entry that comes first
// (where `down`, else last).
template <int M>
__device__ __forceinline__ void exchange(Entry& e, bool down, int lane) {
  const Entry o{newt::xor_lane<M>(e.value), newt::xor_lane<M>(e.id)};
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
  const Entry left{__shfl_up(e.value, 1), __shfl_up(e.id, 1)};
  if (lane > place) e = left;
  if (lane == place) e = c;
}

// The sums over what a lane, a wave or a split has seen.
struct Sums {
  float m, S, U;

  // The same relative to the maximum `to` >= m.
  __device__ __forceinline__ void rescale(float to, float c) {
    if (!(to > m)) return;
    const float d = (m - to) * c;
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
  const float inv = p.inv_temperature;
  // every logit -inf: 0 / 0, as a softmax over them gives
  const float lse = s.S > 0.0f ? __builtin_logf(s.S) : __builtin_nanf("");
  if (lane == 0) {
    const int64_t token = ((const int64_t*)p.tokens)[row];
    float logp = __builtin_nanf("");
    if (token == -1) logp = 0.0f;
    else if (token >= 0 && token < p.vocab)
      logp = (newt::to_f32(((const T*)p.logits)[row * p.stride + token]) - s.m) * inv - lse;
    p.logp[row] = logp;
    p.entropy[row] = lse - kLn2 * (s.U / s.S);
  }
  if (lane < p.top) {
    const bool none = e.id == kNone;
    p.top_logp[row * p.top + lane] = none ? __builtin_nanf("") : (e.value - s.m) * inv - lse;
    p.top_ids[row * p.top + lane] = none ? -1 : e.id;
  }
}

template <typename T>
struct Chunk {
  static constexpr int V = 16 / (int)sizeof(T);
  static constexpr int STEP = 64 * V;  // logits of a wave's chunk
  u32x4 raw;

  // V logits from `at` on, -inf behind `hi`
  __device__ __forceinline__ void load(const T* x, int64_t at, int64_t hi) {
    if (at + V <= hi) {
      raw = *reinterpret_cast<const typename newt::any_vec<T, V>::type*>(x + at);
    } else {
      T t[V];
#pragma unroll
      for (int i = 0; i < V; ++i) t[i] = at + i < hi ? x[at + i] : (T)-kInf;
      raw = __builtin_bit_cast(u32x4, *reinterpret_cast<newt::vec_t<T, V>*>(t));
    }
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
  const int64_t hi;
  const float c;
  Sums s{-kInf, 0.0f, 0.0f};  // m is the wave's, S and U the lane's
  Entry e{-kInf, kNone};
  Entry last{-kInf, kNone};   // the last entry that counts
  bool begun = false;

  // Candidates of a chunk, in the order of their ids. `taken` marks, in the
  // first chunk, the logit that a lane gave to the list already.
  __device__ __forceinline__ void candidates(const float* f, float most, int64_t at, int taken) {
    // `most` may equal the last entry and still come before it, but later ids
    // never come before earlier ones unless there are entries that are none
    const bool equal = taken >= 0 || last.id == kNone;
    u64 found = __ballot(equal ? most >= last.value : most > last.value);
    while (found) {
      const int from = __builtin_ctzll(found);
      found &= found - 1;
      const int skip = __builtin_amdgcn_readlane(taken, from);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const Entry x{uniform(f[i], from), (int)(at + from * V + i)};
        if (i != skip && at + from * V + i < hi && x.before(last)) {  // never NaN
          insert(e, x, lane);
          last = Entry{uniform(e.value, top - 1), __builtin_amdgcn_readlane(e.id, top - 1)};
        }
      }
      if (!equal) found &= __ballot(most > last.value);
    }
  }

  __device__ __forceinline__ void slow(const float* f, float most, int64_t at) {
    const float highest = newt::lane_reduce<newt::Max, 63>(most);
    if (top) {
      int taken = -1;
      if (!begun) {
        begun = true;
        // each lane's first largest logit begins the list
#pragma unroll
        for (int i = V - 1; i >= 0; --i)
          if (f[i] == most && at + lane * V + i < hi) taken = i;
        e = Entry{taken < 0 ? -kInf : most, taken < 0 ? kNone : (int)(at + lane * V + taken)};
        sort(e, lane);
        last = Entry{uniform(e.value, top - 1), __builtin_amdgcn_readlane(e.id, top - 1)};
        if (taken < 0) taken = V;  // nothing to leave out, but this is the first chunk
        most = -kInf;
#pragma unroll
        for (int i = 0; i < V; ++i)
          if (i != taken) most = __builtin_fmaxf(most, f[i]);
      }
      candidates(f, most, at, taken);
    }
    s.rescale(highest, c);
    if (!top) last.value = s.m;
  }

  __device__ __forceinline__ void take(const Chunk<T>& chunk, int64_t at) {
    float f[V];
    chunk.get(f);
    float most = f[0];
#pragma unroll
    for (int i = 1; i < V; ++i) most = __builtin_fmaxf(most, f[i]);
    most = __builtin_fmaxf(most, -kInf);  // of NaN alone: nothing
    // top > 0 and entries missing: anything may still come in
    if (__ballot(most > last.value) || (top && last.id == kNone)) slow(f, most, at);
    const float m = s.m == -kInf ? 0.0f : s.m;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float d = (f[i] - m) * c;
      const float x = __builtin_amdgcn_exp2f(d);  // NaN stays NaN
      s.S += x;
      s.U += x * __builtin_fmaxf(d, -200.0f);  // 2^-inf * -inf counts as 0
    }
  }
};

template <typename T>
__global__ void __launch_bounds__(64 * kWaves)
logprobs_kernel(newt_logprobs_params p, int splits, int64_t per_split) {
  constexpr int STEP = Chunk<T>::STEP, V = Chunk<T>::V;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t row = blockIdx.x / splits;
  const int split = blockIdx.x % splits;
  const int64_t lo = split * per_split;
  const int64_t hi = lo + per_split < p.vocab ? lo + per_split : p.vocab;
  const T* x = (const T*)p.logits + row * p.stride;
  const int top = p.top;
  const float c = kLog2e * p.inv_temperature;

  // chunks of the waves lie side by side; two are on their way while two are
  // worked on
  constexpr int AHEAD = 2;
  Wave<T> w{top, lane, hi, c};
  Chunk<T> next[AHEAD];
  const int64_t step = kWaves * STEP;
  int64_t at = lo + wave * STEP;
#pragma unroll
  for (int i = 0; i < AHEAD; ++i) next[i].load(x, at + i * step + lane * V, hi);
  for (; at < hi; at += AHEAD * step) {
    Chunk<T> now[AHEAD];
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) now[i] = next[i];
#pragma unroll
    for (int i = 0; i < AHEAD; ++i)
      next[i].load(x, at + (AHEAD + i) * step + lane * V, hi);
#pragma unroll
    for (int i = 0; i < AHEAD; ++i)
      if (at + i * step < hi) w.take(now[i], at + i * step);
  }

  Sums s = w.s;
  Entry e = w.e;
  s.join(c);
  __shared__ Sums sums[kWaves];
  __shared__ Entry entries[kWaves][64];
  if (lane == 0) sums[wave] = s;
  entries[wave][lane] = e;
  __syncthreads();
  if (wave != 0) return;
  s = lane < kWaves ? sums[lane] : Sums{-kInf, 0.0f, 0.0f};
  s.join(c);
  if (top)
    for (int i = 1; i < kWaves; ++i) merge(e, entries[i][63 - lane], lane);
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

// One workgroup a row joins its splits: each wave some of their lists, then
// the first wave those of all.
template <typename T>
__global__ void __launch_bounds__(64 * kWaves)
logprobs_join_kernel(newt_logprobs_params p, int splits) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t row = blockIdx.x;
  const int top = p.top;
  const float c = kLog2e * p.inv_temperature;
  const Entry* from = (const Entry*)((const float*)p.workspace + p.rows * splits * 4) +
                      row * splits * top;
  const Entry none{-kInf, kNone};
  Entry e = none;
  if (top) {
    __shared__ Entry entries[kWaves][64];
    if (wave < splits && lane < top) e = from[wave * top + lane];
    for (int i = wave + kWaves; i < splits; i += kWaves)
      merge(e, 63 - lane < top ? from[i * top + 63 - lane] : none, lane);
    entries[wave][lane] = e;
    __syncthreads();
    if (wave != 0) return;
    for (int i = 1; i < kWaves; ++i) merge(e, entries[i][63 - lane], lane);
  } else if (wave != 0) {
    return;
  }
  const float* sums = (const float*)p.workspace + (row * splits + lane) * 4;
  Sums s{-kInf, 0.0f, 0.0f};
  if (lane < splits) s = Sums{sums[0], sums[1], sums[2]};
  s.join(c);
  finish<T>(p, row, s, e, lane);
}

// How a row is shared out: enough workgroups to fill the chip where there are
// few rows, each with at least 4096 logits.
void plan(int64_t rows, int64_t vocab, int* splits, int64_t* per_split) {
  int64_t n = rows ? (1024 + rows - 1) / rows : 1;
  const int64_t most = (vocab + 4095) / 4096;
  n = n < most ? n : most;
  n = n < 1 ? 1 : n < kMostSplits ? n : kMostSplits;
  int64_t per = (vocab + n - 1) / n;
  per = (per + 7) / 8 * 8;
  *splits = (int)((vocab + per - 1) / per);
  *per_split = per;
}

template <typename T>
int launch(const newt_logprobs_params& p, hipStream_t stream) {
  int splits;
  int64_t per;
  plan(p.rows, p.vocab, &splits, &per);
  if (splits > 1 && !p.workspace)
    return fail(NEWT_ERR_INVALID, "newt_token_logprobs: null workspace");
  if (p.rows * splits > 0x7fffffff)
    return fail(NEWT_ERR_INVALID, "newt_token_logprobs: too many rows");
  logprobs_kernel<T><<<dim3((unsigned)(p.rows * splits)), dim3(64 * kWaves), 0, stream>>>(p, splits,
                                                                                          per);
  if (splits > 1)
    logprobs_join_kernel<T><<<dim3((unsigned)p.rows), dim3(64 * kWaves), 0, stream>>>(p, splits);
  return launched("newt_token_logprobs");
}

}  // namespace
}  // namespace newt_ops

extern "C" size_t newt_token_logprobs_workspace(int64_t rows, int64_t vocab, int32_t top, int32_t) {
  if (rows <= 0 || vocab <= 0) return 0;
  int splits;
  int64_t per;
  newt_ops::plan(rows, vocab, &splits, &per);
  return splits > 1 ? (size_t)rows * splits * (2 * top + 4) * sizeof(float) : 0;
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
