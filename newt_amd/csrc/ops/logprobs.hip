// Log probabilities of given tokens, entropy and the largest alternatives:
// with x = logits / T,  m = max x,  S = sum 2^d,  U = sum 2^d d,
// d = (x - m) log2(e):
//   logp = x[token] - m - ln S,  entropy = ln 2 (log2 S - U / S).
// One pass over the logits, which bound it. Each wave keeps m and the list of
// its largest logits so far as wave-uniform state (a lane per list entry), so
// the stream itself costs one comparison a chunk: only a chunk that holds
// something larger than the list's last entry takes the slow path, which
// inserts it and, where the maximum grew, rescales S and U. Expected
// insertions over n logits in no order: top * ln(n / top).
#include "common.h"

namespace newt_ops {
namespace {

constexpr float kLog2e = 1.44269504088896341f;
constexpr float kLn2 = 0.693147180559945309f;
constexpr float kInf = __builtin_inff();
constexpr int kWaves = 4;

// What a wave has seen of a row: m, S and U, and the list's entries, one a
// lane, best first; `n` of them, `last` the value a candidate has to pass.
struct Seen {
  float m = -kInf, S = 0.0f, U = 0.0f;
  float value = -kInf;
  int id = -1;
  int n = 0;

  // m rises to `to`
  __device__ __forceinline__ void rescale(float to, float c) {
    if (!(to > m)) return;
    if (m == -kInf) {
      m = to;
      return;  // nothing but -inf so far: S and U are 0
    }
    const float d = (m - to) * c;
    const float f = __builtin_amdgcn_exp2f(d);
    U = f == 0.0f ? 0.0f : f * (U + S * d);
    S *= f;
    m = to;
  }

  // Candidate (v, at), both the same in every lane, goes behind all entries
  // that are larger or equal with a lower id.
  __device__ __forceinline__ void insert(float v, int at, int top, int lane) {
    const bool before = lane < n && (value > v || (value == v && id < at));
    const int place = __popcll(__ballot(before));
    if (place >= top) return;
    const float left = __shfl_up(value, 1);
    const int left_id = __shfl_up(id, 1);
    if (lane > place) {
      value = left;
      id = left_id;
    }
    if (lane == place) {
      value = v;
      id = at;
    }
    n = n < top ? n + 1 : top;
  }

  __device__ __forceinline__ float last(int top) const {
    return __shfl(value, top - 1);
  }
};

__device__ __forceinline__ float uniform(float v, int lane) {
  return newt::bits_f32(__builtin_amdgcn_readlane(newt::f32_bits(v), lane));
}

// Results of a row whose whole stream `s` holds (S and U already summed).
template <typename T>
__device__ __forceinline__ void finish(const newt_logprobs_params& p, int64_t row, const Seen& s,
                                       int lane) {
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
    p.top_logp[row * p.top + lane] = lane < s.n ? (s.value - s.m) * inv - lse : __builtin_nanf("");
    p.top_ids[row * p.top + lane] = lane < s.n ? s.id : -1;
  }
}

// The partial results of one split of a row, `2 * top + 4` words.
struct Partial {
  u32* at;
  __device__ __forceinline__ void put(const Seen& s, int top, int lane) const {
    if (lane == 0) {
      at[0] = newt::f32_bits(s.m);
      at[1] = newt::f32_bits(s.S);
      at[2] = newt::f32_bits(s.U);
      at[3] = (u32)s.n;
    }
    if (lane < top) {
      at[4 + lane] = newt::f32_bits(s.value);
      at[4 + top + lane] = (u32)s.id;
    }
  }
};

// Adds another wave's or split's results: sums (uniform) and list (a lane an entry).
__device__ __forceinline__ void join(Seen& s, float m, float S, float U, float value, int id, int n,
                                     float c, int top, int lane) {
  s.rescale(m, c);
  if (m == s.m) {
    if (S != 0.0f) {
      s.U += U;
      s.S += S;
    }
  } else if (S != 0.0f) {
    const float d = (m - s.m) * c;
    const float f = __builtin_amdgcn_exp2f(d);
    s.U += f == 0.0f ? 0.0f : f * (U + S * d);
    s.S += S * f;
  }
  for (int e = 0; e < n; ++e) {
    const float v = uniform(value, e);
    if (s.n == top && !(v >= s.last(top))) break;  // no later one is larger
    s.insert(v, __builtin_amdgcn_readlane(id, e), top, lane);
  }
}

template <typename T>
__global__ void __launch_bounds__(64 * kWaves)
logprobs_kernel(newt_logprobs_params p, int splits, int64_t per_split) {
  constexpr int V = 16 / (int)sizeof(T);
  constexpr int STEP = 64 * V;  // logits of a wave's chunk
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t row = blockIdx.x / splits;
  const int split = blockIdx.x % splits;
  const int64_t lo = split * per_split;
  const int64_t hi = lo + per_split < p.vocab ? lo + per_split : p.vocab;
  const T* x = (const T*)p.logits + row * p.stride;
  const int top = p.top;
  const float c = kLog2e * p.inv_temperature;

  Seen s;
  float last = -kInf;   // a chunk without anything above it needs no slow path
  bool filling = top > 0;
  for (int64_t at = lo + wave * STEP; at < hi; at += kWaves * STEP) {
    const int64_t mine = at + lane * V;
    float f[V];
    if (mine + V <= hi) {
      T t[V];
      newt::load_vec<T, V>(x + mine, t, newt::any_align());
#pragma unroll
      for (int i = 0; i < V; ++i) f[i] = newt::to_f32(t[i]);
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) f[i] = mine + i < hi ? newt::to_f32(x[mine + i]) : -kInf;
    }
    float most = f[0];
#pragma unroll
    for (int i = 1; i < V; ++i) most = __builtin_fmaxf(most, f[i]);
    u64 found = __ballot(most > last);
    if (found != 0 || filling) {
      if (top == 0) {
        s.rescale(newt::lane_reduce<newt::Max, 63>(most), c);
        last = s.m;
      } else {
        if (filling) found = ~0ull;
        const float highest = newt::lane_reduce<newt::Max, 63>(most);
        while (found) {
          const int from = __builtin_ctzll(found);
          found &= found - 1;
#pragma unroll
          for (int i = 0; i < V; ++i) {
            const float v = uniform(f[i], from);
            const int64_t id = at + from * V + i;
            // NaN passes neither test
            if (id < hi && (filling ? v == v : v > last)) {
              s.insert(v, (int)id, top, lane);
              if (s.n == top) {
                filling = false;
                last = s.last(top);
              }
            }
          }
          if (!filling) found &= __ballot(most > last);
        }
        s.rescale(highest, c);
      }
    }
    const float m = s.m == -kInf ? 0.0f : s.m;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float d = (f[i] - m) * c;
      const float e = __builtin_amdgcn_exp2f(d);  // NaN stays NaN
      s.S += e;
      s.U += e * __builtin_fmaxf(d, -200.0f);  // 2^-inf * -inf counts as 0
    }
  }
  s.S = newt::lane_reduce<newt::Sum, 63>(s.S);
  s.U = newt::lane_reduce<newt::Sum, 63>(s.U);

  __shared__ float sums[kWaves][4];
  __shared__ float values[kWaves][64];
  __shared__ int ids[kWaves][64];
  if (lane == 0) {
    sums[wave][0] = s.m;
    sums[wave][1] = s.S;
    sums[wave][2] = s.U;
    sums[wave][3] = newt::bits_f32((u32)s.n);
  }
  values[wave][lane] = s.value;
  ids[wave][lane] = s.id;
  __syncthreads();
  if (wave != 0) return;
  for (int w = 1; w < kWaves; ++w)
    join(s, sums[w][0], sums[w][1], sums[w][2], values[w][lane], ids[w][lane],
         __builtin_amdgcn_readfirstlane((int)newt::f32_bits(sums[w][3])), c, top, lane);
  if (splits == 1)
    finish<T>(p, row, s, lane);
  else
    Partial{(u32*)p.workspace + (row * splits + split) * (2 * top + 4)}.put(s, top, lane);
}

// One wave a row joins its splits.
template <typename T>
__global__ void __launch_bounds__(64) logprobs_join_kernel(newt_logprobs_params p, int splits) {
  const int lane = threadIdx.x;
  const int64_t row = blockIdx.x;
  const int top = p.top, words = 2 * top + 4;
  const float c = kLog2e * p.inv_temperature;
  Seen s;
  for (int i = 0; i < splits; ++i) {
    const u32* at = (const u32*)p.workspace + (row * splits + i) * words;
    join(s, newt::bits_f32(at[0]), newt::bits_f32(at[1]), newt::bits_f32(at[2]),
         lane < top ? newt::bits_f32(at[4 + lane]) : -kInf, lane < top ? (int)at[4 + top + lane] : -1,
         __builtin_amdgcn_readfirstlane((int)at[3]), c, top, lane);
  }
  finish<T>(p, row, s, lane);
}

// How a row is shared out: enough workgroups to fill the chip where there are
// few rows, each with at least 8192 logits.
void plan(int64_t rows, int64_t vocab, int* splits, int64_t* per_split) {
  int64_t n = rows ? (1024 + rows - 1) / rows : 1;
  const int64_t most = (vocab + 8191) / 8192;
  n = n < most ? n : most;
  n = n < 1 ? 1 : n;
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
    logprobs_join_kernel<T><<<dim3((unsigned)p.rows), dim3(64), 0, stream>>>(p, splits);
  return launched("newt_token_logprobs");
}

}  // namespace
}  // namespace newt_ops

extern "C" size_t newt_token_logprobs_workspace(int64_t rows, int64_t vocab, int32_t top, int32_t) {
  if (rows <= 0 || vocab <= 0) return 0;
  int splits;
  int64_t per;
  newt_ops::plan(rows, vocab, &splits, &per);
  return splits > 1 ? (size_t)rows * splits * (2 * top + 4) * 4 : 0;
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
