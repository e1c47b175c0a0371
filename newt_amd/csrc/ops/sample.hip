// The next token of each row of logits: weights e^((x - max x) / T), kept by
// top_k, top_p and min_p, and the first id whose running kept weight exceeds u
// times their sum.
// What is kept is the beginning of the logits in falling order, so no order is
// ever made: a histogram over (max - x) / T finds the bin in which the last kept
// one lies, histograms over the bits of its logits find it, and where some but
// not all logits equal to it stay, a search by id finds the last of those. Weights
// are whole numbers of 2^-45 (less for more than 2^17 ids), from exponentials in
// 64 bits: their sums are exact, whatever the order in which atomics add them, so
// the same row gives the same id in every call, and a border is off by 2^-46 of
// the largest weight for each id before it.
#include "common.h"

namespace newt_ops {
namespace {

constexpr int kThreads = 1024, kWaves = kThreads / 64;
constexpr int kBins = 2048;
constexpr int kSegments = 2048;
constexpr float kInf = __builtin_inff();
constexpr u32 kNone = 0xffffffffu;

template <typename T> struct io { static constexpr int V = 16 / (int)sizeof(T); };

// Numbers in the order of the logits; -0 and 0 are equal.
__device__ __forceinline__ u32 key_of(float x) {
  const u32 b = newt::f32_bits(x + 0.0f);
  return b ^ ((u32)((int)b >> 31) | 0x80000000u);
}

// e^y for y <= 0 as a whole number of 2^-shift. y = n ln 2 + r, |r| <= ln 2 / 2;
// the sum's first term left out is r^13 / 13!, 2^-53.
__device__ __forceinline__ u64 weigh(double y, int shift) {
  const double n = __builtin_rint(y * 1.4426950408889634074);
  double r = __builtin_fma(n, -6.93147180559945286e-1, y);
  r = __builtin_fma(n, -2.31904681384629956e-17, r);
  double e = 2.08767569878681e-9;  // 1 / 12!
  e = __builtin_fma(e, r, 2.50521083854417e-8);
  e = __builtin_fma(e, r, 2.75573192239859e-7);
  e = __builtin_fma(e, r, 2.75573192239859e-6);
  e = __builtin_fma(e, r, 2.48015873015873e-5);
  e = __builtin_fma(e, r, 1.98412698412698e-4);
  e = __builtin_fma(e, r, 1.38888888888889e-3);
  e = __builtin_fma(e, r, 8.33333333333333e-3);
  e = __builtin_fma(e, r, 4.16666666666667e-2);
  e = __builtin_fma(e, r, 1.66666666666667e-1);
  e = __builtin_fma(e, r, 0.5);
  e = __builtin_fma(e, r, 1.0);
  e = __builtin_fma(e, r, 1.0);
  // below 2^52 the sum's low bits are the whole number
  const double whole = __builtin_ldexp(e, (int)n + shift) + 4503599627370496.0;
  return __builtin_bit_cast(u64, whole) & 0xfffffffffffffull;
}

template <typename V>
__device__ __forceinline__ V wave_sum(V v) {
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) v += __shfl_xor(v, m);
  return v;
}

// The sum over this lane and those below it.
template <typename V>
__device__ __forceinline__ V wave_scan(V v, int lane) {
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) {
    const V o = __shfl_up(v, m);
    if (lane >= m) v += o;
  }
  return v;
}

struct Shared {
  u64 mass[kBins];     // also a search's segments
  u32 count[kBins];
  u64 part[kWaves];
  u32 part_count[kWaves];
  float top[kWaves];
  int bad[kWaves];
  // what a search found
  u64 before;
  u32 before_count, place, place_count;
  u64 place_mass;
};

template <typename T>
struct Row {
  static constexpr int V = io<T>::V;
  static constexpr int CHUNK = 64 * V;  // of a wave
  const T* x;
  int vocab, chunks, shift;
  int lane, wave;
  Shared& s;
  float top;          // the largest logit
  double by;          // 1 / T
  float bin_scale;

  // V numbers from i on, -inf behind the row's end
  __device__ __forceinline__ void load(int64_t i, float* f) const {
    T t[V];
    if (i + V <= vocab) {
      newt::load_vec<T, V>(x + i, t, newt::any_align());
#pragma unroll
      for (int j = 0; j < V; ++j) f[j] = newt::to_f32(t[j]);
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j) f[j] = i + j < vocab ? newt::to_f32(x[i + j]) : -kInf;
    }
  }
  __device__ __forceinline__ u64 weight(float f) const {
    // e^-1000 is 0 in every shift
    return weigh(__builtin_fmax(((double)f - (double)top) * by, -1000.0), shift);
  }
  // Bins fall with the logit; the last one holds weights of 0 alone.
  __device__ __forceinline__ int bin(float f) const {
    return (int)__builtin_fminf((top - f) * bin_scale, (float)(kBins - 1));
  }
  // f(number) for each of the row, in no order
  template <typename F>
  __device__ __forceinline__ void each(F f) const {
    for (int c = wave; c < chunks; c += kWaves) {
      float v[V];
      load((int64_t)c * CHUNK + lane * V, v);
#pragma unroll
      for (int j = 0; j < V; ++j) f(v[j]);
    }
  }

  __device__ __forceinline__ void clear() const {
    for (int i = threadIdx.x; i < kBins; i += kThreads) {
      s.mass[i] = 0;
      s.count[i] = 0;
    }
    __syncthreads();
  }

  // Of the histogram's bins the first where the running count reaches `k` or the
  // running mass, with `before`, reaches `target`; its place, what lies before
  // it and what is in it to s. All threads call it; the bins are full.
  __device__ __forceinline__ void pick(bool by_mass, u64 k, u64 before, double target) const {
    const int i = threadIdx.x * 2;
    const u64 m0 = s.mass[i], m1 = s.mass[i + 1];
    const u32 c0 = s.count[i], c1 = s.count[i + 1];
    u64 m = wave_scan(m0 + m1, lane);
    u32 c = wave_scan(c0 + c1, lane);
    if (lane == 63) {
      s.part[wave] = m;
      s.part_count[wave] = c;
    }
    if (threadIdx.x == 0) s.place = kNone;
    __syncthreads();
    for (int w = 0; w < wave; ++w) {
      m += s.part[w];
      c += s.part_count[w];
    }
    const u64 mb1 = before + m - m1, mb0 = mb1 - m0;
    const u32 cb1 = c - c1, cb0 = cb1 - c0;
    const auto reached = [&](u64 mass, u32 count) {
      return by_mass ? (double)mass >= target : count >= k;
    };
    // reached with a bin, and not before it
    if (reached(mb1, cb1)) {
      if (!reached(mb0, cb0) && c0) found(i, mb0, cb0, m0, c0);
    } else if (reached(mb1 + m1, c) && c1) {
      found(i + 1, mb1, cb1, m1, c1);
    }
    __syncthreads();
  }
  __device__ __forceinline__ void found(int i, u64 before, u32 before_count, u64 m, u32 c) const {
    s.place = i;
    s.before = before;
    s.before_count = before_count;
    s.place_mass = m;
    s.place_count = c;
  }

  // A logit's key and how many equal ones stay.
  struct Last {
    u32 key, keep, equal;  // `equal`: how many there are
    u64 before;            // the mass of those before it
    u64 each;              // the mass of one
    bool all;              // nothing is left out
  };

  // The last that stays, by count (k > 0) or by mass (target > before).
  __device__ __forceinline__ Last last(bool by_mass, u32 k, double target) const {
    clear();
    each([&](float f) {
      const int b = bin(f);
      if (b < kBins - 1) {
        atomicAdd(&s.count[b], 1u);
        atomicAdd(&s.mass[b], weight(f));
      }
    });
    __syncthreads();
    pick(by_mass, k, 0, target);
    Last r = {0, 0, 0, 0, 0, true};
    if (s.place == kNone) return r;  // among weights of 0, or everything
    r.all = false;
    // the keys of that bin: all at first, then those of a finer histogram's bin
    const int at = s.place;
    u64 before = s.before;
    u32 before_count = s.before_count;
    u32 lo = 0, hi = 0xffffffffu;
    bool first = true;
    for (;;) {
      // the smallest and largest key that are there
      u32 least = 0xffffffffu, most = 0;
      each([&](float f) {
        const u32 key = key_of(f);
        if (first ? bin(f) == at : (key >= lo) & (key <= hi)) {
          least = key < least ? key : least;
          most = key > most ? key : most;
        }
      });
      clear();
      if (threadIdx.x == 0) {
        s.count[0] = 0xffffffffu;
        s.count[1] = 0;
      }
      __syncthreads();
      if (least <= most) {
        atomicMin(&s.count[0], least);
        atomicMax(&s.count[1], most);
      }
      __syncthreads();
      lo = s.count[0];
      hi = s.count[1];
      __syncthreads();
      clear();
      const u32 range = hi - lo;
      const int shift = range < kBins ? 0 : 21 - __builtin_clz(range);  // range >> shift < kBins
      each([&](float f) {
        const u32 key = key_of(f);
        if ((key >= lo) & (key <= hi)) {
          const u32 b = (hi - key) >> shift;
          atomicAdd(&s.count[b], 1u);
          atomicAdd(&s.mass[b], weight(f));
        }
      });
      __syncthreads();
      pick(by_mass, k - before_count, before, target);
      before = s.before;
      before_count += s.before_count;
      const u32 top_key = hi - (s.place << shift);
      if (shift == 0) {
        r.key = top_key;
        r.equal = s.place_count;
        r.before = before;
        r.each = s.place_mass / s.place_count;
        if (by_mass) {
          // those before which less than the target lies
          const double n = __builtin_ceil((target - (double)before) / (double)r.each);
          r.keep = n >= (double)r.equal ? r.equal : n < 1.0 ? 1 : (u32)n;
        } else {
          r.keep = k - before_count;
        }
        __syncthreads();
        return r;
      }
      const u32 width = (1u << shift) - 1;
      hi = top_key;
      lo = hi - lo > width ? hi - width : lo;
      first = false;
      __syncthreads();
    }
  }

  // The sum of f(number, id) over the row, in segments of consecutive chunks that
  // `find` searches.
  template <typename F>
  __device__ __forceinline__ u64 segments(F f) const {
    const int per = (chunks + kSegments - 1) / kSegments;
    const int count = (chunks + per - 1) / per;
    __syncthreads();
    for (int g = wave; g < count; g += kWaves) {
      u64 sum = 0;
      for (int c = g * per; c < chunks && c < (g + 1) * per; ++c) {
        float v[V];
        const int64_t i = (int64_t)c * CHUNK + lane * V;
        load(i, v);
#pragma unroll
        for (int j = 0; j < V; ++j) sum += f(v[j], i + j);
      }
      sum = wave_sum(sum);
      if (lane == 0) s.mass[g] = sum;
    }
    for (int g = count + threadIdx.x; g < kSegments; g += kThreads) s.mass[g] = 0;
    __syncthreads();
    u64 m = wave_sum(s.mass[2 * threadIdx.x] + s.mass[2 * threadIdx.x + 1]);
    if (lane == 0) s.part[wave] = m;
    __syncthreads();
    u64 total = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) total += s.part[w];
    __syncthreads();
    return total;
  }

  // The first id at which the running sum of f exceeds r, below the total that
  // `segments` gave for the same f. One wave's lanes return it.
  template <typename F>
  __device__ __forceinline__ int find(u64 r, F f) const {
    const int per = (chunks + kSegments - 1) / kSegments;
    // the segment, 64 at a time
    int g = 0;
    for (int at = 0; at < kSegments; at += 64) {
      const u64 m = wave_scan(s.mass[at + lane], lane);
      const u64 over = __ballot(m > r);
      if (over) {
        const int l = __builtin_ctzll(over);
        g = at + l;
        if (l) r -= __shfl(m, l - 1);
        break;
      }
      r -= __shfl(m, 63);
    }
    for (int c = g * per; c < chunks; ++c) {
      float v[V];
      u64 w[V], sum = 0;
      const int64_t i = (int64_t)c * CHUNK + lane * V;
      load(i, v);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        w[j] = f(v[j], i + j);
        sum += w[j];
      }
      const u64 m = wave_scan(sum, lane);
      const u64 over = __ballot(m > r);
      if (!over) {
        r -= __shfl(m, 63);
        continue;
      }
      const int l = __builtin_ctzll(over);
      u64 run = m - sum;
      int id = 0;
#pragma unroll
      for (int j = V - 1; j >= 0; --j) {
        u64 upto = run;
#pragma unroll
        for (int n = 0; n <= j; ++n) upto += w[n];
        if (upto > r) id = (int)(i + j);
      }
      return __shfl(id, l);
    }
    return vocab - 1;
  }
};

template <typename T>
__global__ void __launch_bounds__(kThreads) sample_kernel(newt_sample_params p, int shift) {
  __shared__ Shared s;
  const int64_t r = blockIdx.x;
  const int lane = threadIdx.x & 63, wave = wave_id();
  Row<T> row{(const T*)p.logits + r * p.stride, (int)p.vocab, 0, shift, lane, wave, s, 0, 0, 0};
  row.chunks = (int)((p.vocab + Row<T>::CHUNK - 1) / Row<T>::CHUNK);
  const float temperature = p.temperature ? p.temperature[r] : p.temperature_all;
  const float top_p = p.top_p ? p.top_p[r] : p.top_p_all;
  const float min_p = p.min_p ? p.min_p[r] : p.min_p_all;
  const int top_k = p.top_k ? p.top_k[r] : p.top_k_all;
  const float u = p.u[r];

  float top = -kInf;
  int bad = 0;
  row.each([&](float f) {
    top = __builtin_fmaxf(top, f);
    bad |= f != f;
  });
  top = newt::lane_reduce<newt::Max, 63>(top);
  bad = __ballot(bad) != 0;
  if (lane == 0) {
    s.top[wave] = top;
    s.bad[wave] = bad;
  }
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    top = __builtin_fmaxf(top, s.top[w]);
    bad |= s.bad[w];
  }
  __syncthreads();
  bad |= !(__builtin_fabsf(top) < kInf) | !(temperature >= 0.0f && temperature < kInf) |
         (u != u) | (top_p != top_p) | (min_p != min_p);
  if (bad) {
    if (threadIdx.x == 0) p.ids[r] = -1;
    return;
  }
  row.top = top;
  if (temperature == 0.0f || top_k == 1) {
    const auto is_top = [&](float f, int64_t) { return (u64)(f == top); };
    row.segments(is_top);
    if (wave == 0) {
      const int id = row.find(0, is_top);
      if (lane == 0) p.ids[r] = id;
    }
    return;
  }
  row.by = 1.0 / (double)temperature;
  // 64 bins to a factor e in weight, as far as weights reach, 46 ln 2
  row.bin_scale = (float)__builtin_fmin(64.0 * row.by, 1e30);

  u32 key = 0, keep = kNone, equal = kNone;
  if (top_k > 0 && top_k < p.vocab) {
    const auto l = row.last(false, (u32)top_k, 0.0);
    if (!l.all) {
      key = l.key;
      keep = l.keep;
      equal = l.equal;
    }
  }
  const auto equal_ones = [&](float f, int64_t) { return (u64)(key_of(f) == key); };
  int last_id = 0x7fffffff;  // of the logits of that key
  const auto find_last = [&] {
    if (keep >= equal) return;
    row.segments(equal_ones);
    if (wave == 0) {
      const int id = row.find(keep - 1, equal_ones);
      if (lane == 0) s.place = id;
    }
    __syncthreads();
    last_id = (int)s.place;
    __syncthreads();
  };
  const auto stays = [&](float f, int64_t i) {
    const u32 k = key_of(f);
    return (k > key) | ((k == key) & (i <= last_id));
  };
  if (top_p < 1.0f) {
    find_last();
    const u64 mass = row.segments(
        [&](float f, int64_t i) { return stays(f, i) ? row.weight(f) : (u64)0; });
    const double target = (double)top_p * (double)mass;
    // at least the first one
    const auto l = row.last(true, 0, target > 0.0 ? target : 0x1p-60);
    if (!l.all && (l.key > key || (l.key == key && l.keep < keep))) {
      key = l.key;
      keep = l.keep;
      equal = l.equal;
      last_id = 0x7fffffff;
      find_last();
    }
  } else {
    find_last();
  }
  // weights of at least min_p; the largest is 1
  const double least = __builtin_fmin((double)min_p, 1.0) * __builtin_ldexp(1.0, shift);
  const auto kept = [&](float f, int64_t i) {
    if (!stays(f, i)) return (u64)0;
    const u64 w = row.weight(f);
    return (double)w >= least ? w : (u64)0;
  };
  const u64 total = row.segments(kept);
  u64 pass = (u64)((double)__builtin_fmaxf(u, 0.0f) * (double)total);
  pass = pass < total ? pass : total - 1;
  if (wave == 0) {
    const int id = row.find(pass, kept);
    if (lane == 0) p.ids[r] = id;
  }
}

// A weight's bits behind the point: sums of `vocab` of them stay below 2^63.
int weight_bits(int64_t vocab) {
  int bits = 0;
  while (vocab >> bits) ++bits;
  return 62 - bits < 45 ? 62 - bits : 45;
}

const char* wrong(const newt_sample_params& p) {
  if (p.rows < 0 || p.rows > 0x7fffffff) return "bad number of rows";
  if (p.vocab <= 0 || p.vocab >= 1 << 30) return "a row has 1 to 2^30 - 1 logits";
  if (p.dtype != NEWT_F32 && p.dtype != NEWT_F16 && p.dtype != NEWT_BF16) return "unknown dtype";
  if (!p.temperature && !(p.temperature_all >= 0.0f && p.temperature_all < kInf))
    return "temperature has to be 0 or more and finite";
  if (!p.top_p && !(p.top_p_all >= 0.0f)) return "top_p has to be 0 or more";
  if (!p.min_p && !(p.min_p_all >= 0.0f && p.min_p_all <= 1.0f)) return "min_p lies in [0, 1]";
  return nullptr;
}

}  // namespace
}  // namespace newt_ops

extern "C" size_t newt_sample_workspace(int64_t, int64_t, int32_t) { return 0; }

extern "C" int newt_sample(const newt_sample_params* params, void* stream) {
  using namespace newt_ops;
  if (!params) return fail(NEWT_ERR_INVALID, "newt_sample: null params");
  const newt_sample_params& p = *params;
  if (const char* w = wrong(p)) return fail(NEWT_ERR_INVALID, "newt_sample: %s", w);
  if (p.rows == 0) return NEWT_OK;
  if (!p.logits || !p.u || !p.ids) return fail(NEWT_ERR_INVALID, "newt_sample: null tensor");
  hipStream_t s = static_cast<hipStream_t>(stream);
  const int shift = weight_bits(p.vocab);
  const auto go = [&](auto kernel) {
    return run("newt_sample", kernel, p.rows, kThreads, 0, s, p, shift);
  };
  switch (p.dtype) {
    case NEWT_F32: return go(sample_kernel<float>);
    case NEWT_F16: return go(sample_kernel<f16>);
    default: return go(sample_kernel<bf16>);
  }
}
