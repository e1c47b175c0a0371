// The next token of each row of logits: weights e^((x - max x) / T), kept by
// top_k, top_p and min_p, and the first id whose running kept weight exceeds u
// times their sum.
// What is kept is the beginning of the logits in falling order, of which only the
// part around its end is ever put in order: a histogram over (max - x) / T finds
// the bin in which the last kept one lies, and the few logits of that bin are
// sorted in LDS (or, with top_k, all up to it, where LDS holds them). Where a bin
// holds too many, finer histograms over the bits of its logits take its place. A
// token chosen by its running weight is found by sums of segments, of which one is
// read again.
// Weights are whole numbers of 2^-45 (less for more than 2^17 ids), from
// exponentials in 64 bits: their sums are exact, whatever the order in which
// atomics add them, so the same row gives the same id in every call, and a border is
// off by 2^-46 of the largest weight for each id before it.
#include "common.h"

namespace newt_ops {
namespace {

constexpr int kThreads = 1024, kWaves = kThreads / 64;
constexpr int kBins = 2048;
constexpr int kList = 4096;
constexpr float kInf = __builtin_inff();
constexpr u32 kNone = 0xffffffffu;

template <typename T> struct io { static constexpr int V = 16 / (int)sizeof(T); };

// Numbers in the order of the logits; -0 and 0 are equal.
__device__ __forceinline__ u32 key_of(float x) {
  const u32 b = newt::f32_bits(x + 0.0f);
  return b ^ ((u32)((int)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float of_key(u32 k) {
  return newt::bits_f32(k & 0x80000000u ? k ^ 0x80000000u : ~k);
}

// A token's place among all: the largest logit first, the lowest id among equal ones.
__device__ __forceinline__ u64 place_of(float x, u32 id) {
  return ((u64)~key_of(x) << 32) | id;
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
  double table[kBins];  // 2^shift e^(-i / 64)
  u64 mass[kBins];      // a histogram's masses, a search's segments
  u32 count[kBins];
  u64 list[kList];
  u64 part[kWaves];
  u32 part_count[kWaves];
  float top[kWaves];
  int bad[kWaves];
  u32 listed;
  u64 last;
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
  float top;   // the largest logit
  double by;   // 64 / T
  u64 least;   // the smallest weight that min_p keeps

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

  // e^(-i / 64), i = 0..2047, times 2^shift: i / 64 = n ln 2 + r, |r| <= ln 2 / 2;
  // the sum's first term left out is r^13 / 13!, 2^-53.
  __device__ __forceinline__ void fill_table() const {
    for (int i = threadIdx.x; i < kBins; i += kThreads) {
      const double y = i * -0.015625;
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
      s.table[i] = __builtin_ldexp(e, (int)n + shift);
    }
  }
  // (top - x) 64 / T = bin + rest, |rest| <= 1/2; in the last bin weights are 0. Bins
  // fall with the logit.
  struct Point {
    double rest;
    int bin;
  };
  __device__ __forceinline__ Point point(float f) const {
    const double t = __builtin_fmin(((double)top - (double)f) * by, (double)(kBins - 1));
    const double whole = t + 6755399441055744.0;  // 1.5 2^52: the low bits are the bin
    return {t - (whole - 6755399441055744.0), (int)__builtin_bit_cast(u64, whole)};
  }
  // The weight as a whole number: e^(-rest / 64), whose first term left out is
  // (1 / 128)^6 / 6!, 2^-51, times the table's, rounded by 2^52 more.
  __device__ __forceinline__ u64 weight(const Point& a) const {
    double e = -7.76102145512898763e-12;  // -1 / 64^5 / 5!
    e = __builtin_fma(e, a.rest, 2.48352686564127604e-9);
    e = __builtin_fma(e, a.rest, -6.35782877604166667e-7);
    e = __builtin_fma(e, a.rest, 1.220703125e-4);
    e = __builtin_fma(e, a.rest, -0.015625);
    e = __builtin_fma(e, a.rest, 1.0);
    const double whole = __builtin_fma(e, s.table[a.bin], 4503599627370496.0);
    return __builtin_bit_cast(u64, whole) & 0xfffffffffffffull;
  }
  __device__ __forceinline__ u64 weight(float f) const { return weight(point(f)); }

  // f(number, id) for each of the row, in no order, and done(chunk) behind each
  // chunk: a wave loads four chunks, then works on them.
  template <typename F, typename D>
  __device__ __forceinline__ void each(F f, D done) const {
    constexpr int AHEAD = 4;
    const int whole = vocab / CHUNK;
    for (int c = wave; c < whole; c += kWaves * AHEAD) {
      T t[AHEAD][V];
#pragma unroll
      for (int a = 0; a < AHEAD; ++a) {
        const int at = c + a * kWaves < whole ? c + a * kWaves : whole - 1;
        newt::load_vec<T, V>(x + (int64_t)at * CHUNK + lane * V, t[a], newt::any_align());
      }
#pragma unroll
      for (int a = 0; a < AHEAD; ++a) {
        if (c + a * kWaves >= whole) break;
        const int64_t i = (int64_t)(c + a * kWaves) * CHUNK + lane * V;
#pragma unroll
        for (int j = 0; j < V; ++j) f(newt::to_f32(t[a][j]), i + j);
        done(c + a * kWaves);
      }
    }
    if (whole < chunks && whole % kWaves == wave) {
      float v[V];
      const int64_t i = (int64_t)whole * CHUNK + lane * V;
      load(i, v);
#pragma unroll
      for (int j = 0; j < V; ++j) f(v[j], i + j);
      done(whole);
    }
  }
  template <typename F>
  __device__ __forceinline__ void each(F f) const {
    each(f, [](int) {});
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
      if (!reached(mb0, cb0)) found(i, mb0, cb0, m0, c0);
    } else if (reached(mb1 + m1, c)) {
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

  // The mass of all bins.
  __device__ __forceinline__ u64 total() const {
    const u64 m = newt::lane_reduce<newt::Sum, 63>(s.mass[2 * threadIdx.x] + s.mass[2 * threadIdx.x + 1]);
    if (lane == 0) s.part[wave] = m;
    __syncthreads();
    u64 sum = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) sum += s.part[w];
    __syncthreads();
    return sum;
  }

  // The list's first `size`, a power of two, in rising order.
  __device__ __forceinline__ void sort(int size) const {
    for (int k = 2; k <= size; k <<= 1)
      for (int j = k >> 1; j > 0; j >>= 1) {
        __syncthreads();
        for (int i = threadIdx.x; i < size / 2; i += kThreads) {
          const int a = 2 * i - (i & (j - 1)), b = a + j;
          const u64 u = s.list[a], v = s.list[b];
          if ((u > v) == ((a & k) == 0)) {
            s.list[a] = v;
            s.list[b] = u;
          }
        }
      }
    __syncthreads();
  }
  // Rounds the list up to a power of two with entries behind all others.
  __device__ __forceinline__ int fill_up(int n) const {
    int size = 64;
    while (size < n) size <<= 1;
    for (int i = n + threadIdx.x; i < size; i += kThreads) s.list[i] = ~0ull;
    return size;
  }
  // Sums of w over the list's entries before this thread's first, 4 neighbouring
  // ones a thread.
  __device__ __forceinline__ u64 scan(const u64 (&w)[4], u64* sum) const {
    const u64 own = w[0] + w[1] + w[2] + w[3];
    u64 m = wave_scan(own, lane);
    if (lane == 63) s.part[wave] = m;
    __syncthreads();
    u64 all = 0;
#pragma unroll
    for (int i = 0; i < kWaves; ++i) {
      if (i == wave) m += all;
      all += s.part[i];
    }
    __syncthreads();
    *sum = all;
    return m - own;
  }
  __device__ __forceinline__ void append(u64 entry) const {
    const u32 i = atomicAdd(&s.listed, 1u);
    if (i < kList) s.list[i] = entry;
  }
  __device__ __forceinline__ u64 listed_weight(int i, int n) const {
    return i < n ? weight(of_key(~(u32)(s.list[i] >> 32))) : 0;
  }

  // The sums of f(number, id), in segments of consecutive chunks that `find`
  // searches; their sum is `total`.
  template <typename F>
  __device__ __forceinline__ void segments(F f) const {
    const int per = (chunks + kBins - 1) / kBins;
    for (int g = threadIdx.x; g < kBins; g += kThreads) s.mass[g] = 0;
    __syncthreads();
    u64 sum = 0;
    each([&](float v, int64_t i) { sum += f(v, i); }, [&](int c) {
      sum = newt::lane_reduce<newt::Sum, 63>(sum);
      if (per == 1) s.mass[c] = sum;
      else if (lane == 0) atomicAdd(&s.mass[c / per], sum);
      sum = 0;
    });
    __syncthreads();
  }
  __device__ __forceinline__ int segment_of(int64_t id) const {
    return (int)(id / CHUNK) / ((chunks + kBins - 1) / kBins);
  }

  // The first id at which the running sum of f exceeds r, below the total of the
  // segments. One wave's lanes return it.
  template <typename F>
  __device__ __forceinline__ int find(u64 r, F f) const {
    const int per = (chunks + kBins - 1) / kBins;
    // the segment, 64 at a time
    int g = 0;
    for (int at = 0; at < kBins; at += 64) {
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
      bool done = false;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        run += w[j];
        if (!done && run > r) {
          id = (int)(i + j);
          done = true;
        }
      }
      return __shfl(id, l);
    }
    return vocab - 1;
  }

  // The place of the last token that stays, by count or by mass, where a bin holds
  // more than the list: histograms over the keys of the bin, finer and finer, then
  // a search by id. ~0: all stay.
  __device__ __forceinline__ u64 last(bool by_mass, u32 k, double target) const {
    clear();
    each([&](float f, int64_t) {
      const Point a = point(f);
      if (a.bin < kBins - 1) {
        atomicAdd(&s.count[a.bin], 1u);
        atomicAdd(&s.mass[a.bin], weight(a));
      }
    });
    __syncthreads();
    pick(by_mass, k, 0, target);
    if (s.place == kNone) return ~0ull;  // among weights of 0, or everything
    // the keys of that bin: all at first, then those of a finer histogram's bin
    const int at = s.place;
    u64 before = s.before;
    u32 before_count = s.before_count;
    u32 lo = 0, hi = 0xffffffffu;
    bool first = true;
    for (;;) {
      // the smallest and largest key that are there
      u32 least_key = 0xffffffffu, most = 0;
      each([&](float f, int64_t) {
        const u32 key = key_of(f);
        if (first ? point(f).bin == at : (key >= lo) & (key <= hi)) {
          least_key = key < least_key ? key : least_key;
          most = key > most ? key : most;
        }
      });
      clear();
      if (threadIdx.x == 0) {
        s.count[0] = 0xffffffffu;
        s.count[1] = 0;
      }
      __syncthreads();
      if (least_key <= most) {
        atomicMin(&s.count[0], least_key);
        atomicMax(&s.count[1], most);
      }
      __syncthreads();
      lo = s.count[0];
      hi = s.count[1];
      __syncthreads();
      clear();
      const u32 range = hi - lo;
      const int bits = range < kBins ? 0 : 21 - __builtin_clz(range);  // range >> bits < kBins
      each([&](float f, int64_t) {
        const u32 key = key_of(f);
        if ((key >= lo) & (key <= hi)) {
          const u32 b = (hi - key) >> bits;
          atomicAdd(&s.count[b], 1u);
          atomicAdd(&s.mass[b], weight(f));
        }
      });
      __syncthreads();
      pick(by_mass, k - before_count, before, target);
      before = s.before;
      before_count += s.before_count;
      const u32 top_key = hi - (s.place << bits);
      if (bits == 0) {
        const u32 equal = s.place_count;
        u32 keep;
        if (by_mass) {
          // those before which less than the target lies
          const double n = __builtin_ceil((target - (double)before) /
                                          ((double)s.place_mass / (double)equal));
          keep = n >= (double)equal ? equal : n < 1.0 ? 1 : (u32)n;
        } else {
          keep = k - before_count;
        }
        __syncthreads();
        if (keep >= equal) return ((u64)~top_key << 32) | 0xffffffffu;
        const auto equal_ones = [&](float f, int64_t) { return (u64)(key_of(f) == top_key); };
        segments(equal_ones);
        if (wave == 0) {
          const int id = find(keep - 1, equal_ones);
          if (lane == 0) s.place = id;
        }
        __syncthreads();
        const u32 id = s.place;
        __syncthreads();
        return ((u64)~top_key << 32) | id;
      }
      const u32 width = (1u << bits) - 1;
      hi = top_key;
      lo = hi - lo > width ? hi - width : lo;
      first = false;
      __syncthreads();
    }
  }

  __device__ __forceinline__ u64 kept_weight(float f, int64_t i, u64 cut) const {
    if (place_of(f, (u32)i) > cut) return 0;
    const u64 w = weight(f);
    return w >= least ? w : 0;
  }
  // A number below `sum`, u of it.
  __device__ __forceinline__ static u64 share(float u, u64 sum) {
    const u64 r = (u64)((double)__builtin_fmaxf(u, 0.0f) * (double)sum);
    return r < sum ? r : sum - 1;
  }

  // The choice among tokens up to the place `cut`, whose weights the segments
  // hold. One wave's lanes return it.
  __device__ __forceinline__ int choose(float u, u64 cut) const {
    const u64 sum = total();
    if (wave != 0) return 0;
    return find(share(u, sum), [&](float f, int64_t i) { return kept_weight(f, i, cut); });
  }

  // The choice where the list holds all tokens that top_k may keep.
  __device__ __forceinline__ int choose_listed(int n, u32 k, float top_p, float u) const {
    const int size = fill_up(n);
    sort(size);
    const int i = 4 * threadIdx.x;
    u64 w[4], of_k[4], sum, mass;
    u32 id[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      w[j] = listed_weight(i + j, n);
      of_k[j] = i + j < k ? w[j] : 0;
      id[j] = i + j < n ? (u32)s.list[i + j] : 0;
    }
    u64 before = scan(of_k, &mass);
    const double target = (double)top_p * (double)mass;
    u64 entry[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const bool stays = (i + j < k) & ((i + j == 0) | (top_p >= 1.0f) | ((double)before < target)) &
                         (w[j] >= least);
      before += of_k[j];
      // by id, with what finds the weight again
      entry[j] = stays && i + j < n ? ((u64)id[j] << 32) | (u32)(s.list[i + j] >> 32) : ~0ull;
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (i + j < size) s.list[i + j] = entry[j];
    sort(size);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const u64 e = i + j < size ? s.list[i + j] : ~0ull;
      w[j] = e != ~0ull ? weight(of_key(~(u32)e)) : 0;
    }
    u64 run = scan(w, &sum);
    const u64 r = share(u, sum);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (run <= r && run + w[j] > r) s.place = (u32)(s.list[i + j] >> 32);
      run += w[j];
    }
    __syncthreads();
    return (int)s.place;
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
  row.each([&](float f, int64_t) {
    top = __builtin_fmaxf(top, f);
    bad |= f != f;
  });
  top = newt::lane_reduce<newt::Max, 63>(top);
  bad = __ballot(bad) != 0;
  if (lane == 0) {
    s.top[wave] = top;
    s.bad[wave] = bad;
  }
  if (threadIdx.x == 0) s.listed = s.last = 0;
  row.fill_table();
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    top = __builtin_fmaxf(top, s.top[w]);
    bad |= s.bad[w];
  }
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
  row.by = 64.0 / (double)temperature;
  // the largest weight is 2^shift
  row.least = (u64)__builtin_ceil(
      __builtin_fmin(__builtin_fmax((double)min_p, 0.0), 1.0) * __builtin_ldexp(1.0, shift));

  const bool by_count = top_k > 0 && top_k < p.vocab, by_mass = top_p < 1.0f;
  u64 cut = ~0ull;
  if (!by_count && !by_mass) {
    row.segments([&](float f, int64_t i) { return row.kept_weight(f, i, cut); });
    const int id = row.choose(u, cut);
    if (threadIdx.x == 0) p.ids[r] = id;
    return;
  }
  row.clear();
  if (by_count) {
    row.each([&](float f, int64_t) {
      const int b = row.point(f).bin;
      if (b < kBins - 1) atomicAdd(&s.count[b], 1u);
    });
  } else {
    row.each([&](float f, int64_t) {
      const auto a = row.point(f);
      if (a.bin < kBins - 1) atomicAdd(&s.mass[a.bin], row.weight(a));
    });
  }
  __syncthreads();
  // at least the first token
  const double target = by_count ? 0.0
      : __builtin_fmax((double)top_p * (double)row.total(), 0x1p-60);
  row.pick(!by_count, (u64)top_k, 0, target);
  int bin = s.place == kNone ? kBins : (int)s.place;
  const u64 before = s.before;
  const u32 before_count = s.before_count, of_bin = s.place_count;
  if (by_count && bin < kBins && before_count + of_bin <= kList) {
    row.each([&](float f, int64_t i) {
      if (row.point(f).bin <= bin) row.append(place_of(f, (u32)i));
    });
    __syncthreads();
    const int id = row.choose_listed((int)s.listed, (u32)top_k, top_p, u);
    if (threadIdx.x == 0) p.ids[r] = id;
    return;
  }
  bool listed = !(by_count && by_mass) && !(by_count && of_bin > kList);
  if (listed) {
    // what lies before the bin counts at once, what is in it when it is in order
    __syncthreads();
    row.segments([&](float f, int64_t i) -> u64 {
      const auto a = row.point(f);
      if (a.bin < bin) {
        const u64 w = row.weight(a);
        return w >= row.least ? w : 0;
      }
      if (a.bin == bin) row.append(place_of(f, (u32)i));
      return 0;
    });
    listed = s.listed <= kList;
  }
  if (listed) {
    const int n = (int)s.listed;
    if (n) {
      row.sort(row.fill_up(n));
      const int i = 4 * threadIdx.x;
      u64 w[4], sum;
#pragma unroll
      for (int j = 0; j < 4; ++j) w[j] = row.listed_weight(i + j, n);
      u64 run = before + row.scan(w, &sum);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (i + j < n && (by_count ? before_count + i + j < (u32)top_k : (double)run < target)) {
          const u64 entry = s.list[i + j];
          if (w[j] >= row.least) atomicAdd(&s.mass[row.segment_of((u32)entry)], w[j]);
          atomicMax(&s.last, entry);
        }
        run += w[j];
      }
      __syncthreads();
      cut = s.last;
    }
  } else {
    __syncthreads();
    if (by_count) cut = row.last(false, (u32)top_k, 0.0);
    if (by_mass) {
      double mass_target = target;
      if (by_count) {
        row.segments([&](float f, int64_t i) {
          return place_of(f, (u32)i) <= cut ? row.weight(f) : (u64)0;
        });
        mass_target = __builtin_fmax((double)top_p * (double)row.total(), 0x1p-60);
      }
      const u64 by_p = row.last(true, 0, mass_target);
      cut = by_p < cut ? by_p : cut;
    }
    row.segments([&](float f, int64_t i) { return row.kept_weight(f, i, cut); });
  }
  const int id = row.choose(u, cut);
  if (threadIdx.x == 0) p.ids[r] = id;
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
