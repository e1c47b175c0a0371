// The next token of each row of logits: weights e^((x - max x) / T), kept by
// top_k, top_p and min_p, and the first id whose running kept weight exceeds u
// times their sum.
// What is kept is the beginning of the logits in falling order, of which only the
// part around its end is ever put in order: a histogram over (max - x) / T finds
// the bin in which the last kept one lies, and the few logits of that bin are
// sorted in LDS (or, with top_k, all up to it, where LDS holds them). A token chosen
// by its running weight is found by sums of segments, of which one is read again.
// Three kinds of rows go another way (kSlow), over finer and finer histograms of the
// bits of the logits, in one program and without haste:
//   - the bin of the end holds more than a list (all equal, or a huge temperature);
//   - top_k together with top_p, and more than a list up to top_k's end;
//   - top_k together with top_p, and fewer than top_k tokens within 32 temperatures
//     of the largest logit: masked rows, or low temperatures.
// The third is the commonest: by top_k 50 and top_p 0.9 at temperatures of 0.75 / 0.2 /
// 0.05 1 x 128000 bf16 takes 26 / 71 / 160 us, 64 x 32000 fp32 18 / 52 / 53, 256 x 100003
// bf16 38 / 155 / 247. At 0.75 with a top_k of 5000 it is 269, 103 and 389, at 50 by top_p
// alone 405, 58 and 457.
// Long rows are bound by the vector unit, which issues in 64% of the cycles, and by
// LDS: an exponential in 64 bits takes a dozen fp64 instructions (by a table of 2048
// and a polynomial of degree 4), and top_p needs two of them a logit; the histogram's
// 64-bit atomics make two thirds of the LDS' active cycles bank conflicts. bf16 256 x
// 100003 by top_p: 54 us, without a filter 31, greedy, which reads a row twice, 20; 64 x
// 32000 fp32 with settings of each row's own 22, greedy 6; 1 x 128000 with all three
// filters 27, in four kernels of 3 + 5 + 8 + 12 us, each a chain of short steps, greedy
// 11.
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
constexpr int kMostParts = 64;
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

// v of the lane that a DPP control names, 0 where there is none.
template <int CTRL, int ROWS, typename V>
__device__ __forceinline__ V lane_from(V v) {
  if constexpr (sizeof(V) == 4) {
    return (V)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xF, false);
  } else {
    const u32 lo = lane_from<CTRL, ROWS>((u32)v), hi = lane_from<CTRL, ROWS>((u32)(v >> 32));
    return ((V)hi << 32) | lo;
  }
}

// The sum over this lane and those below it: in rows of 16 lanes, then row by row.
template <typename V>
__device__ __forceinline__ V wave_scan(V v) {
  v += lane_from<0x111, 0xF>(v);  // row_shr:1
  v += lane_from<0x112, 0xF>(v);
  v += lane_from<0x114, 0xF>(v);
  v += lane_from<0x118, 0xF>(v);
  v += lane_from<0x142, 0xA>(v);  // row_bcast:15, to rows 1 and 3
  v += lane_from<0x143, 0xC>(v);  // row_bcast:31, to rows 2 and 3
  return v;
}

__device__ __forceinline__ u64 of_lane(u64 v, int lane) {
  return ((u64)(u32)__builtin_amdgcn_readlane((int)(v >> 32), lane) << 32) |
         (u32)__builtin_amdgcn_readlane((int)(u32)v, lane);
}
__device__ __forceinline__ u32 of_lane(u32 v, int lane) {
  return (u32)__builtin_amdgcn_readlane((int)v, lane);
}

// What the waves' parts, one each, are in all and before this wave's.
template <typename V>
struct Offset {
  V all, before;
  __device__ __forceinline__ Offset(const V* part, int lane, int wave) {
    const V v = wave_scan(lane < kWaves ? part[lane] : (V)0);
    all = of_lane(v, kWaves - 1);
    before = wave ? of_lane(v, wave - 1) : (V)0;
  }
};

struct Shared {
  double table[kBins];  // 2^shift e^(-i / 64)
  u64 mass[kBins];      // a histogram's masses, a search's segments
  u32 count[kBins];
  __attribute__((aligned(16))) u64 list[kList];  // places of tokens
  __attribute__((aligned(16))) u64 some[kList];  // those of one bin
  u64 part[kWaves];
  u32 part_count[kWaves];
  float top[kWaves];
  int bad[kWaves];
  u32 listed, picked, first;
  u64 last;
  double edge;  // the table's entry of the bin at the end
  // what a search found
  u64 before;
  u32 before_count, place, place_count;
  u64 place_mass;
};

// A row's settings.
struct Settings {
  float temperature, top_p, min_p, u;
  u32 top_k;
  bool bad, greedy, by_count, by_mass;
  __device__ __forceinline__ Settings(const newt_sample_params& p, int64_t r)
      : temperature(p.temperature ? p.temperature[r] : p.temperature_all),
        top_p(p.top_p ? p.top_p[r] : p.top_p_all),
        min_p(p.min_p ? p.min_p[r] : p.min_p_all), u(p.u[r]) {
    const int k = p.top_k ? p.top_k[r] : p.top_k_all;
    top_k = (u32)k;
    bad = !(temperature >= 0.0f && temperature < kInf) | (u != u) | (top_p != top_p) |
          (min_p != min_p);
    greedy = (temperature == 0.0f) | (k == 1);
    by_count = (k > 0) & (k < p.vocab);
    by_mass = top_p < 1.0f;
  }
};

// What is read of a row behind the histogram, and how the kept ones are found.
enum Mode { kSums, kListed, kSlow };

template <typename T>
struct Row {
  static constexpr int V = io<T>::V;
  static constexpr int CHUNK = 64 * V;  // of a wave
  const T* x;
  int vocab, chunks, shift;
  int from, to;  // the chunks that are this program's
  int lane, wave;
  Shared& s;
  float top;     // the largest logit
  double by;     // 64 / T
  double most;   // of max - x: the last bin
  double reach;  // 64 ln(1 / min_p): of (max - x) 64 / T

  __device__ __forceinline__ Row(const newt_sample_params& p, Shared& s_, int64_t r, int shift_)
      : x((const T*)p.logits + r * p.stride), vocab((int)p.vocab),
        chunks((int)((p.vocab + CHUNK - 1) / CHUNK)), shift(shift_), from(0), to(chunks),
        lane(threadIdx.x & 63), wave(wave_id()), s(s_) {}
  __device__ __forceinline__ void set(const Settings& o, float top_) {
    top = top_;
    by = 64.0 / (double)o.temperature;
    most = (kBins - 1) / by;
    // 2^-46 less of a weight, as little as it is rounded by, still reaches min_p
    reach = o.min_p > 0.0f ? 0x1p-40 - 64.0 * log((double)__builtin_fminf(o.min_p, 1.0f)) : 1e300;
  }

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
    __device__ __forceinline__ bool within(double reach) const { return rest + bin <= reach; }
  };
  __device__ __forceinline__ Point point(float f) const {
    const double d = __builtin_fmin((double)top - (double)f, most);
    // 1.5 2^52 more: the low bits are the bin
    const double whole = __builtin_fma(d, by, 6755399441055744.0);
    return {__builtin_fma(d, by, 6755399441055744.0 - whole), (int)__builtin_bit_cast(u64, whole)};
  }
  // e^(-rest / 64), off by 2^-45 of it, times the table's entry, rounded to a whole
  // number by 2^52 more: its low 52 bits.
  __device__ __forceinline__ static u64 weight_bits(double rest, double entry) {
    double e = 2.483531912468741e-09;
    e = __builtin_fma(e, rest, -6.357848178607495e-07);
    e = __builtin_fma(e, rest, 1.2207031249984305e-04);
    e = __builtin_fma(e, rest, -0.015624999999939368);
    e = __builtin_fma(e, rest, 1.0);
    return __builtin_bit_cast(u64, __builtin_fma(e, entry, 4503599627370496.0));
  }
  static constexpr u64 kWhole = 0x4330000000000000ull;  // the bits of 2^52
  __device__ __forceinline__ u64 weight(const Point& a) const {
    return weight_bits(a.rest, s.table[a.bin]) & 0xfffffffffffffull;
  }
  __device__ __forceinline__ u64 weight(float f) const { return weight(point(f)); }

  // f(number, id) for each of the row, in no order, and done(chunk) behind each
  // chunk: a wave loads four chunks, then works on them.
  template <typename F, typename D>
  __device__ __forceinline__ void each(F f, D done) const {
    constexpr int AHEAD = 4;
    const int whole = to < vocab / CHUNK ? to : vocab / CHUNK;
    for (int c = from + wave; c < whole; c += kWaves * AHEAD) {
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
    if (from <= whole && whole < to && wave == kWaves - 1) {
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

  // The same a number at a time, where there is no hurry.
  template <typename F>
  __device__ __forceinline__ void slowly(F f) const {
#pragma unroll 1
    for (int i = threadIdx.x; i < vocab; i += kThreads) f(newt::to_f32(x[i]), i);
  }

  __device__ __forceinline__ void clear() const {
    for (int i = threadIdx.x; i < kBins; i += kThreads) {
      s.mass[i] = 0;
      s.count[i] = 0;
    }
    __syncthreads();
  }

  // Of the histogram's bins the first where the running count reaches `k` or the
  // running mass, with `before`, reaches `target` (below 0: top_p of all there is);
  // its place, what lies before it and what is in it to s. All threads call it; the
  // bins are full. Returns the target.
  __device__ __forceinline__ double pick(bool by_mass, u64 k, u64 before, double target,
                                         float top_p = 0.0f) const {
    const int i = threadIdx.x * 2;
    const u64 m0 = s.mass[i], m1 = s.mass[i + 1];
    const u32 c0 = s.count[i], c1 = s.count[i + 1];
    u64 m = wave_scan(m0 + m1);
    u32 c = wave_scan(c0 + c1);
    if (lane == 63) {
      s.part[wave] = m;
      s.part_count[wave] = c;
    }
    if (threadIdx.x == 0) s.place = kNone;
    __syncthreads();
    const Offset<u64> masses(s.part, lane, wave);
    const u64 all = masses.all;
    m += masses.before;
    c += Offset<u32>(s.part_count, lane, wave).before;
    // at least the first token
    if (target < 0.0) target = __builtin_fmax((double)top_p * (double)all, 0x1p-60);
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
    return target;
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
    const u64 m =
        newt::lane_reduce<newt::Sum, 63>(s.mass[2 * threadIdx.x] + s.mass[2 * threadIdx.x + 1]);
    if (lane == 0) s.part[wave] = m;
    __syncthreads();
    const u64 sum = Offset<u64>(s.part, lane, wave).all;
    __syncthreads();
    return sum;
  }

  // The first n of `some` in rising order: by counting for few, else bitonic.
  __device__ __forceinline__ void order(int n) const {
    if (n <= 256) {
      const int i = threadIdx.x;
      if (i < 8) s.some[n + i] = ~0ull;
      __syncthreads();
      u64 own = 0;
      int rank = 0;
      if (i < n) {
        own = s.some[i];
        for (int j = 0; j < n; j += 8) {
          u64 other[8];
#pragma unroll
          for (int k = 0; k < 8; ++k) other[k] = s.some[j + k];
#pragma unroll
          for (int k = 0; k < 8; ++k) rank += other[k] < own;
        }
      }
      __syncthreads();
      if (i < n) s.some[rank] = own;
      __syncthreads();
      return;
    }
    int size = 512;
    while (size < n) size <<= 1;
    for (int i = n + threadIdx.x; i < size; i += kThreads) s.some[i] = ~0ull;
    // pairs up to 64 apart are a wave's own, in order without a barrier
    bool wide = true;
    for (int k = 2; k <= size; k <<= 1)
      for (int j = k >> 1; j > 0; j >>= 1) {
        if (wide || j > 64) __syncthreads();
        else __builtin_amdgcn_wave_barrier();
        wide = j > 64;
        for (int i = threadIdx.x; i < size / 2; i += kThreads) {
          const int a = 2 * i - (i & (j - 1)), b = a + j;
          const u64 u = s.some[a], v = s.some[b];
          if ((u > v) == ((a & k) == 0)) {
            s.some[a] = v;
            s.some[b] = u;
          }
        }
      }
    __syncthreads();
  }
  __device__ __forceinline__ static float logit_of(u64 place) {
    return of_key(~(u32)(place >> 32));
  }
  __device__ __forceinline__ void append(u64 place) const {
    const u32 i = atomicAdd(&s.listed, 1u);
    if (i < kList) s.list[i] = place;
  }
  // Moves the list's entries for which f(place) holds to `some`, and counts them.
  template <typename F>
  __device__ __forceinline__ int take(int n, F f) const {
    if (threadIdx.x == 0) s.picked = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += kThreads) {
      const u64 place = s.list[i];
      if (f(place)) s.some[atomicAdd(&s.picked, 1u)] = place;
    }
    __syncthreads();
    return (int)s.picked;
  }
  // The last of `some`, n in order, before which less than the target lies, with
  // `before`, less than it, in front of them all. All have the table entry `entry`.
  __device__ __forceinline__ u64 last_by_mass(int n, u64 before, double target,
                                              double entry) const {
    const int i = 4 * threadIdx.x;
    u64 w[4], own = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      w[j] = i + j < n ? weight_bits(point(logit_of(s.some[i + j])).rest, entry) - kWhole : 0;
      own += w[j];
    }
    u64 run = wave_scan(own);
    if (lane == 63) s.part[wave] = run;
    __syncthreads();
    run += before - own + Offset<u64>(s.part, lane, wave).before;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const u64 next = run + w[j];
      if (i + j < n && (double)run < target && (i + j + 1 == n || !((double)next < target)))
        s.last = s.some[i + j];
      run = next;
    }
    __syncthreads();
    return s.last;
  }

  // The sums of f(number, id), slowly, in segments of consecutive chunks that `find`
  // searches; their sum is `total`.
  template <typename F>
  __device__ __forceinline__ void segments(F f) const {
    clear();
    slowly([&](float v, int64_t i) {
      const u64 w = f(v, i);
      if (w) atomicAdd(&s.mass[segment_of(i)], w);
    });
    __syncthreads();
  }
  __device__ __forceinline__ int segment_of(int64_t id) const {
    return (int)(id / CHUNK) / ((chunks + kBins - 1) / kBins);
  }

  // The first id at which the running sum of f over the row exceeds `share` of the
  // segments' sum, which hold the sums of f. All threads call it; the first wave's
  // get the id.
  template <typename S, typename F>
  __device__ __forceinline__ int find(S share, F f) const {
    const int per = (chunks + kBins - 1) / kBins;
    const u64 m0 = s.mass[2 * threadIdx.x], m1 = s.mass[2 * threadIdx.x + 1];
    u64 m = wave_scan(m0 + m1);
    if (lane == 63) s.part[wave] = m;
    __syncthreads();
    const Offset<u64> sums_of(s.part, lane, wave);
    m += sums_of.before;
    u64 r = share(sums_of.all);
    // the segment in which r lies, and what is left of it there
    const u64 b1 = m - m1, b0 = b1 - m0;
    if (b0 <= r && r < m) {
      s.place = 2 * threadIdx.x + (r >= b1);
      s.before = r - (r >= b1 ? b1 : b0);
    }
    __syncthreads();
    if (wave != 0) return 0;
    const int g = (int)s.place;
    r = s.before;
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
      const u64 upto = wave_scan(sum);
      const u64 over = __ballot(upto > r);
      if (!over) {
        r -= __shfl(upto, 63);
        continue;
      }
      const int l = __builtin_ctzll(over);
      u64 run = upto - sum;
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
    slowly([&](float f, int64_t) {
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
      slowly([&](float f, int64_t) {
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
      slowly([&](float f, int64_t) {
        const u32 key = key_of(f);
        if ((key >= lo) & (key <= hi)) {
          const u32 b = (hi - key) >> bits;
          atomicAdd(&s.count[b], 1u);
          atomicAdd(&s.mass[b], weight(f));
        }
      });
      __syncthreads();
      pick(by_mass, k - before_count, before, target);
      if (s.place == kNone) return ~0ull;  // never: the bin holds the end
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
        const int first = find([&](u64) { return (u64)keep - 1; }, equal_ones);
        __syncthreads();
        if (threadIdx.x == 0) s.place = first;
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

  // A number below `sum`, u of it.
  __device__ __forceinline__ static u64 share(float u, u64 sum) {
    const u64 r = (u64)((double)__builtin_fmaxf(u, 0.0f) * (double)sum);
    return r < sum ? r : sum - 1;
  }

  // The steps, each of all threads of a program, with a barrier at their ends.

  // The largest logit, and whether one is a NaN.
  __device__ __forceinline__ float largest(bool& bad) const {
    float most = -kInf;
    bool nan = false;
    each([&](float f, int64_t) {
      most = __builtin_fmaxf(most, f);
      nan |= f != f;
    });
    most = newt::lane_reduce<newt::Max, 63>(most);
    nan = __ballot(nan) != 0;
    if (lane == 0) {
      s.top[wave] = most;
      s.bad[wave] = nan;
    }
    if (threadIdx.x == 0) {
      s.listed = 0;
      s.first = 0xffffffffu;
    }
    __syncthreads();
    bad = __ballot(lane < kWaves && s.bad[lane]) != 0;
    return newt::lane_reduce<newt::Max, 63>(lane < kWaves ? s.top[lane] : -kInf);
  }

  // Bins' counts, for top_k, or masses, for top_p alone.
  __device__ __forceinline__ void histogram(const Settings& o) const {
    clear();
    if (o.by_count) {
      each([&](float f, int64_t) {
        const int b = point(f).bin;
        if (b < kBins - 1) atomicAdd(&s.count[b], 1u);
      });
    } else {
      each([&](float f, int64_t) {
        const Point a = point(f);
        if (a.bin < kBins - 1) atomicAdd(&s.mass[a.bin], weight(a));
      });
    }
    __syncthreads();
  }

  // What the histogram says of the end of what is kept.
  struct End {
    Mode mode;
    int bin;           // with the last one that top_k and top_p keep (kBins: no such bin)
    int edge;          // kSums: bins before it are kept, those behind it not
    u64 before;
    u32 before_count;
    double target;     // the mass at which top_p ends
  };
  __device__ __forceinline__ End end(const Settings& o) const {
    End e = {kSums, kBins, kBins, 0, 0, 0.0};
    if (o.by_count | o.by_mass) {
      e.target = pick(!o.by_count, o.top_k, 0, -1.0, o.top_p);
      if (s.place != kNone) {
        e.bin = s.place;
        e.before = s.before;
        e.before_count = s.before_count;
        const u32 upto = s.before_count + s.place_count;
        if (o.by_count && upto <= kList) e.mode = kListed;
        else if (o.by_count && (o.by_mass || s.place_count > kList)) e.mode = kSlow;
      } else if (o.by_count && o.by_mass) {
        e.mode = kSlow;
      }
      __syncthreads();
    }
    // bins fall with the logit: what lies before the bin of `reach` is within it
    const int of_min = reach < kBins - 1.5 ? (int)__builtin_rint(reach) : kBins;
    e.edge = e.bin < of_min ? e.bin : of_min;
    return e;
  }

  // Segments' sums of what is certainly kept, and the list of what may be.
  __device__ __forceinline__ void sums(const End& e) const {
    // weights from the edge on come out as 0
    if (threadIdx.x == 0 && e.edge < kBins) s.edge = s.table[e.edge];
    __syncthreads();
    for (int i = e.edge + threadIdx.x; i < kBins; i += kThreads) s.table[i] = 0.0;
    for (int g = threadIdx.x; g < kBins; g += kThreads) s.mass[g] = 0;
    __syncthreads();
    const int per = (chunks + kBins - 1) / kBins;
    u64 sum = 0;
    each([&](float f, int64_t i) {
      const Point a = point(f);
      sum += weight_bits(a.rest, s.table[a.bin]);
      if (a.bin == e.edge) append(place_of(f, (u32)i));
    }, [&](int c) {
      sum = newt::lane_reduce<newt::Sum, 63>(sum - V * kWhole);
      if (per == 1) s.mass[c] = sum;
      else if (lane == 0) atomicAdd(&s.mass[c / per], sum);
      sum = 0;
    });
    __syncthreads();
  }
  // The list of all that top_k may keep.
  __device__ __forceinline__ void candidates(const End& e) const {
    each([&](float f, int64_t i) {
      if (point(f).bin <= e.bin) append(place_of(f, (u32)i));
    });
    __syncthreads();
  }
  // The first id of the largest logit.
  __device__ __forceinline__ void first() const {
    each([&](float f, int64_t i) {
      if (f == top) atomicMin(&s.first, (u32)i);
    });
    __syncthreads();
  }

  // The choice among what the segments hold: of the bins before `edge` all, of that
  // bin places up to `cut` within reach.
  __device__ __forceinline__ int choose(float u, int edge, u64 cut) const {
    return find([&](u64 sum) { return share(u, sum); }, [&](float f, int64_t i) -> u64 {
      const Point a = point(f);
      if (a.bin < edge) return weight(a);
      if (a.bin > edge || place_of(f, (u32)i) > cut || !a.within(reach)) return 0;
      return weight_bits(a.rest, s.edge) - kWhole;
    });
  }

  // The choice after `sums`, whose list holds the edge's bin.
  __device__ __forceinline__ int choose_by_sums(const Settings& o, const End& e) const {
    const int n = (int)s.listed;
    u64 cut = 0;
    if (n) {
      const int m = take(n, [&](u64 place) { return point(logit_of(place)).within(reach); });
      if (m) {
        // places beyond those of top_k and top_p, if their bin is the edge
        cut = ~0ull;
        if (e.bin == e.edge) {
          order(m);
          const u64 left = o.top_k - e.before_count;
          cut = !o.by_count ? last_by_mass(m, e.before, e.target, s.edge)
                : m < left  ? ~0ull
                            : s.some[left - 1];
        }
        for (int i = threadIdx.x; i < m; i += kThreads) {
          const u64 place = s.some[i];
          if (place <= cut)
            atomicAdd(&s.mass[segment_of((u32)place)],
                      weight_bits(point(logit_of(place)).rest, s.edge) - kWhole);
        }
        __syncthreads();
      }
    }
    return choose(o.u, e.edge, cut);
  }

  // The choice after `candidates`.
  __device__ __forceinline__ int choose_listed(const Settings& o, const End& e) const {
    const int n = (int)s.listed;
    const auto bin_of = [&](u64 place) { return point(logit_of(place)).bin; };
    order(take(n, [&](u64 place) { return bin_of(place) == e.bin; }));
    u64 cut = s.some[o.top_k - e.before_count - 1];
    __syncthreads();
    clear();
    if (o.by_mass) {
      for (int i = threadIdx.x; i < n; i += kThreads) {
        const u64 place = s.list[i];
        const Point a = point(logit_of(place));
        if (place <= cut) atomicAdd(&s.mass[a.bin], weight(a));
      }
      __syncthreads();
      const double target = pick(true, 0, 0, -1.0, o.top_p);
      const u32 bin = s.place;
      const u64 before = s.before;
      if (bin != kNone) {
        const int m =
            take(n, [&](u64 place) { return (place <= cut) & ((u32)bin_of(place) == bin); });
        order(m);
        const u64 by_p = last_by_mass(m, before, target, s.table[bin]);
        cut = by_p < cut ? by_p : cut;
      }
      __syncthreads();
      clear();
    }
    for (int i = threadIdx.x; i < n; i += kThreads) {
      const u64 place = s.list[i];
      const Point a = point(logit_of(place));
      if (place <= cut && a.within(reach)) atomicAdd(&s.mass[segment_of((u32)place)], weight(a));
    }
    __syncthreads();
    return find([&](u64 sum) { return share(o.u, sum); }, [&](float f, int64_t i) -> u64 {
      if (place_of(f, (u32)i) > cut) return 0;
      const Point a = point(f);
      return a.within(reach) ? weight(a) : 0;
    });
  }

  // The choice where a bin holds more than a list. The table is whole.
  __device__ __forceinline__ int choose_slowly(const Settings& o) const {
    u64 cut = ~0ull;
    if (o.by_count) cut = last(false, o.top_k, 0.0);
    if (o.by_mass) {
      segments([&](float f, int64_t i) {
        return place_of(f, (u32)i) <= cut ? weight(f) : (u64)0;
      });
      const u64 by_p = last(true, 0, __builtin_fmax((double)o.top_p * (double)total(), 0x1p-60));
      cut = by_p < cut ? by_p : cut;
    }
    const auto kept = [&](float f, int64_t i) -> u64 {
      const Point a = point(f);
      return place_of(f, (u32)i) <= cut && a.within(reach) ? weight(a) : 0;
    };
    segments(kept);
    return find([&](u64 sum) { return share(o.u, sum); }, kept);
  }
};

// A row in one program.
template <typename T>
__global__ void __launch_bounds__(kThreads) sample_kernel(newt_sample_params p, int shift) {
  __shared__ Shared s;
  const int64_t r = blockIdx.x;
  Row<T> row(p, s, r, shift);
  const Settings o(p, r);
  row.fill_table();
  bool bad;
  const float top = row.largest(bad);
  int id = -1;
  if (!(bad | o.bad) && __builtin_fabsf(top) < kInf) {
    row.set(o, top);
    if (o.greedy) {
      row.first();
      id = (int)s.first;
    } else {
      if (o.by_count | o.by_mass) row.histogram(o);
      const auto e = row.end(o);
      if (e.mode == kListed) {
        row.candidates(e);
        id = row.choose_listed(o, e);
      } else {
        if (e.mode == kSums) row.sums(e);
        if (e.mode == kSlow || s.listed > kList) {
          __syncthreads();
          row.fill_table();
          __syncthreads();
          id = row.choose_slowly(o);
        } else {
          id = row.choose_by_sums(o, e);
        }
      }
    }
  }
  if (threadIdx.x == 0) p.ids[r] = id;
}

// A row in several programs: the same steps, a launch each, whose results meet in
// the workspace.
struct Joint {
  float top[kMostParts];
  int bad[kMostParts];
  u32 listed, first;
  u64 bins[kBins];  // masses or counts
  u64 segments[kBins];
  u64 list[kList];
};

template <typename T>
struct Part {
  Joint& j;
  Row<T> row;
  Settings o;
  int parts, part;
  u64 bins[2], segments[2];  // read before what says whether they are needed
  __device__ __forceinline__ void preload() {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      bins[i] = j.bins[2 * threadIdx.x + i];
      segments[i] = j.segments[2 * threadIdx.x + i];
    }
  }
  __device__ __forceinline__ Part(const newt_sample_params& p, Shared& s, int64_t r, int parts_,
                                  int part_, int shift)
      : j(((Joint*)p.workspace)[r]), row(p, s, r, shift), o(p, r), parts(parts_), part(part_) {}
  // this program's chunks, whole segments
  __device__ __forceinline__ void own() {
    const int per = (row.chunks + kBins - 1) / kBins;
    const int each = ((row.chunks + parts - 1) / parts + per - 1) / per * per;
    row.from = part * each < row.chunks ? part * each : row.chunks;
    row.to = row.from + each < row.chunks ? row.from + each : row.chunks;
  }
  // Sets the row's largest logit; false where there is nothing to choose.
  __device__ __forceinline__ bool top() {
    const int i = threadIdx.x & 63;  // of at most 64 parts
    const float most = newt::lane_reduce<newt::Max, 63>(i < parts ? j.top[i] : -kInf);
    const bool bad = o.bad | (__ballot(i < parts && j.bad[i]) != 0);
    if (bad || !(__builtin_fabsf(most) < kInf)) return false;
    row.set(o, most);
    return true;
  }
  __device__ __forceinline__ typename Row<T>::End end() {
    if (o.by_count | o.by_mass) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        row.s.mass[2 * threadIdx.x + i] = o.by_count ? 0 : bins[i];
        row.s.count[2 * threadIdx.x + i] = o.by_count ? (u32)bins[i] : 0;
      }
      __syncthreads();
    }
    return row.end(o);
  }
};

template <typename T>
__global__ void __launch_bounds__(kThreads) part_top_kernel(newt_sample_params p, int parts,
                                                            int shift) {
  __shared__ Shared s;
  Part<T> a(p, s, blockIdx.x / parts, parts, blockIdx.x % parts, shift);
  a.own();
  bool bad;
  const float top = a.row.largest(bad);
  for (int i = a.part * kThreads + threadIdx.x; i < kBins; i += parts * kThreads) a.j.bins[i] = 0;
  if (threadIdx.x == 0) {
    a.j.top[a.part] = top;
    a.j.bad[a.part] = bad;
    if (a.part == 0) {
      a.j.listed = 0;
      a.j.first = 0xffffffffu;
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads) part_histogram_kernel(newt_sample_params p, int parts,
                                                                  int shift) {
  __shared__ Shared s;
  Part<T> a(p, s, blockIdx.x / parts, parts, blockIdx.x % parts, shift);
  a.own();
  a.row.fill_table();  // while the largest logits are on their way
  if (a.o.greedy || !(a.o.by_count | a.o.by_mass) || !a.top()) return;
  a.row.histogram(a.o);
  for (int i = threadIdx.x; i < kBins; i += kThreads) {
    const u64 v = a.o.by_count ? s.count[i] : s.mass[i];
    if (v) atomicAdd(&a.j.bins[i], v);
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads) part_sums_kernel(newt_sample_params p, int parts,
                                                             int shift) {
  __shared__ Shared s;
  Part<T> a(p, s, blockIdx.x / parts, parts, blockIdx.x % parts, shift);
  a.own();
  a.preload();
  a.row.fill_table();
  if (threadIdx.x == 0) {
    s.listed = 0;
    s.first = 0xffffffffu;
  }
  __syncthreads();
  if (!a.top()) return;
  if (a.o.greedy) {
    a.row.first();
    if (threadIdx.x == 0) atomicMin(&a.j.first, s.first);
    return;
  }
  const auto e = a.end();
  if (e.mode == kSlow) return;
  if (e.mode == kListed) {
    a.row.candidates(e);
  } else {
    a.row.sums(e);
    const int per = (a.row.chunks + kBins - 1) / kBins;
    for (int g = a.row.from / per + threadIdx.x; g * per < a.row.to; g += kThreads)
      a.j.segments[g] = s.mass[g];
  }
  if (threadIdx.x == 0) s.place = atomicAdd(&a.j.listed, s.listed);
  __syncthreads();
  const u32 n = s.listed < kList ? s.listed : kList;
  for (u32 i = threadIdx.x; i < n; i += kThreads)
    if (s.place + i < kList) a.j.list[s.place + i] = s.list[i];
}

template <typename T>
__global__ void __launch_bounds__(kThreads) part_choose_kernel(newt_sample_params p, int parts,
                                                               int shift) {
  __shared__ Shared s;
  const int64_t r = blockIdx.x;
  Part<T> a(p, s, r, parts, 0, shift);
  a.preload();
  const u32 n = a.j.listed;
#pragma unroll
  for (int i = 0; i < kList / kThreads; ++i)
    s.list[i * kThreads + threadIdx.x] = a.j.list[i * kThreads + threadIdx.x];
  a.row.fill_table();
  __syncthreads();
  int id = -1;
  if (a.top()) {
    if (a.o.greedy) {
      id = (int)a.j.first;
    } else {
      const auto e = a.end();
      if (e.mode == kSlow || n > kList) {
        id = a.row.choose_slowly(a.o);
      } else {
        if (threadIdx.x == 0) {
          s.listed = n;
          if (e.edge < kBins) s.edge = s.table[e.edge];
        }
        if (e.mode == kSums) {
          const int per = (a.row.chunks + kBins - 1) / kBins;
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int g = 2 * threadIdx.x + i;
            s.mass[g] = g * per < a.row.chunks ? a.segments[i] : 0;
          }
        }
        __syncthreads();
        id = e.mode == kListed ? a.row.choose_listed(a.o, e) : a.row.choose_by_sums(a.o, e);
      }
    }
  }
  if (threadIdx.x == 0) p.ids[r] = id;
}

// How many programs share a row: one where there are rows for half the chip, or
// where rows are so short that four launches cost more than they save; else enough
// to fill the chip, each with work for its waves. us in one and in several:
//   1 x 128000 bf16: no filter 28 / 17, top_p 56 / 37, all three 35 / 34;
//   16 x 128000, settings of each row's own: 74 / 53; 64 x 128000, top_p 69 / 55;
//   64 x 32000 fp32, settings of each row's own: 28 / 37; 16 x 32000 bf16 28 / 36.
// Between the two lengths nothing decided where the border lies: one row by all three
// filters takes 22 us of 50000, 24 of 65535 and 28, in several, of 65536. From 129 rows
// on a row has one program, 129 to 255 of 100003 logits by top_p 50 to 54 us.
int parts_of(int64_t rows, int64_t vocab, int dtype) {
  const int64_t chunk = dtype == NEWT_F32 ? 256 : 512;
  int64_t n = rows && vocab >= 65536 ? 256 / rows : 1;
  const int64_t most = (vocab + chunk * kWaves - 1) / (chunk * kWaves);
  n = n < most ? n : most;
  n = n < kMostParts ? n : kMostParts;
  return n < 2 ? 1 : (int)n;
}

// A weight's bits behind the point: sums of `vocab` of them stay below 2^63.
int weight_bits(int64_t vocab) {
  int bits = 0;
  while (vocab >> bits) ++bits;
  return 62 - bits < 45 ? 62 - bits : 45;
}

template <typename T>
int launch(const newt_sample_params& p, int shift, hipStream_t stream) {
  const char* const what = "newt_sample";
  const int parts = parts_of(p.rows, p.vocab, p.dtype);
  if (parts == 1) {
    int status = NEWT_OK;
    constexpr int64_t kMost = 1 << 21;  // programs of a launch: 2^31 work-items
    for (int64_t r = 0; r < p.rows && status == NEWT_OK; r += kMost) {
      newt_sample_params some = p;
      some.rows = p.rows - r < kMost ? p.rows - r : kMost;
      some.logits = (const T*)p.logits + r * p.stride;
      some.u += r;
      some.ids += r;
      if (p.temperature) some.temperature += r;
      if (p.top_k) some.top_k += r;
      if (p.top_p) some.top_p += r;
      if (p.min_p) some.min_p += r;
      status = run(what, sample_kernel<T>, some.rows, kThreads, 0, stream, some, shift);
    }
    return status;
  }
  if (!p.workspace || ((uintptr_t)p.workspace & 7))
    return fail(NEWT_ERR_INVALID, "newt_sample: null or unaligned workspace");
  int status = run(what, part_top_kernel<T>, p.rows * parts, kThreads, 0, stream, p, parts, shift);
  // settings of the rows' own are on the GPU: a row may need the histogram
  const bool none = !p.top_k && !p.top_p && !(p.top_k_all > 0 && p.top_k_all < p.vocab) &&
                    p.top_p_all >= 1.0f;
  if (status == NEWT_OK && !none)
    status = run(what, part_histogram_kernel<T>, p.rows * parts, kThreads, 0, stream, p, parts,
                 shift);
  if (status == NEWT_OK)
    status = run(what, part_sums_kernel<T>, p.rows * parts, kThreads, 0, stream, p, parts, shift);
  if (status == NEWT_OK)
    status = run(what, part_choose_kernel<T>, p.rows, kThreads, 0, stream, p, parts, shift);
  return status;
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

extern "C" size_t newt_sample_workspace(int64_t rows, int64_t vocab, int32_t dtype) {
  using namespace newt_ops;
  if (rows <= 0 || vocab <= 0 || parts_of(rows, vocab, dtype) == 1) return 0;
  return (size_t)rows * sizeof(Joint);
}

extern "C" int newt_sample(const newt_sample_params* params, void* stream) {
  using namespace newt_ops;
  if (!params) return fail(NEWT_ERR_INVALID, "newt_sample: null params");
  const newt_sample_params& p = *params;
  if (const char* w = wrong(p)) return fail(NEWT_ERR_INVALID, "newt_sample: %s", w);
  if (p.rows == 0) return NEWT_OK;
  if (!p.logits || !p.u || !p.ids) return fail(NEWT_ERR_INVALID, "newt_sample: null tensor");
  hipStream_t s = static_cast<hipStream_t>(stream);
  const int shift = weight_bits(p.vocab);
  switch (p.dtype) {
    case NEWT_F32: return launch<float>(p, shift, s);
    case NEWT_F16: return launch<f16>(p, shift, s);
    default: return launch<bf16>(p, shift, s);
  }
}
