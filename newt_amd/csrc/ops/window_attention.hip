// Causal attention in a sliding window whose first tokens (sinks) stay
// visible, over keys and values in the queries' own type.
//
// A program takes 32 query rows a wave and visits 64 keys at a time, those of
// the sinks first, then the window's; tiles that no row sees are not visited.
// Keys and values are staged in LDS for all of its waves.
//   S^T = K Q^T by v_mfma_f32_32x32x16: a lane holds scores of one query row,
//   so maxima and sums stay in the lane but for one step across its halves;
//   O^T += V^T P^T takes the weights straight from the score accumulators, the
//   value operand read transposed from LDS in the order they hold the keys.
// A value that no query of a program sees is not read, or weighed by 0. 0
// times an infinity or NaN is NaN, so a program whose accumulators end up not
// finite runs again and keeps such values from the rows that do not see them;
// as does one with scores beyond kExact.
// The weights go to the product in the queries' type, as the matrix unit takes
// them; their sum is that of the rounded ones, so that values that are all alike
// come out as they are. That is off by 2^-9 (bf16) or 2^-12 (fp16) of a weight on
// average, beside the output's own rounding, which is as large: against 64 bits
// 0.0021 where rounding the output alone gives 0.0016 (fp16 0.00029 and 0.00021).
// The rest of each weight in a second product, as cached_attention has it for
// fp16, would make half as many products again of the unit that is busiest here.
// bf16 4 x 32 x 4096 x 128 in a window of 1024: 317 us, 762 TFLOP/s of visible
// pairs, MFMA busy 42%. One token of each of 16 sequences over a window of 4096:
// 58 us (4.6 TB/s), where HBM bounds it. 256 head dims do not fit the registers:
// 192 bytes of scratch a lane (264 where rows are not aligned), 388 TFLOP/s for 2
// x 16 x 4096 without a window.
#include "attention.h"

namespace newt_ops {
namespace {

template <typename T> struct frag;
template <> struct frag<bf16> { typedef bf16x8 type; };
template <> struct frag<f16> { typedef f16x8 type; };

// Whole 16-byte pieces of rows go from memory to LDS by themselves (DIRECT)
// where rows and tensors are aligned to them; else through registers.
template <typename T, int D, int WAVES, bool DIRECT>
struct Program {
  typedef typename frag<T>::type TX;
  static constexpr int THREADS = 64 * WAVES;
  static constexpr int ROWS = 32 * WAVES;
  static constexpr int STEPS = D / 16;
  static constexpr int DT = D / 32;
  static constexpr int STAGE = 2 * kTile * D;  // numbers of a stage: keys, then values
  // fp16 weights, and with them their sums and products, are 2^7 times as large,
  // up to 2^(7 + kSlack): those from 2^-21 of the largest on keep all bits of the
  // type, and smaller ones are off by 2^-32 of it at most, where without this a
  // row lost all weights below 2^-25, however many. bf16 has the range by itself.
  static constexpr float kLift = __is_same(T, bf16) ? 0.0f : 7.0f;
  typedef newt::LdsTile<T, D> KTile;
  typedef newt::LdsTileR<T, D> VTile;

  const newt_window_attention_params& p;
  T* even;  // two stages of LDS, two arrays: the compiler then knows that what
  T* odd;   // is on its way into one is not what is read from the other
  const T* k;
  const T* v;
  const Range& range;
  const int wave;
  TX q[STEPS];
  int position;
  float m, l;
  f32x16 acc[DT];

  // A tile's keys and values into stage `to`, rows behind the last visible key
  // as zeros.
  __device__ __forceinline__ void stage(int key, T* k_lds) const {
    constexpr int ROUNDS = kTile * D / 8 / THREADS;
    constexpr int STEP = THREADS / (D / 8);  // rows of a round
    // the swizzles go by 16 rows: rounds that are a multiple of that apart have
    // the same lane offsets, and differ by a scalar
    constexpr int KINDS = STEP < 16 ? 16 / STEP : 1;
    const int rows = range.hi - key;
    const int lane = threadIdx.x & 63;
    T* v_lds = k_lds + kTile * D;
    const T* k_from = k + key * p.k_stride_t;
    const T* v_from = v + key * p.v_stride_t;
#pragma unroll
    for (int c = 0; c < ROUNDS; ++c) {
      // the 16 bytes of LDS at `slot` hold this row and column
      const int kind = c % KINDS, up = (c - kind) * STEP;
      const int first = c * THREADS + 64 * wave, slot = kind * THREADS + 64 * wave + lane;
      int row, d;
      newt::lds_tile_slot<T, D>(slot, row, d);
      put(k_from + up * p.k_stride_t, row, d, p.k_stride_t, row < rows - up,
          k_lds + first * 8);
      VTile::slot(slot, row, d);
      put(v_from + up * p.v_stride_t, row, d, p.v_stride_t, row < rows - up,
          v_lds + first * 8);
    }
  }
  // 8 numbers of a row to this lane's 16 bytes of the wave's at `to`, or zeros.
  __device__ __forceinline__ static void put(const T* from, int row, int d, int64_t stride, bool in,
                                             T* to) {
    if constexpr (DIRECT) {
      newt::lds_dma16_masked(from, (u32)(row * (int)stride + d) * sizeof(T), in, to);
    } else {
      T x[8] = {};
      if (in) newt::load_vec<T, 8>(from + row * stride + d, x, newt::any_align());
      newt::store_vec<T, 8>(to + (threadIdx.x & 63) * 8, x);
    }
  }

  // `to_log2` > 0: the rows' maxima are those of the unscaled scores.
  template <bool CAREFUL>
  __device__ __forceinline__ void attend(int from, int to, float to_log2) {
    m = -kInf;
    l = 0.0f;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) acc[dt] = (f32x16)(0.0f);
    if constexpr (CAREFUL) {
      for (int i = from; i < to; ++i) {
        __syncthreads();
        stage(range.tile(i), even);
        __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0)
        __syncthreads();
        tile<true>(range.tile(i), even, to_log2);
      }
    } else {
      if (from < to) stage(range.tile(from), even);
      for (int i = from; i < to; i += 2) {
        step(i, to, even, odd, to_log2);
        if (i + 1 < to) step(i + 1, to, odd, even, to_log2);
      }
    }
  }

  __device__ __forceinline__ static float add(const bf16x8& w, float l) {
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    const bf16x2 one = {(bf16)1.0f, (bf16)1.0f};
#pragma unroll
    for (int j = 0; j < 8; j += 2)
      l = __builtin_amdgcn_fdot2_f32_bf16(bf16x2{w[j], w[j + 1]}, one, l, false);
    return l;
  }
  __device__ __forceinline__ static float add(const f16x8& w, float l) {
    typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
    const f16x2 one = {(f16)1.0f, (f16)1.0f};
#pragma unroll
    for (int j = 0; j < 8; j += 2)
      l = __builtin_amdgcn_fdot2(f16x2{w[j], w[j + 1]}, one, l, false);
    return l;
  }

  // A tile's scores to weights, masked where a row does not see a key. (The
  // branch costs 32 register moves; a copy of the code behind it for either way,
  // without them, is slower, 352 against 316 us for 4 x 32 x 4096 x 128 in a
  // window of 1024: exponentials then no longer run beside the products.)
  template <bool CAREFUL>
  __device__ __forceinline__ void weigh(f32x16 (&s)[2], int key, float to_log2, TX (&w)[4],
                                        u32& seen) {
    const int half = (threadIdx.x & 63) >> 5;
    if constexpr (CAREFUL) {
      // rounded, in no fma with the maximum
#pragma clang fp contract(off)
      s[0] *= to_log2;
      s[1] *= to_log2;
      to_log2 = 1.0f;
    }
    // bit 16 kh + e: whether the row sees the key of s[kh][e]
    if (CAREFUL || !range.whole(key)) {
      const int at = key + 4 * half;
      const auto offset = [](int kh, int e) { return 32 * kh + 8 * (e / 4) + e % 4; };
      if (!CAREFUL && key >= range.sinks && range.hi > range.last) {
        // no sinks here, and the keys go on to the last query: the window alone
        const int back = position - at;
#pragma unroll
        for (int kh = 0; kh < 2; ++kh)
#pragma unroll
          for (int e = 0; e < 16; ++e)
            s[kh][e] = (u32)(back - offset(kh, e)) < (u32)range.window ? s[kh][e] : -kInf;
      } else {
#pragma unroll
        for (int kh = 0; kh < 2; ++kh)
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const bool sees = range.sees(position, at + offset(kh, e));
            s[kh][e] = sees ? s[kh][e] : -kInf;
            if constexpr (CAREFUL)
              if (!sees) seen &= ~(1u << (16 * kh + e));
          }
      }
    }
    float most = s[0][0];
#pragma unroll
    for (int kh = 0; kh < 2; ++kh)
#pragma unroll
      for (int e = 0; e < 16; ++e) most = __builtin_fmaxf(most, s[kh][e]);
    most = newt::lane_reduce<newt::Max, 32>(most) * to_log2;
    if (__ballot(most > m + (CAREFUL ? 0.0f : kSlack))) {
      const float to_m = __builtin_fmaxf(m, most);
      const float f = m == -kInf ? 0.0f : __builtin_amdgcn_exp2f(m - to_m);
      l *= f;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) acc[dt] *= f;
      m = to_m;
    }
    const float ref = m == -kInf ? 0.0f : m;
#pragma unroll
    for (int kh = 0; kh < 2; ++kh)
#pragma unroll
      for (int e = 0; e < 16; ++e)
        w[2 * kh + e / 8][e % 8] = (T)__builtin_amdgcn_exp2f(
            // maxima beyond kExact would lose the lift to rounding
            CAREFUL ? (s[kh][e] - ref) + kLift
                    : __builtin_fmaf(s[kh][e], to_log2, kLift - ref));
    // the sum of the weights as the product takes them, two at a time
#pragma unroll
    for (int i = 0; i < 4; ++i) l = add(w[i], l);
  }

  // One tile, while the next one is on its way.
  __device__ __forceinline__ void step(int i, int to, T* now, T* next, float to_log2) {
    // this tile's pieces have arrived, and no wave still reads the other stage
    __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0)
    __syncthreads();
    if (i + 1 < to) stage(range.tile(i + 1), next);
    tile<false>(range.tile(i), now, to_log2);
  }

  template <bool CAREFUL>
  __device__ __forceinline__ void tile(int key, const T* k_lds, float to_log2) {
    const int lane = threadIdx.x & 63;
    const T* v_lds = k_lds + kTile * D;
    f32x16 s[2];
#pragma unroll
    for (int kh = 0; kh < 2; ++kh) {
      s[kh] = (f32x16)(0.0f);
#pragma unroll
      for (int st = 0; st < STEPS; ++st)
        s[kh] = newt::mfma_32x32x16(
            __builtin_bit_cast(TX, newt::lds_frag_k<T, D, 32>(k_lds, 32 * kh, 16 * st, lane)),
            q[st], s[kh]);
    }
    u32 seen = ~0u;
    TX w[4];
    weigh<CAREFUL>(s, key, to_log2, w, seen);
#pragma unroll
    for (int ks = 0; ks < 4; ++ks)
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        i16x8 a = newt::lds_frag_r_perm32<T, D>(v_lds, 32 * dt, 16 * ks, lane);
        if constexpr (CAREFUL) a = keep_apart(a, seen >> (8 * ks), acc[dt]);
        acc[dt] = newt::mfma_32x32x16(__builtin_bit_cast(TX, a), w[ks], acc[dt]);
      }
  }

  // The operand without its infinities and NaN, which go into the
  // accumulators of the rows that see them: numbers of +inf and NaN, and of
  // -inf and NaN, among a row's visible keys by a product of 0s and 1s.
  __device__ __forceinline__ i16x8 keep_apart(i16x8 a, u32 seen, f32x16& o) const {
    const int exponent = __is_same(T, bf16) ? 0x7f80 : 0x7c00;
    TX up, down, sees;
    bool found = false;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int bits = (unsigned short)a[j];
      const bool odd = (bits & exponent) == exponent;
      const bool nan = odd && (bits & 0x7fff) != exponent;
      up[j] = (T)(nan || (odd && !(bits & 0x8000)) ? 1.0f : 0.0f);
      down[j] = (T)(nan || (odd && (bits & 0x8000)) ? 1.0f : 0.0f);
      sees[j] = (T)((seen >> j) & 1 ? 1.0f : 0.0f);
      if (odd) a[j] = 0;
      found |= odd;
    }
    if (__ballot(found)) {
      const f32x16 ups = newt::mfma_32x32x16(up, sees, (f32x16)(0.0f));
      const f32x16 downs = newt::mfma_32x32x16(down, sees, (f32x16)(0.0f));
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        if (ups[e] > 0.0f) o[e] += kInf;
        if (downs[e] > 0.0f) o[e] -= kInf;
      }
    }
    return a;
  }
};

template <typename T, int D, int WAVES, bool DIRECT>
__global__ void __launch_bounds__(64 * WAVES, D == 256 ? 1 : 2)
window_attention_kernel(newt_window_attention_params p, int splits, int row_tiles) {
  typedef Program<T, D, WAVES, DIRECT> P;
  __shared__ __attribute__((aligned(16))) T even[P::STAGE];
  __shared__ __attribute__((aligned(16))) T odd[P::STAGE];
  const int lane = threadIdx.x & 63, wave = wave_id(), half = lane >> 5;
  const int program = by_die(blockIdx.x, gridDim.x);
  const int split = program % splits;
  const int unit = program / splits;
  const int row_tile = unit % row_tiles;
  const int group = p.heads / p.kv_heads;
  const int head = unit / row_tiles % p.kv_heads;
  const int b = unit / row_tiles / p.kv_heads;
  const int q_len = (int)p.q_len, all_rows = q_len * group;
  int start = (int)(p.kv_len - p.q_len);
  if (p.q_start) {
    start = p.q_start[b];
    // so that the queries' positions fit an int
    const int most = 0x7ffffffe - q_len;
    start = start < -kLimit ? -kLimit : start > most ? most : start;
  }
  const int r0 = row_tile * P::ROWS;
  const int r1 = r0 + P::ROWS < all_rows ? r0 + P::ROWS : all_rows;
  const Range range(start + r0 / group, start + (r1 - 1) / group, (int)p.kv_len,
                    p.window ? (int)p.window : kNoWindow, (int)p.sinks);

  P t{p, even, odd, (const T*)p.k + b * p.k_stride_b + head * p.k_stride_h,
      (const T*)p.v + b * p.v_stride_b + head * p.v_stride_h, range, wave};
  const int r = r0 + 32 * wave + (lane & 31);
  const bool live = r < all_rows;
  t.position = live ? start + r / group : -1;
  const T* q = (const T*)p.q + (live ? Rows{p.q_stride_b, p.q_stride_h, p.q_stride_t}.at(
                                           b, head * group + r % group, r / group) : 0);
  // a negative scale is taken out of the queries, and one of 0 would make NaN
  // of masked scores: any tiny one gives equal weights
  const bool negative = p.scale < 0.0f;
#pragma unroll
  for (int s = 0; s < P::STEPS; ++s) {
    T x[8];  // rows behind the last one take the first one's, and see nothing
    newt::load_vec<T, 8>(q + 16 * s + 8 * half, x, newt::any_align());
#pragma unroll
    for (int i = 0; i < 8; ++i) t.q[s][i] = negative ? -x[i] : x[i];
  }
  const float to_log2 =
      __builtin_fmaxf(__builtin_fabsf(p.scale) * kLog2e, 1e-37f);

  const int per = (range.tiles + splits - 1) / splits;
  const int from = split * per;
  const int to = from + per < range.tiles ? from + per : range.tiles;
  t.template attend<false>(from, to, to_log2);
  float check = 0.0f;  // NaN where an accumulator is not finite
#pragma unroll
  for (int dt = 0; dt < P::DT; ++dt)
#pragma unroll
    for (int e = 0; e < 16; ++e) check += t.acc[dt][e] * 0.0f;
  if (__syncthreads_or(!(check == 0.0f) | beyond_exact(t.m)))
    t.template attend<true>(from, to, to_log2);

  const float l = newt::lane_reduce<newt::Sum, 32>(t.l);
  if (!live) return;
  if (splits > 1) {
    const Parts parts(p.workspace, (int64_t)(gridDim.x / splits), splits, P::ROWS, D);
    const int64_t at = ((int64_t)unit * splits + split) * P::ROWS + 32 * wave + (lane & 31);
    if (half == 0) {
      parts.m[at] = t.m;
      parts.l[at] = l;
    }
#pragma unroll
    for (int dt = 0; dt < P::DT; ++dt)
#pragma unroll
      for (int e = 0; e < 16; e += 4)
        *(f32x4*)(parts.acc + at * D + 32 * dt + 2 * e + 4 * half) =
            f32x4{t.acc[dt][e], t.acc[dt][e + 1], t.acc[dt][e + 2], t.acc[dt][e + 3]};
    return;
  }
  T* out = (T*)p.out + Rows{p.o_stride_b, p.o_stride_h, p.o_stride_t}.at(
                           b, head * group + r % group, r / group);
#pragma unroll
  for (int dt = 0; dt < P::DT; ++dt)
#pragma unroll
    for (int e = 0; e < 16; e += 4) {
      T x[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) x[j] = (T)(l == 0.0f ? 0.0f : t.acc[dt][e + j] / l);
      newt::store_vec<T, 4>(out + 32 * dt + 2 * e + 4 * half, x, newt::any_align());
    }
}

// Whether every piece of 8 numbers that a tile is staged in is aligned.
bool direct(const newt_window_attention_params& p) {
  const int64_t strides = p.k_stride_b | p.k_stride_h | p.k_stride_t | p.v_stride_b |
                          p.v_stride_h | p.v_stride_t;
  return strides % 8 == 0 && (((uintptr_t)p.k | (uintptr_t)p.v) & 15) == 0 &&
         // and lies within 2^31 bytes of its tile's first
         p.k_stride_t < (1 << 22) && p.v_stride_t < (1 << 22);
}

// Splits of the rows' tiles. Up to 256 programs have a CU each; a program's
// tile takes 0.6 + 0.0052 D us (1.27 for 128 head dims, 0.93 for 64), the kernel
// that joins the splits 3.5 us and what writing and reading the partial results
// at 2.5 TB/s takes: us for 1, 2, 4, 8, 16, 32 splits of
//   one token over 8192 keys, 8 KV heads, 4 query heads each: 162 / 86 / 47 /
//   28 / 18 / 14; 16 sequences, window 4096: 87 / 52 / 49 / 51 / 52 / 63;
//   128 of 4096: 86 / 52 / 34 / 29 / 29 / 41; 512 of 2048, window 512: 20 / 31;
//   3 x 16 heads of 64, 333 of 1999, window 500: 17 / 29.
// The line was drawn through 64 and 128 head dims. Of 256 a tile takes 4.4 us,
// not 1.9, so that the rule, marked *, does not always find the best there:
//   16 sequences, 4 KV heads, window 4096: 297 / 159 / 96 / 107* / 126 / 136;
//   one token over 8192 keys, 8 KV heads: 550 / 281 / 147 / 80 / 48 / 37 (64: 48*);
//   128 of 4096, 16 heads: 283 / 153 / 86 / 56* / 46 / 70;
//   512 of 2048, window 512: 58* / 42 / 38 / 60; 4 x 16, 333 of 1999: 66* / 92.
// From 512 programs of 256 rows on (two for each CU, one after the other), 8
// waves share each tile: 4 x 32 x 4096 x 128 in a window of 1024 327 -> 315 us.
Plan plan(const newt_window_attention_params& p) {
  const int group = p.heads / p.kv_heads;
  Plan r(p.batch, p.q_len, p.kv_heads, group, 256);
  if (p.head_dim <= 128 && r.units >= 512 && direct(p)) return r;
  r = Plan(p.batch, p.q_len, p.kv_heads, group, 128);
  const int64_t span = p.q_len < 128 ? p.q_len : (127 / group) + 2;
  const int64_t tiles = most_tiles(p.kv_len, p.window, p.sinks, span);
  // few rows wait for memory more than for products: two programs to a CU
  int64_t most = r.units ? (r.all_rows <= 32 ? 512 : 256) / r.units : 1;
  most = most < tiles ? most : tiles;
  most = most < kMostSplits ? most : kMostSplits;
  const double tile = 0.6 + p.head_dim * 0.0052;
  const double each = 2.0 * p.batch * p.kv_heads * r.all_rows * (p.head_dim + 2) * 4 / 2.5e6;
  double least = tiles * tile;
  for (int n = 2; n <= most; ++n) {
    const double cost = (tiles + n - 1) / n * tile + 3.5 + n * each;
    if (cost < least) {
      least = cost;
      r.splits = n;
    }
  }
  return r;
}

template <typename T, int D>
int launch(const newt_window_attention_params& p, hipStream_t stream) {
  const Plan r = plan(p);
  if (r.splits > 1 && !p.workspace)
    return fail(NEWT_ERR_INVALID, "newt_window_attention: null workspace");
  if (r.too_large()) return fail(NEWT_ERR_INVALID, "newt_window_attention: too many queries");
  const char* const what = "newt_window_attention";
  const int64_t grid = r.units * r.splits;
  if constexpr (D <= 128)
    if (r.rows == 256)
      return run(what, window_attention_kernel<T, D, 8, true>, grid, 512, 0, stream, p, 1,
                 r.row_tiles);
  const int status =
      direct(p) ? run(what, window_attention_kernel<T, D, 4, true>, grid, 256, 0, stream, p,
                      r.splits, r.row_tiles)
                : run(what, window_attention_kernel<T, D, 4, false>, grid, 256, 0, stream, p,
                      r.splits, r.row_tiles);
  if (status != NEWT_OK || r.splits == 1) return status;
  return join_splits<T, D>(p.workspace, p.out, {p.o_stride_b, p.o_stride_h, p.o_stride_t}, r,
                           p.kv_heads, p.heads / p.kv_heads, stream);
}

template <typename T>
int by_dim(const newt_window_attention_params& p, hipStream_t stream) {
  switch (p.head_dim) {
    case 64: return launch<T, 64>(p, stream);
    case 128: return launch<T, 128>(p, stream);
    default: return launch<T, 256>(p, stream);
  }
}

const char* wrong(const newt_window_attention_params& p) {
  if (p.batch < 0 || p.q_len < 0 || p.kv_len < 0 || p.window < 0 || p.sinks < 0)
    return "negative size";
  if (p.head_dim != 64 && p.head_dim != 128 && p.head_dim != 256)
    return "head_dim is 64, 128 or 256";
  if (p.heads <= 0 || p.kv_heads <= 0 || p.heads % p.kv_heads)
    return "heads have to be a multiple of kv_heads";
  if (p.q_len * p.heads >= kLimit || p.kv_len >= kLimit || p.window >= kLimit || p.sinks >= kLimit)
    return "sizes stay below 2^30";
  if (p.k_stride_t < 0 || p.v_stride_t < 0) return "negative stride";
  return queries_wrong(p, p.head_dim);
}

}  // namespace
}  // namespace newt_ops

extern "C" size_t newt_window_attention_workspace(const newt_window_attention_params* p) {
  using namespace newt_ops;
  if (!p || wrong(*p) || p->batch == 0 || p->q_len == 0) return 0;
  const Plan r = plan(*p);
  return r.splits > 1 ? Parts::bytes(r.units, r.splits, r.rows, p->head_dim) : 0;
}

extern "C" int newt_window_attention(const newt_window_attention_params* params, void* stream) {
  using namespace newt_ops;
  if (!params) return fail(NEWT_ERR_INVALID, "newt_window_attention: null params");
  const newt_window_attention_params& p = *params;
  if (const char* w = wrong(p)) return fail(NEWT_ERR_INVALID, "newt_window_attention: %s", w);
  if (p.batch == 0 || p.q_len == 0) return NEWT_OK;
  if (!p.q || !p.out || (p.kv_len && (!p.k || !p.v)))
    return fail(NEWT_ERR_INVALID, "newt_window_attention: null tensor");
  hipStream_t s = static_cast<hipStream_t>(stream);
  switch (p.dtype) {
    case NEWT_F16: return by_dim<f16>(p, s);
    case NEWT_BF16: return by_dim<bf16>(p, s);
    default: return fail(NEWT_ERR_INVALID, "newt_window_attention: q is fp16 or bf16");
  }
}
