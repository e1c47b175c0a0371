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
// finite runs again and keeps such values from the rows that do not see them.
#include "attention.h"

namespace newt_ops {
namespace {

template <typename T> struct frag;
template <> struct frag<bf16> { typedef bf16x8 type; };
template <> struct frag<f16> { typedef f16x8 type; };

template <typename T, int D, int WAVES>
struct Program {
  typedef typename frag<T>::type TX;
  static constexpr int THREADS = 64 * WAVES;
  static constexpr int ROWS = 32 * WAVES;
  static constexpr int STEPS = D / 16;
  static constexpr int DT = D / 32;
  typedef newt::LdsTile<T, D> KTile;
  typedef newt::LdsTileR<T, D> VTile;

  const newt_window_attention_params& p;
  T* k_lds;
  T* v_lds;
  const T* k;
  const T* v;
  const Range& range;
  TX q[STEPS];
  int64_t position;
  float m, l;
  f32x16 acc[DT];

  // the tile's keys and values from global memory, rows behind the last
  // visible key as zeros
  __device__ __forceinline__ void stage(int64_t key) {
    constexpr int CHUNKS = kTile * D / 8;
#pragma unroll
    for (int c = threadIdx.x; c < CHUNKS; c += THREADS) {
      const int row = c / (D / 8), d = c % (D / 8) * 8;
      T a[8] = {}, b[8] = {};
      if (key + row < range.hi) {
        newt::load_vec<T, 8>(k + (key + row) * p.k_stride_t + d, a, newt::any_align());
        newt::load_vec<T, 8>(v + (key + row) * p.v_stride_t + d, b, newt::any_align());
      }
      newt::store_vec<T, 8>(k_lds + KTile::off(row, d), a);
      newt::store_vec<T, 8>(v_lds + VTile::off(row, d), b);
    }
  }

  template <bool CAREFUL>
  __device__ __forceinline__ void attend(int64_t from, int64_t to) {
    const int lane = threadIdx.x & 63, half = lane >> 5;
    const float to_log2 = p.scale * kLog2e;
    m = -kInf;
    l = 0.0f;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) acc[dt] = (f32x16)(0.0f);
    for (int64_t i = from; i < to; ++i) {
      const int64_t key = range.tile(i);
      __syncthreads();
      stage(key);
      __syncthreads();
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
      const bool masked = !range.whole(key);
      // bit 16 kh + e: whether the row sees the key of s[kh][e]
      u32 seen = ~0u;
      float most = -kInf;
#pragma unroll
      for (int kh = 0; kh < 2; ++kh)
#pragma unroll
        for (int e = 0; e < 16; ++e) s[kh][e] *= to_log2;
      if (masked || CAREFUL) {
#pragma unroll
        for (int kh = 0; kh < 2; ++kh)
#pragma unroll
          for (int e = 0; e < 16; ++e)
            if (!range.sees(position, key + 32 * kh + 8 * (e / 4) + 4 * half + e % 4)) {
              s[kh][e] = -kInf;
              seen &= ~(1u << (16 * kh + e));
            }
      }
#pragma unroll
      for (int kh = 0; kh < 2; ++kh)
#pragma unroll
        for (int e = 0; e < 16; ++e) most = __builtin_fmaxf(most, s[kh][e]);
      most = newt::lane_reduce<newt::Max, 32>(most);
      if (__ballot(most > m + kSlack)) {
        const float to_m = __builtin_fmaxf(m, most);
        const float f = m == -kInf ? 0.0f : __builtin_amdgcn_exp2f(m - to_m);
        l *= f;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) acc[dt] *= f;
        m = to_m;
      }
      const float ref = m == -kInf ? 0.0f : m;
      TX w[4];
#pragma unroll
      for (int kh = 0; kh < 2; ++kh)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const float x = __builtin_amdgcn_exp2f(s[kh][e] - ref);
          l += x;
          w[2 * kh + e / 8][e % 8] = (T)x;
        }
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) {
          i16x8 a = newt::lds_frag_r_perm32<T, D>(v_lds, 32 * dt, 16 * ks, lane);
          if constexpr (CAREFUL) a = keep_apart(a, seen >> (8 * ks), acc[dt]);
          acc[dt] = newt::mfma_32x32x16(__builtin_bit_cast(TX, a), w[ks], acc[dt]);
        }
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

template <typename T, int D, int WAVES>
__global__ void __launch_bounds__(64 * WAVES)
window_attention_kernel(newt_window_attention_params p, int splits, int64_t row_tiles) {
  typedef Program<T, D, WAVES> P;
  __shared__ __attribute__((aligned(16))) T k_lds[kTile * D];
  __shared__ __attribute__((aligned(16))) T v_lds[kTile * D];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5;
  const int split = blockIdx.x % splits;
  const int64_t unit = blockIdx.x / splits;
  const int64_t row_tile = unit % row_tiles;
  const int group = p.heads / p.kv_heads;
  const int head = (int)(unit / row_tiles % p.kv_heads);
  const int64_t b = unit / row_tiles / p.kv_heads;
  const int64_t all_rows = p.q_len * group;
  const int64_t start = p.q_start ? p.q_start[b] : p.kv_len - p.q_len;
  const int64_t r0 = row_tile * P::ROWS;
  const int64_t r1 = r0 + P::ROWS < all_rows ? r0 + P::ROWS : all_rows;
  const Range range(start + r0 / group, start + (r1 - 1) / group, p.kv_len, p.window, p.sinks);

  P t{p, k_lds, v_lds, (const T*)p.k + b * p.k_stride_b + head * p.k_stride_h,
      (const T*)p.v + b * p.v_stride_b + head * p.v_stride_h, range};
  const int64_t r = r0 + 32 * wave + (lane & 31);
  const bool live = r < all_rows;
  t.position = live ? start + r / group : -1;
  const T* q = (const T*)p.q + (live ? Rows{p.q_stride_b, p.q_stride_h, p.q_stride_t}.at(
                                           b, head * group + r % group, r / group) : 0);
#pragma unroll
  for (int s = 0; s < P::STEPS; ++s) {
    T x[8] = {};
    if (live) newt::load_vec<T, 8>(q + 16 * s + 8 * half, x, newt::any_align());
    __builtin_memcpy(&t.q[s], x, 16);
  }

  const int64_t per = (range.tiles + splits - 1) / splits;
  const int64_t from = split * per;
  const int64_t to = from + per < range.tiles ? from + per : range.tiles;
  t.template attend<false>(from, to);
  float check = 0.0f;  // NaN where an accumulator is not finite
#pragma unroll
  for (int dt = 0; dt < P::DT; ++dt)
#pragma unroll
    for (int e = 0; e < 16; ++e) check += t.acc[dt][e] * 0.0f;
  if (__syncthreads_or(!(check == 0.0f))) t.template attend<true>(from, to);

  const float l = newt::lane_reduce<newt::Sum, 32>(t.l);
  if (!live) return;
  if (splits > 1) {
    const Parts parts(p.workspace, (int64_t)(gridDim.x / splits), splits, P::ROWS, D);
    const int64_t at = (unit * splits + split) * P::ROWS + 32 * wave + (lane & 31);
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

struct Plan {
  int64_t row_tiles, units;
  int splits, rows;
};

Plan plan(const newt_window_attention_params& p) {
  Plan r;
  const int64_t rows = p.q_len * (p.heads / p.kv_heads);
  r.rows = 128;
  r.row_tiles = (rows + r.rows - 1) / r.rows;
  r.units = p.batch * p.kv_heads * r.row_tiles;
  r.splits = 1;
  return r;
}

template <typename T, int D>
int launch(const newt_window_attention_params& p, hipStream_t stream) {
  const Plan r = plan(p);
  if (r.splits > 1 && !p.workspace)
    return fail(NEWT_ERR_INVALID, "newt_window_attention: null workspace");
  if (r.units * r.splits > 0x7fffffff)
    return fail(NEWT_ERR_INVALID, "newt_window_attention: too many queries");
  window_attention_kernel<T, D, 4><<<dim3((unsigned)(r.units * r.splits)), dim3(256), 0, stream>>>(
      p, r.splits, r.row_tiles);
  if (r.splits > 1)
    return join_splits<T, D>(p.workspace, p.out, {p.o_stride_b, p.o_stride_h, p.o_stride_t},
                             r.units, r.splits, r.rows, r.row_tiles, p.q_len, p.kv_heads,
                             p.heads / p.kv_heads, stream);
  return launched("newt_window_attention");
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
  return nullptr;
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
