// Attention of a step's tokens over the 8-bit cache.
//
// A wave takes 64 tokens at a time and keeps everything in registers: with
// keys stored token by token and values transposed, both products read their
// cache operand straight from memory in 16-byte pieces, so nothing goes
// through LDS until the waves' results are joined.
//   S^T = K Q^T by v_mfma_f32_16x16x32: lane (g, n) (g = lane / 16, n = lane %
//   16) gives key row n and takes scores of query row n. Key row n of score
//   tile t is token 16 (n / 4) + 4 t + n % 4, so that the 16 scores a lane ends
//   up with are those of tokens 16 g .. 16 g + 15 in order; within a row, lane
//   group g feeds head dims D/4 g .. D/4 (g + 1) to the products.
//   O^T += V^T P^T: k-slot (g, j) of step u is token 16 g + 8 u + j: the lane's
//   own scores as they are, and 16 consecutive bytes of a value row.
// e4m3 numbers are exact in bf16 and fp16. The blocks' scales multiply scores
// and weights in fp32; weights times scales are taken to bf16, whose range
// holds any scale, and where the queries are fp16 the rest of each weight goes
// through a second product, for a result as exact as fp16 asks for.
// HBM bounds it: the visible blocks are read once per KV head.
#include "attention.h"

namespace newt_ops {
namespace {

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

// 8 e4m3 bytes to an MFMA operand
template <typename T> struct from_bytes;
template <> struct from_bytes<bf16> {
  __device__ __forceinline__ static bf16x8 get(u32 lo, u32 hi) {
    const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, false);
    const bf16x2 b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, true);
    const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, false);
    const bf16x2 d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, true);
    return bf16x8{a.x, a.y, b.x, b.y, c.x, c.y, d.x, d.y};
  }
};
template <> struct from_bytes<f16> {
  __device__ __forceinline__ static f16x8 get(u32 lo, u32 hi) {
    const f16x2 a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, false);
    const f16x2 b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, true);
    const f16x2 c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, false);
    const f16x2 d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, true);
    return f16x8{a.x, a.y, b.x, b.y, c.x, c.y, d.x, d.y};
  }
};

template <typename T> struct frag;
template <> struct frag<bf16> { typedef bf16x8 type; };
template <> struct frag<f16> { typedef f16x8 type; };

// bytes that are NaN (0x7f or 0xff) as 0x80, others 0
__device__ __forceinline__ u32 nan_bytes(u32 w) {
  return ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
}

constexpr int kWaves = 4;

template <typename T, int D, int MT>
__global__ void __launch_bounds__(64 * kWaves)
cached_attention_kernel(newt_cached_attention_params p, int splits, int row_tiles) {
  typedef typename frag<T>::type TX;
  constexpr bool kExact = sizeof(T) == 2 && !__is_same(T, bf16);
  constexpr int ROWS = 16 * MT;
  constexpr int STEPS = D / 32;   // of the score product
  constexpr int DT = D / 16;      // tiles of head dims
  constexpr int KV4 = D / 64;     // 16-byte pieces of a key row a lane holds
  const int lane = threadIdx.x & 63, wave = wave_id();
  const int n = lane & 15, g = lane >> 4;
  const int split = blockIdx.x % splits;
  const int unit = blockIdx.x / splits;
  const int row_tile = unit % row_tiles;
  const int kv_heads = p.cache.kv_heads, group = p.heads / kv_heads;
  const int head = unit / row_tiles % kv_heads;
  const int b = unit / row_tiles / kv_heads;
  const int size = p.cache.block_size, shift = __builtin_ctz(size);
  const int q_len = (int)p.q_len, all_rows = q_len * group;

  const int len = p.lens[b] > 0 ? p.lens[b] : 0;
  const int held = (int)(p.table_width * size);  // positions that the table has
  const int r0 = row_tile * ROWS;
  const int r1 = r0 + ROWS < all_rows ? r0 + ROWS : all_rows;
  const Range range(len - q_len + r0 / group, len - q_len + (r1 - 1) / group,
                    len < held ? len : held, p.window ? (int)p.window : kNoWindow, (int)p.sinks);

  // queries, and each lane's rows' positions
  TX q[MT][STEPS];
  int position[MT];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    const int r = r0 + 16 * mt + n;
    const bool live = r < all_rows;
    position[mt] = live ? len - q_len + r / group : -1;
    const T* from = (const T*)p.q + (live ? Rows{p.q_stride_b, p.q_stride_h, p.q_stride_t}.at(
                                                b, head * group + r % group, r / group) : 0) +
                    D / 4 * g;
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
      T t[8];  // rows behind the last one take the first one's, and see nothing
      newt::load_vec<T, 8>(from + 8 * s, t, newt::any_align());
      __builtin_memcpy(&q[mt][s], t, 16);
    }
  }

  float m[MT], l[MT];
  f32x4 acc[MT][DT];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    m[mt] = -kInf;
    l[mt] = 0.0f;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) acc[mt][dt] = (f32x4)(0.0f);
  }
  const float to_log2 = p.scale * kLog2e;
  const int32_t* table = p.table + b * p.table_stride;

  const int per = (range.tiles + splits - 1) / splits;
  const int end = (split + 1) * per < range.tiles ? (split + 1) * per : range.tiles;
  for (int i = split * per + wave; i < end; i += kWaves) {
    const int key = range.tile(i);
    const bool whole = range.whole(key);
    // the blocks of this lane's keys (tokens 16 (n / 4) on) and values (16 g on)
    int64_t page[2];
    bool in[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int token = key + 16 * (j ? g : n >> 2);
      const int slot = token >> shift;
      in[j] = token < range.hi;
      int32_t block = in[j] ? table[slot] : 0;
      if (block < 0 || block >= p.cache.blocks) {
        in[j] = false;
        block = 0;
      }
      page[j] = (int64_t)block * kv_heads + head;
    }
    const bool bad = __ballot(!in[1]) != 0;  // values' groups cover the whole tile
    const unsigned char* k = (const unsigned char*)p.cache.k +
                             (page[0] * size + ((key + 16 * (n >> 2)) & (size - 1)) + (n & 3)) * D +
                             D / 4 * g;
    const unsigned char* v = (const unsigned char*)p.cache.v + (page[1] * D + n) * size +
                             ((key + 16 * g) & (size - 1));
    u32x4 kb[4][KV4], vb[DT];
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int c = 0; c < KV4; ++c) kb[t][c] = *(const u32x4*)(k + 4 * t * D + 16 * c);
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) vb[dt] = *(const u32x4*)(v + 16 * dt * size);
    float k_scale = p.cache.k_scale[page[1]] * to_log2;
    float v_scale = p.cache.v_scale[page[1]];

    f32x4 s[MT][4];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) s[mt][t] = (f32x4)(0.0f);
#pragma unroll
      for (int st = 0; st < STEPS; ++st) {
        const TX a = from_bytes<T>::get(kb[t][st / 2][st % 2 * 2], kb[t][st / 2][st % 2 * 2 + 1]);
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) s[mt][t] = newt::mfma_16x16x32(a, q[mt][st], s[mt][t]);
      }
    }
    const bool masked = !whole || bad;
    bool nan_values = false;
    if (masked) {
      // bytes of tokens that no row sees may hold anything: as zeros
      u32 keep[4];
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        keep[w] = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (in[1] && range.any(key + 16 * g + 4 * w + j)) keep[w] |= 0xffu << (8 * j);
      }
      u32 nans = 0;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          vb[dt][w] &= keep[w];
          nans |= nan_bytes(vb[dt][w]);
        }
      nan_values = __ballot(nans != 0) != 0;
    }
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      float x[16];
      float most = -kInf;
      u32 seen = 0xffffu;
#pragma unroll
      for (int j = 0; j < 16; ++j) x[j] = s[mt][j / 4][j % 4] * k_scale;
      if (masked) {
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          if (!(in[1] && range.sees(position[mt], key + 16 * g + j))) {
            x[j] = -kInf;
            seen &= ~(1u << j);
          }
        }
      }
#pragma unroll
      for (int j = 0; j < 16; ++j) most = __builtin_fmaxf(most, x[j]);
      most = newt::lane_reduce<newt::Max, 48>(most);
      if (__ballot(most > m[mt] + kSlack)) {
        const float to = __builtin_fmaxf(m[mt], most);
        const float f = m[mt] == -kInf ? 0.0f : __builtin_amdgcn_exp2f(m[mt] - to);
        l[mt] *= f;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) acc[mt][dt] *= f;
        m[mt] = to;
      }
      const float ref = m[mt] == -kInf ? 0.0f : m[mt];
      bf16x8 hi[2], lo[2];
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const float w = __builtin_amdgcn_exp2f(x[j] - ref);
        l[mt] += w;
        // a token that is not seen weighs nothing, whatever its block's scale
        const float scaled = (seen >> j) & 1 ? w * v_scale : 0.0f;
        hi[j / 8][j % 8] = (bf16)scaled;
        if constexpr (kExact) lo[j / 8][j % 8] = (bf16)(scaled - (float)hi[j / 8][j % 8]);
      }
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          u32 a0 = vb[dt][2 * u], a1 = vb[dt][2 * u + 1];
          if (nan_values) {
            // a NaN reaches the rows that see its token and no others
            const u32 n0 = nan_bytes(a0), n1 = nan_bytes(a1);
            if (__ballot((n0 | n1) != 0)) {
              bf16x8 is, sees;
#pragma unroll
              for (int j = 0; j < 8; ++j) {
                is[j] = (bf16)(((j < 4 ? n0 : n1) >> (8 * (j % 4) + 7)) & 1 ? 1.0f : 0.0f);
                sees[j] = (bf16)((seen >> (8 * u + j)) & 1 ? 1.0f : 0.0f);
              }
              f32x4 count = newt::mfma_16x16x32(is, sees, (f32x4)(0.0f));
#pragma unroll
              for (int e = 0; e < 4; ++e)
                if (count[e] > 0.0f) acc[mt][dt][e] = __builtin_nanf("");
              a0 &= ~(n0 | (n0 - (n0 >> 7)));
              a1 &= ~(n1 | (n1 - (n1 >> 7)));
            }
          }
          const bf16x8 a = from_bytes<bf16>::get(a0, a1);
          acc[mt][dt] = newt::mfma_16x16x32(a, hi[u], acc[mt][dt]);
          if constexpr (kExact) acc[mt][dt] = newt::mfma_16x16x32(a, lo[u], acc[mt][dt]);
        }
    }
  }

  // the waves' results joined through LDS, a row tile at a time
  constexpr int PITCH = D + 4;
  __shared__ float sm[kWaves][16], sl[kWaves][16];
  __shared__ float sacc[kWaves][16 * PITCH];
  const Parts parts(p.workspace, (int64_t)(gridDim.x / splits), splits, ROWS, D);
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    if (mt) __syncthreads();
    const float sum = newt::lane_reduce<newt::Sum, 48>(l[mt]);
    if (g == 0) {
      sm[wave][n] = m[mt];
      sl[wave][n] = sum;
    }
    __syncthreads();
    float M = sm[0][n];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) M = newt::Max::op(M, sm[w][n]);
    const float f = m[mt] == -kInf ? 0.0f : __builtin_amdgcn_exp2f(m[mt] - M);
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
      *(f32x4*)&sacc[wave][n * PITCH + 16 * dt + 4 * g] = acc[mt][dt] * f;
    __syncthreads();
    // 16 threads a row, each D / 16 of its dims in runs of 4
    const int row = threadIdx.x >> 4, part = threadIdx.x & 15;
    const int r = r0 + 16 * mt + row;
    if (r < all_rows) {
      float most = sm[0][row];
#pragma unroll
      for (int w = 1; w < kWaves; ++w) most = newt::Max::op(most, sm[w][row]);
      float total = 0.0f;
#pragma unroll
      for (int w = 0; w < kWaves; ++w)
        total += sm[w][row] == -kInf ? sl[w][row]
                                     : sl[w][row] * __builtin_amdgcn_exp2f(sm[w][row] - most);
      const int64_t at = ((int64_t)unit * splits + split) * ROWS + 16 * mt + row;
      if (splits > 1 && part == 0) {
        parts.m[at] = most;
        parts.l[at] = total;
      }
      T* to = (T*)p.out + Rows{p.o_stride_b, p.o_stride_h, p.o_stride_t}.at(
                              b, head * group + r % group, r / group);
#pragma unroll
      for (int c = 0; c < D / 64; ++c) {
        const int d = 64 * c + 4 * part;
        f32x4 o = *(const f32x4*)&sacc[0][row * PITCH + d];
#pragma unroll
        for (int w = 1; w < kWaves; ++w) o += *(const f32x4*)&sacc[w][row * PITCH + d];
        if (splits > 1) {
          *(f32x4*)(parts.acc + at * D + d) = o;
        } else {
          T t[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) t[e] = (T)(total == 0.0f ? 0.0f : o[e] / total);
          newt::store_vec<T, 4>(to + d, t, newt::any_align());
        }
      }
    }
  }
}

// Rows of a program and splits of its tiles, from sizes that the host knows:
// the table's width bounds the lengths.
Plan plan(const newt_cached_attention_params& p) {
  const int group = p.heads / p.cache.kv_heads;
  Plan r(p.batch, p.q_len, p.cache.kv_heads, group, p.q_len * group > 16 ? 32 : 16);
  const int64_t tiles = most_tiles(p.table_width * p.cache.block_size, p.window, p.sinks, p.q_len);
  r.splits = split_count(r.units, tiles, 1024, kWaves);
  return r;
}

template <typename T, int D>
int launch(const newt_cached_attention_params& p, hipStream_t stream) {
  const Plan r = plan(p);
  if (r.splits > 1 && !p.workspace)
    return fail(NEWT_ERR_INVALID, "newt_cached_attention: null workspace");
  if (r.too_large()) return fail(NEWT_ERR_INVALID, "newt_cached_attention: too many queries");
  const dim3 grid((unsigned)(r.units * r.splits)), block(64 * kWaves);
  if (r.rows == 16)
    cached_attention_kernel<T, D, 1><<<grid, block, 0, stream>>>(p, r.splits, r.row_tiles);
  else
    cached_attention_kernel<T, D, 2><<<grid, block, 0, stream>>>(p, r.splits, r.row_tiles);
  if (r.splits > 1)
    return join_splits<T, D>(p.workspace, p.out, {p.o_stride_b, p.o_stride_h, p.o_stride_t}, r,
                             p.cache.kv_heads, p.heads / p.cache.kv_heads, stream);
  return launched("newt_cached_attention");
}

template <typename T>
int by_dim(const newt_cached_attention_params& p, hipStream_t stream) {
  switch (p.cache.head_dim) {
    case 64: return launch<T, 64>(p, stream);
    case 128: return launch<T, 128>(p, stream);
    default: return launch<T, 256>(p, stream);
  }
}

const char* wrong(const newt_cached_attention_params& p) {
  if (const char* w = cache_wrong(p.cache)) return w;
  if (p.batch < 0 || p.q_len < 0 || p.table_width < 0 || p.window < 0 || p.sinks < 0)
    return "negative size";
  if (p.heads <= 0 || p.heads % p.cache.kv_heads) return "heads have to be a multiple of kv_heads";
  if (p.q_len * p.heads >= kLimit || p.table_width * p.cache.block_size >= kLimit ||
      p.window >= kLimit || p.sinks >= kLimit)
    return "sizes stay below 2^30";
  return nullptr;
}

}  // namespace
}  // namespace newt_ops

extern "C" size_t newt_cached_attention_workspace(const newt_cached_attention_params* p) {
  using namespace newt_ops;
  if (!p || wrong(*p) || p->batch == 0 || p->q_len == 0) return 0;
  const Plan r = plan(*p);
  return r.splits > 1 ? Parts::bytes(r.units, r.splits, r.rows, p->cache.head_dim) : 0;
}

extern "C" int newt_cached_attention(const newt_cached_attention_params* params, void* stream) {
  using namespace newt_ops;
  if (!params) return fail(NEWT_ERR_INVALID, "newt_cached_attention: null params");
  const newt_cached_attention_params& p = *params;
  if (const char* w = wrong(p)) return fail(NEWT_ERR_INVALID, "newt_cached_attention: %s", w);
  if (p.batch == 0 || p.q_len == 0) return NEWT_OK;
  if (!p.q || !p.out || !p.lens || (p.table_width && !p.table))
    return fail(NEWT_ERR_INVALID, "newt_cached_attention: null tensor");
  if (p.cache.blocks == 0 && p.table_width)
    return fail(NEWT_ERR_INVALID, "newt_cached_attention: a cache without blocks");
  hipStream_t s = static_cast<hipStream_t>(stream);
  switch (p.dtype) {
    case NEWT_F16: return by_dim<f16>(p, s);
    case NEWT_BF16: return by_dim<bf16>(p, s);
    default: return fail(NEWT_ERR_INVALID, "newt_cached_attention: q is fp16 or bf16");
  }
}
