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
// through a second product, for a result as exact as fp16 asks for (0.00021 from
// 64 bits). For bf16 queries a weight rounded by 2^-9 adds no more than the
// output's own rounding (0.0022 for 0.0016); there the second product would take
// the batch below from 122.3 to 123.7 us and the single sequence from 14.1 to 14.5.
// HBM bounds large batches: the visible blocks are read once per KV head. bf16, 64
// sequences of up to 8192 tokens, 32 heads of 128 over 8: 122 us (5.6 TB/s), 5 of
// them the join. Small ones wait for memory: 1 sequence of 8191 tokens 14 us.
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

// Waves that share a SIMD's registers.
constexpr int occupancy(int D, int MT) { return D * MT <= 128 ? 2 : 1; }

// How a launch's tiles are dealt out, from the sequences' lengths, which only
// the GPU knows. A unit is a sequence, a row tile and a head; its tiles are
// those of the sequence (at least one, so that every unit is visited). Of
// `shares` programs
//   - where an even share of all tiles is kLong and more, each takes an even
//     run of the line of all tiles, unit behind unit: a batch of any lengths
//     keeps every CU busy to the end (64 sequences of 2048 to 8192 tokens: 148
//     -> 120 us against equal splits of each), at the cost of a start and an
//     end in each unit that a run touches;
//   - else each takes an even part of one unit, units in as many parts as their
//     lengths ask for.
// With `shares` 0 each program takes a unit. Runs / parts, us, for 8 heads of 128
// (u: lengths from a quarter on), by the tiles of an even share:
//   9: 8 sequences of 8192 u 24.4 / 23.6, 2 of 65536 u 26.7 / 24.0;
//   16: 1 of 65536 33.6 / 34.1, 8 of 8192 30.6 / 35.8;
//   18: 16 of 8192 u 37.0 / 43.4, 32 of 4096 u 36.5 / 41.3;
//   32: 8 of 16384 51.0 / 60.7, 16 of 8192 50.8 / 51.2, 32 of 4096 49.6 / 49.6;
//   38: 16 of 16384 u 62.6 / 89.9; 60: 48 of 8192 u 89.4 / 130.
// So runs are the better ones from about 12 on; kLong is above that.
constexpr int kLong = 24;

struct Deal {
  const int32_t* lens;
  int batch, units_each;  // units of a sequence
  int q_len, held, window, sinks, shares;

  int lane, len0;  // the lane's own sequence of the first 64, its length

  __device__ __forceinline__ Deal(const newt_cached_attention_params& p, int row_tiles, int shares_)
      : lens(p.lens), batch((int)p.batch), units_each(row_tiles * p.cache.kv_heads),
        q_len((int)p.q_len), held((int)(p.table_width * p.cache.block_size)),
        window(p.window ? (int)p.window : kNoWindow), sinks((int)p.sinks), shares(shares_),
        lane(threadIdx.x & 63), len0(lane < batch ? lens[lane] : 0) {}

  // Lengths may be any number. Those near 2^31 are taken a little shorter, so
  // that the key numbers of tiles asked for ahead, up to 10 tiles behind the
  // range, fit an int; tables hold fewer than 2^30 tokens, so nothing else
  // changes.
  __device__ __forceinline__ static int bounded(int n) {
    constexpr int most = 0x7fffffff - 16 * kTile;
    return n < 0 ? 0 : n < most ? n : most;
  }
  // A length, by the same wave-wide load for all that ask where there are up to
  // 64 sequences.
  __device__ __forceinline__ int length(int b) const {
    return bounded(b < 64 ? lane_of(len0, b) : lens[b]);
  }
  // tiles of a sequence, for all of its row tiles
  __device__ __forceinline__ int tiles_of(int len) const {
    const Range r(len - q_len, len - 1, len < held ? len : held, window, sinks);
    return r.tiles > 0 ? r.tiles : 1;
  }
  // those of the lane's own sequence of 64 from `c` on
  __device__ __forceinline__ int own_tiles(int c) const {
    if (c + lane >= batch) return 0;
    return tiles_of(bounded(c ? lens[c + lane] : len0));
  }
  struct Tiles {
    __device__ __forceinline__ int operator()(int tiles) const { return tiles; }
  };
  // t of the lanes up to this one
  __device__ __forceinline__ static int up_to(int t) {
    t += __builtin_amdgcn_update_dpp(0, t, 0x111, 0xF, 0xF, false);  // row_shr:1, 2, 4, 8
    t += __builtin_amdgcn_update_dpp(0, t, 0x112, 0xF, 0xF, false);
    t += __builtin_amdgcn_update_dpp(0, t, 0x114, 0xF, 0xF, false);
    t += __builtin_amdgcn_update_dpp(0, t, 0x118, 0xF, 0xF, false);
    t += __builtin_amdgcn_update_dpp(0, t, 0x142, 0xA, 0xF, false);  // row_bcast:15 to rows 1, 3
    t += __builtin_amdgcn_update_dpp(0, t, 0x143, 0xC, 0xF, false);  // row_bcast:31 to rows 2, 3
    return t;
  }
  __device__ __forceinline__ static int lane_of(int v, int lane) {
    return __builtin_amdgcn_readlane(v, lane);
  }
  // Something of each sequence, summed over all, and over those before
  // `b` if that is one. Every lane of a wave.
  template <typename F>
  __device__ __forceinline__ int sum(F of, int b, int& before) const {
    int all = 0;
    for (int c = 0; c < batch; c += 64) {
      const int own = of(own_tiles(c)), t = up_to(own);
      if (b >= c && b < c + 64) before = all + lane_of(t - own, b - c);
      all += lane_of(t, 63);
    }
    return all;
  }
  // The sequence within whose units place `at` of a line lies, each of them
  // `of(tiles)` long, and the first place of the sequence's.
  template <typename F>
  __device__ __forceinline__ int sequence(F of, int at, int& first) const {
    int all = 0;
    for (int c = 0; c < batch; c += 64) {
      const int own = of(own_tiles(c)), t = up_to(own);
      const u64 past = __ballot((all + t) * units_each > at);
      if (past) {
        const int l = __builtin_ctzll(past);
        first = (all + lane_of(t - own, l)) * units_each;
        return c + l;
      }
      all += lane_of(t, 63);
    }
    return -1;  // behind the line
  }
  // An even share of `places`, of one tile a wave at least.
  __device__ __forceinline__ int share(int places) const {
    const int n = (int)(((u32)places + shares - 1) / (u32)shares);
    return n > kWaves ? n : kWaves;
  }
  // Whether units are cut into parts, rather than the line into runs.
  __device__ __forceinline__ bool parts(int share) const {
    return share < kLong && batch * units_each < shares;
  }
  // Parts of a unit: one, and of the programs left its share by its tiles,
  // rounded down, so that all together are at most `shares`.
  struct Parts {
    float each;
    __device__ __forceinline__ int operator()(int tiles) const {
      const int n = (int)((float)tiles * each), most = (tiles + kWaves - 1) / kWaves;
      return tiles == 0 ? 0 : n < 1 ? 1 : n < most ? n : most;
    }
  };
  __device__ __forceinline__ Parts parts_of(int places) const {
    return {(float)(shares - batch * units_each) / (float)places * 0.9999f};
  }
};

// What a wave does of a unit.
template <typename T, int D, int MT>
struct Wave {
  typedef typename frag<T>::type TX;
  static constexpr bool kExact = !__is_same(T, bf16);
  static constexpr int ROWS = 16 * MT;
  static constexpr int STEPS = D / 32;  // of the score product
  static constexpr int DT = D / 16;     // tiles of head dims
  static constexpr int KV4 = D / 64;    // 16-byte pieces of a key row a lane holds

  const newt_cached_attention_params& p;
  const int lane, n, g, size, shift, kv_heads;
  int head;
  const int32_t* table;
  TX q[MT][STEPS];
  int position[MT];
  float m[MT], l[MT];
  f32x4 acc[MT][DT];
  // the tile at hand and, for the next, what is on its way
  u32x4 kb[4][KV4], vb[DT];
  int k_entry, v_entry;  // blocks of tokens 16 (n / 4) on, for keys, and 16 g on, for values
  float next_k_scale, next_v_scale;
  bool in, next_in;      // whether there are the tokens from 16 g on
  int64_t values_page;   // the block and head that hold them

  __device__ __forceinline__ Wave(const newt_cached_attention_params& p_)
      : p(p_), lane(threadIdx.x & 63), n(lane & 15), g(lane >> 4), size(p.cache.block_size),
        shift(__builtin_ctz(size)), kv_heads(p.cache.kv_heads) {}

  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      m[mt] = -kInf;
      l[mt] = 0.0f;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) acc[mt][dt] = (f32x4)(0.0f);
    }
  }

  // Queries and positions of the unit's rows.
  __device__ __forceinline__ void begin(int b, int head_, int r0, int len) {
    head = head_;
    table = p.table + b * p.table_stride;
    const int group = p.heads / kv_heads, all_rows = (int)p.q_len * group;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      const int r = r0 + 16 * mt + n;
      const bool live = r < all_rows;
      position[mt] = live ? len - (int)p.q_len + r / group : -1;
      const T* from = (const T*)p.q + (live ? Rows{p.q_stride_b, p.q_stride_h, p.q_stride_t}.at(
                                                  b, head * group + r % group, r / group) : 0) +
                      D / 4 * g;
#pragma unroll
      for (int s = 0; s < STEPS; ++s) {
        T t[8];  // rows behind the last one take the first one's, and see nothing
        newt::load_vec<T, 8>(from + 8 * s, t, newt::any_align());
#pragma unroll
        for (int i = 0; i < 8; ++i) q[mt][s][i] = p.scale < 0.0f ? -t[i] : t[i];
      }
    }
    clear();
  }

  // A row tile's blocks are read by it alone where there is one row tile: then
  // they need not stay in the caches (read at 6.65 TB/s so, 5.95 without).
  __device__ __forceinline__ static u32x4 load(const unsigned char* at) {
    if constexpr (MT == 1) return __builtin_nontemporal_load((const u32x4*)at);
    else return *(const u32x4*)at;
  }

  __device__ __forceinline__ void ask_blocks(int key, int hi) {
    const int k_token = key + 16 * (n >> 2), v_token = key + 16 * g;
    k_entry = table[k_token < hi ? k_token >> shift : 0];
    v_entry = table[v_token < hi ? v_token >> shift : 0];
  }
  __device__ __forceinline__ void ask_keys(int key, int hi) {
    // a block that is not there: another one is read in its place
    const bool k_in = (key + 16 * (n >> 2) < hi) & ((u32)k_entry < (u32)p.cache.blocks);
    next_in = (key + 16 * g < hi) & ((u32)v_entry < (u32)p.cache.blocks);
    const int64_t page = (int64_t)(k_in ? k_entry : 0) * kv_heads + head;
    values_page = (int64_t)(next_in ? v_entry : 0) * kv_heads + head;
    const unsigned char* k = (const unsigned char*)p.cache.k +
                             (page * size + ((key + 16 * (n >> 2)) & (size - 1)) + (n & 3)) * D +
                             D / 4 * g;
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int c = 0; c < KV4; ++c) kb[t][c] = load(k + 4 * t * D + 16 * c);
    next_k_scale = p.cache.k_scale[values_page];
    next_v_scale = p.cache.v_scale[values_page];
  }
  __device__ __forceinline__ void ask_values(int key) {
    const unsigned char* v = (const unsigned char*)p.cache.v + (values_page * D + n) * size +
                             ((key + 16 * g) & (size - 1));
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) vb[dt] = load(v + 16 * dt * size);
    in = next_in;
  }

  // The tile from `key` on. With MORE there is a next one, whose keys are asked
  // for when this one's are used up and whose values when those are: with a
  // branch in MORE's place the waits for values would be for the next keys too.
  template <bool MORE, bool CAREFUL>
  __device__ __forceinline__ void tile(const Range& range, int key, int next, int after) {
    const bool bad = __ballot(!in) != 0;  // the groups of 16 cover the whole tile
    float k_scale = next_k_scale * (__builtin_fabsf(p.scale) * kLog2e), v_scale = next_v_scale;
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
    if constexpr (MORE) {
      ask_keys(next, range.hi);
      ask_blocks(after, range.hi);
    }
    // bit j: whether the row sees this lane's j-th token
    u32 seen[MT];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) seen[mt] = 0xffffu;
    if constexpr (CAREFUL) {
      // rounded, in no fma with the maximum
#pragma clang fp contract(off)
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int t = 0; t < 4; ++t) s[mt][t] *= k_scale;
      k_scale = 1.0f;
    } else {
      // scores of 0 times the scale, and masked ones, stay what they are
      k_scale = k_scale < 1e-37f ? 1e-37f : k_scale;
    }
    if (CAREFUL || bad || !range.whole(key)) {
      const int at = key + 16 * g;
      if (!CAREFUL && !bad && key >= range.sinks && range.hi > range.last) {
        // no sinks here, and the tokens go on to the last query's: the window alone
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          const int back = position[mt] - at;
#pragma unroll
          for (int j = 0; j < 16; ++j)
            s[mt][j / 4][j % 4] =
                (u32)(back - j) < (u32)range.window ? s[mt][j / 4][j % 4] : -kInf;
        }
      } else {
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            const bool sees = in & range.sees(position[mt], at + j);
            s[mt][j / 4][j % 4] = sees ? s[mt][j / 4][j % 4] : -kInf;
            if constexpr (CAREFUL) seen[mt] &= sees ? ~0u : ~(1u << j);
          }
      }
      // bytes of tokens that no row sees may hold anything: as zeros; and so
      // may the scales of a block that holds no other
      bool any = false;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        u32 keep = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const bool one = in & range.any(at + 4 * w + j);
          keep |= one ? 0xffu << (8 * j) : 0u;
          any |= one;
        }
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) vb[dt][w] &= keep;
      }
      k_scale = any ? k_scale : 1.0f;
      v_scale = any ? v_scale : 0.0f;
      if constexpr (CAREFUL) keep_apart(seen);
    }
    bf16x8 hi[MT][2], lo[MT][2];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      float most = s[mt][0][0];
#pragma unroll
      for (int j = 1; j < 16; ++j) most = __builtin_fmaxf(most, s[mt][j / 4][j % 4]);
      most = newt::lane_reduce<newt::Max, 48>(most * k_scale);
      if (__ballot(most > m[mt] + (CAREFUL ? 0.0f : kSlack))) {
        const float to = __builtin_fmaxf(m[mt], most);
        const float f = m[mt] == -kInf ? 0.0f : __builtin_amdgcn_exp2f(m[mt] - to);
        l[mt] *= f;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) acc[mt][dt] *= f;
        m[mt] = to;
      }
      const float ref = m[mt] == -kInf ? 0.0f : m[mt];
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const float w = __builtin_amdgcn_exp2f(__builtin_fmaf(s[mt][j / 4][j % 4], k_scale, -ref));
        l[mt] += w;
        float scaled = w * v_scale;
        // a token that is not seen weighs nothing, whatever its block's scale
        if constexpr (CAREFUL) scaled = (seen[mt] >> j) & 1 ? scaled : 0.0f;
        hi[mt][j / 8][j % 8] = (bf16)scaled;
        if constexpr (kExact)
          lo[mt][j / 8][j % 8] = (bf16)(scaled - (float)hi[mt][j / 8][j % 8]);
      }
    }
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        const bf16x8 a = from_bytes<bf16>::get(vb[dt][2 * u], vb[dt][2 * u + 1]);
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          acc[mt][dt] = newt::mfma_16x16x32(a, hi[mt][u], acc[mt][dt]);
          if constexpr (kExact) acc[mt][dt] = newt::mfma_16x16x32(a, lo[mt][u], acc[mt][dt]);
        }
      }
    if constexpr (MORE) ask_values(next);
  }

  // Takes NaN out of the values, into the accumulators of the rows that see
  // them: their number among a row's visible tokens by a product of 0s and 1s.
  __device__ __forceinline__ void keep_apart(const u32* seen) {
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const u32 n0 = nan_bytes(vb[dt][2 * u]), n1 = nan_bytes(vb[dt][2 * u + 1]);
        if (!__ballot((n0 | n1) != 0)) continue;
        bf16x8 is;
#pragma unroll
        for (int j = 0; j < 8; ++j)
          is[j] = (bf16)(((j < 4 ? n0 : n1) >> (8 * (j % 4) + 7)) & 1 ? 1.0f : 0.0f);
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          bf16x8 sees;
#pragma unroll
          for (int j = 0; j < 8; ++j)
            sees[j] = (bf16)((seen[mt] >> (8 * u + j)) & 1 ? 1.0f : 0.0f);
          const f32x4 count = newt::mfma_16x16x32(is, sees, (f32x4)(0.0f));
#pragma unroll
          for (int e = 0; e < 4; ++e)
            acc[mt][dt][e] = count[e] > 0.0f ? __builtin_nanf("") : acc[mt][dt][e];
        }
        vb[dt][2 * u] &= ~(n0 | (n0 - (n0 >> 7)));
        vb[dt][2 * u + 1] &= ~(n1 | (n1 - (n1 >> 7)));
      }
  }

  // Every kWaves-th of the tiles [from, to).
  __device__ __forceinline__ void attend(const Range& range, int from, int to) {
    if (from >= to) return;
    ask_blocks(range.tile(from), range.hi);
    ask_keys(range.tile(from), range.hi);
    ask_blocks(range.tile(from + kWaves), range.hi);
    ask_values(range.tile(from));
    int i = from;
    for (; i + kWaves < to; i += kWaves)
      tile<true, false>(range, range.tile(i), range.tile(i + kWaves), range.tile(i + 2 * kWaves));
    tile<false, false>(range, range.tile(i), 0, 0);
    // 0 times NaN is NaN: where there is any in a sum or an accumulator, again,
    // with the NaN among values and scales kept from the rows that do not see
    // them; and where scores are beyond kExact
    float check = 0.0f;
    bool again = false;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      check += l[mt] * 0.0f;
      again |= beyond_exact(m[mt]);
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int e = 0; e < 4; ++e) check += acc[mt][dt][e] * 0.0f;
    }
    if (!__ballot(!(check == 0.0f) | again)) return;
    clear();
    for (i = from; i < to; i += kWaves) {
      ask_blocks(range.tile(i), range.hi);
      ask_keys(range.tile(i), range.hi);
      ask_values(range.tile(i));
      tile<false, true>(range, range.tile(i), 0, 0);
    }
  }
};

// Partial results of a share: of the unit that it does not begin (0), and of
// the one that it begins and does not end (1).
template <int D, int ROWS>
struct Slots {
  float* acc;
  float* m;
  float* l;
  __host__ __device__ Slots(void* workspace, int shares) {
    acc = (float*)workspace;
    m = acc + (int64_t)2 * shares * ROWS * D;
    l = m + (int64_t)2 * shares * ROWS;
  }
  static size_t bytes(int shares) { return (size_t)2 * shares * ROWS * (D + 2) * sizeof(float); }
};

template <typename T, int D, int MT>
__global__ void __launch_bounds__(64 * kWaves, occupancy(D, MT))
cached_attention_kernel(newt_cached_attention_params p, int row_tiles, int shares) {
  typedef Wave<T, D, MT> W;
  constexpr int ROWS = W::ROWS, PITCH = D + 4;
  __shared__ float sm[kWaves][16], sl[kWaves][16];
  __shared__ float sacc[kWaves][16 * PITCH];
  const int wave = wave_id(), lane = threadIdx.x & 63;
  const int kv_heads = p.cache.kv_heads, group = p.heads / kv_heads;
  const int q_len = (int)p.q_len, all_rows = q_len * group;
  const Deal deal(p, row_tiles, shares);
  const Slots<D, ROWS> slots(p.workspace, shares);

  // the share's place in the line, and how much of it is left
  int b, unit, from, left;  // a sequence, one of its units, a tile of that
  if (shares) {
    int first = 0;
    const int places = deal.sum(Deal::Tiles(), -1, first) * deal.units_each;
    const int share = deal.share(places);
    if (deal.parts(share)) {
      const Deal::Parts parts = deal.parts_of(places);
      b = deal.sequence(parts, blockIdx.x, first);
      if (b < 0) return;
      const int tiles = deal.tiles_of(deal.length(b));
      const u32 n = parts(tiles), part = (blockIdx.x - first) % n;
      unit = (blockIdx.x - first) / n;
      from = (u32)tiles * part / n;
      left = (u32)tiles * (part + 1) / n - from;
    } else {
      const u32 at = (u32)blockIdx.x * share;  // at most `shares` tiles behind the line
      if (at >= (u32)places) return;
      left = places - (int)at < share ? places - (int)at : share;
      b = deal.sequence(Deal::Tiles(), (int)at, first);
      const u32 tiles = deal.tiles_of(deal.length(b));
      unit = ((int)at - first) / tiles;
      from = ((int)at - first) % tiles;
    }
  } else {
    b = blockIdx.x / deal.units_each;
    unit = blockIdx.x % deal.units_each;
    from = 0;
    left = 0x7fffffff;
  }
  W w(p);
  for (;;) {
    const int len = deal.length(b), tiles = deal.tiles_of(len);
    const int to = tiles - from < left ? tiles : from + left;
    const int head = unit % kv_heads, r0 = unit / kv_heads * ROWS;
    const int r1 = r0 + ROWS < all_rows ? r0 + ROWS : all_rows;
    const Range range(len - q_len + r0 / group, len - q_len + (r1 - 1) / group,
                      len < deal.held ? len : deal.held, deal.window, deal.sinks);
    w.begin(b, head, r0, len);
    // the line has as many tiles for each row tile as for all together
    w.attend(range, from + wave, to < range.tiles ? to : range.tiles);

    // the waves' results joined through LDS, 16 rows at a time
    const bool part = from > 0 || to < tiles;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      const int n = lane & 15, g = lane >> 4;
      const float sum = newt::lane_reduce<newt::Sum, 48>(w.l[mt]);
      if (g == 0) {
        sm[wave][n] = w.m[mt];
        sl[wave][n] = sum;
      }
      __syncthreads();
      float M = sm[0][n];
#pragma unroll
      for (int i = 1; i < kWaves; ++i) M = newt::Max::op(M, sm[i][n]);
      const float f = w.m[mt] == -kInf ? 0.0f : __builtin_amdgcn_exp2f(w.m[mt] - M);
#pragma unroll
      for (int dt = 0; dt < W::DT; ++dt)
        *(f32x4*)&sacc[wave][n * PITCH + 16 * dt + 4 * g] = w.acc[mt][dt] * f;
      __syncthreads();
      // 16 threads a row, each D / 16 of its dims in runs of 4
      const int row = threadIdx.x >> 4, piece = threadIdx.x & 15;
      const int r = r0 + 16 * mt + row;
      if (r < all_rows) {
        float most = sm[0][row];
#pragma unroll
        for (int i = 1; i < kWaves; ++i) most = newt::Max::op(most, sm[i][row]);
        float total = 0.0f;
#pragma unroll
        for (int i = 0; i < kWaves; ++i)
          total += sm[i][row] == -kInf ? sl[i][row]
                                       : sl[i][row] * __builtin_amdgcn_exp2f(sm[i][row] - most);
        const int64_t at = ((int64_t)2 * blockIdx.x + (from == 0)) * ROWS + 16 * mt + row;
        if (part && piece == 0) {
          slots.m[at] = most;
          slots.l[at] = total;
        }
        T* out = (T*)p.out + Rows{p.o_stride_b, p.o_stride_h, p.o_stride_t}.at(
                                 b, head * group + r % group, r / group);
#pragma unroll
        for (int c = 0; c < D / 64; ++c) {
          const int d = 64 * c + 4 * piece;
          f32x4 o = *(const f32x4*)&sacc[0][row * PITCH + d];
#pragma unroll
          for (int i = 1; i < kWaves; ++i) o += *(const f32x4*)&sacc[i][row * PITCH + d];
          if (part) {
            *(f32x4*)(slots.acc + at * D + d) = o;
          } else {
            T t[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) t[e] = (T)(total == 0.0f ? 0.0f : o[e] / total);
            newt::store_vec<T, 4>(out + d, t, newt::any_align());
          }
        }
      }
      __syncthreads();
    }
    left -= to - from;
    if (!shares || left <= 0) return;
    from = 0;
    if (++unit == deal.units_each) {
      unit = 0;
      ++b;
    }
  }
}

// The units that several shares did: o = sum acc 2^(m - M) / sum l 2^(m - M).
// One wave a row.
template <typename T, int D, int ROWS>
__global__ void __launch_bounds__(256)
cached_join_kernel(newt_cached_attention_params p, int row_tiles, int shares) {
  const int lane = threadIdx.x & 63;
  const int kv_heads = p.cache.kv_heads, group = p.heads / kv_heads;
  const int all_rows = (int)p.q_len * group;
  const u32 w = blockIdx.x * 4 + wave_id();
  if (w >= (u32)p.batch * kv_heads * all_rows) return;
  const int r = w % all_rows, head = w / all_rows % kv_heads, b = w / all_rows / kv_heads;
  const Deal deal(p, row_tiles, shares);
  int before = 0;
  const int places = deal.sum(Deal::Tiles(), b, before) * deal.units_each;
  const u32 share = deal.share(places), tiles = deal.tiles_of(deal.length(b));
  const int unit = r / ROWS * kv_heads + head;
  int w0, splits;
  if (deal.parts(share)) {
    const Deal::Parts parts = deal.parts_of(places);
    deal.sum(parts, b, before);
    splits = parts(tiles);
    w0 = before * deal.units_each + unit * splits;
  } else {
    const u32 first = before * deal.units_each + unit * tiles;
    w0 = first / share;
    splits = (int)((first + tiles - 1) / share) - w0 + 1;
  }
  if (splits == 1) return;  // its program has written it

  const Slots<D, ROWS> slots(p.workspace, shares);
  // the unit's first share has begun it, the others have not
  const auto slot = [&](int s) { return (2 * (w0 + s) + (s == 0)) * ROWS + r % ROWS; };
  // 16 bytes a lane: the wave reads SIDE shares at a time, AT_ONCE such pieces
  // without waiting in between
  constexpr int WIDE = D / 4, SIDE = 64 / WIDE, AT_ONCE = 8;
  const int side = lane / WIDE, d = lane % WIDE * 4;
  float M = -kInf, total = 0.0f;
  f32x4 acc = (f32x4)(0.0f);
  for (int s = side; s - side < splits; s += SIDE * AT_ONCE) {
    f32x4 a[AT_ONCE];
    float m[AT_ONCE], l[AT_ONCE];
#pragma unroll
    for (int j = 0; j < AT_ONCE; ++j) {
      const bool in = s + j * SIDE < splits;
      const int at = slot(in ? s + j * SIDE : 0);
      a[j] = *(const f32x4*)(slots.acc + (int64_t)at * D + d);
      m[j] = slots.m[at];
      l[j] = slots.l[at];
      if (!in) {
        a[j] = (f32x4)(0.0f);
        m[j] = -kInf;
        l[j] = 0.0f;
      }
    }
    float most = M;
#pragma unroll
    for (int j = 0; j < AT_ONCE; ++j) most = newt::Max::op(most, m[j]);
    const float old = M == -kInf ? 0.0f : __builtin_amdgcn_exp2f(M - most);
    total *= old;
    acc *= old;
    M = most;
#pragma unroll
    for (int j = 0; j < AT_ONCE; ++j) {
      // without a maximum a share has seen nothing, or NaN
      const float f = m[j] == -kInf ? 0.0f : __builtin_amdgcn_exp2f(m[j] - M);
      total += m[j] == -kInf ? l[j] : l[j] * f;
      acc += a[j] * f;
    }
  }
  // and the sides', each relative to its own maximum
  float most = M;
  if constexpr (SIDE > 2) most = newt::lane_reduce<newt::Max, 16>(most);
  if constexpr (SIDE > 1) most = newt::lane_reduce<newt::Max, 32>(most);
  const float own = M == -kInf ? 0.0f : __builtin_amdgcn_exp2f(M - most);
  total = M == -kInf ? total : total * own;
  acc *= own;
  const auto sides = [](float v) {
    if constexpr (SIDE > 2) v = newt::lane_reduce<newt::Sum, 16>(v);
    if constexpr (SIDE > 1) v = newt::lane_reduce<newt::Sum, 32>(v);
    return v;
  };
  total = sides(total);
#pragma unroll
  for (int i = 0; i < 4; ++i) acc[i] = sides(acc[i]);
  if (side) return;
  T t[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) t[i] = (T)(total == 0.0f ? 0.0f : acc[i] / total);
  T* to = (T*)p.out + Rows{p.o_stride_b, p.o_stride_h, p.o_stride_t}.at(
                          b, head * group + r % group, r / group) + d;
  newt::store_vec<T, 4>(to, t, newt::any_align());
}

struct Launch {
  int rows, row_tiles, shares;
  int64_t units;
};

// The shape of a launch, from sizes that the host knows: the table's width
// bounds the lengths. A program a unit (first) or tiles dealt out by the lengths
// (second; * what the rule takes), us, 32 heads of 128 over 8, one token:
//   1 sequence of 256, 512, 768, 1024 tokens: 5.6* 7.9, 7.5* 10.5, 9.4 12.2*, 12.7
//   12.7*; 24 of them: 6.9* 9.1, 9.7* 12.1, 12.3 14.9*, 14.9 17.4*;
//   32 of 1024 and 1536: 15.7* 18.3, 20.6 23.1*; 128: 47.8* 52.2, 67.7 72.3*;
//   64 of any length up to 1024 and 2048: 21.6* 48.8, 34.6 57.7*;
//   256 of 2048 and of up to 2048: 172 184*, 103 156*;
//   512 of 2048 and of up to 2048: 339* 365, 194* 265;
//   1, 8, 64 of 8192: 64 14*, 67 34*, 170 173*; 64 of 2048 to 8192: 137 117*.
// Dealing out pays for few units and long ones; the rule does it sooner than that.
Launch launch_of(const newt_cached_attention_params& p) {
  Launch r;
  const int64_t rows = p.q_len * (p.heads / p.cache.kv_heads);
  // two tiles of 16 rows share what is read; with head_dim 256 they would not
  // fit the registers
  r.rows = rows > 16 && p.cache.head_dim < 256 ? 32 : 16;
  r.row_tiles = (int)((rows + r.rows - 1) / r.rows);
  r.units = p.batch * p.cache.kv_heads * r.row_tiles;
  const int64_t tiles = most_tiles(p.table_width * p.cache.block_size, p.window, p.sinks, p.q_len);
  int64_t shares = 256 * occupancy(p.cache.head_dim, r.rows / 16);
  const int64_t most = (r.units * tiles + kWaves - 1) / kWaves;
  shares = shares < most ? shares : most;
  const bool whole = tiles <= 8 || (r.units >= 256 && tiles <= 16) || r.units >= 4096 ||
                     r.units * tiles >= kLimit;
  r.shares = whole ? 0 : (int)shares;
  return r;
}

template <int D>
size_t workspace_of(const Launch& r) {
  return r.rows == 16 ? Slots<D, 16>::bytes(r.shares) : Slots<D, 32>::bytes(r.shares);
}

template <typename T, int D, int MT>
int launch(const newt_cached_attention_params& p, const Launch& r, hipStream_t stream) {
  const char* const what = "newt_cached_attention";
  const int status = run(what, cached_attention_kernel<T, D, MT>, r.shares ? r.shares : r.units,
                         64 * kWaves, 0, stream, p, r.row_tiles, r.shares);
  if (status != NEWT_OK || !r.shares) return status;
  const int64_t waves = p.batch * p.heads * p.q_len;
  return run(what, cached_join_kernel<T, D, 16 * MT>, (waves + 3) / 4, 256, 0, stream, p,
             r.row_tiles, r.shares);
}

template <typename T, int D>
int by_rows(const newt_cached_attention_params& p, hipStream_t stream) {
  const Launch r = launch_of(p);
  if (r.shares && !p.workspace)
    return fail(NEWT_ERR_INVALID, "newt_cached_attention: null workspace");
  if (r.units > 0x7fffffff || p.batch * p.heads * p.q_len > 0x7fffffff)
    return fail(NEWT_ERR_INVALID, "newt_cached_attention: too many queries");
  if constexpr (D < 256)
    if (r.rows == 32) return launch<T, D, 2>(p, r, stream);
  return launch<T, D, 1>(p, r, stream);
}

template <typename T>
int by_dim(const newt_cached_attention_params& p, hipStream_t stream) {
  switch (p.cache.head_dim) {
    case 64: return by_rows<T, 64>(p, stream);
    case 128: return by_rows<T, 128>(p, stream);
    default: return by_rows<T, 256>(p, stream);
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
  return queries_wrong(p, p.cache.head_dim);
}

}  // namespace
}  // namespace newt_ops

extern "C" size_t newt_cached_attention_workspace(const newt_cached_attention_params* p) {
  using namespace newt_ops;
  if (!p || wrong(*p) || p->batch == 0 || p->q_len == 0) return 0;
  const Launch r = launch_of(*p);
  if (!r.shares) return 0;
  switch (p->cache.head_dim) {
    case 64: return workspace_of<64>(r);
    case 128: return workspace_of<128>(r);
    default: return workspace_of<256>(r);
  }
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
