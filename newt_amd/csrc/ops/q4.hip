// Products with 4-bit weights and a scale for each group of columns, up to 48 rows
// of x (more: q4_many.hip):
//   y[m][n] = sum_g s[n][g] (sum_k x[m][k] q[n][k] - z[n][g] sum_k x[m][k])
// and, for a gated feed-forward block, act(y of the gate) * (y of the rest).
// The weights' bytes bound it: each is read once, 16 bytes a lane in the order in
// which the matrix unit takes it, and no number of it goes through LDS. A weight
// becomes a 16-bit number without a conversion: its 4 bits are put below the point of
// a number in [1, 2), (16 + q) / 16, exactly. The products begin with minus the sum of
// x, which comes from one more product, of x and -1, for all rows of weights that a
// wave has; zeros take a sixteenth of it each:
//   sum_k x (q - z) = 16 ((sum_k x (16 + q) / 16 - sum_k x) - z / 16 sum_k x)
// Everything up to the output's rounding is fp32; the factor 16 comes last, and for
// bf16 all of it is held 2^-12 times as large (kUnit), so that no group's sums overflow
// for any finite x and nothing does that the result does not. Where x holds an
// infinity its sum does, and the difference is no number.
// A wave takes NT tiles of 16 weight rows, MT tiles of 16 rows of x and every
// WAVES-th block of 128 columns; the waves' sums are joined in LDS in their order.
// bf16, groups of 128, three sets of weights in turn: 1 x 4096 x 6144 5.8 us (2.3 TB/s);
// gated 1 x 4096 x 2 x 12288 11.6 us (4.6 TB/s); 4 x 4096 x 128000 to fp32 53.8 us
// (5.1 TB/s; the same weights again 45).
#include "q4.h"

namespace newt_ops {
namespace {

template <typename T, int NT, int MT, int WAVES, int GROUP, bool GATED>
__global__ void __launch_bounds__(64 * WAVES)
q4_kernel(newt_q4_params p, int n_blocks) {
  typedef typename frag<T>::type TX;
  constexpr int STEPS = GROUP / 32, PER = 128 / GROUP;  // of a group, groups of a block
  constexpr int SIZE = NT * MT * 256;                   // sums of a wave
  __shared__ __attribute__((aligned(16))) float sums[WAVES * SIZE];
  const int lane = threadIdx.x & 63, wave = wave_id(), part = lane >> 4, col = lane & 15;
  const int n_block = blockIdx.x % n_blocks, m_block = blockIdx.x / n_blocks;
  const int blocks = (int)((p.cols + 127) / 128), groups = blocks * PER;
  const int64_t tiles = (p.outputs + 15) / 16 * (GATED ? 2 : 1);
  const int64_t tile = (int64_t)n_block * NT;

  const u32x4* q[NT];
  int64_t at[NT];  // of scales and zeros
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int64_t t = tile + n < tiles ? tile + n : tiles - 1;
    q[n] = (const u32x4*)p.q + t * blocks * 64 + lane;
    at[n] = t * groups * 16 + 4 * part;
  }
  // Rows of x behind the last one are that one again, and columns behind the last
  // one the first ones: their sums are not stored, and multiplied by scales of 0.
  const T* x[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    const int64_t row = ((int64_t)m_block * MT + m) * 16 + col;
    x[m] = (const T*)p.x + (row < p.rows ? row : p.rows - 1) * p.x_stride + 8 * part;
  }
  const Widen<T> widen;
  TX minus;
#pragma unroll
  for (int i = 0; i < 8; ++i) minus[i] = (T)-kUnit<T>;
  f32x4 acc[NT][MT];
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int m = 0; m < MT; ++m) acc[n][m] = (f32x4)(0.0f);

  const auto all_blocks = [&](auto scale_type) {
    typedef decltype(scale_type) S;
    for (int b = wave; b < blocks; b += WAVES) {
      u32x4 w[NT];
      S s[PER][NT][4];
      u32 z[PER][NT];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        w[n] = q[n][(int64_t)b * 64];
#pragma unroll
        for (int g = 0; g < PER; ++g) {
          const int64_t i = at[n] + (int64_t)(b * PER + g) * 16;
          // 0 for a group behind the last column, which a block's first one never is: 0 to 5%
          // of a call; a branch around such groups takes up to a third, zeros for x 12%
          u32x2 bits = *(const u32x2*)((const S*)p.scales + i);
          if (g > 0) bits &= b * 128 + g * GROUP < (int)p.cols ? ~0u : 0u;
          __builtin_memcpy(s[g][n], &bits, 8);
          z[g][n] = p.zeros ? *(const u32*)((const unsigned char*)p.zeros + i) : 0x08080808u;
        }
      }
      TX v[MT][4];
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int k = b * 128 + 32 * j < (int)p.cols ? b * 128 + 32 * j : 0;
          T t[8];
          newt::load_vec<T, 8>(x[m] + k, t, newt::any_align());
          v[m][j] = __builtin_bit_cast(
              TX, newt::pack8(t[0], t[1], t[2], t[3], t[4], t[5], t[6], t[7]));
        }
#pragma unroll
      for (int g = 0; g < PER; ++g) {
        // minus the sum of x, the same in all rows, and a sixteenth of it
        f32x4 less[MT];
        float part_of[MT];
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          less[m] = (f32x4)(0.0f);
#pragma unroll
          for (int j = 0; j < STEPS; ++j)
            less[m] = newt::mfma_16x16x32(minus, v[m][g * STEPS + j], less[m]);
          part_of[m] = less[m][0] * 0.0625f;
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          f32x4 sum[MT];  // of x q / 16
#pragma unroll
          for (int m = 0; m < MT; ++m) sum[m] = less[m];
#pragma unroll
          for (int j = 0; j < STEPS; ++j) {
            const TX a = widen(w[n][g * STEPS + j]);
#pragma unroll
            for (int m = 0; m < MT; ++m)
              sum[m] = newt::mfma_16x16x32(a, v[m][g * STEPS + j], sum[m]);
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float scale = newt::to_f32(s[g][n][i]);
            const float zero = (float)((z[g][n] >> (8 * i)) & 255);
#pragma unroll
            for (int m = 0; m < MT; ++m)
              acc[n][m][i] = __builtin_fmaf(__builtin_fmaf(part_of[m], zero, sum[m][i]), scale,
                                            acc[n][m][i]);
          }
        }
      }
    }
  };
  if (p.scale_dtype == NEWT_F16) all_blocks(f16());
  else all_blocks(bf16());
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int m = 0; m < MT; ++m)
      *(f32x4*)(sums + wave * SIZE + ((n * MT + m) * 64 + lane) * 4) = acc[n][m];
  __syncthreads();
  // 4 neighbouring outputs of a row of x at a time
  constexpr int OUT = GATED ? NT / 2 : NT;
  const auto joined = [&](int n, int m, int l) {
    f32x4 t = (f32x4)(0.0f);
#pragma unroll
    for (int i = 0; i < WAVES; ++i)
      t += *(const f32x4*)(sums + i * SIZE + ((n * MT + m) * 64 + l) * 4);
    return t * kWhole<T>;
  };
  for (int e = threadIdx.x; e < OUT * MT * 64; e += 64 * WAVES) {
    const int l = e & 63, m = e / 64 % MT, n = e / 64 / MT;
    const int64_t row = ((int64_t)m_block * MT + m) * 16 + (l & 15);
    const int64_t first = ((int64_t)n_block * OUT + n) * 16 + 4 * (l >> 4);
    if (row >= p.rows || first >= p.outputs) continue;
    f32x4 y;
    if constexpr (GATED) {
      const f32x4 gate = joined(2 * n, m, l), up = joined(2 * n + 1, m, l);
#pragma unroll
      for (int i = 0; i < 4; ++i) y[i] = activate(gate[i], p.act) * up[i];
    } else {
      y = joined(n, m, l);
    }
    store4<T>(p, row, first, y);
  }
}

template <typename T, int GROUP, bool GATED>
int launch(const newt_q4_params& p, hipStream_t stream) {
  const int64_t tiles = (p.outputs + 15) / 16 * (GATED ? 2 : 1);
  const auto go = [&](auto nt, auto mt, auto waves) {
    constexpr int NT = decltype(nt)::value, MT = decltype(mt)::value;
    constexpr int WAVES = decltype(waves)::value;
    const int64_t n_blocks = (tiles + NT - 1) / NT, m_blocks = (p.rows + 16 * MT - 1) / (16 * MT);
    if (n_blocks * m_blocks > 0x7fffffff)
      return fail(NEWT_ERR_INVALID, "newt_q4_matmul: too many rows");
    return run("newt_q4_matmul", q4_kernel<T, NT, MT, WAVES, GROUP, GATED>, n_blocks * m_blocks,
               64 * WAVES, 0, stream, p, (int)n_blocks);
  };
#define NEWT_TILE(NT, MT, WAVES)                                           \
  go(std::integral_constant<int, NT>(), std::integral_constant<int, MT>(), \
     std::integral_constant<int, WAVES>())
  // Wide programs read x less often, narrow ones of many waves have more of the
  // weights on their way where there are few: us of (NT, WAVES) for bf16, groups of 128,
  //   1 x 16384 x 2048: (1, 16) 9.7, (2, 16) 13.3, (2, 8) 15.3, (4, 8) 24;
  //   1 x 4096 x 6144: (1, 16) 6.7, (2, 8) 6.3, (4, 8) 8.7; 16 rows 11.2 / 7.9 / 9.8;
  //   gated 1 x 4096 x 2 x 12288: (2, 8) 11.9, (4, 8) 13.5, (4, 4) 15.3;
  //   16 x 4096 x 28672: (2, 8) 22, (4, 4) 17; 4 x 4096 x 128000: 62, 57;
  //   gated 32 x 2048 x 2 x 5504 fp16, groups of 64: (2, 8) 12.3, (4, 4) 12.2, (4, 8) 9.7;
  //   of 48 rows: 17.5, 15.4, 11.6.
  // Two blocks at a time take as long as one or longer: waves, not the loads of a
  // wave, hide the memory's latency (6.3 and 6.3, 13.5 and 11.9, 63.7 and 62.4 us).
  if (p.rows <= 16) {
    if constexpr (!GATED)
      if (tiles <= 128) return NEWT_TILE(1, 1, 16);
    if (tiles > 2048 || (tiles > 1024 && p.rows > 4)) return NEWT_TILE(4, 1, 4);
    return NEWT_TILE(2, 1, 8);
  }
  if constexpr (GROUP > 32)  // whose scales would not fit the registers
    if (tiles >= 512) return p.rows <= 32 ? NEWT_TILE(4, 2, 8) : NEWT_TILE(4, 3, 8);
  return p.rows <= 32 ? NEWT_TILE(2, 2, 8) : NEWT_TILE(2, 3, 8);
#undef NEWT_TILE
}

template <typename T, bool GATED>
int by_group(const newt_q4_params& p, hipStream_t stream) {
  switch (p.group) {
    case 32: return launch<T, 32, GATED>(p, stream);
    case 64: return launch<T, 64, GATED>(p, stream);
    default: return launch<T, 128, GATED>(p, stream);
  }
}

template <typename T>
int by_act(const newt_q4_params& p, hipStream_t stream) {
  return p.act == NEWT_ACT_NONE ? by_group<T, false>(p, stream) : by_group<T, true>(p, stream);
}

// more take the tiles of q4_many.hip: us for 64 rows, gated, 4096 x 2 x 12288 bf16 44
// here, 32 there; 2048 x 2 x 5504 fp16, groups of 64, 17 and 22; 48 rows of the first
// 31 and 31, of the second 11.6 and 19.7. One border for all sizes is a compromise: 48
// rows here and 49 there take 34 and 33 for the first, 11.5 and 20 for the second, 16 and
// 20 for 4096 x 6144, 143 and 93 for 4096 x 128000.
constexpr int64_t kFewRows = 48;

const char* wrong(const newt_q4_params& p) {
  if (p.rows < 0 || p.outputs < 0 || p.cols <= 0) return "bad size";
  if (p.rows >= 1 << 30 || p.outputs >= 1 << 30 || p.cols >= 1 << 30)
    return "sizes stay below 2^30";
  if (p.group != 32 && p.group != 64 && p.group != 128)
    return "groups are of 32, 64 or 128 columns";
  if (p.cols % p.group) return "columns have to be whole groups";
  if (p.act != NEWT_ACT_NONE && p.act != NEWT_ACT_SILU && p.act != NEWT_ACT_GELU)
    return "unknown activation";
  if (p.act != NEWT_ACT_NONE && p.bias) return "a gated product has no bias";
  if (p.dtype != NEWT_F16 && p.dtype != NEWT_BF16) return "x is fp16 or bf16";
  if (p.scale_dtype != NEWT_F16 && p.scale_dtype != NEWT_BF16) return "scales are fp16 or bf16";
  if (p.out_dtype != p.dtype && p.out_dtype != NEWT_F32) return "out is of x's type or fp32";
  if (p.rows > 1 && p.out_stride < p.outputs) return "rows of out overlap";
  return nullptr;
}

}  // namespace
}  // namespace newt_ops

extern "C" size_t newt_q4_matmul_workspace(const newt_q4_params* p) {
  using namespace newt_ops;
  if (!p || wrong(*p) || p->rows <= kFewRows || p->outputs == 0) return 0;
  return q4_many_workspace(*p);
}

extern "C" int newt_q4_matmul(const newt_q4_params* params, void* stream) {
  using namespace newt_ops;
  if (!params) return fail(NEWT_ERR_INVALID, "newt_q4_matmul: null params");
  const newt_q4_params& p = *params;
  if (const char* w = wrong(p)) return fail(NEWT_ERR_INVALID, "newt_q4_matmul: %s", w);
  if (p.rows == 0 || p.outputs == 0) return NEWT_OK;
  if (!p.x || !p.q || !p.scales || !p.out)
    return fail(NEWT_ERR_INVALID, "newt_q4_matmul: null tensor");
  if (((uintptr_t)p.q | (uintptr_t)p.scales | (uintptr_t)p.zeros) & 15)
    return fail(NEWT_ERR_INVALID, "newt_q4_matmul: weights are not aligned");
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (p.rows > kFewRows) return q4_many(p, s);
  if (out_meets(p)) return fail(NEWT_ERR_INVALID, "newt_q4_matmul: out overlaps x or bias");
  return p.dtype == NEWT_F16 ? by_act<f16>(p, s) : by_act<bf16>(p, s);
}
