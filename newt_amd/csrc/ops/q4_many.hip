// Products with 4-bit weights for many rows of x, which the matrix unit bounds.
// A program takes 64 rows of x and 256 rows of weights, each of its 4 waves 64 of
// those: 128 columns of x are staged in LDS for all waves, while the weights go
// from memory to the wave that multiplies them and become operands there,
//   S[n][m] += W[n][k] x[m][k] by v_mfma_f32_32x32x16,
// so that a word of weights is widened once for 64 rows and a piece of x is read
// from LDS twice for 128 rows of weights. As for few rows the sums hold (16 + z) /
// 16 times the sum of x too much. That is taken off within the matrix unit: one
// more step multiplies -1 and -z / 16, which bf16 holds exactly for any byte z, by
// the sum of x in three bf16 parts, exactly what fp32 holds; on the vector unit it
// would take as long as widening the weights. Each wave sums 16 rows of x for all, a
// block ahead, between its products. A group's sums then take their scales on the
// way into the accumulators, in fp32; up to the output all is held kUnit / 16 times
// as large.
// Few programs split the columns; a second kernel adds the parts in their order.
// bf16 512 x 4096 x 2 x 12288, gated, groups of 128: 123 us, 838 TFLOP/s (119 on
// another card); groups of 64 154, of 32 213 us. The products alone, with nothing
// loaded, widened or scaled, took 83 us of 121 (an eighth of them is what is taken
// off): under them the chip's power lets the clock fall to 1.5 GHz or so. Beside
// that, one at a time, the scales cost 8%, loading x 6%, its sums 5% (before they
// went between the products), widening and the operands' reads 7%, the weights'
// loads 1%. fp16 333 x 8192 x 2003 in groups of 32: 42 us (261 TFLOP/s), of 128 30
// us.
#include "q4.h"

namespace newt_ops {
namespace {

constexpr int kRows = 64, kTiles = 16, kBlock = 128;

template <typename T, typename S, int GROUP, bool DIRECT>
__global__ void __launch_bounds__(256, 2)
q4_many_kernel(newt_q4_params p, int m_blocks, int n_blocks, int per) {
  typedef typename frag<T>::type TX;
  constexpr int PER = kBlock / GROUP, STEPS = GROUP / 16;
  // three stages of x, [row][column], and of each wave's scales and zeros, [tile]
  // [group][16]
  constexpr int SCALES = 4 * PER * 2, ZEROS = 4 * PER;  // pieces of 16 bytes
  __shared__ __attribute__((aligned(16))) T x0[kRows * kBlock];
  __shared__ __attribute__((aligned(16))) T x1[kRows * kBlock];
  __shared__ __attribute__((aligned(16))) T x2[kRows * kBlock];
  __shared__ __attribute__((aligned(16))) unsigned char levels0[4 * 2048];
  __shared__ __attribute__((aligned(16))) unsigned char levels1[4 * 2048];
  __shared__ __attribute__((aligned(16))) unsigned char levels2[4 * 2048];
  __shared__ __attribute__((aligned(16))) bf16x4 sums[2][PER * kRows];
  const int lane = threadIdx.x & 63, wave = wave_id(), half = lane >> 5;
  const int program = by_die(blockIdx.x, gridDim.x);
  const int split = program / (m_blocks * n_blocks), unit = program % (m_blocks * n_blocks);
  const int n_block = unit / m_blocks, m_block = unit % m_blocks;
  const bool gated = p.act != NEWT_ACT_NONE;
  const int blocks = (int)((p.cols + kBlock - 1) / kBlock), groups = blocks * PER;
  const int tiles = (int)((p.outputs + 15) / 16) * (gated ? 2 : 1);
  const int tile = n_block * kTiles + wave * 4;
  const int from = split * per, to = from + per < blocks ? from + per : blocks;
  const int64_t m0 = (int64_t)m_block * kRows;
  const int rows = p.rows - m0 < kRows ? (int)(p.rows - m0) : kRows;

  // a lane's row of the two times 32 that its wave has
  const auto at = [&](int t) { return (int64_t)(t < tiles ? t : tiles - 1); };
  const char* const q = (const char*)p.q + at(tile) * blocks * 1024;
  u32 q_at[2];  // fewer than 2^19 blocks
#pragma unroll
  for (int f = 0; f < 2; ++f)
    q_at[f] = (u32)(at(tile + 2 * f + ((lane >> 4) & 1)) - at(tile)) * (u32)blocks * 1024 +
              (16 * half + (lane & 15)) * 16;
  // the pieces of its wave's scales and zeros that a lane stages
  const char* const levels_of[2] = {
      (const char*)p.scales + at(tile) * groups * 32,
      (const char*)(p.zeros ? p.zeros : p.scales) + at(tile) * groups * 16};
  const auto level_at = [&](int per) {  // pieces of a tile in a block
    return (u32)(at(tile + lane / per % 4) - at(tile)) * (u32)(blocks * per) * 16 + lane % per * 16;
  };
  const u32 scale_at = level_at(2 * PER), zero_at = level_at(PER);

  int row0, k0;
  newt::lds_tile_slot<T, kBlock>(threadIdx.x, row0, k0);
  const u32 x_at = (u32)(row0 * (int)p.x_stride + k0) * 2;
  const auto stage = [&](int b, T* to_lds, unsigned char* levels) {
    newt::lds_dma16_masked(levels_of[0] + (int64_t)b * (2 * PER * 16), scale_at, lane < SCALES,
                           levels + 2048 * wave);
    newt::lds_dma16_masked(levels_of[1] + (int64_t)b * (PER * 16), zero_at, lane < ZEROS,
                           levels + 2048 * wave + 1024);
    const T* base = (const T*)p.x + m0 * p.x_stride + b * kBlock;
    const int cols = (int)(p.cols - (int64_t)b * kBlock);
#pragma unroll
    for (int c = 0; c < kRows / 16; ++c) {
      // 16 rows on, a lane's place in them is the same
      const bool in = (row0 < rows - 16 * c) & (k0 < cols);
      if constexpr (DIRECT) {
        newt::lds_dma16_masked(base + 16 * c * p.x_stride, x_at, in,
                               to_lds + (c * 256 + 64 * wave) * 8);
      } else {
        T t[8] = {};
        if (in)
          newt::load_vec<T, 8>(base + (row0 + 16 * c) * p.x_stride + k0, t, newt::any_align());
        newt::store_vec<T, 8>(to_lds + (c * 256 + threadIdx.x) * 8, t);
      }
    }
  };

  f32x16 acc[2][2];
#pragma unroll
  for (int f = 0; f < 2; ++f)
#pragma unroll
    for (int m = 0; m < 2; ++m) acc[f][m] = (f32x16)(0.0f);
  const Widen<T> widen;
  const TX ones = __builtin_bit_cast(TX, widen.ones);

  // A block's x, scales, zeros and weights.
  const auto load = [&](int b, u32x4 (&w)[2][2], T* to_lds, unsigned char* levels) {
    b = b < to ? b : to - 1;
    stage(b, to_lds, levels);
#pragma unroll
    for (int f = 0; f < 2; ++f)
#pragma unroll
      for (int i = 0; i < 2; ++i)
        w[f][i] = *(const u32x4*)(q + (int64_t)b * 1024 + q_at[f] + 512 * i);
  };

  // The sums of 16 rows over 32 columns, times kUnit, and a group's in three parts.
  const auto add_32 = [&](const T* x_lds, int k, f32x4 all) {
    const TX x = __builtin_bit_cast(TX, newt::lds_frag_k<T, kBlock, 16>(x_lds, 16 * wave, k, lane));
    return newt::mfma_16x16x32(ones, x, all);
  };
  const auto keep = [&](const f32x4& all, bf16x4* to_sums) {
    const bf16 hi = (bf16)all[0];
    const float rest = all[0] - (float)hi;
    const bf16 mid = (bf16)rest;
    if (lane < 16)
      to_sums[16 * wave + lane] = bf16x4{hi, mid, (bf16)(rest - (float)mid), (bf16)0.0f};
  };

  // One block, while the one after the next is on its way: the next one is there,
  // and its sums come one block ahead, so that they need no barrier of their own.
  const auto step = [&](int b, const T* now, const unsigned char* levels, u32x4 (&v)[2][2],
                        const T* after, T* next, unsigned char* next_levels, u32x4 (&w)[2][2],
                        const bf16x4* own_sums, bf16x4* next_sums) {
    newt::wait_vmcnt<0>();
    __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0)
    newt::barrier_nofence();
    load(b + 2, w, next, next_levels);
    // not unrolled: groups side by side would not fit the registers
#pragma unroll 1
    for (int g = 0; g < PER; ++g) {
      f32x16 part[2][2];
#pragma unroll
      for (int f = 0; f < 2; ++f)
#pragma unroll
        for (int m = 0; m < 2; ++m) part[f][m] = (f32x16)(0.0f);
      // a step's operands are made while the one before it is multiplied
      TX x[2][2], a[2][2];
      const auto operands = [&](int i) {
#pragma unroll
        for (int m = 0; m < 2; ++m)
          x[i & 1][m] = __builtin_bit_cast(
              TX, newt::lds_frag_k<T, kBlock, 32>(now, 32 * m, 16 * (g * STEPS + i), lane));
#pragma unroll
        for (int f = 0; f < 2; ++f) a[i & 1][f] = widen(v[f][i & 1][i / 2]);
      };
      operands(0);
      f32x4 all = (f32x4)(0.0f);
#pragma unroll
      for (int i = 0; i < STEPS; ++i) {
        if (i + 1 < STEPS) operands(i + 1);
        if (i & 1) all = add_32(after, 16 * (g * STEPS + i - 1), all);
#pragma unroll
        for (int f = 0; f < 2; ++f)
#pragma unroll
          for (int m = 0; m < 2; ++m)
            part[f][m] = newt::mfma_32x32x16(a[i & 1][f], x[i & 1][m], part[f][m]);
        __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);  // LDS reads
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);  // a product
          __builtin_amdgcn_sched_group_barrier(0x002, 4, 0);  // vector instructions
        }
      }
      keep(all, next_sums + g * kRows);
      bf16x8 less_x[2];
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        const bf16x4 t = own_sums[g * kRows + 32 * m + (lane & 31)];
#pragma unroll
        for (int i = 0; i < 8; ++i) less_x[m][i] = half == 0 ? t[i & 3] : (bf16)0.0f;
      }
#pragma unroll
      for (int f = 0; f < 2; ++f) {
        // the lane's own row's zero, and the scales of the rows whose sums it has
        const int own = 2 * f;
        const u32 zero =
            p.zeros ? levels[2048 * wave + 1024 +
                             ((own + ((lane >> 4) & 1)) * PER + g) * 16 + (lane & 15)]
                    : 8;
        float scale[16];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          S t[4];
          newt::load_vec<S, 4>((const S*)(levels + 2048 * wave) + ((own + i / 2) * PER + g) * 16 +
                                   8 * (i & 1) + 4 * half,
                               t);
#pragma unroll
          for (int j = 0; j < 4; ++j) scale[4 * i + j] = newt::to_f32(t[j]);
        }
        const bf16 part_of = (bf16)(-0.0625f * (float)zero);
        bf16x8 less_a;  // by the three parts and 0, twice
#pragma unroll
        for (int i = 0; i < 8; ++i) less_a[i] = i < 4 ? (bf16)-1.0f : part_of;
#pragma unroll
        for (int m = 0; m < 2; ++m) {
          part[f][m] = newt::mfma_32x32x16(less_a, less_x[m], part[f][m]);
#pragma unroll
          for (int e = 0; e < 16; ++e)
            acc[f][m][e] = __builtin_fmaf(part[f][m][e], scale[e], acc[f][m][e]);
        }
        // the next group's weights to the front
        if constexpr (PER == 4) {
#pragma unroll
          for (int i = 0; i < 2; ++i) v[f][i] = u32x4{v[f][i][1], v[f][i][2], v[f][i][3], 0};
        } else if constexpr (PER == 2) {
#pragma unroll
          for (int i = 0; i < 2; ++i) v[f][i] = u32x4{v[f][i][2], v[f][i][3], 0, 0};
        }
      }
    }
  };
  u32x4 w0[2][2], w1[2][2], w2[2][2];
  load(from, w0, x0, levels0);
  load(from + 1, w1, x1, levels1);
  newt::wait_vmcnt<0>();
  __syncthreads();
#pragma unroll 1
  for (int g = 0; g < PER; ++g) {
    f32x4 all = (f32x4)(0.0f);
#pragma unroll
    for (int k = 0; k < GROUP; k += 32) all = add_32(x0, g * GROUP + k, all);
    keep(all, sums[0] + g * kRows);
  }
  for (int b = from; b < to; b += 6) {
#define NEWT_STEP(i, X, AFTER, NEXT, S)                                                        \
  if (b + i < to)                                                                              \
  step(b + i, x##X, levels##X, w##X, x##AFTER, x##NEXT, levels##NEXT, w##NEXT, sums[S], sums[1 - S])
    NEWT_STEP(0, 0, 1, 2, 0);
    NEWT_STEP(1, 1, 2, 0, 1);
    NEWT_STEP(2, 2, 0, 1, 0);
    NEWT_STEP(3, 0, 1, 2, 1);
    NEWT_STEP(4, 1, 2, 0, 0);
    NEWT_STEP(5, 2, 0, 1, 1);
#undef NEWT_STEP
  }
  newt::wait_vmcnt<0>();

  const bool whole = per >= blocks;
#pragma unroll
  for (int f = 0; f < 2; ++f)
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      const int row = 32 * m + (lane & 31);
      if (row >= rows) continue;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int t = tile + 2 * f + i / 2, in_tile = 8 * (i & 1) + 4 * half;
        if (t >= tiles) continue;
        const auto part_of = [&](int j) {
          return f32x4{acc[f][m][4 * j], acc[f][m][4 * j + 1], acc[f][m][4 * j + 2],
                       acc[f][m][4 * j + 3]};
        };
        if (!whole) {
          float* to_part = (float*)p.workspace + ((int64_t)split * p.rows + m0 + row) * tiles * 16;
          *(f32x4*)(to_part + t * 16 + in_tile) = part_of(i);
        } else if (!gated) {
          const int64_t first = (int64_t)t * 16 + in_tile;
          if (first < p.outputs) store4<T>(p, m0 + row, first, part_of(i) * kWhole<T>);
        } else if (i < 2) {
          const int64_t first = (int64_t)(t / 2) * 16 + in_tile;
          f32x4 y = part_of(i + 2) * kWhole<T>;
          const f32x4 gate = part_of(i) * kWhole<T>;
#pragma unroll
          for (int c = 0; c < 4; ++c) y[c] *= activate(gate[c], p.act);
          if (first < p.outputs) store4<T>(p, m0 + row, first, y);
        }
      }
    }
}

// The splits' sums, 4 outputs a thread, in the splits' order.
template <typename T>
__global__ void __launch_bounds__(256) q4_join_kernel(newt_q4_params p, int splits) {
  const bool gated = p.act != NEWT_ACT_NONE;
  const u32 quads = (u32)((p.outputs + 15) / 16) * 4;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t row = i / quads, first = i % quads * 4;
  if (row >= p.rows || first >= p.outputs) return;
  const int64_t width = (int64_t)quads * (gated ? 8 : 4);
  const auto joined = [&](int64_t at) {
    const float* from = (const float*)p.workspace + row * width + at;
    f32x4 y = *(const f32x4*)from;
    for (int s = 1; s < splits; ++s) y += *(const f32x4*)(from + s * p.rows * width);
    return y * kWhole<T>;
  };
  if (!gated) {
    store4<T>(p, row, first, joined(first));
  } else {
    const int64_t at = first / 16 * 32 + first % 16;
    const f32x4 gate = joined(at);
    f32x4 y = joined(at + 16);
#pragma unroll
    for (int c = 0; c < 4; ++c) y[c] *= activate(gate[c], p.act);
    store4<T>(p, row, first, y);
  }
}

struct Plan {
  int64_t m_blocks, n_blocks, tiles, per, splits;
  explicit Plan(const newt_q4_params& p) {
    const int64_t blocks = (p.cols + kBlock - 1) / kBlock;
    tiles = (p.outputs + 15) / 16 * (p.act != NEWT_ACT_NONE ? 2 : 1);
    m_blocks = (p.rows + kRows - 1) / kRows;
    n_blocks = (tiles + kTiles - 1) / kTiles;
    const int64_t units = m_blocks * n_blocks;
    // us for a block of one program on a CU, and of two side by side, by the group: 512 x
    // 4096, gated, takes 48 / 78 us for 2 x 2048 and 2 x 8192 columns in groups of 128, 69
    // / 98 of 64, 107 / 136 of 32. 333 x 8192 x 2003 in groups of 32 takes 189 us in one
    // part, 74 in 3, 51 in 5, 44 in 10, 47 in 16 and in 20; in groups of 128 76, 36, 29, 31, 33.
    const double one = p.group == 128 ? 1.2 : p.group == 64 ? 1.9 : 3.0;
    const double two = p.group == 128 ? 2.2 : p.group == 64 ? 2.7 : 3.9;
    const double each = 2.0 * p.rows * tiles * 16 * 4 / 4e6;  // for a split's sums
    double least = 1e30;
    for (int64_t n = 1; n <= 32 && n <= blocks; ++n) {
      const int64_t some = (blocks + n - 1) / n, parts = (blocks + some - 1) / some;
      const int64_t rounds = units * parts / 512, rest = units * parts % 512;
      const double cost = (rounds * two + (rest > 256 ? two : rest ? one : 0.0)) * (some + 2) +
                          (parts > 1 ? 4.0 + each * parts : 0.0);
      if (cost < least) {
        least = cost;
        per = some;
        splits = parts;
      }
    }
  }
};

template <typename T, typename S, int GROUP>
int launch(const newt_q4_params& p, hipStream_t stream) {
  const Plan r(p);
  const int64_t grid = r.m_blocks * r.n_blocks * r.splits;
  if (p.cols >= 1 << 25) return fail(NEWT_ERR_INVALID, "newt_q4_matmul: too many columns");
  if (grid > 0x7fffffff) return fail(NEWT_ERR_INVALID, "newt_q4_matmul: too many rows");
  if (r.splits > 1 && (!p.workspace || ((uintptr_t)p.workspace & 15)))
    return fail(NEWT_ERR_INVALID, "newt_q4_matmul: null or unaligned workspace");
  if (out_meets(p)) return fail(NEWT_ERR_INVALID, "newt_q4_matmul: out overlaps x or bias");
  // whole pieces of 16 bytes, within 2^31 bytes of a program's first
  const bool direct = p.x_stride % 8 == 0 && ((uintptr_t)p.x & 15) == 0 && p.x_stride >= 0 &&
                      p.x_stride < 1 << 23;
  const auto kernel =
      direct ? q4_many_kernel<T, S, GROUP, true> : q4_many_kernel<T, S, GROUP, false>;
  const int status = run("newt_q4_matmul", kernel, grid, 256, 0, stream, p, (int)r.m_blocks,
                         (int)r.n_blocks, (int)r.per);
  if (status != NEWT_OK || r.splits == 1) return status;
  const int64_t threads = p.rows * ((p.outputs + 15) / 16) * 4;
  return run("newt_q4_matmul", q4_join_kernel<T>, (threads + 255) / 256, 256, 0, stream, p,
             (int)r.splits);
}

template <typename T, typename S>
int by_group(const newt_q4_params& p, hipStream_t stream) {
  switch (p.group) {
    case 32: return launch<T, S, 32>(p, stream);
    case 64: return launch<T, S, 64>(p, stream);
    default: return launch<T, S, 128>(p, stream);
  }
}

template <typename T>
int by_scale(const newt_q4_params& p, hipStream_t stream) {
  return p.scale_dtype == NEWT_F16 ? by_group<T, f16>(p, stream) : by_group<T, bf16>(p, stream);
}

}  // namespace

size_t q4_many_workspace(const newt_q4_params& p) {
  const Plan r(p);
  return r.splits > 1 ? (size_t)r.splits * p.rows * r.tiles * 16 * sizeof(float) : 0;
}

int q4_many(const newt_q4_params& p, hipStream_t stream) {
  return p.dtype == NEWT_F16 ? by_scale<f16>(p, stream) : by_scale<bf16>(p, stream);
}

}  // namespace newt_ops
