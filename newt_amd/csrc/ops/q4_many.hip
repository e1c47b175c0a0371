// Products with 4-bit weights for many rows of x, which the matrix unit bounds.
// A program takes 64 rows of x and 256 rows of weights, each of its 4 waves 64 of
// those: 128 columns of x are staged in LDS for all waves, while the weights go
// from memory to the wave that multiplies them and become operands there,
//   S[n][m] += W[n][k] x[m][k] by v_mfma_f32_32x32x16,
// so that a word of weights is widened once for 64 rows and a piece of x is read
// from LDS twice for 128 rows of weights. As for few rows the sums hold (16 + z) /
// 16 times the sum of x too much. That is taken off within the matrix unit: one
// more step multiplies -(16 + z) / 16, which bf16 holds exactly, by the sum of x
// in three bf16 parts, exactly what fp32 holds; on the vector unit it would take
// as long as widening the weights. Each wave sums 16 rows of x for all.
// A group's sums then take their scales on the way into the accumulators, in fp32.
#include "q4.h"

namespace newt_ops {
namespace {

constexpr int kRows = 64, kTiles = 16, kBlock = 128;

template <typename T, typename S, int GROUP, bool DIRECT>
__global__ void __launch_bounds__(256, 2)
q4_many_kernel(newt_q4_params p, int m_blocks, int n_blocks, int per) {
  typedef typename frag<T>::type TX;
  constexpr int PER = kBlock / GROUP, STEPS = GROUP / 16;
  __shared__ __attribute__((aligned(16))) T even[kRows * kBlock];
  __shared__ __attribute__((aligned(16))) T odd[kRows * kBlock];
  __shared__ __attribute__((aligned(16))) bf16x4 sums[PER * kRows];
  // a block's scales and zeros, [tile][group][16]
  constexpr int SCALES = kTiles * PER * 2, ZEROS = kTiles * PER;  // pieces of 16 bytes
  constexpr int LEVELS = (SCALES + ZEROS + 63) / 64 * 64 * 16;
  __shared__ __attribute__((aligned(16))) unsigned char levels_even[LEVELS];
  __shared__ __attribute__((aligned(16))) unsigned char levels_odd[LEVELS];
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
  const u32x4* q[2];
#pragma unroll
  for (int f = 0; f < 2; ++f)
    q[f] = (const u32x4*)p.q + at(tile + 2 * f + ((lane >> 4) & 1)) * blocks * 64 + 16 * half +
           (lane & 15);
  // the piece of a block's scales or zeros that a thread stages
  const int piece = threadIdx.x;
  const unsigned char* level = nullptr;
  int level_step = 0;
  if (piece < SCALES) {
    level = (const unsigned char*)p.scales +
            (at(n_block * kTiles + piece / (2 * PER)) * groups * 2 + piece % (2 * PER)) * 16;
    level_step = 2 * PER * 16;
  } else if (piece < SCALES + ZEROS && p.zeros) {
    const int i = piece - SCALES;
    level = (const unsigned char*)p.zeros +
            (at(n_block * kTiles + i / PER) * groups + i % PER) * 16;
    level_step = PER * 16;
  }

  const auto stage = [&](int b, T* to_lds, unsigned char* levels) {
    if (level) newt::lds_dma16(level + (int64_t)b * level_step, levels + 64 * wave * 16);
    const T* base = (const T*)p.x + m0 * p.x_stride + b * kBlock;
    const int cols = (int)(p.cols - (int64_t)b * kBlock);
#pragma unroll
    for (int c = 0; c < kRows * kBlock / 8 / 256; ++c) {
      const int first = c * 256 + 64 * wave;
      int row, k;
      newt::lds_tile_slot<T, kBlock>(first + lane, row, k);
      const bool in = (row < rows) & (k < cols);
      if constexpr (DIRECT) {
        newt::lds_dma16_masked(base, (u32)(row * (int)p.x_stride + k) * 2, in, to_lds + first * 8);
      } else {
        T t[8] = {};
        if (in) newt::load_vec<T, 8>(base + row * p.x_stride + k, t, newt::any_align());
        newt::store_vec<T, 8>(to_lds + (first + lane) * 8, t);
      }
    }
  };

  f32x16 acc[2][2];
#pragma unroll
  for (int f = 0; f < 2; ++f)
#pragma unroll
    for (int m = 0; m < 2; ++m) acc[f][m] = (f32x16)(0.0f);
  TX ones;
#pragma unroll
  for (int i = 0; i < 8; ++i) ones[i] = (T)1.0f;

  const auto load = [&](int b, u32x4 (&w)[2][2]) {
#pragma unroll
    for (int f = 0; f < 2; ++f)
#pragma unroll
      for (int i = 0; i < 2; ++i) w[f][i] = q[f][(int64_t)b * 64 + 32 * i];
  };

  // One block, while the next one is on its way.
  const auto step = [&](int b, const T* now, T* next, const unsigned char* levels,
                        unsigned char* next_levels, u32x4 (&v)[2][2], u32x4 (&w)[2][2]) {
    newt::wait_vmcnt<0>();
    __syncthreads();
    if (b + 1 < to) {
      stage(b + 1, next, next_levels);
      load(b + 1, w);
    }
    f32x4 all = (f32x4)(0.0f);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const TX x = __builtin_bit_cast(TX, newt::lds_frag_k<T, kBlock, 16>(now, 16 * wave, 32 * j, lane));
      all = newt::mfma_16x16x32(ones, x, all);
      if ((j + 1) % (GROUP / 32) == 0) {
        const bf16 hi = (bf16)all[0];
        const float rest = all[0] - (float)hi;
        const bf16 mid = (bf16)rest;
        if (lane < 16)
          sums[j / (GROUP / 32) * kRows + 16 * wave + lane] =
              bf16x4{hi, mid, (bf16)(rest - (float)mid), (bf16)0.0f};
        all = (f32x4)(0.0f);
      }
    }
    // the sums are there; what is on its way to the other stage need not be
    __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0)
    newt::barrier_nofence();
    // not unrolled: groups side by side would not fit the registers
#pragma unroll 1
    for (int g = 0; g < PER; ++g) {
      f32x16 part[2][2];
#pragma unroll
      for (int f = 0; f < 2; ++f)
#pragma unroll
        for (int m = 0; m < 2; ++m) part[f][m] = (f32x16)(0.0f);
#pragma unroll
      for (int i = 0; i < STEPS; ++i) {
        const int st = g * STEPS + i;
        TX x[2];
#pragma unroll
        for (int m = 0; m < 2; ++m)
          x[m] = __builtin_bit_cast(TX, newt::lds_frag_k<T, kBlock, 32>(now, 32 * m, 16 * st, lane));
#pragma unroll
        for (int f = 0; f < 2; ++f) {
          const TX a = widen<T>(v[f][i & 1][i / 2]);
#pragma unroll
          for (int m = 0; m < 2; ++m) part[f][m] = newt::mfma_32x32x16(a, x[m], part[f][m]);
        }
      }
      bf16x8 x[2];
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        const bf16x4 t = sums[g * kRows + 32 * m + (lane & 31)];
#pragma unroll
        for (int i = 0; i < 8; ++i) x[m][i] = i < 3 && half == 0 ? t[i] : (bf16)0.0f;
      }
#pragma unroll
      for (int f = 0; f < 2; ++f) {
        // the lane's own row's zero, and the scales of the rows whose sums it has
        const int own = 4 * wave + 2 * f;
        const u32 zero =
            p.zeros ? levels[SCALES * 16 + ((own + ((lane >> 4) & 1)) * PER + g) * 16 + (lane & 15)] : 8;
        float scale[16];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          S t[4];
          newt::load_vec<S, 4>(
              (const S*)levels + ((own + i / 2) * PER + g) * 16 + 8 * (i & 1) + 4 * half, t);
#pragma unroll
          for (int j = 0; j < 4; ++j) scale[4 * i + j] = newt::to_f32(t[j]);
        }
        const bf16 less = (bf16)(-1.0f - 0.0625f * (float)zero);
        bf16x8 a;
#pragma unroll
        for (int i = 0; i < 8; ++i) a[i] = i < 3 ? less : (bf16)0.0f;
#pragma unroll
        for (int m = 0; m < 2; ++m) {
          part[f][m] = newt::mfma_32x32x16(a, x[m], part[f][m]);
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
  u32x4 v[2][2], w[2][2];
  if (from < to) {
    stage(from, even, levels_even);
    load(from, v);
  }
  for (int b = from; b < to; b += 2) {
    step(b, even, odd, levels_even, levels_odd, v, w);
    if (b + 1 < to) step(b + 1, odd, even, levels_odd, levels_even, w, v);
  }

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
        const auto quad = [&](int j) {
          return f32x4{acc[f][m][4 * j], acc[f][m][4 * j + 1], acc[f][m][4 * j + 2],
                       acc[f][m][4 * j + 3]} * 16.0f;
        };
        if (!whole) {
          float* to_part = (float*)p.workspace + ((int64_t)split * p.rows + m0 + row) * tiles * 16;
          *(f32x4*)(to_part + t * 16 + in_tile) = quad(i);
        } else if (!gated) {
          const int64_t first = (int64_t)t * 16 + in_tile;
          if (first < p.outputs) store4<T>(p, m0 + row, first, quad(i));
        } else if (i < 2) {
          const int64_t first = (int64_t)(t / 2) * 16 + in_tile;
          f32x4 y = quad(i + 2);
          const f32x4 gate = quad(i);
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
    return y;
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
    const double each = 2.0 * p.rows * tiles * 16 * 4 / 4e6;  // us for a split's sums
    double least = 1e30;
    for (int64_t n = 1; n <= 32 && n <= blocks; ++n) {
      const int64_t some = (blocks + n - 1) / n, parts = (blocks + some - 1) / some;
      const double cost = (double)((units * parts + 255) / 256) * (double)(some + 1) * 0.6 +
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
  if (grid > 0x7fffffff) return fail(NEWT_ERR_INVALID, "newt_q4_matmul: too many rows");
  if (r.splits > 1 && !p.workspace)
    return fail(NEWT_ERR_INVALID, "newt_q4_matmul: null workspace");
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
