// Root-mean-square norm of rows, with the residual's addition in front and an
// optional 8-bit output behind:
//   h = round(x + residual), y = h * rsqrt(mean(h^2) + eps) * w,
//   e4m3: scale = max(amax |y| / 448, 2^-126) over a group or the row,
//         q = round(y / scale).
// HBM bounds it (each input read once, each output written once), so a row is
// held in registers between the sum of squares and the output, and every
// access is 16 bytes a lane at whatever alignment the row has. bf16 4096 x 8192
// with a residual, three sets of inputs in turn: 44 us (6.1 TB/s) to bf16, 40
// (5.8) to e4m3 with a scale a row, 42 (5.6) with one for each 128 columns; a
// copy reaches 5.77 TB/s over 4.3 GB and 7.1 over 268 MB.
// Squares are summed in fp32 as they are: a row of numbers around 1e19 has an
// infinite sum, and its y is 0.
#include "common.h"

namespace newt_ops {
namespace {

constexpr float kTiny = 1.17549435e-38f;  // 2^-126

template <typename T> struct io {
  static constexpr int V = 16 / (int)sizeof(T);  // elements of a 16-byte access
};

// V elements from column c of a row, 0 behind its end
template <typename T>
__device__ __forceinline__ void load_cols(const T* row, int64_t c, int64_t cols, float* f) {
  constexpr int V = io<T>::V;
  T t[V];
  if (c + V <= cols) {
    newt::load_vec<T, V>(row + c, t, newt::any_align());
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) t[i] = c + i < cols ? row[c + i] : (T)0.0f;
  }
#pragma unroll
  for (int i = 0; i < V; ++i) f[i] = newt::to_f32(t[i]);
}

template <typename T>
__device__ __forceinline__ void store_cols(T* row, int64_t c, int64_t cols, const float* f) {
  constexpr int V = io<T>::V;
  T t[V];
#pragma unroll
  for (int i = 0; i < V; ++i) t[i] = (T)f[i];
  if (c + V <= cols) {
    newt::store_vec<T, V>(row + c, t, newt::any_align());
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (c + i < cols) row[c + i] = t[i];
  }
}

template <typename T>
__device__ __forceinline__ void store_e4m3(unsigned char* row, int64_t c, int64_t cols,
                                           const float* f, float scale) {
  constexpr int V = io<T>::V;
  // a product with the reciprocal is off by 2^-23 of the quotient, which the
  // rounding to 4 bits sees at one number in 2^19; with divisions 4096 x 8192 bf16
  // with a residual takes 42.8 us instead of 41.1, 2730 x 12288 48.0 instead of 41.8
  const float by = 1.0f / scale;
  u32 w[V / 4];
#pragma unroll
  for (int i = 0; i < V; i += 4)
    w[i / 4] = to_e4m3x4(f[i] * by, f[i + 1] * by, f[i + 2] * by, f[i + 3] * by);
  if (c + V <= cols) {
    unsigned char b[V];
    __builtin_memcpy(b, w, V);
    newt::store_vec<unsigned char, V>(row + c, b, newt::any_align());
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (c + i < cols) row[c + i] = (unsigned char)(w[i / 4] >> (8 * (i % 4)));
  }
}

// amax over the `lanes` (4 to 64, a power of two) neighbouring lanes that hold a
// group, on the VALU: each step's partner holds the maximum of the other half.
__device__ __forceinline__ float group_max(float v, int lanes) {
  v = newt::lane_reduce<newt::Max, 3>(v);
  if (lanes >= 8) v = newt::Max::op(v, newt::mirror_lane<8>(v));
  if (lanes >= 16) v = newt::Max::op(v, newt::mirror_lane<16>(v));
  float lo, hi;
  if (lanes >= 32) {
    newt::pair_lanes<16>(v, lo, hi);
    v = newt::Max::op(lo, hi);
  }
  if (lanes >= 64) {
    newt::pair_lanes<32>(v, lo, hi);
    v = newt::Max::op(lo, hi);
  }
  return v;
}

template <typename T, typename W>
__device__ __forceinline__ void load_w(const W* w, int64_t c, int64_t cols, float* f) {
  constexpr int V = io<T>::V;
  if constexpr (sizeof(W) == sizeof(T)) {
    load_cols<W>(w, c, cols, f);
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) f[i] = c + i < cols ? newt::to_f32(w[c + i]) : 0.0f;
  }
}

// LANES threads hold a row of up to LANES * V * CHUNKS columns. Rows of up to
// a wave share a workgroup of 256 threads.
template <typename T, typename W, bool E4M3, int LANES, int CHUNKS>
__global__ void __launch_bounds__(LANES < 256 ? 256 : LANES)
rmsnorm_kernel(newt_rmsnorm_params p) {
  constexpr int V = io<T>::V;
  constexpr int ROWS = LANES < 256 ? 256 / LANES : 1;
  constexpr int WAVES = LANES > 64 ? LANES / 64 : 1;
  __shared__ float slot[2 * WAVES * (LANES > 64 ? ROWS : 1)];
  const int lane = threadIdx.x % LANES;
  const int in_block = threadIdx.x / LANES;
  const int64_t row = (int64_t)blockIdx.x * ROWS + in_block;
  const bool live = row < p.rows;
  const int64_t r = live ? row : 0;
  const int64_t cols = live ? p.cols : 0;
  const T* x = (const T*)p.x + r * p.x_stride;
  const T* residual = (const T*)p.residual + r * p.residual_stride;
  T* hidden = (T*)p.hidden + r * p.hidden_stride;

  float h[CHUNKS][V];
  float sum = 0.0f;
#pragma unroll
  for (int c = 0; c < CHUNKS; ++c) load_cols<T>(x, (int64_t)(c * LANES + lane) * V, cols, h[c]);
  if (p.residual) {
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
      const int64_t at = (int64_t)(c * LANES + lane) * V;
      float f[V];
      load_cols<T>(residual, at, cols, f);
#pragma unroll
      for (int i = 0; i < V; ++i) h[c][i] = newt::to_f32((T)(h[c][i] + f[i]));
      store_cols<T>(hidden, at, cols, h[c]);
    }
  }
#pragma unroll
  for (int c = 0; c < CHUNKS; ++c)
#pragma unroll
    for (int i = 0; i < V; ++i) sum += h[c][i] * h[c][i];
  if constexpr (LANES >= 64) sum = block_reduce<newt::Sum, WAVES>(sum, slot);
  else sum = newt::lane_reduce<newt::Sum, LANES - 1>(sum);
  const float rstd = 1.0f / __builtin_sqrtf(sum / (float)p.cols + p.eps);
  float top = 0.0f;
#pragma unroll
  for (int c = 0; c < CHUNKS; ++c) {
    const int64_t at = (int64_t)(c * LANES + lane) * V;
    float f[V];
    load_w<T, W>((const W*)p.w, at, cols, f);
#pragma unroll
    for (int i = 0; i < V; ++i) h[c][i] = h[c][i] * rstd * f[i];
    if constexpr (!E4M3) {
      store_cols<T>((T*)p.out + r * p.out_stride, at, cols, h[c]);
    } else if (p.group == 0) {
#pragma unroll
      for (int i = 0; i < V; ++i) top = newt::Max::op(top, __builtin_fabsf(h[c][i]));
    }
  }
  if constexpr (E4M3) {
    unsigned char* out = (unsigned char*)p.out + r * p.out_stride;
    if (p.group == 0) {
      if constexpr (LANES >= 64) top = block_reduce<newt::Max, WAVES>(top, slot + WAVES);
      else top = newt::lane_reduce<newt::Max, LANES - 1>(top);
      const float scale = __builtin_fmaxf(top / 448.0f, kTiny);
      if (live && lane == 0) p.scale[r] = scale;
#pragma unroll
      for (int c = 0; c < CHUNKS; ++c)
        store_e4m3<T>(out, (int64_t)(c * LANES + lane) * V, cols, h[c], scale);
    } else {
      const int lanes = p.group / V;
#pragma unroll
      for (int c = 0; c < CHUNKS; ++c) {
        const int64_t at = (int64_t)(c * LANES + lane) * V;
        top = 0.0f;
#pragma unroll
        for (int i = 0; i < V; ++i) top = newt::Max::op(top, __builtin_fabsf(h[c][i]));
        const float scale = __builtin_fmaxf(group_max(top, lanes) / 448.0f, kTiny);
        if (at < cols && at % p.group == 0) p.scale[r * (p.cols / p.group) + at / p.group] = scale;
        store_e4m3<T>(out, at, cols, h[c], scale);
      }
    }
  }
}

// Rows longer than registers hold: the row is read again (from the caches,
// mostly) for the output, and once more for a scale of the whole row.
template <typename T, typename W, bool E4M3>
__global__ void __launch_bounds__(1024) rmsnorm_long_kernel(newt_rmsnorm_params p) {
  constexpr int V = io<T>::V;
  __shared__ float slot[32];
  const int64_t r = blockIdx.x;
  const int64_t cols = p.cols;
  const int64_t step = 1024 * V;
  const int64_t first = (int64_t)threadIdx.x * V;
  // the row's end rounded up to a step, so that every lane of a wave makes the
  // same trips and takes part in group_max
  const int64_t end = (cols + step - 1) / step * step;
  const T* x = (const T*)p.x + r * p.x_stride;
  const T* residual = (const T*)p.residual + r * p.residual_stride;
  T* hidden = (T*)p.hidden + r * p.hidden_stride;
  float sum = 0.0f;
  for (int64_t c = first; c < cols; c += step) {
    float h[V], f[V];
    load_cols<T>(x, c, cols, h);
    if (p.residual) {
      load_cols<T>(residual, c, cols, f);
#pragma unroll
      for (int i = 0; i < V; ++i) h[i] = newt::to_f32((T)(h[i] + f[i]));
      store_cols<T>(hidden, c, cols, h);
    }
#pragma unroll
    for (int i = 0; i < V; ++i) sum += h[i] * h[i];
  }
  sum = block_reduce<newt::Sum, 16>(sum, slot);
  const float rstd = 1.0f / __builtin_sqrtf(sum / (float)cols + p.eps);
  // each thread reads the columns that it wrote itself
  const T* source = p.residual ? hidden : x;
  const auto value = [&](int64_t c, float* h) {
    float f[V];
    load_cols<T>(source, c, cols, h);
    load_w<T, W>((const W*)p.w, c, cols, f);
#pragma unroll
    for (int i = 0; i < V; ++i) h[i] = h[i] * rstd * f[i];
  };
  if constexpr (!E4M3) {
    for (int64_t c = first; c < cols; c += step) {
      float h[V];
      value(c, h);
      store_cols<T>((T*)p.out + r * p.out_stride, c, cols, h);
    }
  } else {
    unsigned char* out = (unsigned char*)p.out + r * p.out_stride;
    float scale = 0.0f;
    if (p.group == 0) {
      float top = 0.0f;
      for (int64_t c = first; c < cols; c += step) {
        float h[V];
        value(c, h);
#pragma unroll
        for (int i = 0; i < V; ++i) top = newt::Max::op(top, __builtin_fabsf(h[i]));
      }
      top = block_reduce<newt::Max, 16>(top, slot + 16);
      scale = __builtin_fmaxf(top / 448.0f, kTiny);
      if (threadIdx.x == 0) p.scale[r] = scale;
    }
    for (int64_t c = first; c < end; c += step) {
      float h[V];
      value(c, h);
      if (p.group) {
        float top = 0.0f;
#pragma unroll
        for (int i = 0; i < V; ++i) top = newt::Max::op(top, __builtin_fabsf(h[i]));
        scale = __builtin_fmaxf(group_max(top, p.group / V) / 448.0f, kTiny);
        if (c < cols && c % p.group == 0) p.scale[r * (cols / p.group) + c / p.group] = scale;
      }
      store_e4m3<T>(out, c, cols, h, scale);
    }
  }
}

template <typename T, typename W, bool E4M3>
int launch(const newt_rmsnorm_params& p, hipStream_t stream) {
  constexpr int V = io<T>::V;
  const int64_t vecs = (p.cols + V - 1) / V;
  const auto go = [&](auto lanes, auto chunks) {
    constexpr int L = decltype(lanes)::value, C = decltype(chunks)::value;
    constexpr int rows = L < 256 ? 256 / L : 1;
    return run("newt_rmsnorm", rmsnorm_kernel<T, W, E4M3, L, C>, (p.rows + rows - 1) / rows,
               L < 256 ? 256 : L, 0, stream, p);
  };
  // enough lanes for a row in one or two pieces each (up to four of the longest)
#define NEWT_ROWS(L, C) \
  if (vecs <= L * C) return go(std::integral_constant<int, L>(), std::integral_constant<int, C>())
  NEWT_ROWS(8, 1);
  NEWT_ROWS(16, 1);
  NEWT_ROWS(32, 1);
  NEWT_ROWS(64, 1);
  NEWT_ROWS(64, 2);
  NEWT_ROWS(256, 1);
  NEWT_ROWS(384, 1);
  NEWT_ROWS(256, 2);
  NEWT_ROWS(384, 2);
  NEWT_ROWS(512, 2);
  NEWT_ROWS(768, 2);
  NEWT_ROWS(1024, 2);
  NEWT_ROWS(1024, 4);
#undef NEWT_ROWS
  return run("newt_rmsnorm", rmsnorm_long_kernel<T, W, E4M3>, p.rows, 1024, 0, stream, p);
}

template <typename T, typename W>
int by_out(const newt_rmsnorm_params& p, hipStream_t stream) {
  return p.out_dtype == NEWT_E4M3 ? launch<T, W, true>(p, stream) : launch<T, W, false>(p, stream);
}

template <typename T>
int by_weight(const newt_rmsnorm_params& p, hipStream_t stream) {
  if (p.w_dtype == p.dtype) return by_out<T, T>(p, stream);
  if (p.w_dtype == NEWT_F32) return by_out<T, float>(p, stream);
  return fail(NEWT_ERR_INVALID, "newt_rmsnorm: w is of x's type or fp32");
}

}  // namespace
}  // namespace newt_ops

extern "C" int newt_rmsnorm(const newt_rmsnorm_params* params, void* stream) {
  using namespace newt_ops;
  if (!params) return fail(NEWT_ERR_INVALID, "newt_rmsnorm: null params");
  const newt_rmsnorm_params& p = *params;
  if (p.rows == 0) return NEWT_OK;
  const bool e4m3 = p.out_dtype == NEWT_E4M3;
  if (!p.x || !p.w || !p.out || (p.residual && !p.hidden) || (e4m3 && !p.scale))
    return fail(NEWT_ERR_INVALID, "newt_rmsnorm: null tensor");
  if (p.rows < 0 || p.rows > 0x7fffffff || p.cols <= 0)
    return fail(NEWT_ERR_INVALID, "newt_rmsnorm: %lld rows of %lld columns", (long long)p.rows,
                (long long)p.cols);
  if (p.out_dtype != p.dtype && !e4m3)
    return fail(NEWT_ERR_INVALID, "newt_rmsnorm: out is of x's type or e4m3");
  if (p.group != 0 && (!e4m3 || (p.group != 32 && p.group != 64 && p.group != 128 &&
                                 p.group != 256) || p.cols % p.group))
    return fail(NEWT_ERR_INVALID, "newt_rmsnorm: no groups of %d in %lld columns", p.group,
                (long long)p.cols);
  hipStream_t s = static_cast<hipStream_t>(stream);
  switch (p.dtype) {
    case NEWT_F32: return by_weight<float>(p, s);
    case NEWT_F16: return by_weight<f16>(p, s);
    case NEWT_BF16: return by_weight<bf16>(p, s);
    default: return fail(NEWT_ERR_INVALID, "newt_rmsnorm: unknown dtype %d", p.dtype);
  }
}
