// New tokens' keys and values into the 8-bit cache. Each block and head has
// one scale, a power of two: the smallest s with amax |x| <= 448 s over the
// block's tokens so far. e4m3 is a floating format, so a finer scale would gain
// no precision, and under a power of two a block whose scale grows keeps its
// older tokens' values exactly, but for those that fall below 2^-6 of the new
// scale and lose low bits there.
// Keys lie token by token, values transposed, head_dim rows of block_size
// tokens, the order in which the two products of the attention that reads
// them take them into matrix operands.
// Reading the tokens once and writing a byte for each number bounds it: bf16, 8
// sequences of 2048 tokens, 8 heads of 128, takes 25 us (3.3 TB/s) where no cache
// has them, 20 on the same ones again, waves waiting 53% of their cycles; one
// token of each of 64 sequences 4.4.
#include "common.h"

namespace newt_ops {
namespace {

constexpr int kLowest = -100;  // scales start at 2^-100; an empty block's scale is that

// exponent e of the smallest 2^e with top <= 448 * 2^e = 1.75 * 2^(e + 8)
__device__ __forceinline__ int scale_exponent(float top) {
  const u32 b = newt::f32_bits(top);
  const int e = (int)(b >> 23) - 127 - 8 + ((b & 0x7fffffu) > 0x600000u ? 1 : 0);
  return e < kLowest ? kLowest : e;
}

__device__ __forceinline__ float power_of_two(int e) { return newt::bits_f32((u32)(e + 127) << 23); }

// amax counts numbers only; infinities and NaN become NaN (0x7f)
__device__ __forceinline__ float finite_abs(float x) {
  const float a = __builtin_fabsf(x);
  return a < __builtin_inff() ? a : 0.0f;
}
__device__ __forceinline__ float or_nan(float x) {
  return __builtin_fabsf(x) < __builtin_inff() ? x : __builtin_nanf("");
}

// four e4m3 bytes times f
__device__ __forceinline__ u32 scaled(u32 w, float f) {
  return to_e4m3x4(__builtin_amdgcn_cvt_f32_fp8((int)w, 0) * f,
                   __builtin_amdgcn_cvt_f32_fp8((int)w, 1) * f,
                   __builtin_amdgcn_cvt_f32_fp8((int)w, 2) * f,
                   __builtin_amdgcn_cvt_f32_fp8((int)w, 3) * f);
}

// The part of a call that one workgroup does: one block of one sequence, one
// head, its keys or its values.
template <typename T>
struct Part {
  bool live = false;
  bool values;
  int held, end;     // the block's tokens [0, held) are older, [held, end) new
  const T* x;        // where the block's token 0 would be among the new ones
  int64_t stride;
  unsigned char* out;
  float* scale;

  __device__ __forceinline__ Part(const newt_kv_append_params& p, int slots) {
    const u32 heads = p.cache.kv_heads, at_head = blockIdx.x >> 1;
    const u32 head = at_head % heads, slot_of = at_head / heads % (u32)slots;
    const u32 b = at_head / heads / (u32)slots;
    const int size = p.cache.block_size, D = p.cache.head_dim;
    values = blockIdx.x & 1;
    const int64_t start = p.start[b];
    int64_t count = p.count ? p.count[b] : p.tokens;
    count = count < p.tokens ? count : p.tokens;
    if (start < 0 || count <= 0) return;
    const int64_t at = start / size + slot_of;  // the block's place in the sequence
    const int64_t first = at * size;
    if (first >= start + count || at >= p.table_width) return;
    const int64_t block = p.table[b * p.table_stride + at];
    if (block < 0 || block >= p.cache.blocks) return;
    live = true;
    held = start > first ? (int)(start - first) : 0;
    end = start + count < first + size ? (int)(start + count - first) : size;
    stride = values ? p.v_stride_t : p.k_stride_t;
    x = (values ? (const T*)p.v + b * p.v_stride_b + head * p.v_stride_h
                : (const T*)p.k + b * p.k_stride_b + head * p.k_stride_h) +
        (first - start) * stride;
    const int64_t page = block * p.cache.kv_heads + head;
    out = (unsigned char*)(values ? p.cache.v : p.cache.k) + page * size * D;
    scale = (values ? p.cache.v_scale : p.cache.k_scale) + page;
  }

  // The block's scale, from the new tokens' amax; older tokens are taken to it
  // where it grew. All of a workgroup's threads.
  template <int THREADS>
  __device__ __forceinline__ float rescale(float top, int size, int D) const {
    __shared__ float slot[THREADS / 64];
    top = block_reduce<newt::Max, THREADS / 64>(top, slot);
    float to = power_of_two(scale_exponent(top));
    const float had = held > 0 ? *scale : to;
    if (had > to) to = had;
    if (held > 0 && !(had >= to)) {
      const float f = had / to;
      if (values) {
        // rows of `size` bytes, their first `held`; whole pieces of 16 are
        // written, with the bytes behind as they were
        const int units = (held + 15) / 16;
        for (int i = threadIdx.x; i < units * D; i += THREADS) {
          u32x4* o = (u32x4*)(out + (i / units) * size + i % units * 16);
          u32x4 w = *o;
          const int n = held - i % units * 16;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int left = n - 4 * j;
            const u32 keep = left >= 4 ? 0u : left <= 0 ? ~0u : ~0u << (8 * left);
            w[j] = (w[j] & keep) | (scaled(w[j], f) & ~keep);
          }
          *o = w;
        }
      } else {
        for (int i = threadIdx.x; i < held * D / 16; i += THREADS) {
          u32x4 w = ((u32x4*)out)[i];
#pragma unroll
          for (int j = 0; j < 4; ++j) w[j] = scaled(w[j], f);
          ((u32x4*)out)[i] = w;
        }
      }
    }
    // the old scale is read and the old bytes are written before new ones are
    __syncthreads();
    if (threadIdx.x == 0) *scale = to;
    return to;
  }
};

// A few tokens: one wave, a number at a time.
template <typename T, int D>
__global__ void __launch_bounds__(64) kv_append_few_kernel(newt_kv_append_params p, int slots) {
  const Part<T> part(p, slots);
  if (!part.live) return;
  const int size = p.cache.block_size;
  constexpr int N = D / 64;  // numbers of a token a lane holds
  const int d = threadIdx.x * N;
  float top = 0.0f;
  for (int t = part.held; t < part.end; ++t) {
    T x[N];
    newt::load_vec<T, N>(part.x + t * part.stride + d, x, newt::any_align());
#pragma unroll
    for (int i = 0; i < N; ++i) top = newt::Max::op(top, finite_abs(newt::to_f32(x[i])));
  }
  const float scale = part.template rescale<64>(top, size, D);
  for (int t = part.held; t < part.end; ++t) {
    T x[N];
    newt::load_vec<T, N>(part.x + t * part.stride + d, x, newt::any_align());
    float f[4] = {};
#pragma unroll
    for (int i = 0; i < N; ++i) f[i] = or_nan(newt::to_f32(x[i]) / scale);
    const u32 w = to_e4m3x4(f[0], f[1], f[2], f[3]);
#pragma unroll
    for (int i = 0; i < N; ++i)
      part.out[part.values ? (d + i) * size + t : t * D + d + i] = (unsigned char)(w >> (8 * i));
  }
}

// Many tokens. A thread holds CHUNKS pieces of 8 numbers, of 4 neighbouring
// tokens each, so that it has 4 tokens' bytes of a head dim together; values
// are transposed through LDS and written in rows. The LDS rows of each 8 head
// dims begin 16 bytes further, which spreads a wave's 4-byte writes over all
// banks.
template <typename T, int D, int THREADS, int CHUNKS>
__global__ void __launch_bounds__(THREADS) kv_append_kernel(newt_kv_append_params p, int slots) {
  extern __shared__ __attribute__((aligned(16))) unsigned char lds[];
  const Part<T> part(p, slots);
  if (!part.live) return;
  const int size = p.cache.block_size;
  constexpr int WIDE = D / 8;            // pieces of a token
  constexpr int GROUPS = THREADS / WIDE; // groups of 4 tokens that the workgroup holds at a time
  const int d = threadIdx.x % WIDE * 8;
  const int group = threadIdx.x / WIDE;

  T x[CHUNKS][8];
  float top = 0.0f;
#pragma unroll
  for (int c = 0; c < CHUNKS; ++c) {
    const int t = (c / 4 * GROUPS + group) * 4 + c % 4;
    if (t >= part.held && t < part.end) {
      newt::load_vec<T, 4>(part.x + t * part.stride + d, x[c], newt::any_align());
      newt::load_vec<T, 4>(part.x + t * part.stride + d + 4, x[c] + 4, newt::any_align());
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) x[c][i] = (T)0.0f;
    }
  }
#pragma unroll
  for (int c = 0; c < CHUNKS; ++c)
#pragma unroll
    for (int i = 0; i < 8; ++i) top = newt::Max::op(top, finite_abs(newt::to_f32(x[c][i])));
  const float scale = part.template rescale<THREADS>(top, size, D);
  // the scales made here are powers of two, whose reciprocals are exact; a
  // larger one that the block came with need not be
  const float by = 1.0f / scale;
  const bool power = (newt::f32_bits(scale) & 0x7fffffu) == 0;
  const auto put = [&](int c, int i) {
    const float v = newt::to_f32(x[c][i]);
    return or_nan(power ? v * by : v / scale);
  };

  if (!part.values) {
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
      const int t = (c / 4 * GROUPS + group) * 4 + c % 4;
      if (t >= part.held && t < part.end)
        *(u32x2*)(part.out + t * D + d) =
            u32x2{to_e4m3x4(put(c, 0), put(c, 1), put(c, 2), put(c, 3)),
                  to_e4m3x4(put(c, 4), put(c, 5), put(c, 6), put(c, 7))};
    }
    return;
  }
  const auto row = [&](int at) { return lds + at * size + at / 8 * 16; };
#pragma unroll
  for (int c = 0; c < CHUNKS; c += 4) {
    const int t = (c / 4 * GROUPS + group) * 4;
    if (t < size)
#pragma unroll
      for (int i = 0; i < 8; ++i)
        *(u32*)(row(d + i) + t) = to_e4m3x4(put(c, i), put(c + 1, i), put(c + 2, i), put(c + 3, i));
  }
  __syncthreads();
  const int units = size / 16;
  for (int i = threadIdx.x; i < units * D; i += THREADS) {
    const int at = i / units, t = i % units * 16;
    if (t >= part.end || t + 16 <= part.held) continue;
    const u32x4 w = *(const u32x4*)(row(at) + t);
    unsigned char* o = part.out + at * size + t;
    if (t >= part.held && t + 16 <= part.end) {
      *(u32x4*)o = w;
    } else {
#pragma unroll
      for (int j = 0; j < 16; ++j)
        if (t + j >= part.held && t + j < part.end) o[j] = (unsigned char)(w[j / 4] >> (8 * (j % 4)));
    }
  }
}

template <typename T, int D>
int launch(const newt_kv_append_params& p, hipStream_t stream) {
  const int size = p.cache.block_size;
  // blocks that `tokens` consecutive ones can reach
  const int64_t slots = (p.tokens + size - 2) / size + 1;
  // one program for each of them, each head, keys and values
  const int64_t grid = slots * p.batch * p.cache.kv_heads * 2;
  if (grid > 0x7fffffff) return fail(NEWT_ERR_INVALID, "newt_kv_append: too many tokens");
  const unsigned lds = size * D + D / 8 * 16;
  const char* const what = "newt_kv_append";
  if (p.tokens <= 4) return run(what, kv_append_few_kernel<T, D>, grid, 64, 0, stream, p, (int)slots);
  if (size * D <= 8192)
    return run(what, kv_append_kernel<T, D, 256, 4>, grid, 256, lds, stream, p, (int)slots);
  if (size * D <= 16384)
    return run(what, kv_append_kernel<T, D, 256, 8>, grid, 256, lds, stream, p, (int)slots);
  return run(what, kv_append_kernel<T, D, 1024, 8>, grid, 1024, lds, stream, p, (int)slots);
}

template <typename T>
int by_dim(const newt_kv_append_params& p, hipStream_t stream) {
  switch (p.cache.head_dim) {
    case 64: return launch<T, 64>(p, stream);
    case 128: return launch<T, 128>(p, stream);
    default: return launch<T, 256>(p, stream);
  }
}

}  // namespace
}  // namespace newt_ops

extern "C" int newt_kv_append(const newt_kv_append_params* params, void* stream) {
  using namespace newt_ops;
  if (!params) return fail(NEWT_ERR_INVALID, "newt_kv_append: null params");
  const newt_kv_append_params& p = *params;
  if (const char* wrong = cache_wrong(p.cache)) return fail(NEWT_ERR_INVALID, "newt_kv_append: %s", wrong);
  if (p.batch < 0 || p.tokens < 0 || p.table_width < 0)
    return fail(NEWT_ERR_INVALID, "newt_kv_append: negative size");
  if (p.batch == 0 || p.tokens == 0 || p.table_width == 0 || p.cache.blocks == 0) return NEWT_OK;
  if (!p.k || !p.v || !p.table || !p.start)
    return fail(NEWT_ERR_INVALID, "newt_kv_append: null tensor");
  hipStream_t s = static_cast<hipStream_t>(stream);
  switch (p.dtype) {
    case NEWT_F32: return by_dim<float>(p, s);
    case NEWT_F16: return by_dim<f16>(p, s);
    case NEWT_BF16: return by_dim<bf16>(p, s);
    default: return fail(NEWT_ERR_INVALID, "newt_kv_append: unknown dtype %d", p.dtype);
  }
}
