// New tokens' keys and values into the 8-bit cache. Each block and head has
// one scale, a power of two: the smallest s with amax |x| <= 448 s over the
// block's tokens so far. e4m3 is a floating format, so a finer scale would gain
// no precision, and under a power of two a block whose scale grows keeps its
// older tokens' values exactly, but for those that fall below 2^-6 of the new
// scale and lose low bits there.
// Keys lie token by token, values transposed, head_dim rows of block_size
// tokens, the order in which the two products of the attention that reads
// them take them into matrix operands.
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

__device__ __forceinline__ void from_e4m3x4(u32 w, float* f) {
  f[0] = __builtin_amdgcn_cvt_f32_fp8((int)w, 0);
  f[1] = __builtin_amdgcn_cvt_f32_fp8((int)w, 1);
  f[2] = __builtin_amdgcn_cvt_f32_fp8((int)w, 2);
  f[3] = __builtin_amdgcn_cvt_f32_fp8((int)w, 3);
}

// One workgroup: one block of one sequence, one head, keys (blockIdx.z 0) or
// values (1).
template <typename T, int THREADS>
__global__ void __launch_bounds__(THREADS) kv_append_kernel(newt_kv_append_params p, int slots) {
  __shared__ float slot[THREADS / 64 > 0 ? THREADS / 64 : 1];
  const int b = blockIdx.x / slots;
  const int head = blockIdx.y;
  const bool values = blockIdx.z != 0;
  const int size = p.cache.block_size, D = p.cache.head_dim;
  int64_t start = p.start[b];
  int64_t count = p.count ? p.count[b] : p.tokens;
  count = count < p.tokens ? count : p.tokens;
  if (start < 0 || count <= 0) return;
  const int64_t at = start / size + blockIdx.x % slots;  // the block's place in the sequence
  const int64_t first = at * size;
  if (first >= start + count || at >= p.table_width) return;
  const int64_t block = p.table[b * p.table_stride + at];
  if (block < 0 || block >= p.cache.blocks) return;
  // the block's tokens [0, held) are older, [held, end) new
  const int held = start > first ? (int)(start - first) : 0;
  const int end = start + count < first + size ? (int)(start + count - first) : size;
  const int64_t token = first + held - start;  // the first new one's index in the call
  const T* x = values ? (const T*)p.v + b * p.v_stride_b + head * p.v_stride_h + token * p.v_stride_t
                      : (const T*)p.k + b * p.k_stride_b + head * p.k_stride_h + token * p.k_stride_t;
  const int64_t stride = values ? p.v_stride_t : p.k_stride_t;
  const int64_t page = block * p.cache.kv_heads + head;
  unsigned char* out = (unsigned char*)(values ? p.cache.v : p.cache.k) + page * size * D;
  float* scales = values ? p.cache.v_scale : p.cache.k_scale;

  const int n = (end - held) * D;
  float top = 0.0f;
  for (int i = threadIdx.x; i < n; i += THREADS)
    top = newt::Max::op(top, finite_abs(newt::to_f32(x[(int64_t)(i / D) * stride + i % D])));
  top = block_reduce<newt::Max, THREADS / 64>(top, slot);
  float scale = power_of_two(scale_exponent(top));
  if (held > 0) {
    const float had = scales[page];
    if (had >= scale) {
      scale = had;
    } else {
      // older tokens in the new scale
      const float f = had / scale;
      for (int i = threadIdx.x; i < held * D; i += THREADS) {
        unsigned char* o = values ? out + (i / held) * size + i % held : out + i;
        const float v = __builtin_amdgcn_cvt_f32_fp8((int)*o, 0) * f;
        *o = (unsigned char)to_e4m3x4(v, 0.0f, 0.0f, 0.0f);
      }
    }
  }
  for (int i = threadIdx.x; i < n; i += THREADS) {
    const int t = i / D, d = i % D;
    const float v = or_nan(newt::to_f32(x[(int64_t)t * stride + d]) / scale);
    out[values ? d * size + held + t : (held + t) * D + d] =
        (unsigned char)to_e4m3x4(v, 0.0f, 0.0f, 0.0f);
  }
  // every thread has read the old scale before block_reduce's barrier or, with
  // one wave, in program order before this
  __syncthreads();
  if (threadIdx.x == 0) scales[page] = scale;
}

template <typename T>
int launch(const newt_kv_append_params& p, hipStream_t stream) {
  // blocks that `tokens` consecutive ones can reach
  const int64_t slots = (p.tokens + p.cache.block_size - 2) / p.cache.block_size + 1;
  if (slots * p.batch > 0x7fffffff)
    return fail(NEWT_ERR_INVALID, "newt_kv_append: too many tokens");
  const dim3 grid((unsigned)(slots * p.batch), (unsigned)p.cache.kv_heads, 2);
  if (p.tokens <= 4)
    kv_append_kernel<T, 64><<<grid, dim3(64), 0, stream>>>(p, (int)slots);
  else
    kv_append_kernel<T, 256><<<grid, dim3(256), 0, stream>>>(p, (int)slots);
  return launched("newt_kv_append");
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
    case NEWT_F32: return launch<float>(p, s);
    case NEWT_F16: return launch<f16>(p, s);
    case NEWT_BF16: return launch<bf16>(p, s);
    default: return fail(NEWT_ERR_INVALID, "newt_kv_append: unknown dtype %d", p.dtype);
  }
}
