// Rotary positions of queries and keys:
//   (a, b) -> amplitude (a cos pf - b sin pf, b cos pf + a sin pf)
// for the pairs of a head, f the pair's frequency, p the token's position.
// Angles are fractions of a turn: with f / 2 pi held as a 64-bit fraction the
// product with p modulo 2^64 is the fraction of a turn that is left, whatever the
// position, off by 2^-34 of a turn at most; its upper 32 bits, rounded, give the quadrant
// and, exactly, the rest of at most pi/4, whose sine and cosine are short sums.
// HBM bounds it, each number read and written once. A thread keeps the angles of
// its pairs for a token and turns two heads by them. What it reads it reads past the
// caches (non-temporal), which leaves them to the outputs: bf16 4 x (32 + 8) x 4096 x
// 128 as slices of one product, outputs in the same memory every time, 56 us (6.0 TB/s)
// and 67 without; in other memory every time 64 (5.3 TB/s) and 70. Outputs past the
// caches too take 63 either way, but the next operator would find them in HBM.
#include "common.h"

namespace newt_ops {
namespace {

// cos and sin of 2 pi turns / 2^32: |x| <= pi/4 and the quadrant. The sums'
// first terms left out are x^12 / 12! and x^11 / 11!, below 2^-29.
__device__ __forceinline__ void cos_sin(u32 turns, float& c, float& s) {
  const u32 quadrant = (turns + 0x20000000u) >> 30;
  const float x = (float)(int)(turns - (quadrant << 30)) * 1.46291807926715968e-9f;  // 2 pi / 2^32
  const float y = x * x;
  float ps = 2.7557319e-6f, pc = -2.7557319e-7f;
  ps = __builtin_fmaf(ps, y, -1.9841270e-4f);
  pc = __builtin_fmaf(pc, y, 2.4801587e-5f);
  ps = __builtin_fmaf(ps, y, 8.3333333e-3f);
  pc = __builtin_fmaf(pc, y, -1.3888889e-3f);
  ps = __builtin_fmaf(ps, y, -1.6666667e-1f);
  pc = __builtin_fmaf(pc, y, 4.1666667e-2f);
  pc = __builtin_fmaf(pc, y, -0.5f);
  ps = __builtin_fmaf(ps * y, x, x);
  pc = __builtin_fmaf(pc, y, 1.0f);
  c = quadrant & 1 ? ps : pc;
  s = quadrant & 1 ? pc : ps;
  if ((quadrant + 1) & 2) c = -c;
  if (quadrant & 2) s = -s;
}

// A unit is V pairs of a head; what is behind them is copied, V numbers a unit.
template <typename T, int V, bool INTERLEAVED>
__global__ void __launch_bounds__(256)
rotate_kernel(newt_rotate_params p, u32 slots, u32 units, u32 threads) {
  const u32 i = blockIdx.x * 256 + threadIdx.x;
  if (i >= threads) return;
  const u32 unit = i % units, rest = i / units;
  const u32 slot = rest % slots, token = rest / slots;
  const u32 t = token % (u32)p.tokens, b = token / (u32)p.tokens;
  const u32 heads = (u32)(p.heads + p.kv_heads);
  const int half = (int)p.rot_dim / 2, D = (int)p.head_dim;
  const int turned = half / V;  // units of pairs, then those that are copied
  const T* q = (const T*)p.q + b * p.q_stride_b + t * p.q_stride_t;
  const T* k = (const T*)p.k + b * p.k_stride_b + t * p.k_stride_t;
  T* qo = (T*)p.q_out + b * p.qo_stride_b + t * p.qo_stride_t;
  T* ko = (T*)p.k_out + b * p.ko_stride_b + t * p.ko_stride_t;
  const auto from = [&](u32 h) {
    return h < (u32)p.heads ? q + h * p.q_stride_h : k + (h - (u32)p.heads) * p.k_stride_h;
  };
  const auto to = [&](u32 h) {
    return h < (u32)p.heads ? qo + h * p.qo_stride_h : ko + (h - (u32)p.heads) * p.ko_stride_h;
  };
  if ((int)unit >= turned) {
    const int d = 2 * half + ((int)unit - turned) * V;
#pragma unroll 4
    for (u32 h = slot; h < heads; h += slots) {
      const T* x = from(h) + d;
      T* y = to(h) + d;
      if (d + V <= D) {
        T v[V];
        newt::load_vec_nt<T, V>(x, v, newt::any_align());
        newt::store_vec<T, V>(y, v, newt::any_align());
      } else {
        for (int j = 0; d + j < D; ++j) y[j] = x[j];
      }
    }
    return;
  }
  const int position = p.positions[b * p.position_stride_b + (p.each ? t * p.position_stride_t : 0)];
  const u64 at = (u64)((long long)position + (p.each ? 0 : (long long)t));
  // Two pieces of V numbers, half of what turns apart: neighbouring lanes read
  // neighbouring pieces. They hold the two sides of V pairs, or V / 2 pairs each (one
  // pair where V is 1).
  constexpr bool PAIRS = INTERLEAVED && V > 1;
  const int d0 = (int)unit * V * (INTERLEAVED && !PAIRS ? 2 : 1);
  const int d1 = d0 + (INTERLEAVED && !PAIRS ? 1 : half);
  float c[V], s[V];
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const int pair = !PAIRS ? (int)unit * V + j : j < V / 2 ? d0 / 2 + j : d1 / 2 + j - V / 2;
    const u64 turns = at * p.turns[pair];
    cos_sin((u32)((turns + 0x80000000ull) >> 32), c[j], s[j]);
    c[j] *= p.amplitude;
    s[j] *= p.transposed ? -p.amplitude : p.amplitude;
  }
#pragma unroll 4
  for (u32 h = slot; h < heads; h += slots) {
    const T* x = from(h);
    T* y = to(h);
    T v[2 * V];
    newt::load_vec_nt<T, V>(x + d0, v, newt::any_align());
    newt::load_vec_nt<T, V>(x + d1, v + V, newt::any_align());
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int ia = PAIRS ? 2 * j : j, ib = PAIRS ? 2 * j + 1 : j + V;
      const float a = newt::to_f32(v[ia]), e = newt::to_f32(v[ib]);
      v[ia] = (T)(a * c[j] - e * s[j]);
      v[ib] = (T)(e * c[j] + a * s[j]);
    }
    newt::store_vec<T, V>(y + d0, v, newt::any_align());
    newt::store_vec<T, V>(y + d1, v + V, newt::any_align());
  }
}

template <typename T, int V>
int launch(const newt_rotate_params& p, hipStream_t stream) {
  const int64_t units = p.rot_dim / 2 / V + (p.head_dim - p.rot_dim + V - 1) / V;
  const int64_t heads = p.heads + p.kv_heads, tokens = p.batch * p.tokens;
  // two heads a thread, or one where the threads would not fill the chip: us of 1, 2, 4
  // and 8 in the large case above, outputs in other memory every time, 71 / 65 / 67 /
  // 68, interleaved 64 / 63 / 65 / 66, of 2 x 40 x 4096 x 128 in fp32 60 / 63 / 65 / 69
  int64_t each = units * tokens * heads / (256 * 1024);
  each = each < 1 ? 1 : each > 2 ? 2 : each;
  const int64_t slots = (heads + each - 1) / each, threads = units * tokens * slots;
  if (threads > 0xffffffffll - 256 || units > 0x7fffffff)
    return fail(NEWT_ERR_INVALID, "newt_rotate: too many tokens");
  const auto kernel = p.interleaved ? rotate_kernel<T, V, true> : rotate_kernel<T, V, false>;
  return run("newt_rotate", kernel, (threads + 255) / 256, 256, 0, stream, p, (u32)slots,
             (u32)units, (u32)threads);
}

template <typename T>
int by_width(const newt_rotate_params& p, hipStream_t stream) {
  // 16 bytes an access where the pairs divide into such pieces
  constexpr int WIDE = 16 / (int)sizeof(T);
  if (p.rot_dim % (2 * WIDE) == 0) return launch<T, WIDE>(p, stream);
  if (p.rot_dim % 8 == 0) return launch<T, 4>(p, stream);
  return launch<T, 1>(p, stream);
}

const char* wrong(const newt_rotate_params& p) {
  if (p.batch < 0 || p.tokens < 0 || p.heads < 0 || p.kv_heads < 0) return "negative size";
  if (p.head_dim <= 0 || p.head_dim >= 1 << 20) return "head_dim is 1 to 2^20";
  if (p.rot_dim < 2 || p.rot_dim % 2 || p.rot_dim > p.head_dim)
    return "rot_dim is even, from 2 to head_dim";
  if (p.batch >= 1 << 30 || p.tokens >= 1 << 30 || p.heads >= 1 << 30 || p.kv_heads >= 1 << 30 ||
      p.batch * p.tokens >= 1ll << 31)
    return "too many tokens";
  if ((double)(p.batch * p.tokens) * (double)(p.heads + p.kv_heads) * (double)p.head_dim > 0x1p50)
    return "too many tokens";
  if (!(__builtin_fabsf(p.amplitude) < __builtin_inff())) return "amplitude has to be finite";
  const int D = (int)p.head_dim;
  if ((p.heads && rows_overlap(D, p.batch, p.qo_stride_b, p.heads, p.qo_stride_h, p.tokens,
                               p.qo_stride_t)) ||
      (p.kv_heads && rows_overlap(D, p.batch, p.ko_stride_b, p.kv_heads, p.ko_stride_h, p.tokens,
                                  p.ko_stride_t)))
    return "rows of an output overlap";
  return nullptr;
}

}  // namespace
}  // namespace newt_ops

extern "C" int newt_rotate(const newt_rotate_params* params, void* stream) {
  using namespace newt_ops;
  if (!params) return fail(NEWT_ERR_INVALID, "newt_rotate: null params");
  const newt_rotate_params& p = *params;
  if (const char* w = wrong(p)) return fail(NEWT_ERR_INVALID, "newt_rotate: %s", w);
  if (p.dtype != NEWT_F32 && p.dtype != NEWT_F16 && p.dtype != NEWT_BF16)
    return fail(NEWT_ERR_INVALID, "newt_rotate: unknown dtype %d", p.dtype);
  if (p.batch == 0 || p.tokens == 0 || p.heads + p.kv_heads == 0) return NEWT_OK;
  if ((p.heads && (!p.q || !p.q_out)) || (p.kv_heads && (!p.k || !p.k_out)) || !p.turns ||
      !p.positions)
    return fail(NEWT_ERR_INVALID, "newt_rotate: null tensor");
  hipStream_t s = static_cast<hipStream_t>(stream);
  switch (p.dtype) {
    case NEWT_F32: return by_width<float>(p, s);
    case NEWT_F16: return by_width<f16>(p, s);
    default: return by_width<bf16>(p, s);
  }
}
