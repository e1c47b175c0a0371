// What the products with 4-bit weights share: from a word of weights to an operand
// of the matrix unit, and from sums to outputs.
#pragma once
#include "byte_rows.h"
#include "common.h"

namespace newt_ops {

template <typename T> struct frag;
template <> struct frag<bf16> { typedef bf16x8 type; };
template <> struct frag<f16> { typedef f16x8 type; };

// What weights are multiplied by as operands, a power of two: sums hold this times
// x (16 + q) / 16 for the columns of a group. Where x is bf16 they would leave fp32's
// range long before the result does; of 128 columns and zeros of any byte none comes
// to 2^128 this way (16 x 2^7 x 2^128 / 2^12). Sums below 2^-110 pay: they
// lose up to 2^-133 an addition.
template <typename T> constexpr float kUnit = __is_same(T, bf16) ? 0x1p-12f : 1.0f;
// A group's sum (q - z) x from what is summed.
template <typename T> constexpr float kWhole = 16.0f / kUnit<T>;

// 8 weights to kUnit (16 + q) / 16: the 4 bits go below the point of a number in
// [kUnit, 2 kUnit), by one shift and one v_and_or_b32 for two of them. That
// instruction takes one constant from a scalar register and none from the code, so
// both are kept from the compiler, which would rather use two instructions with
// constants in them.
template <typename T>
struct Widen {
  u32 mask;
  u32x4 ones;  // kUnit in both halves: an operand of these, too
  __device__ __forceinline__ Widen() {
    constexpr bool B = __is_same(T, bf16);  // the upper 4 of 7 bits, or of 10
    mask = B ? 0x00780078u : 0x03c003c0u;
    ones = (u32x4)(B ? 0x39803980u : 0x3c003c00u);
    asm("" : "+s"(mask));
    asm("" : "+v"(ones));
  }
  __device__ __forceinline__ typename frag<T>::type operator()(u32 w) const {
    const u32 one = ones[0];
    u32x4 r;
    if constexpr (__is_same(T, bf16)) {
      r[0] = (w & mask) | one;
      r[1] = ((w >> 4) & mask) | one;
      r[2] = ((w >> 8) & mask) | one;
      r[3] = (__builtin_amdgcn_alignbit(w, w, 12) & mask) | one;
    } else {
      r[0] = ((w << 3) & mask) | one;
      r[1] = ((w >> 1) & mask) | one;
      r[2] = ((w >> 5) & mask) | one;
      r[3] = (__builtin_amdgcn_alignbit(w, w, 9) & mask) | one;
    }
    return __builtin_bit_cast(typename frag<T>::type, r);
  }
};

__device__ __forceinline__ float activate(float v, int act) {
  if (act == NEWT_ACT_SILU) return v / (1.0f + __builtin_expf(-v));
  // 1 + erf cancels below 0: 4% off at -5. 512 x 4096 x 2 x 12288 takes 129 us with erfc, 125
  // with erf, one row 12 with either.
  return 0.5f * v * erfcf(v * -0.70710678f);
}

// 4 neighbouring outputs of a row from `first` on.
template <typename T>
__device__ __forceinline__ void store4(const newt_q4_params& p, int64_t row, int64_t first,
                                       f32x4 y) {
  const int count = p.outputs - first < 4 ? (int)(p.outputs - first) : 4;
  if (p.bias) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i < count) y[i] += newt::to_f32(((const T*)p.bias)[first + i]);
  }
  if (p.out_dtype == NEWT_F32) {
    float* out = (float*)p.out + row * p.out_stride + first;
    const float t[4] = {y[0], y[1], y[2], y[3]};
    if (count == 4) newt::store_vec<float, 4>(out, t, newt::any_align());
    else for (int i = 0; i < count; ++i) out[i] = t[i];
  } else {
    T* out = (T*)p.out + row * p.out_stride + first;
    const T t[4] = {(T)y[0], (T)y[1], (T)y[2], (T)y[3]};
    if (count == 4) newt::store_vec<T, 4>(out, t, newt::any_align());
    else for (int i = 0; i < count; ++i) out[i] = t[i];
  }
}

// Whether out lies over x or bias, which programs read while others write.
inline bool out_meets(const newt_q4_params& p) {
  const int64_t size = p.out_dtype == NEWT_F32 ? 4 : 2;
  const ByteRows out(p.out, p.rows, p.out_stride * size, p.outputs * size);
  return rows_meet(out, ByteRows(p.x, p.rows, p.x_stride * 2, p.cols * 2)) ||
         rows_meet(out, ByteRows(p.bias, p.bias ? 1 : 0, 0, p.outputs * 2));
}

// q4_many.hip: products with many rows of x.
size_t q4_many_workspace(const newt_q4_params& p);
int q4_many(const newt_q4_params& p, hipStream_t stream);

}  // namespace newt_ops
