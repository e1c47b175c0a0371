// What the operators of libnewt_ops.so share: error reporting at the C entries,
// element conversions and reductions over a workgroup. Device templates
// (vector accesses, wave64 butterflies, MFMA wrappers, LDS tiles) come from
// newt_gfx950.h, the header of the compiled kernels.
#pragma once
#include <hip/hip_runtime.h>

#include <type_traits>

#include "../../../include/newt_ops.h"
#include "newt_gfx950.h"

namespace newt_ops {

// Keeps the message of the calling thread's last failure; fixed storage, so
// that reporting an error cannot fail itself.
int fail(int status, const char* format, ...) __attribute__((format(printf, 2, 3)));

int hip_fail(hipError_t e, const char* what);

template <typename T> struct same { typedef T type; };

// Launches a kernel and gives this launch's own status: what other code's
// calls have left behind is not looked at.
template <typename... P>
int run(const char* what, void (*kernel)(P...), int64_t grid, int block, unsigned lds,
        hipStream_t stream, typename same<P>::type... args) {
  void* list[] = {static_cast<void*>(&args)...};
  const hipError_t e = hipLaunchKernel(reinterpret_cast<const void*>(kernel),
                                       dim3((unsigned)grid), dim3((unsigned)block), list, lds,
                                       stream);
  return e == hipSuccess ? NEWT_OK : hip_fail(e, what);
}

// What is wrong with a cache's description, or null.
const char* cache_wrong(const newt_kv_cache& c);

// ---------------------------------------------------------------------------
// workgroup reductions: each wave's partial through LDS, read back by all.
// `slot` needs one float per wave; a second reduction takes another slot or a
// barrier between.
// ---------------------------------------------------------------------------
template <typename Op, int WAVES>
__device__ __forceinline__ float block_reduce(float v, float* slot) {
  v = newt::lane_reduce<Op, 63>(v);
  if constexpr (WAVES > 1) {
    if ((threadIdx.x & 63) == 0) slot[threadIdx.x >> 6] = v;
    __syncthreads();
    v = slot[0];
#pragma unroll
    for (int i = 1; i < WAVES; ++i) v = Op::op(v, slot[i]);
  }
  return v;
}

// The wave's index in its workgroup, as a number that the compiler knows to be
// the same in all of its lanes.
__device__ __forceinline__ int wave_id() {
  return __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
}

// Four floats to four e4m3 bytes, rounded to nearest even by the hardware.
__device__ __forceinline__ u32 to_e4m3x4(float a, float b, float c, float d) {
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return (u32)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
}

}  // namespace newt_ops
