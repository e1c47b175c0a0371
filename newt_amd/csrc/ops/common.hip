// Error reporting of libnewt_ops.so (include/newt_ops.h).
#include <cstdarg>
#include <cstdio>

#include "common.h"

namespace newt_ops {

namespace {
thread_local char last_error[512] = "";
}

int fail(int status, const char* format, ...) {
  va_list args;
  va_start(args, format);
  std::vsnprintf(last_error, sizeof last_error, format, args);
  va_end(args);
  return status;
}

int hip_fail(hipError_t e, const char* what) {
  return fail(static_cast<int>(e), "%s: %s (%s)", what, hipGetErrorName(e), hipGetErrorString(e));
}

const char* cache_wrong(const newt_kv_cache& c) {
  const int s = c.block_size;
  if (s != 16 && s != 32 && s != 64 && s != 128 && s != 256)
    return "blocks hold 16, 32, 64, 128 or 256 tokens";
  if (c.head_dim != 64 && c.head_dim != 128 && c.head_dim != 256)
    return "head_dim is 64, 128 or 256";
  if (c.blocks < 0 || c.kv_heads <= 0 || c.kv_heads > 65535) return "bad number of blocks or heads";
  if (c.blocks && (!c.k || !c.v || !c.k_scale || !c.v_scale)) return "null cache tensor";
  if (((uintptr_t)c.k | (uintptr_t)c.v) & 15) return "keys and values have to be aligned to 16 bytes";
  return nullptr;
}

}  // namespace newt_ops

extern "C" {
int newt_ops_abi_version(void) { return NEWT_OPS_ABI_VERSION; }
const char* newt_ops_last_error(void) { return newt_ops::last_error; }
}
