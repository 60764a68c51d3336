// Error plumbing and runtime queries of the C ABI (include/coopt_amd.h).
#include "common.h"

namespace coopt {

static thread_local std::string g_last_error;

void set_error(const std::string& msg) { g_last_error = msg; }
void clear_error() { g_last_error.clear(); }

int check_launch(const char* what) {
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) {
    set_error(std::string(what) + ": " + hipGetErrorString(e));
    return COOPT_EHIP;
  }
  return COOPT_OK;
}

const char* cache_write_error(int cache_dtype, const void* k_cache, const void* v_cache,
                              int64_t c_blk_stride, int64_t c_tok_stride, int64_t c_head_stride,
                              const void* k_scale, const void* v_scale) {
  // a lane stores 16 bytes of a bf16 row, 8 of an INT8 row, 4 of an INT4 row; strides count
  // elements (INT4: bytes)
  const uintptr_t bytes = cache_dtype == COOPT_DT_BF16 ? 16 : cache_dtype == COOPT_DT_I8 ? 8 : 4;
  const int64_t step = cache_dtype == COOPT_DT_I4 ? 4 : 8;
  if (cache_dtype != COOPT_DT_BF16) {
    if (!k_scale || !v_scale)
      return cache_dtype == COOPT_DT_I8 ? "INT8 cache needs k_scale and v_scale" : "INT4 cache needs k_scale and v_scale";
    if (((reinterpret_cast<uintptr_t>(k_scale) | reinterpret_cast<uintptr_t>(v_scale)) & 1u) != 0)
      return "scales must be 2-byte aligned";
  }
  if (((reinterpret_cast<uintptr_t>(k_cache) | reinterpret_cast<uintptr_t>(v_cache)) & (bytes - 1)) != 0 ||
      c_blk_stride % step || c_tok_stride % step || c_head_stride % step)
    return cache_dtype == COOPT_DT_BF16  ? "bf16 cache rows must be 16-byte aligned"
           : cache_dtype == COOPT_DT_I8 ? "INT8 cache rows must be 8-byte aligned"
                                         : "INT4 cache rows must be 4-byte aligned";
  return nullptr;
}

}  // namespace coopt

extern "C" const char* coopt_last_error(void) { return coopt::g_last_error.c_str(); }

extern "C" int coopt_hip_runtime_version(int* version) {
  COOPT_REQUIRE(version != nullptr, "null version pointer");
  hipError_t e = hipRuntimeGetVersion(version);
  if (e != hipSuccess) {
    coopt::set_error(std::string("hipRuntimeGetVersion: ") + hipGetErrorString(e));
    return COOPT_EHIP;
  }
  return COOPT_OK;
}
