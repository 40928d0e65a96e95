// What the C entry points share: error reporting and checks of arguments.
#pragma once

#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdarg>
#include <cstdio>

#include "../../include/pal_hip.h"
#include "pal_hip_internal.h"
#include "pal_log.h"

namespace {

inline int fail(int code, const char* fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof(buf), fmt, ap);
  va_end(ap);
  pal::set_last_error(buf);
  return code;
}

inline int ok() {
  pal::clear_last_error();
  return PAL_OK;
}

inline int hip_status(hipError_t err, const char* what) {
  if (err == hipSuccess) return ok();
  return fail(PAL_ERR_HIP, "[%s] HIP error: %s", what, hipGetErrorString(err));
}

inline bool valid_dtype(int dtype) { return dtype == PAL_DTYPE_FLOAT16 || dtype == PAL_DTYPE_BFLOAT16; }
inline bool valid_pool_dtype(int dtype) { return valid_dtype(dtype) || dtype == PAL_DTYPE_FP8_E4M3; }
inline int pool_elem_bytes(int dtype) { return dtype == PAL_DTYPE_FP8_E4M3 ? 1 : 2; }

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

inline float scale_log2_for(int head_dim) {
  return static_cast<float>(1.4426950408889634 / std::sqrt(static_cast<double>(head_dim)));
}

inline size_t align256(size_t n) { return (n + 255) & ~static_cast<size_t>(255); }

constexpr int kMaxPageSize = 1024;  // prefill's run-time page sizes (multiples of 8)

// Checks shared by every attention entry point; returns PAL_OK or an error.
inline int check_attention_dims(const char* op, int dtype, int num_q_heads, int num_kv_heads, int head_dim,
                                int tokens_per_page, int64_t num_pages, int64_t page_table_width,
                                bool any_page_size = false) {
  if (!valid_dtype(dtype)) return fail(PAL_ERR_INVALID_ARGUMENT, "[%s] unsupported dtype code %d", op, dtype);
  if (num_q_heads <= 0 || num_kv_heads <= 0 || head_dim <= 0 || tokens_per_page <= 0 || num_pages < 0 ||
      page_table_width < 0)
    return fail(PAL_ERR_INVALID_ARGUMENT, "[%s] negative or zero dimension", op);
  if (num_q_heads % num_kv_heads != 0)
    return fail(PAL_ERR_RUNTIME, "num_q_heads must be divisible by num_kv_heads (%d %% %d != 0)", num_q_heads,
                num_kv_heads);
  if (any_page_size) {  // prefill over 16-bit pools: any multiple of 8 up to kMaxPageSize
    if (tokens_per_page % 8 != 0 || tokens_per_page > kMaxPageSize)
      return fail(PAL_ERR_RUNTIME, "[%s] no kernel for tokens_per_page %d (supported: multiples of 8 up to %d)", op,
                  tokens_per_page, kMaxPageSize);
  } else if (tokens_per_page != 16 && tokens_per_page != 32) {
    return fail(PAL_ERR_RUNTIME, "[%s] no kernel for tokens_per_page %d (supported: 16, 32)", op, tokens_per_page);
  }
  return PAL_OK;
}

}  // namespace
