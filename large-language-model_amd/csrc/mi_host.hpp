// mi_host.hpp -- host state that every C entry point shares (held in mi_gemm.hip): the error
// text of the calling thread, the check of the current device and its CU count.
#pragma once
#include <stdarg.h>
#include <stdint.h>
#include <stdio.h>

#include "../../include/mi_gemm.h"

namespace mig {

int host_error(int code, const char* text);  // stores mi_last_error's text, returns code
int host_device();                           // MI_OK if the current device is a gfx950
int host_cus();                              // CUs of the current device

// Workgroups of `threads` that a launch may have: its threads are counted in 32 bits.
inline int64_t host_most_groups(int threads) { return UINT32_MAX / (uint32_t)threads; }

inline int host_fail(int code, const char* fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof(buf), fmt, ap);
  va_end(ap);
  return host_error(code, buf);
}

}  // namespace mig
