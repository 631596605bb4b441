// What the launch layers share: the calling thread's last error.
#pragma once

#include <hip/hip_runtime.h>

#include "triton_ext/tx_dot.h"

namespace txk {

// Sets the calling thread's last error (tx_get_last_error) and returns `code`.
int fail(int code, const char *fmt, ...) __attribute__((format(printf, 2, 3)));
void clearError();

} // namespace txk

#define TX_HIP_CHECK(expr)                                                     \
  do {                                                                         \
    hipError_t e_ = (expr);                                                    \
    if (e_ != hipSuccess)                                                      \
      return fail(TX_ERR_HIP, "%s failed: %s", #expr, hipGetErrorString(e_));  \
  } while (0)
