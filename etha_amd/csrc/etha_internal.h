// What the library's source files share: error reporting of the C ABI and the launch counter.
#ifndef ETHA_INTERNAL_H
#define ETHA_INTERNAL_H

#include <hip/hip_runtime.h>

#include <atomic>
#include <cstdarg>
#include <cstdio>
#include <exception>
#include <new>

#include "etha_reshard.h"

namespace etha_internal {

// message of the calling thread's last failure; a fixed buffer, so that reporting a failure (out of host memory
// among them) allocates nothing
inline thread_local char g_err[512] = "";

inline std::atomic<uint64_t> g_kernel_launches{0};

inline int fail(int code, const char* fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(g_err, sizeof(g_err), fmt, ap);
  va_end(ap);
  return code;
}

// Body of an entry point that builds host-side containers: no C++ exception leaves the library (the ABI is
// plain C); running out of host memory becomes ETHA_ERR_NOMEM.
template <typename F>
int guarded(const char* what, F&& body) {
  try {
    return body();
  } catch (const std::bad_alloc&) {
    return fail(ETHA_ERR_NOMEM, "%s: out of host memory", what);
  } catch (const std::exception& e) {
    return fail(ETHA_ERR_INVALID, "%s: %s", what, e.what());
  } catch (...) {
    return fail(ETHA_ERR_INVALID, "%s: unexpected exception", what);
  }
}

}  // namespace etha_internal

#define HIP_TRY(expr)                                                                                    \
  do {                                                                                                   \
    hipError_t e_ = (expr);                                                                              \
    if (e_ != hipSuccess)                                                                                \
      return etha_internal::fail(ETHA_ERR_HIP, "%s: %s", #expr, hipGetErrorString(e_));                  \
  } while (0)

#endif  // ETHA_INTERNAL_H
