// Host-side helpers every translation unit of libhecka shares: the calling thread's error message, launch checks, alignment.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>
#include <stdio.h>

#include "../../include/hecka.h"

namespace hecka {

inline thread_local char g_err[256] = "";

inline int fail(int code, const char* fmt, const char* a = "", long long x = 0, long long y = 0) {
  snprintf(g_err, sizeof(g_err), fmt, a, x, y);
  return code;
}
inline int check_launch(const char* what) {
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return fail(HECKA_ELAUNCH, "%s: launch failed (%lld)", what, (long long)e);
  return HECKA_OK;
}
// hipGetLastError is sticky per thread: drop whatever an earlier, unrelated runtime call left behind so
// that check_launch reports only this launch.
inline void clear_error() { (void)hipGetLastError(); }
inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace hecka
