// Error reporting and checks shared by the C ABI's files.
#pragma once

#include <hip/hip_runtime.h>

#include <cstddef>
#include <cstdint>

#include "omx_gdn.h"

namespace omx {

// sets the calling thread's message and returns `code`; clears it and returns OMX_GDN_OK
int fail(int code, const char* fmt, ...) __attribute__((format(printf, 2, 3)));
int ok();
int launch_status(hipError_t e, const char* what);

inline bool aligned(const void* p, size_t a) { return (reinterpret_cast<uintptr_t>(p) % a) == 0; }

}  // namespace omx

#define REQUIRE(cond, ...) \
  do {                     \
    if (!(cond)) return omx::fail(OMX_GDN_EINVAL, __VA_ARGS__); \
  } while (0)
