// Error reporting shared by the files of C entry points (defined in bg_api.hip): the calling thread's
// last message and a BG_E_* code, and whether a stream is being captured.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace bg {
int32_t api_fail(int32_t code, const char* msg);
int32_t api_hip_fail(hipError_t e, const char* what);
bool api_capturing(hipStream_t st);
}  // namespace bg
