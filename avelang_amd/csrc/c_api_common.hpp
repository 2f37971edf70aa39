// Error text shared by the translation units of the C ABI (defined in c_api.hip).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace ave {

int fail_inval(const char* fmt, ...) __attribute__((format(printf, 1, 2)));   // AVE_FP4_EINVAL
int finish(hipError_t e, const char* what);                                   // 0, or the hipError_t with its message
void clear_error();
inline bool aligned(const void* p, size_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

}  // namespace ave
