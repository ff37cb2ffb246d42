// dpft_internal.h -- what the translation units of libdpft_ic.so share.
#ifndef DPFT_INTERNAL_H
#define DPFT_INTERNAL_H

#include <hip/hip_runtime.h>

// Sets dpft_last_error()'s thread-local message and returns `code`.
__attribute__((visibility("hidden"), format(printf, 2, 3))) int dpft_fail(int code, const char* fmt, ...);
// DPFT_OK, or DPFT_E_HIP with the name of the launch that failed.
__attribute__((visibility("hidden"))) int dpft_hip_check(const char* what);

#endif  // DPFT_INTERNAL_H
