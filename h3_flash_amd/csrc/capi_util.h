// Shared by the files of C entry points: the per-thread message and the CU count.
#pragma once

#include <stdint.h>

namespace h3a {

// Sets the calling thread's message and returns `code`.
int fail(int code, const char* fmt, ...);
void clear_error();

// CU count of the current device, cached per device (0: unknown).
int device_cus();

inline bool aligned16(const void* p) { return ((uintptr_t)p & 15u) == 0; }
inline bool aligned4(const void* p) { return ((uintptr_t)p & 3u) == 0; }

}  // namespace h3a
