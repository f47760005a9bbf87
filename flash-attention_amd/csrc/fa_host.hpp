// What the library's translation units share on the host side: the calling thread's error text and the event-timed
// launch.  Not exported.
#pragma once
#include <hip/hip_runtime.h>

#define FA_HIDDEN __attribute__((visibility("hidden")))

namespace fa_host {

// Sets fa_last_error()'s text for the calling thread and returns `code`.
FA_HIDDEN int fail(int code, const char* text);
FA_HIDDEN void clear_error();
// Runs `launch(arg)` on `stream`; with elapsed_ms non-null it is bracketed by events and waited for.
FA_HIDDEN int timed(hipStream_t stream, float* elapsed_ms, int (*launch)(void*), void* arg);
// Compute units of the current device.
FA_HIDDEN int device_cus();

}  // namespace fa_host
