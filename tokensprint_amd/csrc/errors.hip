#include <stdarg.h>
#include "common.h"

static thread_local char g_error[512] = "";

void ts_set_error(const char* fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(g_error, sizeof(g_error), fmt, ap);
  va_end(ap);
}

extern "C" const char* ts_last_error() { return g_error; }

// Version of the C interface; the Python loader refuses a library with another one.
extern "C" int ts_abi_version() { return 3; }

// Which capture the stream's work goes into: a number that no other capture has, or 0.
extern "C" int64_t ts_capture_id(hipStream_t stream) {
  hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
  unsigned long long id = 0;
  if (hipStreamGetCaptureInfo(stream, &status, &id) != hipSuccess) {
    (void)hipGetLastError();
    return 0;
  }
  return status == hipStreamCaptureStatusActive ? (int64_t)id : 0;
}
