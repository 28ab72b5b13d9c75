// Library identity and thread-local error reporting for the C ABI.
#include <string.h>

#include "abi_util.h"

namespace tbf16 {

static thread_local char g_err[512] = "";

void set_error(const char* fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(g_err, sizeof(g_err), fmt, ap);
  va_end(ap);
}

int64_t num_cus() {
  static int64_t cache[64] = {};
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) return 256;
  if (cache[dev] == 0) {
    int n = 0;
    if (hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || n <= 0) n = 256;
    cache[dev] = n;
  }
  return cache[dev];
}

}  // namespace tbf16

extern "C" int tbf16_abi_version(void) { return TBF16_ABI_VERSION; }

extern "C" const char* tbf16_last_error(void) { return tbf16::g_err; }
