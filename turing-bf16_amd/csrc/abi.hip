// Library identity and thread-local error reporting for the C ABI.
#include <string.h>

#include <atomic>

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
  static std::atomic<int> cache[64];
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) return 256;
  int n = cache[dev].load(std::memory_order_relaxed);
  if (n == 0) {
    if (hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || n <= 0) n = 256;
    cache[dev].store(n, std::memory_order_relaxed);
  }
  return n;
}

}  // namespace tbf16

extern "C" int tbf16_abi_version(void) { return TBF16_ABI_VERSION; }

extern "C" const char* tbf16_last_error(void) { return tbf16::g_err; }
