// serving_runtime.cu -- error state and fault counter of the serving library
// (declared in include/sm120norm_b200_serving.h). Its kernels follow the
// process-wide switches of the norm library, sm120n_set_programmatic_launch and
// sm120n_set_wait_limit.
#include <cstdarg>
#include <cstdio>
#include <string>

#include "runtime.h"
#include "sm120norm_b200_serving.h"

namespace sm120n {
namespace {
thread_local std::string g_last_error;
}

int fail(int status, const char* fmt, ...) {
  char buffer[512];
  va_list args;
  va_start(args, fmt);
  vsnprintf(buffer, sizeof buffer, fmt, args);
  va_end(args);
  g_last_error = buffer;
  return status;
}

void clear_error() { g_last_error.clear(); }

bool programmatic_launch_enabled() { return sm120n_get_programmatic_launch() != 0; }

uint32_t wait_poll_limit() { return sm120n_get_wait_limit(); }

}  // namespace sm120n

extern "C" {

int sm120s_abi_version(void) { return SM120S_ABI_VERSION; }

const char* sm120s_last_error(void) { return sm120n::g_last_error.c_str(); }

}  // extern "C"
