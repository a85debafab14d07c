// runtime.cu -- error state and process-wide switches of the C ABI (declared
// in include/sm120norm_b200.h and csrc/runtime.h).
#include <atomic>
#include <cstdarg>
#include <cstdio>
#include <string>

#include "runtime.h"

namespace sm120n {
namespace {

thread_local std::string g_last_error;
std::atomic<bool> g_programmatic_launch{true};
std::atomic<uint32_t> g_wait_polls{kDefaultWaitPolls};

}  // namespace

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

bool programmatic_launch_enabled() { return g_programmatic_launch.load(std::memory_order_relaxed); }

uint32_t wait_poll_limit() { return g_wait_polls.load(std::memory_order_relaxed); }

}  // namespace sm120n

extern "C" {

int sm120n_abi_version(void) { return SM120N_ABI_VERSION; }

const char* sm120n_last_error(void) { return sm120n::g_last_error.c_str(); }

const char* sm120n_status_string(int status) {
  switch (status) {
    case SM120N_OK: return "ok";
    case SM120N_ERR_INVALID_ARGUMENT: return "invalid argument";
    case SM120N_ERR_UNSUPPORTED: return "unsupported";
    case SM120N_ERR_CUDA: return "CUDA error";
    default: return "unknown status";
  }
}

void sm120n_set_programmatic_launch(int enabled) { sm120n::g_programmatic_launch.store(enabled != 0); }

int sm120n_get_programmatic_launch(void) { return sm120n::g_programmatic_launch.load() ? 1 : 0; }

void sm120n_set_wait_limit(uint32_t polls) {
  sm120n::g_wait_polls.store(polls == 0 || polls > sm120n::kDefaultWaitPolls
                                 ? sm120n::kDefaultWaitPolls
                                 : polls);
}

uint32_t sm120n_get_wait_limit(void) { return sm120n::g_wait_polls.load(); }

}  // extern "C"
