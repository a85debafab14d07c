// device_caches.cu -- per-device properties, occupancy and shared-memory grants
// behind csrc/runtime.h, asked of the CUDA runtime once, and the wait for a
// device; linked into both libraries.
#include <map>
#include <mutex>
#include <tuple>

#include "runtime.h"

namespace sm120n {
namespace {

constexpr int kMaxDevices = 64;
std::mutex g_cache_mutex;
int g_sm_count[kMaxDevices] = {0};
std::map<std::tuple<int, const void*, int, size_t>, int> g_occupancy;
std::map<std::pair<int, const void*>, size_t> g_smem_optin;
size_t g_block_smem[kMaxDevices] = {0};

}  // namespace

int current_device_info(DeviceInfo* info) {
  int device = 0;
  cudaError_t err = cudaGetDevice(&device);
  if (err != cudaSuccess) {
    return fail(SM120N_ERR_CUDA, "cudaGetDevice failed: %s", cudaGetErrorString(err));
  }
  if (device < 0 || device >= kMaxDevices) {
    return fail(SM120N_ERR_UNSUPPORTED, "device ordinal %d is out of range", device);
  }
  std::lock_guard<std::mutex> lock(g_cache_mutex);
  if (g_sm_count[device] == 0) {
    int sms = 0;
    err = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device);
    if (err != cudaSuccess || sms <= 0) {
      return fail(SM120N_ERR_CUDA, "cannot query the SM count of device %d: %s", device,
                  cudaGetErrorString(err));
    }
    g_sm_count[device] = sms;
  }
  info->device = device;
  info->sm_count = g_sm_count[device];
  return SM120N_OK;
}

int wait_for_device() {
  const cudaError_t err = cudaDeviceSynchronize();
  return err == cudaSuccess ? SM120N_OK
                            : fail(SM120N_ERR_CUDA, "waiting for the device failed: %s",
                                   cudaGetErrorString(err));
}

int max_resident_ctas(const void* kernel, int threads, size_t smem, int* out) {
  int device = 0;
  cudaError_t err = cudaGetDevice(&device);
  if (err != cudaSuccess) {
    return fail(SM120N_ERR_CUDA, "cudaGetDevice failed: %s", cudaGetErrorString(err));
  }
  const auto key = std::make_tuple(device, kernel, threads, smem);
  {
    std::lock_guard<std::mutex> lock(g_cache_mutex);
    auto it = g_occupancy.find(key);
    if (it != g_occupancy.end()) {
      *out = it->second;
      return SM120N_OK;
    }
  }
  int ctas = 0;
  err = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&ctas, kernel, threads, smem);
  if (err != cudaSuccess) {
    return fail(SM120N_ERR_CUDA, "occupancy query failed: %s", cudaGetErrorString(err));
  }
  if (ctas < 1) ctas = 1;
  std::lock_guard<std::mutex> lock(g_cache_mutex);
  g_occupancy[key] = ctas;
  *out = ctas;
  return SM120N_OK;
}

int allow_dynamic_smem(const void* kernel, size_t bytes) {
  int device = 0;
  cudaError_t err = cudaGetDevice(&device);
  if (err != cudaSuccess) {
    return fail(SM120N_ERR_CUDA, "cudaGetDevice failed: %s", cudaGetErrorString(err));
  }
  std::lock_guard<std::mutex> lock(g_cache_mutex);
  size_t& granted = g_smem_optin[std::make_pair(device, kernel)];
  if (granted >= bytes) return SM120N_OK;
  err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             static_cast<int>(bytes));
  if (err != cudaSuccess) {
    return fail(SM120N_ERR_CUDA, "cannot grant %zu bytes of shared memory: %s", bytes,
                cudaGetErrorString(err));
  }
  granted = bytes;
  return SM120N_OK;
}

int max_block_smem(size_t* bytes) {
  int device = 0;
  cudaError_t err = cudaGetDevice(&device);
  if (err != cudaSuccess) {
    return fail(SM120N_ERR_CUDA, "cudaGetDevice failed: %s", cudaGetErrorString(err));
  }
  if (device < 0 || device >= kMaxDevices) {
    return fail(SM120N_ERR_UNSUPPORTED, "device ordinal %d is out of range", device);
  }
  std::lock_guard<std::mutex> lock(g_cache_mutex);
  if (g_block_smem[device] == 0) {
    int value = 0;
    err = cudaDeviceGetAttribute(&value, cudaDevAttrMaxSharedMemoryPerBlockOptin, device);
    if (err != cudaSuccess || value <= 0) {
      return fail(SM120N_ERR_CUDA, "cannot query shared memory per block: %s",
                  cudaGetErrorString(err));
    }
    g_block_smem[device] = static_cast<size_t>(value);
  }
  *bytes = g_block_smem[device];
  return SM120N_OK;
}

}  // namespace sm120n
