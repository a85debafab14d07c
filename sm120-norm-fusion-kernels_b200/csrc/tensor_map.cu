// tensor_map.cu -- see csrc/tensor_map.h; linked into both libraries.
#include "tensor_map.h"

#include <mutex>

#include "runtime.h"

namespace sm120n {

PFN_cuTensorMapEncodeTiled_v12000 tensor_map_encoder(int* rc) {
  static std::once_flag once;
  static PFN_cuTensorMapEncodeTiled_v12000 encode = nullptr;
  static cudaError_t status = cudaSuccess;
  std::call_once(once, [] {
    cudaDriverEntryPointQueryResult query;
    status = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", reinterpret_cast<void**>(&encode),
                                     cudaEnableDefault, &query);
    if (status == cudaSuccess && query != cudaDriverEntryPointSuccess) status = cudaErrorNotSupported;
  });
  *rc = status == cudaSuccess && encode != nullptr
            ? SM120N_OK
            : fail(SM120N_ERR_CUDA, "cuTensorMapEncodeTiled is not available: %s",
                   cudaGetErrorString(status));
  return encode;
}

}  // namespace sm120n
