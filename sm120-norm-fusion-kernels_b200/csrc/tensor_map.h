// tensor_map.h -- the driver's encoder of TMA tensor maps.
#pragma once

#include <cuda.h>
#include <cudaTypedefs.h>

namespace sm120n {

// The encoder, or null with an error status in *rc.
PFN_cuTensorMapEncodeTiled_v12000 tensor_map_encoder(int* rc);

}  // namespace sm120n
