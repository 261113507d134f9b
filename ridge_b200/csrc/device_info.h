// What the launchers outside gemm_host.cu need of the per-device state it keeps.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>
#include <cudaTypedefs.h>

#include <cstdint>

namespace ridge_b200 {

struct DeviceInfo {
    int device;
    int num_sms;
    int* err_word;  // device error word written by kernels whose bounded waits expire
};

// The current device; RIDGE_ENOTSUP when it is not sm_100, or a CUDA error.
int device_info(DeviceInfo* out);

// cuTensorMapEncodeTiled, or null where the driver has none.
PFN_cuTensorMapEncodeTiled_v12000 tensor_map_encode_fn();

}  // namespace ridge_b200
