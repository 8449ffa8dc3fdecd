// Host helpers shared by the files that implement the C ABI (defined in capi.cu).
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>

namespace smb {

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                  const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

struct DeviceInfo {
  int sms = 0;
  bool sm100 = false;
};

// Keeps the error's text for smb_last_cuda_error and returns SMB_ERR_CUDA.
int cuda_fail(cudaError_t err);
// The driver's tensor-map encoder, looked up at run time (null without a driver).
EncodeTiledFn encode_fn();
// Facts of the current device, filled once per device.
int device_info(DeviceInfo* out);
// Whether launches use programmatic dependent launch.
bool pdl_enabled();

}  // namespace smb
