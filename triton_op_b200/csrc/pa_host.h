// What the library's translation units share on the host side.
#pragma once

#include <cuda_runtime.h>

namespace pa_host {

struct DeviceInfo {
  int sm_count = 0;
  int max_smem_optin = 0;
  bool ready = false;
};

// Remembers the error for pa_last_cuda_error() and returns PA_ERR_CUDA.
int cuda_fail(cudaError_t e);
// Attributes of the current device; a PaStatus.
int device_info(DeviceInfo** out);

}  // namespace pa_host
