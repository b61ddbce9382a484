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

// Lets a kernel use all the dynamic shared memory that a CTA of the device can have; `declared` are at least the
// bytes that it declares statically.  The limit belongs to the kernel and the device, not to a call: a limit of
// just this call's size could be lowered by another host thread's smaller call between here and the launch, which then
// fails.  So every call sets the same value.
template <typename K>
inline cudaError_t raise_dynamic_smem(K* kernel, const DeviceInfo& dev, int declared = 0) {
  return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, dev.max_smem_optin - declared);
}

}  // namespace pa_host
