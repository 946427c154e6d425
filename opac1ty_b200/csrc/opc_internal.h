// opc_internal.h -- what the library's translation units share on the host: the error message of
// the calling thread, device properties and the device error word (all defined in opc_lib.cu).
#pragma once

#include <cudaTypedefs.h>
#include <cuda_runtime.h>

namespace opc_host {

// Record the thread's error message (opc_last_error) and return `code`.
__attribute__((visibility("hidden"), format(printf, 2, 3))) int fail(int code, const char* fmt, ...);
__attribute__((visibility("hidden"))) int cuda_fail(cudaError_t e, const char* what);

struct Device {
  int sm_count = 0;
  int max_smem_optin = 0;
  int* error_word = nullptr;  // device address of the word opc_take_device_error reads
};
// Properties of the current device (looked up once per device).
__attribute__((visibility("hidden"))) int current_device(Device* out);

// cuTensorMapEncodeTiled (NULL where the driver has none).
__attribute__((visibility("hidden"))) PFN_cuTensorMapEncodeTiled_v12000 tensor_map_encoder();

}  // namespace opc_host
