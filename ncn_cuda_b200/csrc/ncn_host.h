// What the host side of the library shares between its translation units: facts of a device, the error of a CUDA call.
#pragma once
#include <cuda_runtime.h>

namespace ncn {

struct DevInfo {
  int dev = -1, sms = 0, smem_optin = 0;
  int* status = nullptr;  // the device status word that a kernel with an abandoned wait writes
};

int get_dev(DevInfo& out);
int cuda_fail(cudaError_t e);  // records the text for ncn_last_cuda_error and clears the error; NCN_ERR_CUDA

}  // namespace ncn
