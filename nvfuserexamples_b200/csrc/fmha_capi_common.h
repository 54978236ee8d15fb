// fmha_capi_common.h — what the files of extern "C" entry points share (defined in fmha_capi.cu).  Internal to the library.
#pragma once
#include <cuda.h>
#include <cudaTypedefs.h>
#include <cuda_runtime.h>

namespace fmha {

int cuda_fail(cudaError_t e);   // keeps the error for fmha_sm100_last_cuda_error and returns FMHA_ERR_LAUNCH
int check_device();             // binds the current device's context to the thread; FMHA_ERR_NO_DEVICE unless it is an sm_100
PFN_cuTensorMapEncodeTiled_v12000 get_encode_fn();   // cuTensorMapEncodeTiled, null if the driver has none

}  // namespace fmha
