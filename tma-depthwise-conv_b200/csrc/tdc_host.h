// tdc_host.h — what the host halves of libtdc_sm100.so share.
#pragma once

namespace tdc {
namespace host {

// Records a failed CUDA call for tdc_last_cuda_error; returns TDC_ERR_CUDA.
int cuda_fail(int cuda_error);

// Checks that the current device is an sm_100 one and that no earlier launch
// on it reported a failed pipeline wait; TDC_OK or a TDC_ERR_* code.
int prepare_device();

}  // namespace host
}  // namespace tdc
