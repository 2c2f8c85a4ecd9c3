// tdc_host.h — what the host halves of libtdc_sm100.so share.
#pragma once

#include <cstdint>

namespace tdc {
namespace host {

// Records a failed CUDA call for tdc_last_cuda_error; returns TDC_ERR_CUDA.
int cuda_fail(int cuda_error);

// Checks that the current device is an sm_100 one and that no earlier launch
// on it reported a failed pipeline wait; TDC_OK or a TDC_ERR_* code.
int prepare_device();

// Limit and failure record of the bounded waits of launches on the current
// device (after prepare_device): the device's status words, and its slot of
// the mapped host page or null.
struct WaitRecord {
  uint64_t timeout_ns;
  int* words;
  int* host;
};
int wait_record(WaitRecord* r);

}  // namespace host
}  // namespace tdc
