// What the rest of the library sees of linear_api.cu beside the entry points in include/spmm_b200.h.
#pragma once

namespace spmm_b200 {

// The status word of the linear-layer kernels on the current device (spmm_b200_device_status reports it with its own):
// 1 after a bounded wait has given up, minus a cudaError_t if it cannot be read.
int linear_status(int reset);

}  // namespace spmm_b200
