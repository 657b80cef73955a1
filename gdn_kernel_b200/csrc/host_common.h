// What the library's translation units share on the host: one error message per
// thread, and one status word per device (gdn_b200.cu defines both).
#pragma once

#include <cuda_runtime.h>

namespace gdn {

// Record `msg` as the calling thread's last error; returns `code`.
int lib_fail(int code, const char* msg) noexcept;
int lib_cuda_fail(cudaError_t e, const char* what) noexcept;
void lib_clear_error() noexcept;

// One-time setup of the current device: its status word and SM count.
int lib_device(unsigned int** status, int* sm_count) noexcept;

}  // namespace gdn
