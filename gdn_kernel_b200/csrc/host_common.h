// What the library's translation units share on the host: one error message per
// thread, and one status word per device (gdn_b200.cu defines both).
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>

namespace gdn {

// Record `msg` as the calling thread's last error; returns `code`.
int lib_fail(int code, const char* msg) noexcept;
int lib_cuda_fail(cudaError_t e, const char* what) noexcept;
void lib_clear_error() noexcept;

// One-time setup of the current device: its status word and SM count.
int lib_device(unsigned int** status, int* sm_count) noexcept;

// Tensor map over packed bf16 tokens [tokens, heads, width], tokens `stride`
// elements apart, heads adjacent; the box is box_tokens x 1 head x 64 features
// (128 bytes, the 128-byte-swizzle span).  Loads past the tokens read zeros.
int lib_token_map(CUtensorMap* m, const void* base, int width, int heads, long long tokens,
                  long long stride, int box_tokens) noexcept;

}  // namespace gdn
