// pl_kv8.h -- what pl_attn.cu and pl_kv8.cu, the two translation units of
// libpl_attn.so, share.
#pragma once
#include <cstddef>
#include <cstdint>
#include <cuda_runtime.h>

namespace pl_module {

// Device allocation of the module (pl_attn.cu), with its failure injection.
cudaError_t alloc(void** p, size_t bytes);

// Bound on the device-side waits of the 8-bit cache's kernels on the current
// device (pl_kv8.cu), whose constants are apart from pl_attn.cu's.
cudaError_t kv8_wait_limit(uint64_t ns);

}  // namespace pl_module
