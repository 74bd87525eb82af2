// host_common.h — what the library's translation units share on the host: the thread's error
// message and the per-device lookups (defined in mlxp_attn.cu).
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>
#include <cudaTypedefs.h>

#define MLXP_INTERNAL __attribute__((visibility("hidden")))

namespace mlxp {

// Positions a sequence's block table may reach, and query rows a call may have, in the cache
// kernels, whose indexes are 32-bit: room for a few tiles past the last one.
constexpr long long kMaxCacheIndex = 0x7fffffffLL - 1023;

// Records the message of mlxp_last_error and returns `code`.
MLXP_INTERNAL int fail(int code, const char* fmt, ...);
MLXP_INTERNAL int cuda_fail(cudaError_t e, const char* what);
MLXP_INTERNAL int current_device(int& dev);
// Device status word and SM count of the current device; either may be null.
MLXP_INTERNAL int device_info(int** status, int* sms);

// The driver's tensor-map encoder.
MLXP_INTERNAL int tensor_map_encoder(PFN_cuTensorMapEncodeTiled_v12000* fn);
// Limit of every bounded device-side wait (mlxp_set_wait_timeout_ns).
MLXP_INTERNAL unsigned long long wait_timeout_ns();

}  // namespace mlxp
