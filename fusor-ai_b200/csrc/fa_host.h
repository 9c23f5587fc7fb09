// What the C ABI's translation units share on the host: the calling thread's last error, the
// per-device state and the check of caller pointers (all defined in fa_attn.cu).
#pragma once

#include <cuda_runtime.h>

namespace fa {
namespace host {

// Records a failure message for fa_last_error and returns `code`.
int fail(int code, const char* fmt, ...) __attribute__((format(printf, 2, 3)));
int cuda_fail(cudaError_t e, const char* what);

// The SM count and the device error word of `device` (allocated at its first use).
int device_info(int device, int* sms, unsigned** err);

// Whether kernels on `device` may address `ptr` (null passes): see check_ptr in fa_attn.cu.
int pointer_on(const void* ptr, int device, const char* what);

}  // namespace host
}  // namespace fa
