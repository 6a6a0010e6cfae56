// Shared by the policy operators' translation units: element types, error reporting, launch checks.
#pragma once
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../../include/urgym_ops.h"

typedef __bf16 bf16;
typedef _Float16 f16;

// formats the message of this thread's last failed call; returns -1
__attribute__((visibility("hidden"))) int uo_fail(const char* fmt, ...);
// the error of the launches since the last check, as a return code
__attribute__((visibility("hidden"))) int uo_launched(const char* what);

#define UO_WAVE 64

__device__ __forceinline__ float uo_wave_sum(float x) {
#pragma unroll
    for (int m = 32; m; m >>= 1) x += __shfl_xor(x, m);
    return x;
}
