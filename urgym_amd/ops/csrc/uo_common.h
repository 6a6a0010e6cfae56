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

template <int CTRL>
__device__ __forceinline__ float uo_dpp(float x) {
    return __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(x), CTRL, 0xf, 0xf, true));
}

// the sum over groups of G neighbouring lanes (2 .. 64), the same in all of them: each step adds the mirror image, so both sides
// add the same two numbers
template <int G>
__device__ __forceinline__ float uo_group_sum(float x) {
    if constexpr (G >= 2) x += uo_dpp<0xB1>(x);   // lane ^ 1
    if constexpr (G >= 4) x += uo_dpp<0x4E>(x);   // lane ^ 2
    if constexpr (G >= 8) x += uo_dpp<0x141>(x);  // the mirror in 8: the other quad
    if constexpr (G >= 16) x += uo_dpp<0x140>(x); // the mirror in 16
    if constexpr (G >= 32) x += __shfl_xor(x, 16);
    if constexpr (G >= 64) x += __shfl_xor(x, 32);
    return x;
}
