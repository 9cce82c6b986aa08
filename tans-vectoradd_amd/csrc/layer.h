// What the layer kernels (rows.hip, linear.hip) share: vector types, buffer
// resources, bf16 and E4M3FN conversions, host-side checks.
#ifndef TANS_LAYER_H
#define TANS_LAYER_H

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <string>

#include "../../include/tans_amd.h"

extern "C" void tans_internal_set_error(const char* msg);  // codec.cpp

namespace {

constexpr int kLanes = 64;

typedef uint32_t v4u __attribute__((ext_vector_type(4)));
typedef uint32_t v2u __attribute__((ext_vector_type(2)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef float v2f __attribute__((ext_vector_type(2)));
typedef __bf16 v2bf __attribute__((ext_vector_type(2)));

typedef __amdgpu_buffer_rsrc_t Rsrc;

// Raw buffer of `bytes` bytes: loads past its end return zero.
__device__ __forceinline__ Rsrc rsrc(const void* base, uint32_t bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), (short)0, (int)bytes,
                                             0x00020000);
}

__device__ __forceinline__ float bf16_lo(uint32_t u) { return __builtin_bit_cast(float, u << 16); }
__device__ __forceinline__ float bf16_hi(uint32_t u) {
    return __builtin_bit_cast(float, u & 0xFFFF0000u);
}

// Two floats to bf16, round to nearest even, a in the low half (a NaN stays one).
__device__ __forceinline__ uint32_t bf16_pack(float a, float b) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(v2f{a, b}, v2bf));
}

// Host side ---------------------------------------------------------------

inline int fail(int code, const std::string& msg) {
    tans_internal_set_error(msg.c_str());
    return code;
}

inline int hip_check(hipError_t e, const char* what) {
    if (e == hipSuccess) return TANS_OK;
    return fail(TANS_EHIP, std::string(what) + ": " + hipGetErrorString(e));
}

inline bool aligned(const void* p, uintptr_t a) { return reinterpret_cast<uintptr_t>(p) % a == 0; }

}  // namespace

#endif  // TANS_LAYER_H
