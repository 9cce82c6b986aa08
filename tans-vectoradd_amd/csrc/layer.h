// What the layer kernels (rows.hip, linear.hip, positions.hip, attention.hip) share:
// vector types, buffer resources, bf16 and E4M3FN conversions, the rounding of a row
// to 8 bits, host-side checks.
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

// Rows to 8 bits: scale = max(max |y|, 2^-100) / 448, q = E4M3FN(y / scale).
constexpr float kFp8Max = 448.0f;
constexpr uint32_t kAmaxMinBits = (127 - 100) << 23;   // 2^-100
constexpr int kVec = 8;            // elements of a 16-byte load of bf16

struct Max {   // of non-negative floats' bits: a NaN is the largest
    static __device__ __forceinline__ float join(float a, float b) {
        const uint32_t x = __builtin_bit_cast(uint32_t, a), y = __builtin_bit_cast(uint32_t, b);
        return __builtin_bit_cast(float, x > y ? x : y);
    }
    static constexpr float kNone = 0.0f;
};

template <class Op, int CTRL>
__device__ __forceinline__ float dpp_join(float v) {
    return Op::join(v, __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(
                           0, __builtin_bit_cast(int, v), CTRL, 0xF, 0xF, false)));
}

__device__ __forceinline__ void unpack(const v4u& u, float (&f)[kVec]) {
    #pragma unroll
    for (int i = 0; i < 4; i++) {
        f[2 * i] = bf16_lo(u[i]);
        f[2 * i + 1] = bf16_hi(u[i]);
    }
}

__device__ __forceinline__ float amax8(const float (&y)[kVec], float top) {
    #pragma unroll
    for (int i = 0; i < kVec; i++)
        top = Max::join(top, __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, y[i]) & 0x7FFFFFFFu));
    return top;
}

// E4M3FN(y / sc), inv = 1 / sc: the quotient by the reciprocal and one
// correction, since bf16 rows often divide to the middle between two bytes
__device__ __forceinline__ v2u to_fp8(const float (&y)[kVec], float sc, float inv) {
    float t[kVec];
    #pragma unroll
    for (int i = 0; i < kVec; i++) {
        t[i] = y[i] * inv;
        t[i] = __builtin_fmaf(__builtin_fmaf(-t[i], sc, y[i]), inv, t[i]);
    }
    v2u r;
    #pragma unroll
    for (int j = 0; j < 2; j++) {
        int b = __builtin_amdgcn_cvt_pk_fp8_f32(t[4 * j], t[4 * j + 1], 0, false);
        r[j] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(t[4 * j + 2], t[4 * j + 3], b, true);
    }
    return r;
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
