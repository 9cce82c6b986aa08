// Row kernels of a layer (gfx950): the root-mean-square norm with the
// residual's addition and an 8-bit output, and the 8-bit rounding of rows.
// No counterpart in the reference.
//
//   h = x + residual                       (32 bits; also stored as bf16)
//   y = h * weight / sqrt(mean(h^2) + eps) (norm; y = x for the rounding)
//   scale = max(max |y|, 2^-100) / 448
//   q = E4M3FN(y / scale)
//
// h^2 is summed from the unrounded h.  The maximum is taken over the bits of
// |y| as unsigned numbers, in which a NaN is larger than infinity: a row that
// holds one, or an infinity, comes out with a NaN or infinite scale and NaN
// bytes.
#include "layer.h"

namespace {

constexpr float kFp8Max = 448.0f;
constexpr uint32_t kAmaxMinBits = (127 - 100) << 23;   // 2^-100
constexpr int kRowBlock = 256;

template <bool MAX>
__device__ __forceinline__ uint32_t block_reduce(uint32_t v, uint32_t* part) {
    auto join = [](uint32_t a, uint32_t b) -> uint32_t {
        if constexpr (MAX) return a > b ? a : b;
        else return __builtin_bit_cast(uint32_t, __builtin_bit_cast(float, a) +
                                                     __builtin_bit_cast(float, b));
    };
    #pragma unroll
    for (int m = 32; m >= 1; m >>= 1) v = join(v, __shfl_xor(v, m, kLanes));
    if ((threadIdx.x & (kLanes - 1)) == 0) part[threadIdx.x / kLanes] = v;
    __syncthreads();
    v = part[0];
    for (int w = 1; w < kRowBlock / kLanes; w++) v = join(v, part[w]);
    __syncthreads();
    return v;
}

// One workgroup a row.
template <bool NORM, bool RES>
__global__ __launch_bounds__(kRowBlock) void rows_kernel(
    const uint16_t* x, const uint16_t* residual,
    const uint16_t* __restrict__ weight, int64_t D, float eps, uint8_t* __restrict__ q,
    float* __restrict__ scale, uint16_t* h) {
    __shared__ uint32_t part[kRowBlock / kLanes];
    const int64_t row = blockIdx.x;
    auto sum_at = [&](int64_t i) {
        float v = bf16_lo(x[row * D + i]);
        if (RES) v += bf16_lo(residual[row * D + i]);
        return v;
    };
    float inv = 1.0f;
    if (NORM) {
        float s = 0.0f;
        for (int64_t i = threadIdx.x; i < D; i += kRowBlock) {
            const float v = sum_at(i);
            s += v * v;
        }
        s = __builtin_bit_cast(float, block_reduce<false>(__builtin_bit_cast(uint32_t, s), part));
        inv = 1.0f / sqrtf(s / (float)D + eps);
    }
    auto y_at = [&](int64_t i) { return NORM ? sum_at(i) * inv * bf16_lo(weight[i]) : sum_at(i); };
    uint32_t top = kAmaxMinBits;
    for (int64_t i = threadIdx.x; i < D; i += kRowBlock) {
        const uint32_t u = __builtin_bit_cast(uint32_t, y_at(i)) & 0x7FFFFFFFu;
        top = u > top ? u : top;
    }
    const float sc = __builtin_bit_cast(float, block_reduce<true>(top, part)) / kFp8Max;
    const float to_q = 1.0f / sc;
    for (int64_t i = threadIdx.x; i < D; i += kRowBlock) {
        q[row * D + i] = (uint8_t)__builtin_amdgcn_cvt_pk_fp8_f32(y_at(i) * to_q, 0.0f, 0, false);
        if (RES) h[row * D + i] = (uint16_t)bf16_pack(sum_at(i), 0.0f);   // h may be the residual
    }
    if (threadIdx.x == 0) scale[row] = sc;
}

int rows_check(const char* what, const void* x, int64_t M, int64_t D, const void* q,
               const void* scale) {
    const std::string op(what);
    if (M < 0 || M > INT32_MAX) return fail(TANS_EINVAL, op + ": M must be 0 .. 2^31 - 1");
    if (D < 16 || D % 16 || D > (int64_t(1) << 24))
        return fail(TANS_EINVAL, op + ": D must be a multiple of 16, 16 .. 2^24");
    if (M == 0) return TANS_OK;
    if (!x || !q || !scale) return fail(TANS_EINVAL, op + ": null pointer");
    if (!aligned(x, 16) || !aligned(q, 16) || !aligned(scale, 4))
        return fail(TANS_EINVAL, op + ": misaligned buffer (rows 16, scale 4 bytes)");
    return TANS_OK;
}

}  // namespace

extern "C" {

int tans_fp8_rmsnorm(const void* x, const void* residual, const void* weight, int64_t M, int64_t D,
                     float eps, void* q, float* scale, void* h, void* stream) {
    const int rc = rows_check("rmsnorm", x, M, D, q, scale);
    if (rc != TANS_OK || M == 0) return rc;
    if (!weight || (residual && !h)) return fail(TANS_EINVAL, "rmsnorm: null pointer");
    if (!aligned(weight, 16) || !aligned(residual, 16) || !aligned(h, 16))
        return fail(TANS_EINVAL, "rmsnorm: misaligned buffer (rows and weight 16 bytes)");
    if (!(eps >= 0.0f)) return fail(TANS_EINVAL, "rmsnorm: eps must not be negative");
    auto launch = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, dim3((unsigned)M), dim3(kRowBlock), 0, (hipStream_t)stream,
                           (const uint16_t*)x, (const uint16_t*)residual, (const uint16_t*)weight,
                           D, eps, (uint8_t*)q, scale, (uint16_t*)h);
    };
    if (residual) launch(rows_kernel<true, true>); else launch(rows_kernel<true, false>);
    return hip_check(hipGetLastError(), "rows_kernel launch");
}

int tans_fp8_quantize_rows(const void* x, int64_t M, int64_t D, void* q, float* scale,
                           void* stream) {
    const int rc = rows_check("quantize_rows", x, M, D, q, scale);
    if (rc != TANS_OK || M == 0) return rc;
    hipLaunchKernelGGL((rows_kernel<false, false>), dim3((unsigned)M), dim3(kRowBlock), 0,
                       (hipStream_t)stream, (const uint16_t*)x, (const uint16_t*)nullptr,
                       (const uint16_t*)nullptr, D, 0.0f, (uint8_t*)q, scale, (uint16_t*)nullptr);
    return hip_check(hipGetLastError(), "rows_kernel launch");
}

}  // extern "C"
