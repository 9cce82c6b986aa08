// Matrix product of FP8 rows with FP8 weights, its epilogue included
// (gfx950).  No counterpart in the reference.
//
//   v[m][n] = a_scale[m] * w_scale[n] * scale * sum_k a[m][k] w[n][k] + bias[n]
//   y[m][n] = act(v[m][n]) + residual[m][n]
//   gated: y[m][j] = act(v[m][j]) * v[m][F + j] + residual[m][j], F = R / 2
//
// a and w hold E4M3FN bytes; the products of v_mfma_f32_16x16x128_f8f6f4 are
// exact and summed in 32 bits; y is rounded once, to bf16.
#include "layer.h"

namespace {

typedef int v8i __attribute__((ext_vector_type(8)));

constexpr int64_t kMaxCols = int64_t(1) << 22;   // a tile's rows stay below 2^32 bytes

struct Epilogue {
    const float* a_scale;        // [M] or null (1)
    const float* w_scale;        // [R] or null (1)
    const uint16_t* bias;        // bf16 [R] or null
    const uint16_t* residual;    // bf16 [M, N] or null
    uint16_t* y;                 // bf16 [M, N]
    float scale;
    int act;
};

__device__ __forceinline__ float activate(float v, int act) {
    switch (act) {
        case TANS_ACT_RELU: return v < 0.0f ? 0.0f : v;   // a NaN stays one
        case TANS_ACT_SILU: return v / (1.0f + expf(-v));
        case TANS_ACT_GELU: return 0.5f * v * (1.0f + erff(v * 0.70710678f));
        case TANS_ACT_GELU_TANH:
            return 0.5f * v * (1.0f + tanhf(0.79788456f * (v + 0.044715f * v * v * v)));
        default: return v;
    }
}

// A wave computes 16 rows of a times 16 outputs; 4 waves of a workgroup take
// consecutive groups of 16 outputs.  Operands go from memory straight to
// registers: lane l holds row l % 16 of either and, of each 128 columns,
// columns 32 (l / 16) .. + 31.  Of the 16 x 16 products, lane l gets those of
// a's row l % 16 with weight rows 4 (l / 16) .. + 3.
template <bool GATED>
__global__ __launch_bounds__(256) void linear_kernel(const uint8_t* __restrict__ a,
                                                     const uint8_t* __restrict__ w, int64_t M,
                                                     int64_t N, int64_t C, Epilogue e) {
    const int lane = threadIdx.x & (kLanes - 1);
    const int r = lane & 15, g = lane >> 4;
    const int64_t blocks = (N + 63) / 64;   // of 64 outputs, for each 16 rows
    const int64_t m = blockIdx.x / blocks * 16 + r;
    const int64_t n0 = (blockIdx.x % blocks * 4 + threadIdx.x / kLanes) * 16;
    if (n0 >= N) return;
    const int64_t n = n0 + r < N ? n0 + r : N - 1;   // in bounds; not stored
    const uint8_t* pa = a + (m < M ? m : M - 1) * C;
    const uint8_t* pw = w + n * C;
    const uint8_t* pu = w + (N + n) * C;
    auto load = [&](const uint8_t* p, int64_t k) {
        v4u lo = {0, 0, 0, 0}, hi = {0, 0, 0, 0};
        if (k < C) lo = *reinterpret_cast<const v4u*>(p + k);          // C % 16 == 0
        if (k + 16 < C) hi = *reinterpret_cast<const v4u*>(p + k + 16);
        return v8i{(int)lo.x, (int)lo.y, (int)lo.z, (int)lo.w,
                   (int)hi.x, (int)hi.y, (int)hi.z, (int)hi.w};
    };
    v4f acc = {0, 0, 0, 0}, up = {0, 0, 0, 0};
    for (int64_t k = 32 * g; k < C + 32 * g; k += 128) {
        const v8i av = load(pa, k);
        acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(load(pw, k), av, acc, 0, 0, 0, 0, 0, 0);
        if (GATED)
            up = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(load(pu, k), av, up, 0, 0, 0, 0, 0, 0);
    }
    if (m >= M) return;
    const float sa = e.a_scale ? e.a_scale[m] : 1.0f;
    for (int i = 0; i < 4; i++) {
        const int64_t c = n0 + 4 * g + i;
        if (c >= N) break;
        auto scaled = [&](float v, int64_t col) {
            v = v * sa * ((e.w_scale ? e.w_scale[col] : 1.0f) * e.scale);
            return e.bias ? v + bf16_lo(e.bias[col]) : v;
        };
        float v = activate(scaled(acc[i], c), e.act);
        if (GATED) v *= scaled(up[i], N + c);
        if (e.residual) v += bf16_lo(e.residual[m * N + c]);
        e.y[m * N + c] = (uint16_t)bf16_pack(v, 0.0f);
    }
}

}  // namespace

extern "C" {

int tans_fp8_linear_workspace(int64_t M, int64_t R, int64_t C, int32_t gated, int64_t* bytes) {
    if (!bytes) return fail(TANS_EINVAL, "linear: null pointer");
    if (M < 0 || R < 1 || M > INT32_MAX || R > INT32_MAX || (gated && R % 2))
        return fail(TANS_EINVAL, "linear: need M >= 0 and R >= 1 below 2^31, R even if gated");
    if (C < 16 || C % 16 || C > kMaxCols)
        return fail(TANS_EINVAL, "linear: C must be a multiple of 16, 16 .. 2^22");
    *bytes = 0;
    return TANS_OK;
}

int tans_fp8_linear(const void* a, const float* a_scale, const void* w, const float* w_scale,
                    float scale, const void* bias, const void* residual, int32_t activation,
                    int32_t gated, int64_t M, int64_t R, int64_t C, void* workspace,
                    int64_t workspace_bytes, void* y, void* stream) {
    int64_t need = 0;
    const int rc = tans_fp8_linear_workspace(M, R, C, gated, &need);
    if (rc != TANS_OK) return rc;
    if (activation < 0 || activation > TANS_ACT_GELU_TANH)
        return fail(TANS_EINVAL, "linear: activation must be 0 .. 4");
    if (M == 0) return TANS_OK;
    if (!a || !w || !y) return fail(TANS_EINVAL, "linear: null pointer");
    if (!aligned(a, 16) || !aligned(w, 16) || !aligned(y, 16) || !aligned(residual, 16) ||
        !aligned(bias, 16) || !aligned(a_scale, 4) || !aligned(w_scale, 4))
        return fail(TANS_EINVAL, "linear: misaligned buffer (scales 4, others 16 bytes)");
    if (need > 0 && (!workspace || !aligned(workspace, 16) || workspace_bytes < need))
        return fail(TANS_EINVAL, "linear: workspace too small, null or misaligned (16 bytes)");
    const int64_t N = gated ? R / 2 : R;
    const int64_t blocks = (N + 63) / 64 * ((M + 15) / 16);
    if (blocks > UINT32_MAX / 256) return fail(TANS_EINVAL, "linear: too many outputs for one call");
    const dim3 grid((unsigned)blocks);
    const Epilogue e = {a_scale, w_scale, (const uint16_t*)bias, (const uint16_t*)residual,
                        (uint16_t*)y, scale, activation};
    auto launch = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, grid, dim3(256), 0, (hipStream_t)stream, (const uint8_t*)a,
                           (const uint8_t*)w, M, N, C, e);
    };
    if (gated) launch(linear_kernel<true>); else launch(linear_kernel<false>);
    return hip_check(hipGetLastError(), "linear_kernel launch");
}

}  // extern "C"
