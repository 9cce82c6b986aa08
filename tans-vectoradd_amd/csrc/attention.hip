// Attention of a batch's new tokens over a paged cache (gfx950).  No counterpart in
// the reference.
//
//   s_j = scale * q . k_j            for the slots j that the token sees
//   o = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m),  m = max_j s_j
//
// A token sees the slots before its sequence's new tokens and, of those, the ones that
// its row of the mask names (without a mask those up to itself).  One that sees nothing
// has o = 0.
#include <math.h>

#include "cache.h"
#include "launch.h"

namespace {

struct Caches { const void *k, *v; const float *k_scale, *v_scale; };

// One wave for each token and head, one slot after the other.
template <int D, bool FP8>
__global__ __launch_bounds__(256) void attend_kernel(const uint16_t* q, int64_t q_stride, Caches cache, Batch batch,
                                                     const uint8_t* mask, int W, int Hq, float scale,
                                                     uint16_t* out) {
    const int lane = threadIdx.x & (kLanes - 1);
    const int64_t id = (int64_t)blockIdx.x * 4 + threadIdx.x / kLanes;
    const int n = (int)(id / Hq), h = (int)(id % Hq);
    if (n >= batch.N) return;
    const int b = find_sequence(batch, n);
    if (b < 0 || n >= batch.start(b + 1)) return;
    const int t = n - batch.start(b), T = batch.tokens(b), c = batch.context(b);
    const int hk = h / (Hq / (int)batch.heads);
    constexpr int E = D / kLanes;
    float x[E], o[E] = {};
    for (int i = 0; i < E; i++) x[i] = bf16_lo(q[n * q_stride + h * D + lane * E + i]);
    float m = -INFINITY, l = 0.0f;
    const int64_t all = (int64_t)c + T < batch.capacity() ? (int64_t)c + T : batch.capacity();
    for (int s = 0; s < all; s++) {
        const int j = s - c;
        if (j >= 0 && !(mask ? j < W && mask[(int64_t)n * W + j] : j <= t)) continue;
        uint32_t row;
        if (!batch.row(b, s, hk, row)) continue;
        float d = 0.0f, val[E];
        for (int i = 0; i < E; i++) {
            const int64_t e = (int64_t)row * D + lane * E + i;
            float key;
            if constexpr (FP8) {
                key = __builtin_amdgcn_cvt_f32_fp8(((const uint8_t*)cache.k)[e], 0) * cache.k_scale[row];
                val[i] = __builtin_amdgcn_cvt_f32_fp8(((const uint8_t*)cache.v)[e], 0) * cache.v_scale[row];
            } else {
                key = bf16_lo(((const uint16_t*)cache.k)[e]);
                val[i] = bf16_lo(((const uint16_t*)cache.v)[e]);
            }
            d += x[i] * key;
        }
        for (int i = 1; i < kLanes; i *= 2) d += __shfl_xor(d, i);
        d *= scale;
        const float top = fmaxf(m, d), old = m == -INFINITY ? 0.0f : expf(m - top), p = expf(d - top);
        l = l * old + p;
        for (int i = 0; i < E; i++) o[i] = o[i] * old + p * val[i];
        m = top;
    }
    for (int i = 0; i < E; i++)
        out[((int64_t)n * Hq + h) * D + lane * E + i] = (uint16_t)bf16_pack(m == -INFINITY ? 0.0f : o[i] / l, 0.0f);
}

}  // namespace

extern "C" {

int tans_tree_attention_workspace(int64_t N, int64_t B, int64_t q_heads, int64_t heads, int64_t dim,
                                  int64_t slots, int64_t max_tokens, int64_t* bytes) {
    if (!bytes) return fail(TANS_EINVAL, "tree_attention: null pointer");
    *bytes = 0;
    return TANS_OK;
}

int tans_tree_attention(const void* q, int64_t q_stride, const void* k_cache, const void* v_cache,
                        const float* k_scale, const float* v_scale, int64_t pages, int64_t heads,
                        int64_t page, int64_t dim, const int32_t* table, int64_t per,
                        const int32_t* starts, const int32_t* lens, int64_t B, const void* mask,
                        int64_t mask_cols, int64_t N, int64_t q_heads, float scale, int64_t max_tokens,
                        void* workspace, int64_t workspace_bytes, void* out, void* stream) {
    const std::string op = "tree_attention";
    int rc = batch_check(op, k_cache, v_cache, k_scale, v_scale, pages, heads, page, dim, table, per,
                         starts, lens, B, N, q_heads);
    if (rc != TANS_OK) return rc;
    if (mask && (mask_cols < 0 || mask_cols > INT32_MAX))
        return fail(TANS_EINVAL, op + ": the mask must have 0 .. 2^31 - 1 columns");
    if (!(scale > 0.0f) || scale > 3.0e38f) return fail(TANS_EINVAL, op + ": scale must be positive and finite");
    if (N == 0 || B == 0) return TANS_OK;
    if (!q || !out) return fail(TANS_EINVAL, op + ": null pointer");
    rc = stride_check(op, "q", q, q_stride, q_heads * dim);
    if (rc == TANS_OK && !aligned(out, 16)) rc = fail(TANS_EINVAL, op + ": out is misaligned (16 bytes)");
    if (rc != TANS_OK) return rc;
    const Batch batch = {table, starts, lens, (int)B, (int)per, (int)N,
                         (uint32_t)pages, (uint32_t)heads, (uint32_t)page};
    auto launch = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, dim3((unsigned)((N * q_heads + 3) / 4)), dim3(256), 0, (hipStream_t)stream,
                           (const uint16_t*)q, q_stride, Caches{k_cache, v_cache, k_scale, v_scale}, batch,
                           (const uint8_t*)mask, (int)mask_cols, (int)q_heads, scale, (uint16_t*)out);
        return hip_check(hipGetLastError(), "attend_kernel launch");
    };
    if (dim == 64) return k_scale ? launch(attend_kernel<64, true>) : launch(attend_kernel<64, false>);
    if (dim == 128) return k_scale ? launch(attend_kernel<128, true>) : launch(attend_kernel<128, false>);
    return k_scale ? launch(attend_kernel<256, true>) : launch(attend_kernel<256, false>);
}

}  // extern "C"
