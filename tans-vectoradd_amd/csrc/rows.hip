// Row kernels of a layer (gfx950): the root-mean-square norm with the
// residual's addition and an 8-bit output, and the 8-bit rounding of rows.
// No counterpart in the reference.
//
//   h = x + residual                       (32 bits; also stored as bf16)
//   y = h * weight / sqrt(mean(h^2) + eps) (norm; y = x for the rounding)
//   scale = max(max |y|, 2^-100) / 448
//   q = E4M3FN(y / scale)                (the operand of the FP8 products)
//
// Sums, maximum and scale are 32-bit.  h is kept as bf16 because the next layer
// reads it as its residual; y only as 8 bits, with a scale for each row.
//
// h^2 is summed from the unrounded h.  Where mean(h^2) + eps is outside 2^-100 ..
// 2^128 (a 32-bit square has overflowed, or lost bits below 2^-126 that count),
// the sum is taken again of h times a power of two, so that the norm of any
// finite row is right.  The maximum is taken over the bits of |y| as unsigned
// numbers, in which a NaN is larger than infinity: a row that holds one, or an
// infinity, comes out with a scale that is not finite and NaN bytes.
#include <algorithm>

#include "layer.h"

namespace {

constexpr int kMaxWaves = 16;      // of a workgroup
constexpr int kMaxVecs = 7;        // of a row that a thread holds: 57344 elements a row

struct Sum {
    static __device__ __forceinline__ float join(float a, float b) { return a + b; }
    static constexpr float kNone = 0.0f;
};

// Over each row of 16 lanes; all of them get the result.
template <class Op>
__device__ __forceinline__ float join16(float v) {
    v = dpp_join<Op, 0xB1>(v);    // lane ^ 1
    v = dpp_join<Op, 0x4E>(v);    // lane ^ 2
    v = dpp_join<Op, 0x141>(v);   // mirrored in halves of the row
    return dpp_join<Op, 0x140>(v);   // mirrored in the row
}

template <class Op>
__device__ __forceinline__ float wave_join(float v) {
    v = join16<Op>(v);
    // the swap of a register with itself gives each lane its own row's value
    // and its neighbour row's, then the halves'; read through a 64-bit cast
    uint32_t u = __builtin_bit_cast(uint32_t, v);
    uint64_t p = __builtin_bit_cast(uint64_t, __builtin_amdgcn_permlane16_swap(u, u, false, false));
    v = Op::join(__builtin_bit_cast(float, (uint32_t)p), __builtin_bit_cast(float, (uint32_t)(p >> 32)));
    u = __builtin_bit_cast(uint32_t, v);
    p = __builtin_bit_cast(uint64_t, __builtin_amdgcn_permlane32_swap(u, u, false, false));
    return Op::join(__builtin_bit_cast(float, (uint32_t)p), __builtin_bit_cast(float, (uint32_t)(p >> 32)));
}

// Over the nw waves that share a row, in a fixed order.  One barrier; each
// call of a kernel has a `part` of its own.
template <class Op>
__device__ __forceinline__ float row_join(float v, float (&part)[kMaxWaves], int nw) {
    v = wave_join<Op>(v);
    if (nw == 1) return v;
    const int lane = threadIdx.x & (kLanes - 1);
    if (lane == 0) part[threadIdx.x / kLanes] = v;
    __syncthreads();
    return join16<Op>((lane & 15) < nw ? part[lane & 15] : Op::kNone);
}

// Whether mean(h^2) + eps can be trusted: sums of squares that overflow are
// infinite, and squares below 2^-126 lose at most 2^-126 each, 2^-26 of the
// least mean here.  Alike in all lanes that share a row, so one scalar branch.
__device__ __forceinline__ bool in_range(float mean) {
    constexpr uint32_t kLeast = (127 - 100) << 23, kInf = 255u << 23;
    const uint32_t u = (uint32_t)__builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, mean));
    return u - kLeast < kInf - kLeast;
}

// A power of two that brings a row's largest |h| to 1 .. 4, or by 2^100 at most:
// then a square is never lost beside the row's largest, nor does eps f^2 overflow
// where the mean was too small (eps < 2^-100).
__device__ __forceinline__ float rescale(float top) {
    const int e = (int)(__builtin_bit_cast(uint32_t, top) >> 23);   // 255 with NaN and infinity
    const int f = 254 - e < 1 ? 1 : 254 - e > 227 ? 227 : 254 - e;
    return __builtin_bit_cast(float, (uint32_t)f << 23);
}

template <bool NORM, bool RES>
struct Row {
    // vector i of the row: h, and the residual's sum as it is stored
    static __device__ __forceinline__ v4u load(const uint16_t* p, int64_t i) {
        return *reinterpret_cast<const v4u*>(p + i * kVec);
    }
    static __device__ __forceinline__ void sum(const v4u& x, const v4u& r, float (&h)[kVec]) {
        unpack(x, h);
        if constexpr (RES) {
            float f[kVec];
            unpack(r, f);
            #pragma unroll
            for (int k = 0; k < kVec; k++) h[k] += f[k];
        }
    }
    static __device__ __forceinline__ float squares(const float (&h)[kVec], float s) {
        #pragma unroll
        for (int k = 0; k < kVec; k++) s = __builtin_fmaf(h[k], h[k], s);
        return s;
    }
    static __device__ __forceinline__ void scale_by(float (&h)[kVec], float f) {
        #pragma unroll
        for (int k = 0; k < kVec; k++) h[k] *= f;
    }
    static __device__ __forceinline__ void normed(float (&h)[kVec], const v4u& w, float inv) {
        if constexpr (NORM) {
            float f[kVec];
            unpack(w, f);
            #pragma unroll
            for (int k = 0; k < kVec; k++) h[k] = h[k] * inv * f[k];
        }
    }
    static __device__ __forceinline__ void store(uint16_t* p, int64_t i, const float (&h)[kVec]) {
        *reinterpret_cast<v4u*>(p + i * kVec) = v4u{bf16_pack(h[0], h[1]), bf16_pack(h[2], h[3]),
                                                   bf16_pack(h[4], h[5]), bf16_pack(h[6], h[7])};
    }
};

// Bound by memory: each element is read once and written once.  8192 x 5120 with
// residual 46.8 us for 294 MB (6.3 TB/s; 52 a call among others), the rounding
// of 8192 x 17408 73.8 us for 428 MB (5.8).  The first kernel here took three passes
// over the row (131 and 246 us).  One row takes 2.9 us, a launch and two
// dependent latencies; the call's 8 .. 10 us are the host's.
//
// A row is read once and held in registers, NV vectors of 8 a thread (vector
// t + T j for thread t of the T that share the row).  Workgroups of nw > 1
// waves take one row; with nw == 1 each of a workgroup's waves takes a row of
// its own and nothing waits at a barrier.  All loads are issued before the
// first is used.
template <bool NORM, bool RES, int NV>
__global__ __launch_bounds__(kMaxWaves * kLanes) void rows_kernel(
    const uint16_t* x, const uint16_t* residual, const uint16_t* __restrict__ weight, int64_t M,
    int V, int nw, float eps, uint8_t* __restrict__ q, float* __restrict__ scale, uint16_t* h) {
    using P = Row<NORM, RES>;
    __shared__ float part_s[kMaxWaves], part_m[kMaxWaves], part_h[kMaxWaves], part_t[kMaxWaves];
    const bool solo = nw == 1;
    const int T = nw * kLanes;
    const int t = solo ? threadIdx.x & (kLanes - 1) : threadIdx.x;
    const int64_t row = solo ? (int64_t)blockIdx.x * (blockDim.x / kLanes) + threadIdx.x / kLanes
                             : blockIdx.x;
    if (row >= M) return;   // whole waves, and only where none waits for another
    const int64_t D = (int64_t)V * kVec;
    v4u xv[NV], rv[NV], wv[NV];
    #pragma unroll
    for (int j = 0; j < NV; j++) {
        const int i = t + j * T;
        xv[j] = rv[j] = wv[j] = v4u{0, 0, 0, 0};
        if (i < V) {
            xv[j] = P::load(x + row * D, i);
            if (RES) rv[j] = P::load(residual + row * D, i);
        }
    }
    if (NORM) {
        #pragma unroll
        for (int j = 0; j < NV; j++) {
            const int i = t + j * T;
            if (i < V) wv[j] = P::load(weight, i);
        }
    }
    float y[NV][kVec];
    float s = 0.0f;
    #pragma unroll
    for (int j = 0; j < NV; j++) {
        P::sum(xv[j], rv[j], y[j]);
        if (RES && t + j * T < V) P::store(h + row * D, t + j * T, y[j]);
        if (NORM) s = P::squares(y[j], s);
    }
    float inv = 1.0f;
    if (NORM) {
        float mean = row_join<Sum>(s, part_s, nw) / (float)D + eps;
        if (!in_range(mean)) {
            float most = 0.0f;
            #pragma unroll
            for (int j = 0; j < NV; j++) most = amax8(y[j], most);
            const float f = rescale(row_join<Max>(most, part_h, nw));
            s = 0.0f;
            #pragma unroll
            for (int j = 0; j < NV; j++) {
                P::scale_by(y[j], f);
                s = P::squares(y[j], s);
            }
            mean = row_join<Sum>(s, part_t, nw) / (float)D + eps * f * f;
        }
        inv = 1.0f / sqrtf(mean);
    }
    float top = __builtin_bit_cast(float, kAmaxMinBits);
    #pragma unroll
    for (int j = 0; j < NV; j++) {
        P::normed(y[j], wv[j], inv);
        // past the row's end h is zero, and an infinite inv would make it NaN
        if (t + j * T < V) top = amax8(y[j], top);
    }
    const float sc = row_join<Max>(top, part_m, nw) / kFp8Max;
    const float to_q = 1.0f / sc;
    #pragma unroll
    for (int j = 0; j < NV; j++) {
        const int i = t + j * T;
        if (i < V) *reinterpret_cast<v2u*>(q + row * D + (int64_t)i * kVec) = to_fp8(y[j], sc, to_q);
    }
    if (t == 0) scale[row] = sc;
}

// Rows longer than a workgroup holds in registers (57344 elements): three
// passes (five where the squares leave their range), the later ones reading what
// the first left in the caches.
template <bool NORM, bool RES>
__global__ __launch_bounds__(kMaxWaves * kLanes) void long_rows_kernel(
    const uint16_t* x, const uint16_t* residual, const uint16_t* __restrict__ weight, int V,
    float eps, uint8_t* __restrict__ q, float* __restrict__ scale, uint16_t* h) {
    using P = Row<NORM, RES>;
    __shared__ float part_s[kMaxWaves], part_m[kMaxWaves], part_h[kMaxWaves], part_t[kMaxWaves];
    constexpr int T = kMaxWaves * kLanes;
    const int64_t row = blockIdx.x;
    const int64_t D = (int64_t)V * kVec;
    auto sum_at = [&](int i, float (&f)[kVec]) {
        const v4u xv = P::load(x + row * D, i);
        P::sum(xv, RES ? P::load(residual + row * D, i) : xv, f);
    };
    float inv = 1.0f, by = 1.0f;   // of h's power of two
    float f[kVec];
    if (NORM) {
        float s = 0.0f;
        for (int i = threadIdx.x; i < V; i += T) {
            sum_at(i, f);
            s = P::squares(f, s);
        }
        float mean = row_join<Sum>(s, part_s, kMaxWaves) / (float)D + eps;
        if (!in_range(mean)) {
            float most = 0.0f;
            for (int i = threadIdx.x; i < V; i += T) {
                sum_at(i, f);
                most = amax8(f, most);
            }
            by = rescale(row_join<Max>(most, part_h, kMaxWaves));
            s = 0.0f;
            for (int i = threadIdx.x; i < V; i += T) {
                sum_at(i, f);
                P::scale_by(f, by);
                s = P::squares(f, s);
            }
            mean = row_join<Sum>(s, part_t, kMaxWaves) / (float)D + eps * by * by;
        }
        inv = 1.0f / sqrtf(mean);
    }
    auto y_at = [&](int i) {
        if (NORM) P::scale_by(f, by);
        P::normed(f, NORM ? P::load(weight, i) : v4u{0, 0, 0, 0}, inv);
    };
    float top = __builtin_bit_cast(float, kAmaxMinBits);
    for (int i = threadIdx.x; i < V; i += T) {
        sum_at(i, f);
        y_at(i);
        top = amax8(f, top);
    }
    const float sc = row_join<Max>(top, part_m, kMaxWaves) / kFp8Max;
    const float to_q = 1.0f / sc;
    for (int i = threadIdx.x; i < V; i += T) {
        sum_at(i, f);
        if (RES) P::store(h + row * D, i, f);   // h may be x or the residual
        y_at(i);
        *reinterpret_cast<v2u*>(q + row * D + (int64_t)i * kVec) = to_fp8(f, sc, to_q);
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

// Waves per row: up to 8 (512 threads) while 4 vectors a thread hold the row,
// else up to 16, so that longer rows keep their registers.  us per call with
// at most 8 / 16 waves, norm with residual: 8192 x 5120 52.4 / 55.8, 8192 x
// 17408 175.1 / 172.8 (7 bytes an element: 5.6 and 5.8 TB/s, where a 1 GiB copy
// reaches 5.2); rounding alone: 8192 x 5120 23.7 / 31.5, 8192 x 17408 77.9 /
// 73.5.  Up to some hundred rows a call takes the 4.0 .. 4.5 us of a launch at
// either.
template <bool NORM, bool RES>
int rows_launch(const uint16_t* x, const uint16_t* residual, const uint16_t* weight, int64_t M,
                int64_t D, float eps, uint8_t* q, float* scale, uint16_t* h, hipStream_t stream) {
    const int V = (int)(D / kVec);
    if (V > kMaxVecs * kMaxWaves * kLanes) {
        hipLaunchKernelGGL((long_rows_kernel<NORM, RES>), dim3((unsigned)M),
                           dim3(kMaxWaves * kLanes), 0, stream, x, residual, weight, V, eps, q,
                           scale, h);
        return hip_check(hipGetLastError(), "long_rows_kernel launch");
    }
    const int waves1 = (V + kLanes - 1) / kLanes;   // waves at one vector a thread
    const int most = waves1 <= 8 * 4 ? 8 : kMaxWaves;
    const int nv = std::min(kMaxVecs, (waves1 + most - 1) / most);
    const int nw = (waves1 + nv - 1) / nv;
    const int solo_rows = 4;                        // rows of one wave: 4 a workgroup
    const unsigned blocks = nw == 1 ? (unsigned)((M + solo_rows - 1) / solo_rows) : (unsigned)M;
    const unsigned threads = (nw == 1 ? solo_rows : nw) * kLanes;
    auto launch = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, dim3(blocks), dim3(threads), 0, stream, x, residual, weight, M, V,
                           nw, eps, q, scale, h);
    };
    switch (nv) {
        case 1: launch(rows_kernel<NORM, RES, 1>); break;
        case 2: launch(rows_kernel<NORM, RES, 2>); break;
        case 3: launch(rows_kernel<NORM, RES, 3>); break;
        case 4: launch(rows_kernel<NORM, RES, 4>); break;
        case 5: launch(rows_kernel<NORM, RES, 5>); break;
        case 6: launch(rows_kernel<NORM, RES, 6>); break;
        default: launch(rows_kernel<NORM, RES, 7>); break;
    }
    return hip_check(hipGetLastError(), "rows_kernel launch");
}

// All rows, in calls of at most kCallRows: a launch has fewer than 2^32 threads.
constexpr int64_t kCallRows = int64_t(1) << 21;   // of up to 1024 threads

template <bool NORM, bool RES>
int rows_all(const void* x, const void* residual, const void* weight, int64_t M, int64_t D,
             float eps, void* q, float* scale, void* h, void* stream) {
    for (int64_t m = 0; m < M; m += kCallRows) {
        const int rc = rows_launch<NORM, RES>(
            (const uint16_t*)x + m * D, RES ? (const uint16_t*)residual + m * D : nullptr,
            (const uint16_t*)weight, std::min(M - m, kCallRows), D, eps, (uint8_t*)q + m * D,
            scale + m, RES ? (uint16_t*)h + m * D : nullptr, (hipStream_t)stream);
        if (rc != TANS_OK) return rc;
    }
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
    return residual ? rows_all<true, true>(x, residual, weight, M, D, eps, q, scale, h, stream)
                    : rows_all<true, false>(x, nullptr, weight, M, D, eps, q, scale, nullptr, stream);
}

int tans_fp8_quantize_rows(const void* x, int64_t M, int64_t D, void* q, float* scale,
                           void* stream) {
    const int rc = rows_check("quantize_rows", x, M, D, q, scale);
    if (rc != TANS_OK || M == 0) return rc;
    return rows_all<false, false>(x, nullptr, nullptr, M, D, 0.0f, q, scale, nullptr, stream);
}

}  // extern "C"
