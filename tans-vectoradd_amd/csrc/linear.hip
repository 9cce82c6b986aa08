// Matrix product of FP8 rows with FP8 weights, its epilogue included
// (gfx950).  No counterpart in the reference.
//
//   v[m][n] = a_scale[m] * w_scale[n] * scale * sum_k a[m][k] w[n][k] + bias[n]
//   y[m][n] = act(v[m][n]) + residual[m][n]
//   gated: y[m][j] = act(v[m][j]) * v[m][F + j] + residual[m][j], F = R / 2
//
// a and w hold E4M3FN bytes, whose products are exact.  The FP8 matrix
// instructions (v_mfma_f32_16x16x128_f8f6f4 and 32x32x64) add them in groups of 8
// columns, each product cut off at 2^-13 of its group's largest, and the groups
// in 32 bits (measured with sums that cancel, alike for every FP8 form).  The
// bf16 instruction, to which the bytes convert exactly, cuts off at 2^-24:
// over 4096 random columns the relative 2-norm of its error is 9e-8, as that of a
// sum in 32 bits, and the FP8 form's 1.3e-5.  The FP8 form is the choice here:
// its rate is 2.5 to 3 times the other's (4.4 against 1.4 .. 1.7 PFLOP/s in a loop
// of nothing else), with half of the operands' bytes and no conversions, and y's
// rounding to bf16, 2^-9, is a hundred times as large.  A single output whose
// products nearly cancel can be off by several percent of itself.
//
// Everything after the sum is 32-bit; y is rounded once, to bf16, the type in
// which a model keeps what lies between its layers.
//
// Three kernels, by what bounds them: few rows of a stream w past them (the
// memory's rate), some rows share tiles of w (the rate at which tiles reach
// LDS), many rows are a matrix product (the matrix cores at the board's power
// limit).  linear_plan.h chooses.
#include <math.h>

#include <algorithm>
#include <type_traits>

#include "launch.h"
#include "layer.h"
#include "linear_plan.h"

namespace {

using namespace tans_linear;

typedef int v8i __attribute__((ext_vector_type(8)));

template <int V>
constexpr std::integral_constant<int, V> kInt{};

// of w: the rows of y that the lanes of a store or residual load take beside each
// other, up to 15 of kMaxRows or, gated, 31 of half as many elements, stay within
// 32 bits (store_staged)
constexpr int64_t kMaxRows = int64_t(1) << 27;
constexpr int64_t kMaxCols = int64_t(1) << 22;   // a tile's rows stay below 2^32 bytes

// An offset past every tile's bytes (256 rows of kMaxCols: 2^30), also with a
// row's offset added
constexpr uint32_t kOut = 0x80000000u;

constexpr float kLog2e = 1.44269504f;

struct Epilogue {
    const float* a_scale;        // [M] or null (1)
    const float* w_scale;        // [R] or null (1)
    const uint16_t* bias;        // bf16 [R] or null
    const uint16_t* residual;    // bf16 [M, N] or null
    uint16_t* y;                 // bf16 [M, N]
    float scale;
    float lo;                    // kClip: the least value
};

// The activations in four forms, each a kernel of its own:
//   kClip  max(v, lo): none (lo = -infinity) and ReLU (a NaN stays one)
//   kSilu  v sigmoid(v)
//   kTanh  GELU's tanh form: (1 + tanh(u)) / 2 = sigmoid(2 u)
//   kErf   v Phi(v), erfc by Abramowitz and Stegun 7.1.26 (absolute error
//          below 1.5e-7)
enum Act { kClip, kSilu, kTanh, kErf };

template <int ACT>
__device__ __forceinline__ float activate(float v, const Epilogue& e) {
    if constexpr (ACT == kClip) {
        return __builtin_elementwise_maximum(v, e.lo);
    } else if constexpr (ACT == kSilu) {
        return v * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-kLog2e * v));
    } else if constexpr (ACT == kTanh) {
        constexpr float c1 = 2.0f * 0.79788456f * kLog2e;   // 2 sqrt(2 / pi), to base 2
        const float x = v * __builtin_fmaf(0.044715f * c1, v * v, c1);
        return v * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-x));
    } else {
        const float x = __builtin_fabsf(v) * 0.70710678f;
        const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.3275911f, x, 1.0f));
        float p = __builtin_fmaf(1.061405429f, t, -1.453152027f);
        p = __builtin_fmaf(p, t, 1.421413741f);
        p = __builtin_fmaf(p, t, -0.284496736f);
        p = __builtin_fmaf(p, t, 0.254829592f) * t;
        const float half_erfc = 0.5f * p * __builtin_amdgcn_exp2f(-1.44269504f * x * x);
        return v * (v < 0.0f ? half_erfc : 1.0f - half_erfc);
    }
}

constexpr int kNT = 2;   // cache policy: non-temporal

// 16 bytes a lane from memory to LDS, lane l's to lds + 16 l; zeros from
// offsets out of range.
template <int POLICY>
__device__ __forceinline__ void load_lds(const Rsrc& src, uint8_t* lds, uint32_t offset) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(src, (__attribute__((address_space(3))) void*)lds, 16,
                                             (int)offset, 0, 0, POLICY);
}

// Waits until at most N of the wave's loads (those issued last) are under way.
template <int N>
__device__ __forceinline__ void wait_loads() {
    static_assert(N < 64, "a 6-bit counter");
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt((N & 15) | (N >> 4) << 14 | 0xF70);
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
}

// Between a wave's writes to LDS and its reads of what other lanes wrote, and
// back: the hardware keeps a wave's LDS accesses in order, the compiler only
// those of one lane.
__device__ __forceinline__ void wave_sync() {
    __builtin_amdgcn_sched_barrier(0);   // (registers for one chunk at a time)
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    __builtin_amdgcn_sched_barrier(0);
}

__device__ __forceinline__ v8i join(const v4u& lo, const v4u& hi) {
    return v8i{(int)lo.x, (int)lo.y, (int)lo.z, (int)lo.w,
               (int)hi.x, (int)hi.y, (int)hi.z, (int)hi.w};
}

// Scale and bias of w's rows first + c .. first + c + CN - 1, of which those
// with c + i < N exist (the others are repeats of the last).
template <int CN, bool WHOLE = false>
__device__ __forceinline__ void columns(const Epilogue& e, int64_t first, int64_t c, int64_t N,
                                        float (&ws)[CN], float (&bs)[CN]) {
    #pragma unroll
    for (int i = 0; i < CN; i++) {
        ws[i] = 1.0f;
        bs[i] = 0.0f;
    }
    uint16_t b[CN];
    if (WHOLE || c + CN <= N) {
        if (e.w_scale) __builtin_memcpy(ws, e.w_scale + first + c, sizeof(ws));
        if (e.bias) __builtin_memcpy(b, e.bias + first + c, sizeof(b));
    } else {
        #pragma unroll
        for (int i = 0; i < CN; i++) {
            const int64_t n = first + (c + i < N ? c + i : N - 1);
            if (e.w_scale) ws[i] = e.w_scale[n];
            if (e.bias) b[i] = e.bias[n];
        }
    }
    #pragma unroll
    for (int i = 0; i < CN; i++) {
        ws[i] *= e.scale;
        if (e.bias) bs[i] = bf16_lo(b[i]);
    }
}

// ---------------------------------------------------------------------
// Few rows of a: w streamed from memory to registers.
// ---------------------------------------------------------------------

// Bound by w's bytes, read once: 34816 x 5120 (178 MB) by one row 28.7 .. 30.3 us,
// 5.9 .. 6.2 TB/s, by 8 rows 31; 5120 x 17408 (89 MB) by one row 17.1, by 7 18
// (4.9 .. 5.2 TB/s, of which some 3 us are the first loads' latency and the
// join).  w loaded to registers instead of LDS, as the operands need it, takes
// 16 bytes of 16 rows an instruction, and half of a cache line each: 42 us for
// one row by 34816 x 5120.  With LDS, 2 waves and a pipeline of 4 steps, or 4
// waves and 2, are within 3%; one wave a workgroup takes 47 us by 5120 x 17408.
//
// Products of up to 8 MA rows of a.  A workgroup takes 16 NF rows of w (gated:
// NF / 2 groups of 16 gate rows and the value rows that belong to them); its KW
// waves share the columns, wave k steps k, k + KW, ... of 128.  Each wave streams
// its steps through LDS of its own, PIPE steps deep, and waits for its own loads
// only.  A load brings 8 rows of 128 bytes, whole cache lines; lane l the 16
// bytes that belong at position l % 8 of row l / 8, a row's pieces permuted by an
// exclusive or with a key of the row so that 16 rows' reads of a piece touch all
// banks.  Lane (g, r) then reads, of row r of a group of 16, the pieces g and
// 4 + g, the same for a and w, and gets of the 16 x 16 products of an
// instruction those of a's row r with w's rows 4 g .. 4 g + 3.  The waves' sums
// are added in wave order through LDS.
template <bool GATED, int ACT, int MA, int NF, int KW, int PIPE>
__global__ __launch_bounds__(KW * kLanes) void linear_stream_kernel(
    const uint8_t* __restrict__ a, const uint8_t* __restrict__ w, int64_t M, int64_t N, int64_t C,
    Epilogue e) {
    constexpr int NO = GATED ? NF / 2 : NF;   // groups of 16 outputs
    constexpr int MF = (MA + 1) / 2;          // groups of 16 rows of a
    constexpr int kWave = (MF + NF) * 16 * kStep;   // bytes of a wave's step
    // (arrays of their own, so that a read waits for its own step's loads only)
    __shared__ __attribute__((aligned(1024))) uint8_t ring0[KW * kWave], ring1[KW * kWave],
        ring2[PIPE > 2 ? KW * kWave : 1], ring3[PIPE > 3 ? KW * kWave : 1];
    __shared__ float part[KW][MF * NF * 4][kLanes];
    const int lane = threadIdx.x & (kLanes - 1);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kLanes);
    const int r = lane & 15, g = lane >> 4;
    const int64_t n0 = (int64_t)blockIdx.x * (16 * NO);
    const uint32_t row_bytes = (uint32_t)C;
    const uint32_t rows = (uint32_t)(N - n0 < 16 * NO ? N - n0 : 16 * NO);
    const Rsrc asrc = rsrc(a, (uint32_t)M * row_bytes);
    const Rsrc wsrc = rsrc(w + n0 * C, rows * row_bytes);
    const Rsrc usrc = rsrc(w + (GATED ? N + n0 : n0) * C, rows * row_bytes);
    // rows 8 j + lane / 8 of a group: key (row / 2) % 8, another one for odd j
    const int lrow = lane >> 3, lpos = lane & 7;
    const uint32_t lcol[2] = {(uint32_t)(lpos ^ (lrow >> 1)) * 16, (uint32_t)(lpos ^ (lrow >> 1) ^ 4) * 16};
    const uint32_t lbase = (uint32_t)lrow * row_bytes;
    auto load = [&](int step, uint8_t* ring) {
        uint8_t* to = ring + wave * kWave;
        uint32_t o[2];
        #pragma unroll
        for (int h = 0; h < 2; h++) {
            const uint32_t c = (uint32_t)step * kStep + lcol[h];
            o[h] = c < row_bytes ? lbase + c : kOut;
        }
        #pragma unroll
        for (int j = 0; j < 2 * NF; j++)
            load_lds<kNT>(GATED && j >= 2 * NO ? usrc : wsrc, to + j * 1024,
                          o[j & 1] + (uint32_t)(GATED ? j % (2 * NO) : j) * 8 * row_bytes);
        #pragma unroll
        for (int j = 0; j < MA; j++)
            load_lds<0>(asrc, to + NF * 2048 + j * 1024, o[j & 1] + (uint32_t)j * 8 * row_bytes);
    };
    const uint32_t fbase = (uint32_t)wave * kWave + r * kStep + (uint32_t)(g ^ (r >> 1)) * 16;
    auto frag = [&](const uint8_t* ring, int i) {   // group i of the step
        return join(*reinterpret_cast<const v4u*>(ring + i * 2048 + fbase),
                    *reinterpret_cast<const v4u*>(ring + i * 2048 + (fbase ^ 64)));
    };
    v4f acc[MF][NF];
    #pragma unroll
    for (int i = 0; i < MF; i++)
        #pragma unroll
        for (int j = 0; j < NF; j++) acc[i][j] = v4f{0, 0, 0, 0};
    auto multiply = [&](int next, uint8_t* ring) {
        wait_loads<(PIPE - 1) * (2 * NF + MA)>();   // all but the later steps' have come
        v8i fa[MF], fw[NF];
        #pragma unroll
        for (int i = 0; i < NF; i++) fw[i] = frag(ring, i);
        #pragma unroll
        for (int i = 0; i < MF; i++) fa[i] = frag(ring, NF + i);
        #pragma unroll
        for (int j = 0; j < NF; j++)
            #pragma unroll
            for (int i = 0; i < MF; i++)
                acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(fw[j], fa[i], acc[i][j],
                                                                             0, 0, 0, 0, 0, 0);
        // (the products have waited for the reads: their slot is free)
        __builtin_amdgcn_sched_barrier(0);
        asm volatile("" ::: "memory");
        load(next, ring);
        __builtin_amdgcn_sched_barrier(0);
    };
    // (steps past the last load zeros)
    const int steps = (int)((C + kStep - 1) / kStep);
    load(wave, ring0);
    load(wave + KW, ring1);
    if (PIPE > 2) load(wave + 2 * KW, ring2);
    if (PIPE > 3) load(wave + 3 * KW, ring3);
    for (int s = wave; s < steps; s += PIPE * KW) {
        multiply(s + PIPE * KW, ring0);
        multiply(s + (PIPE + 1) * KW, ring1);
        if (PIPE > 2) multiply(s + (PIPE + 2) * KW, ring2);
        if (PIPE > 3) multiply(s + (PIPE + 3) * KW, ring3);
    }
    #pragma unroll
    for (int i = 0; i < MF; i++)
        #pragma unroll
        for (int j = 0; j < NF; j++)
            #pragma unroll
            for (int c = 0; c < 4; c++) part[wave][(i * NF + j) * 4 + c][lane] = acc[i][j][c];
    wait_loads<0>();   // (loads past the last step still write into the ring)
    __syncthreads();
    // one output a thread, consecutive ones along a row of y
    const int n_rows = (int)M;
    for (int t = threadIdx.x; t < n_rows * 16 * NO; t += KW * kLanes) {
        const int m = t / (16 * NO), n = t % (16 * NO);
        if (n >= (int)rows) continue;
        auto sum = [&](int j) {   // of group j: w's row n % 16 of it
            float v = 0.0f;
            #pragma unroll
            for (int k = 0; k < KW; k++)
                v += part[k][(m / 16 * NF + j) * 4 + n % 4][n % 16 / 4 * 16 + m % 16];
            return v;
        };
        const float sm = e.a_scale ? e.a_scale[m] : 1.0f;
        auto scaled = [&](float v, int64_t col) {
            v = v * sm * ((e.w_scale ? e.w_scale[col] : 1.0f) * e.scale);
            return e.bias ? v + bf16_lo(e.bias[col]) : v;
        };
        float v = activate<ACT>(scaled(sum(n / 16), n0 + n), e);
        if (GATED) v *= scaled(sum(NO + n / 16), N + n0 + n);
        const int64_t o = (int64_t)m * N + n0 + n;
        if (e.residual) v += bf16_lo(e.residual[o]);
        e.y[o] = (uint16_t)bf16_pack(v, 0.0f);
    }
}

// ---------------------------------------------------------------------
// Some rows of a: tiles of 32 MI rows of a by 32 NW rows of w.
// ---------------------------------------------------------------------
typedef float v16f __attribute__((ext_vector_type(16)));

__device__ __forceinline__ v16f mfma(const v8i& w, const v8i& a, const v16f& c) {
    return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(w, a, c, 0, 0, 0, 0, 0, 0);
}

// x, of which the compiler knows nothing any more
__device__ __forceinline__ uint32_t opaque_s(uint32_t x) {
    asm volatile("" : "+s"(x));
    return x;
}
__device__ __forceinline__ uint32_t opaque_v(uint32_t x) {
    asm volatile("" : "+v"(x));
    return x;
}

// A barrier for which all but each wave's last N loads into LDS have arrived,
// and its LDS reads (the compiler's own waits cover a wave's own loads only;
// __syncthreads would wait for all of them).
template <int N>
__device__ __forceinline__ void arrive() {
    static_assert(N < 64, "a 6-bit counter");
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt((N & 15) | (N >> 4) << 14 | 0x070);   // vmcnt(N), lgkmcnt(0)
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
}

// Outputs go through LDS, some rows of W sums of a wave's own (gated: W / 2
// gates, then their values): a lane's sums lie in a row each, 32 rows to an
// instruction, and stored from there outputs would be 16-byte writes all over y.
// 16-byte pieces of a row are permuted by an exclusive or with a key of the row,
// so that 16 rows' writes of a piece, and a row's reads, touch all banks.
template <int W>
__device__ __forceinline__ int staged(int row, int piece) {   // in floats
    const int key = W >= 64 ? row & 15 : (row >> 1) & 7;
    return row * W + (piece ^ key) * 4;
}

__device__ __forceinline__ v4f quad(const v16f& v, int b, float by) {
    return v4f{v[4 * b] * by, v[4 * b + 1] * by, v[4 * b + 2] * by, v[4 * b + 3] * by};
}

// What W columns (gated W / 2) from c0 on and ROWS rows from m0 on need besides
// the sums, loaded before any of them is stored: loads and stores count as one
// sequence, and a load between stores would wait for them.  A lane takes eight
// columns of every 512 / W-th row (gated 1024 / W).  WHOLE: all of them exist,
// and nothing is masked (a masked load or store ends a run of code in which the
// compiler can leave loads under way).
template <bool GATED, int W>
struct Columns {
    float ws[8], bs[8], wu[8], bu[8];
    template <bool WHOLE>
    __device__ __forceinline__ void load(const Epilogue& e, int lane, int64_t c0, int64_t N) {
        const int64_t c = c0 + lane % ((GATED ? W / 2 : W) / 8) * 8;
        if (!WHOLE && c >= N) return;   // (nothing of it is stored)
        columns<8, WHOLE>(e, 0, c, N, ws, bs);
        if (GATED) columns<8, WHOLE>(e, N, c, N, wu, bu);
    }
};

template <int CW, int ROWS>
struct Residual {
    static constexpr int per_row = CW / 8, Q = ROWS * per_row / kLanes;
    v4u u[Q];
    template <bool WHOLE>
    __device__ __forceinline__ void load(const Epilogue& e, int lane, int64_t m0, int64_t M, int64_t c0,
                                         int64_t N) {
        const int64_t c = c0 + lane % per_row * 8;
        const uint32_t mine = (uint32_t)(lane / per_row) * (uint32_t)N + lane % per_row * 8;
        #pragma unroll
        for (int q = 0; q < Q; q++) {
            // (a uniform part and 32 bits a lane)
            const uint16_t* p = e.residual + (m0 + q * (kLanes / per_row)) * N + c0 + mine;
            const int64_t m = m0 + q * (kLanes / per_row) + lane / per_row;
            if (WHOLE || (m < M && c + 8 <= N)) {
                __builtin_memcpy(&u[q], p, 16);   // (rows of y need not be aligned)
            } else {
                u[q] = v4u{0, 0, 0, 0};
                #pragma unroll
                for (int i = 0; i < 8; i++)
                    if (m < M && c + i < N) u[q][i / 2] |= (uint32_t)p[i] << (i % 2 * 16);
            }
        }
    }
};

template <bool GATED, int ACT, int W, int ROWS, bool WHOLE>
__device__ __forceinline__ void store_staged(const float* stage, const Epilogue& e,
                                             const Columns<GATED, W>& k,
                                             const Residual<(GATED ? W / 2 : W), ROWS>& res,
                                             int lane, int64_t m0, int64_t M, int64_t c0, int64_t N) {
    using Res = Residual<(GATED ? W / 2 : W), ROWS>;
    static_assert((kLanes / Res::per_row - 1) * (GATED ? kMaxRows / 2 : kMaxRows) + 64 <=
                      (int64_t)UINT32_MAX, "`mine`, here and in Residual, in elements");
    const int p = lane % Res::per_row * 2;
    const int64_t c = c0 + p * 4;
    const uint32_t mine = (uint32_t)(lane / Res::per_row) * (uint32_t)N + p * 4;
    wave_sync();
    #pragma unroll
    for (int q = 0; q < Res::Q; q++) {
        const int row = q * (kLanes / Res::per_row) + lane / Res::per_row;
        const int64_t m = m0 + row;
        float v[8];
        #pragma unroll
        for (int h = 0; h < 2; h++) {
            const v4f x = *reinterpret_cast<const v4f*>(stage + staged<W>(row, p + h));
            #pragma unroll
            for (int i = 0; i < 4; i++)
                v[4 * h + i] = activate<ACT>(x[i] * k.ws[4 * h + i] + k.bs[4 * h + i], e);
            if constexpr (GATED) {
                const v4f u = *reinterpret_cast<const v4f*>(stage + staged<W>(row, W / 8 + p + h));
                #pragma unroll
                for (int i = 0; i < 4; i++) v[4 * h + i] *= u[i] * k.wu[4 * h + i] + k.bu[4 * h + i];
            }
        }
        if (e.residual) {
            #pragma unroll
            for (int i = 0; i < 4; i++) {
                v[2 * i] += bf16_lo(res.u[q][i]);
                v[2 * i + 1] += bf16_hi(res.u[q][i]);
            }
        }
        const v4u out = {bf16_pack(v[0], v[1]), bf16_pack(v[2], v[3]), bf16_pack(v[4], v[5]),
                         bf16_pack(v[6], v[7])};
        uint16_t* y = e.y + (m0 + q * (kLanes / Res::per_row)) * N + c0 + mine;
        if (WHOLE || (m < M && c + 8 <= N)) {
            __builtin_memcpy(y, &out, 16);
        } else {
            #pragma unroll
            for (int i = 0; i < 8; i++)
                if (m < M && c + i < N) y[i] = (uint16_t)(out[i / 2] >> (i % 2 * 16));
        }
    }
    wave_sync();
}

struct MidMap {
    int tiles_m, tiles_n, splits;
    int64_t Np;       // outputs of a row of partial sums, a multiple of 16
    float* sums;      // splits > 1: [splits][M][1 or, gated, 2][Np]
};

// Workgroup: NW waves, each 32 rows of w (gated: 16 gate and 16 value rows) times
// 32 MI rows of a; `splits` workgroups share a tile's columns and leave 32-bit
// partial sums.  Each wave loads its own rows of w and its part of a's, PIPE - 1
// steps of 128 columns ahead; one barrier a step.  Pieces, keys and banks as in
// linear_tile_kernel below.
//
// A step of 128 columns takes a workgroup 0.3 us (32 x 64 rows) to 1.2 (128 x
// 256).  Over the ten tiles that goes with the bytes that reach LDS, 40 .. 46 GB/s
// a CU while all CUs load (11 TB/s together); the products take a SIMD 512 cycles
// of some 2000 (1024 where two waves share it, NW > 4) and the LDS reads, 4.4
// cycles each of 16 bytes a lane, 355 (128 x 128) to 700 (128 x 256), and nothing
// here lays one over the other.  So the best tile is the one that covers the
// product in the fewest bytes a CU: 97 rows by 34816 x 5120 (gated) 39.4 .. 40.7 us
// with 128 x 160 (one round of 218 workgroups), 43.4 with 128 x 192, 61.7 with 128 x
// 128 (two rounds), 62.3 with 64 x 128; 192 rows 52.5 with 192 x 160, 70 with 256 x
// 256 on half of the CUs.  w is not kept in the caches (non-temporal): a tile's
// workgroups run at the same time on one XCD and share it while it passes.  That
// holds for a small w too, which the XCDs then fetch more than once (1003 rows by
// 2187 x 1296: 14 MiB read of 3.9).  A product of few tiles is split along its
// columns: 64 rows by 5120 x 17408 26.0 us in 6 parts, 33.0 in 3 and 68.6 whole; 160
// by 460 x 14672 15.7 in 12 parts of 32 x 128 and 75.7 whole.
//
// With PIPE = 2 two workgroups share a CU, and one's products hide the other's
// loads and epilogue: for products of few steps, which are mostly those
// (linear_plan.h has what it gains).
template <bool GATED, int ACT, int MI, int NW, int PIPE>
__global__ __launch_bounds__(NW * kLanes, PIPE == 2 ? 2 : 1) void linear_mid_kernel(
    const uint8_t* __restrict__ a, const uint8_t* __restrict__ w, int64_t M, int64_t N, int64_t C,
    MidMap map, Epilogue e) {
    constexpr int kLoadsA = (4 * MI + NW - 1) / NW;   // of 8 rows; the last ones may be past a's
    constexpr int kA = kLoadsA * NW * 1024, kW = NW * 32 * kStep;
    constexpr int kLoads = kLoadsA + 4;         // of a wave and step
    static_assert(PIPE >= 2 && PIPE <= 4, "slots");
    __shared__ __attribute__((aligned(1024))) uint8_t slot0[kA + kW], slot1[kA + kW],
        slot2[PIPE > 2 ? kA + kW : 1], slot3[PIPE > 3 ? kA + kW : 1];
    const int lane = threadIdx.x & (kLanes - 1);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kLanes);
    const int r = lane & 31, g = lane >> 5;
    const uint32_t row_bytes = (uint32_t)C;
    // the row tiles of a tile of w and their parts are neighbours on one XCD
    const int item = xcd_order(blockIdx.x, gridDim.x);
    const int tm = item % map.tiles_m, rest = item / map.tiles_m;
    const int split = rest % map.splits, tn = rest / map.splits;
    const int64_t m0 = (int64_t)tm * (32 * MI);
    const int64_t n0 = ((int64_t)tn * NW + wave) * (GATED ? 16 : 32);   // the wave's
    const int steps_all = (int)((C + kStep - 1) / kStep);
    const int k_first = (int)((int64_t)steps_all * split / map.splits);
    const int k_end = (int)((int64_t)steps_all * (split + 1) / map.splits);
    const uint32_t col_end = (uint32_t)(k_end * (int64_t)kStep < C ? k_end * (int64_t)kStep : C);

    auto rows = [&](int64_t have, int most) {
        return (uint32_t)(have < 0 ? 0 : have < most ? have : most) * row_bytes;
    };
    const uint32_t wbytes = rows(N - n0, GATED ? 16 : 32);
    const Rsrc asrc = rsrc(a + m0 * C, rows(M - m0, 32 * MI));
    const Rsrc wsrc = rsrc(wbytes ? w + n0 * C : w, wbytes);
    const Rsrc usrc = rsrc(GATED && wbytes ? w + (N + n0) * C : w, GATED ? wbytes : 0);
    // of w: rows 8 j + lane / 8 of the wave's, key from rows' bits 1, 4 and 2
    const int lrow = lane >> 3, lpos = lane & 7;
    const uint32_t acol = (uint32_t)(lpos ^ (lane >> 4)) * 16;   // of an even group of 8 rows
    uint32_t wcol[2];   // j / 2 even, odd
    #pragma unroll
    for (int h = 0; h < 2; h++)
        wcol[h] = (uint32_t)(lpos ^ (((lane >> 4) & 1) | (h << 1) | ((lane >> 5) << 2))) * 16;
    auto fetch = [&](int k, uint8_t* slot) {
        const uint32_t k0 = (uint32_t)(k_first + k) * kStep;
        const uint32_t to = opaque_s((uint32_t)wave * (32 * kStep));
        #pragma unroll
        for (int j = 0; j < 4; j++) {
            // rows 8 j ..: gated, the gate's 16, then the value's
            const int row = GATED ? j % 2 * 8 : 8 * j;
            const uint32_t c = k0 + wcol[j / 2];
            load_lds<kNT>(GATED && j / 2 ? usrc : wsrc, slot + kA + to + j * 1024,
                          (c < col_end ? (uint32_t)lrow * row_bytes + c : kOut) + (uint32_t)row * row_bytes);
        }
        #pragma unroll
        for (int j = 0; j < kLoadsA; j++) {
            const uint32_t group = opaque_s((uint32_t)(j * NW + wave));
            const uint32_t c = k0 + (acol ^ (group & 1) << 6);
            load_lds<0>(asrc, slot + group * 1024,
                        (c < col_end ? (uint32_t)lrow * row_bytes + c : kOut) + group * 8 * row_bytes);
        }
    };
    // Operand row r of w is row 16 b + 4 i + c of its 32 for r = 8 i + 4 b + c, so
    // that lane (g, r) gets 16 consecutive outputs; gated, 16 (i / 2) + 8 b +
    // 4 (i % 2) + c: 8 consecutive gates, and their values.
    const int i4 = r >> 3, b1 = (r >> 2) & 1, c4 = r & 3;
    const int wrow = GATED ? i4 / 2 * 16 + b1 * 8 + i4 % 2 * 4 + c4 : b1 * 16 + i4 * 4 + c4;
    const int wkey = ((wrow >> 1) & 1) | ((wrow >> 4) << 1) | (((wrow >> 2) & 1) << 2);
    uint32_t abase[4], wbase[4];
    #pragma unroll
    for (int q = 0; q < 4; q++) {
        abase[q] = opaque_v(r * kStep + (uint32_t)((2 * q + g) ^ ((r >> 1) & 7)) * 16);
        wbase[q] = opaque_v(kA + (uint32_t)wave * (32 * kStep) + wrow * kStep +
                            (uint32_t)((2 * q + g) ^ wkey) * 16);
    }
    v16f acc[MI];
    #pragma unroll
    for (int i = 0; i < MI; i++)
        #pragma unroll
        for (int c = 0; c < 16; c++) acc[i][c] = 0.0f;
    auto read = [](const uint8_t* p, const uint32_t (&base)[4], int h) {
        return join(*reinterpret_cast<const v4u*>(p + base[2 * h]),
                    *reinterpret_cast<const v4u*>(p + base[2 * h + 1]));
    };
    // step k in `slot`; the slot of the step before is refilled
    auto step = [&](int k, uint8_t* slot, uint8_t* before) {
        arrive<(PIPE - 2) * kLoads>();
        fetch(k + PIPE - 1, before);
        #pragma unroll
        for (int h = 0; h < 2; h++) {
            const v8i fw = read(slot, wbase, h);
            v8i fa[MI];
            #pragma unroll
            for (int i = 0; i < MI; i++) fa[i] = read(slot + i * 4096, abase, h);
            #pragma unroll
            for (int i = 0; i < MI; i++) acc[i] = mfma(fw, fa[i], acc[i]);
        }
    };
    fetch(0, slot0);
    if (PIPE > 2) fetch(1, slot1);
    if (PIPE > 3) fetch(2, slot2);
    // (steps past the split's last are zeros)
    for (int k = 0; k < k_end - k_first; k += PIPE) {
        if constexpr (PIPE == 2) {
            step(k, slot0, slot1);
            step(k + 1, slot1, slot0);
        } else if constexpr (PIPE == 3) {
            step(k, slot0, slot2);
            step(k + 1, slot1, slot0);
            step(k + 2, slot2, slot1);
        } else {
            step(k, slot0, slot3);
            step(k + 1, slot1, slot0);
            step(k + 2, slot2, slot1);
            step(k + 3, slot3, slot2);
        }
    }
    // the slots are free: 4 KiB of them for each wave's sums
    arrive<0>();
    if (n0 >= N) return;
    float* stage = reinterpret_cast<float*>(slot0 + wave * 4096);
    // gated: the gates' 16 columns, then the values'
    auto put = [&](int i, float by) {
        #pragma unroll
        for (int b = 0; b < 4; b++)
            *reinterpret_cast<v4f*>(stage + staged<32>(r, GATED ? b / 2 * 4 + g * 2 + b % 2 : g * 4 + b)) =
                quad(acc[i], b, by);
    };
    if (map.splits > 1) {
        float* to = map.sums + (int64_t)split * M * (GATED ? 2 : 1) * map.Np;
        #pragma unroll
        for (int i = 0; i < MI; i++) {
            put(i, 1.0f);
            wave_sync();
            #pragma unroll
            for (int q = 0; q < 4; q++) {
                const int row = q * 8 + lane / 8, piece = lane % 8;
                const int64_t m = m0 + i * 32 + row;
                const v4f v = *reinterpret_cast<const v4f*>(stage + staged<32>(row, piece));
                const int64_t c = n0 + (GATED ? piece % 4 : piece) * 4;
                if (m < M && c < map.Np)
                    *reinterpret_cast<v4f*>(to + (m * (GATED ? 2 : 1) + (GATED ? piece / 4 : 0)) * map.Np + c) = v;
            }
            wave_sync();
        }
        return;
    }
    float sm[MI];
    #pragma unroll
    for (int i = 0; i < MI; i++) {
        const int64_t m = m0 + i * 32 + r;
        sm[i] = e.a_scale ? e.a_scale[m < M ? m : M - 1] : 1.0f;
    }
    auto finish = [&](auto WHOLE) {
        constexpr bool whole = decltype(WHOLE)::value;
        Columns<GATED, 32> cols;
        cols.template load<whole>(e, lane, n0, N);
        Residual<(GATED ? 16 : 32), 32> res[MI];
        if (e.residual) {
            #pragma unroll
            for (int i = 0; i < MI; i++) res[i].template load<whole>(e, lane, m0 + i * 32, M, n0, N);
        }
        #pragma unroll
        for (int i = 0; i < MI; i++) {
            put(i, sm[i]);
            store_staged<GATED, ACT, 32, 32, whole>(stage, e, cols, res[i], lane, m0 + i * 32, M, n0, N);
        }
    };
    if (m0 + MI * 32 <= M && n0 + (GATED ? 16 : 32) <= N) finish(std::true_type{});
    else finish(std::false_type{});
}

// y from the splits' sums, added in their order (no atomics: every call gives
// the same bits).  A thread takes 4 consecutive outputs.  Bound by its launch:
// 2.9 us beside the sums' bytes, which lie in the caches.
template <bool GATED, int ACT>
__global__ __launch_bounds__(256) void linear_join_kernel(MidMap map, int64_t M, int64_t N, Epilogue e) {
    const int64_t quads = map.Np / 4;
    const int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int64_t m = t / quads, n = t % quads * 4;
    if (m >= M || n >= N) return;
    const int64_t row = (GATED ? 2 : 1) * map.Np, stride = M * row;
    const float* p = map.sums + m * row + n;
    v4f s = {0, 0, 0, 0}, u = {0, 0, 0, 0};
    for (int k = 0; k < map.splits; k++) {
        s += *reinterpret_cast<const v4f*>(p + k * stride);
        if (GATED) u += *reinterpret_cast<const v4f*>(p + k * stride + map.Np);
    }
    float ws[4], bs[4], wu[4], bu[4];
    columns(e, 0, n, N, ws, bs);
    if (GATED) columns(e, N, n, N, wu, bu);
    const float sm = e.a_scale ? e.a_scale[m] : 1.0f;
    #pragma unroll
    for (int i = 0; i < 4; i++) {
        if (n + i >= N) break;
        float v = activate<ACT>(s[i] * sm * ws[i] + bs[i], e);
        if (GATED) v *= u[i] * sm * wu[i] + bu[i];
        if (e.residual) v += bf16_lo(e.residual[m * N + n + i]);
        e.y[m * N + n + i] = (uint16_t)bf16_pack(v, 0.0f);
    }
}

// ---------------------------------------------------------------------
// Tiles of 256 rows of a by 256 rows of w, for products with many rows.
//
// Four waves of 128 x 128 outputs, 256 sums a lane, the most that the registers
// hold: a step of 128 columns brings 64 KiB to LDS for 32 products of 32 x 32 x
// 64 a wave.  8 waves of 64 x 128, or 16 x 16 x 128 products, read more of LDS
// per product (8192^3 425 us with the latter, whose sums the compiler also moves
// between registers in the loop).  Two steps lie in LDS, in units that are
// refilled as soon as they are read; loads and LDS reads are spread over the
// products (8192^3 467 us before, 431 after that).  A step takes 2230 cycles,
// 2048 of them in the matrix cores (92%).  The workgroups are persistent, so that
// the next tile's first steps load during the epilogue.
//
// 8192^3 takes 370 .. 400 us by the operands' values, 2.75 .. 2.98 PFLOP/s; 8192 by
// 34816 x 5120 (gated) 1105 .. 1160 by the board, 2.52 .. 2.65; 2048 by 5120 x 17408
// 152 .. 158, 2.3 .. 2.4.  Bound by the board's power: the clock falls to 1.65 ..
// 1.75 GHz of 2.4 within the loop.  Besides, a tile's epilogue takes 20,000 cycles
// in which nothing is multiplied: 17 tiles a CU by 34816 x 5120, 18% of the
// time, most of it the issue of 27 vector instructions an output.
// ---------------------------------------------------------------------
constexpr int kTile = 256;          // rows of either operand
constexpr int kHalf = 128;          // w's rows come in two halves (gated: gate and value)
constexpr int kUnit = kHalf * kStep;
constexpr int kTileWaves = 4;

// GY: groups of 32 rows of w's second half that a wave takes (2, or 1 for tiles
// of 192 rows of w, which fit products of few tiles better: 2048 rows by 5120 x
// 17408 are 216 of them, one round at 156 us, or 160 of 256 rows at 172).
template <bool GATED, int ACT, int GY>
__global__ __launch_bounds__(kTileWaves * kLanes, 1) void linear_tile_kernel(
    const uint8_t* __restrict__ a, const uint8_t* __restrict__ w, int64_t M, int64_t N, int64_t C,
    TileMap map, Epilogue e) {
    // Two steps' operands, each in units of its own (128 rows, 16 KiB; the
    // compiler tells loads into different arrays apart, and waits for none
    // that a read does not need): s<operand><half><step % 2>
    __shared__ __attribute__((aligned(1024))) uint8_t sa00[kUnit], sa10[kUnit], sw00[kUnit], sw10[kUnit * GY / 2];
    __shared__ __attribute__((aligned(1024))) uint8_t sa01[kUnit], sa11[kUnit], sw01[kUnit], sw11[kUnit * GY / 2];
    __shared__ __attribute__((aligned(1024))) float out_stage[kTileWaves][32 * 64];
    static_assert(GY == 2 || (GY == 1 && !GATED), "a gated tile's halves belong together");
    constexpr int kWide = kHalf + 64 * GY;      // rows of w
    constexpr int kW0 = 4, kW1 = 2 * GY;        // loads of a wave for w's halves; a's are 4
    const int lane = threadIdx.x & (kLanes - 1);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kLanes);
    const int wm = wave >> 1, wn = wave & 1;
    const uint32_t row_bytes = (uint32_t)C;
    const int steps = (int)((C + 2 * kStep - 1) / (2 * kStep)) * 2;   // even

    // Lane (g, r) is lane 32 g + r.  Its addresses are computed for each tile
    // from an opaque lane number: kept over a tile's epilogue they would be
    // spilled, and the loop would wait for their reloads, and with them for all
    // loads issued before, in every step.
    //
    // Loads: one instruction brings 8 rows of 128 bytes, lane l the 16 bytes
    // that belong at position l % 8 of row l / 8.  A row's 16-byte pieces are
    // permuted by an exclusive or with a key of the row.
    //
    // Fragments: of each group of 32 rows lane (g, r) takes the pieces g, 2 + g,
    // 4 + g and 6 + g of one, two for each of two products.  Of the 32 x 32
    // products of an instruction it gets those of a's row r with w's rows
    // 8 i + 4 g + c (i, c = 0 .. 3) of the operand; w's row 16 g + 4 i + c is put
    // there, so that a lane's 16 outputs are consecutive.
    uint32_t acol, wcol, lbase, abase[4], wbase[2][4];
    auto aim = [&]() {
        const uint32_t l = opaque_v((uint32_t)lane), r = l & 31, g = l >> 5;
        acol = ((l & 7) ^ (((l >> 4) & 3) | ((wave & 1) << 2))) * 16;
        wcol = ((l & 7) ^ (((l >> 4) & 1) | ((wave >> 1) << 1) | ((l >> 5) << 2))) * 16;
        lbase = (wave * 8 + (l >> 3)) * row_bytes;
        const uint32_t wrow = ((r >> 2) & 1) * 16 + (r >> 3) * 4 + (r & 3);
        #pragma unroll
        for (int q = 0; q < 4; q++) {
            const uint32_t piece = ((2 * q + g) ^ ((r >> 1) & 7)) * 16;
            abase[q] = opaque_v((wm * 64 + r) * 128 + piece);
            wbase[0][q] = opaque_v((wn * 64 + wrow) * 128 + piece);
            wbase[1][q] = GY == 2 ? wbase[0][q] : opaque_v((wn * 32 + wrow) * 128 + piece);
        }
    };

    struct Src { Rsrc a, w0, w1; int64_t m0, n0; } cur, nxt;
    auto source = [&](int t) {
        Src s;
        if (t < 0) {   // nothing: every load is out of range
            s.a = s.w0 = s.w1 = rsrc(a, 0);
            s.m0 = s.n0 = 0;
            return s;
        }
        int tm, tn;
        map.place(t, tm, tn);
        s.m0 = (int64_t)tm * kTile;
        s.n0 = (int64_t)tn * (GATED ? kHalf : kWide);
        auto rows = [&](int64_t have, int most) {
            return (uint32_t)(have < 0 ? 0 : have < most ? have : most) * row_bytes;
        };
        s.a = rsrc(a + s.m0 * C, rows(M - s.m0, kTile));
        s.w0 = rsrc(w + s.n0 * C, rows(N - s.n0, kHalf));
        const int64_t second = GATED ? N + s.n0 : s.n0 + kHalf;
        const uint32_t bytes1 = rows(GATED ? N - s.n0 : N - second, 64 * GY);
        s.w1 = rsrc(bytes1 ? w + second * C : w, bytes1);
        return s;
    };
    // Half h of a's or w's rows of step k into a unit, in 4 loads (j) of each
    // wave; columns past C come as zeros.  a's half h is rows 64 h .. of each
    // 128, w's half h rows 128 h ...
    auto fetch_a = [&](const Src& s, int k, int h, uint8_t* unit, int j) {
        const uint32_t c = (uint32_t)k * kStep + acol;
        load_lds<0>(s.a, unit + opaque_s(wave * 1024) + j * 4096,
                 (c < row_bytes ? lbase + c : kOut) +
                     (uint32_t)((j >> 1) * 128 + h * 64 + (j & 1) * 32) * row_bytes);
    };
    auto fetch_w = [&](const Src& s, int k, int h, uint8_t* unit, int j) {
        const uint32_t c = (uint32_t)k * kStep + wcol;
        load_lds<0>(h ? s.w1 : s.w0, unit + opaque_s(wave * 1024) + j * 4096,
                 (c < row_bytes ? lbase + c : kOut) + (uint32_t)j * 32 * row_bytes);
    };

    v8i fa[4][2], fw[2 + GY][2];     // [2 h + group of 32 rows][product]: half h
    v16f acc[4][2 + GY];
    auto zero = [&]() {
        #pragma unroll
        for (int i = 0; i < 4; i++)
            #pragma unroll
            for (int j = 0; j < 2 + GY; j++)
                #pragma unroll
                for (int c = 0; c < 16; c++) acc[i][j][c] = 0.0f;
    };
    // piece s % 4 of group s / 4 of a half, s = 0 .. 7
    auto set = [](v8i& f, int half, const v4u& u) {
        #pragma unroll
        for (int i = 0; i < 4; i++) f[4 * half + i] = (int)u[i];
    };
    auto read_a = [&](int h, const uint8_t* unit, int s) {
        set(fa[2 * h + s / 4][s % 4 / 2], s % 2, *reinterpret_cast<const v4u*>(unit + s / 4 * 4096 + abase[s % 4]));
    };
    auto read_w = [&](int h, const uint8_t* unit, int s) {
        set(fw[2 * h + s / 4][s % 4 / 2], s % 2, *reinterpret_cast<const v4u*>(unit + s / 4 * 4096 + wbase[h][s % 4]));
    };
    // The products of halves HA and HW, with `reads` LDS reads for the next phase
    // and `loads` loads spread over them.
    auto multiply = [&](auto HA, auto HW, auto READS, auto&& read, auto LOADS, auto&& load) {
        constexpr int ha = decltype(HA)::value, hw = decltype(HW)::value;
        constexpr int ng = hw ? GY : 2, n = 4 * ng;   // groups of w, products
        constexpr int reads = decltype(READS)::value, loads = decltype(LOADS)::value;
        #pragma unroll
        for (int s = 0; s < n; s++) {
            #pragma unroll
            for (int o = s * reads / n; o < (s + 1) * reads / n; o++) read(o);
            #pragma unroll
            for (int o = s * loads / n; o < (s + 1) * loads / n; o++) load(o);
            const int kh = s / (2 * ng), i = s / ng % 2, f = s % ng;
            v16f& c = acc[2 * ha + i][2 * hw + f];
            c = mfma(fw[2 * hw + f][kh], fa[2 * ha + i][kh], c);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    constexpr std::integral_constant<int, 0> I0{};
    constexpr std::integral_constant<int, 1> I1{};
    // A step in two halves, on its units a0, a1, x, y (w's halves X and Y) and
    // the next step's a0n, yn; a's half 0 and w's half X are in registers.  Each
    // half reads two units and refills the two that the half before has read
    // with the step after the next (k2 of s2), so that a load has two to three
    // half steps to arrive in.  Leaves a's half 0 and w's half Y of the next step
    // in registers.
    auto step = [&](auto X, auto Y, uint8_t* a0, uint8_t* a1, uint8_t* x, uint8_t* y, uint8_t* a0n,
                    uint8_t* yn, const Src& s2, int k2) {
        constexpr int hx = decltype(X)::value, hy = decltype(Y)::value;
        constexpr int wx = hx ? kW1 : kW0, wy = hy ? kW1 : kW0;
        arrive<8 + kW0 + kW1>();         // (all but the two half steps' before)
        multiply(I0, X, kInt<2 * wy>, [&](int s) { read_w(hy, y, s); },
                 kInt<4>, [&](int j) { fetch_a(s2, k2, 0, a0, j); });
        multiply(I0, Y, kInt<8>, [&](int s) { read_a(1, a1, s); },
                 kInt<wx>, [&](int j) { fetch_w(s2, k2, hx, x, j); });
        arrive<8 + 2 * wx>();
        multiply(I1, Y, kInt<8>, [&](int s) { read_a(0, a0n, s); },
                 kInt<wy>, [&](int j) { fetch_w(s2, k2, hy, y, j); });
        multiply(I1, X, kInt<2 * wy>, [&](int s) { read_w(hy, yn, s); },
                 kInt<4>, [&](int j) { fetch_a(s2, k2, 1, a1, j); });
    };

    int i = 0;
    int t = map.at(0, blockIdx.x, gridDim.x);
    if (t < 0) return;
    cur = source(t);
    aim();
    auto fetch = [](auto LOADS, auto&& load) {
        #pragma unroll
        for (int j = 0; j < decltype(LOADS)::value; j++) load(j);
    };
    // in the order in which they are read
    fetch(kInt<4>, [&](int j) { fetch_a(cur, 0, 0, sa00, j); });
    fetch(kInt<kW0>, [&](int j) { fetch_w(cur, 0, 0, sw00, j); });
    fetch(kInt<kW1>, [&](int j) { fetch_w(cur, 0, 1, sw10, j); });
    fetch(kInt<4>, [&](int j) { fetch_a(cur, 0, 1, sa10, j); });
    fetch(kInt<4>, [&](int j) { fetch_a(cur, 1, 0, sa01, j); });
    fetch(kInt<kW1>, [&](int j) { fetch_w(cur, 1, 1, sw11, j); });
    fetch(kInt<kW0>, [&](int j) { fetch_w(cur, 1, 0, sw01, j); });
    fetch(kInt<4>, [&](int j) { fetch_a(cur, 1, 1, sa11, j); });
    arrive<16 + 2 * kW1>();
    while (true) {
        const int t_next = map.at(++i, blockIdx.x, gridDim.x);
        nxt = source(t_next);
        if (i > 1) aim();
        // (the last step of a tile before has read these pieces too, but not
        // kept them over the epilogue)
        #pragma unroll
        for (int s = 0; s < 8; s++) {
            read_a(0, sa00, s);
            read_w(0, sw00, s);
        }
        zero();
        for (int k = 2; k <= steps; k += 2) {
            // the last two steps fetch the next tile's first two
            const Src& s2 = k == steps ? nxt : cur;
            const int k2 = k == steps ? 0 : k;
            step(I0, I1, sa00, sa10, sw00, sw10, sa01, sw11, s2, k2);
            step(I1, I0, sa01, sa11, sw11, sw01, sa00, sw00, s2, k2 + 1);
        }

        float* stage = out_stage[wave];
        // Lane (g, r) has, of each 32 of w's rows (f), 16 consecutive sums of row
        // r.  32 rows at a time by a half's 64 columns, or gated by 32 gates and
        // their values.
        const int64_t first = cur.m0 + wm * 128;
        // (opaque: else the lane's addresses are kept, and spilled, over the loop)
        const int ln = (int)opaque_v((uint32_t)lane), er = ln & 31, eg = ln >> 5;
        float sm[4];
        #pragma unroll
        for (int i = 0; i < 4; i++) {
            const int64_t m = first + i * 32 + er;
            sm[i] = e.a_scale ? e.a_scale[m < M ? m : M - 1] : 1.0f;
        }
        wait_loads<0>();   // (left to the compiler, some are waited for in the loop)
        // part: w's half, or gated the first or second 32 of the wave's outputs
        auto finish = [&](auto PART) {
            constexpr int part = decltype(PART)::value;
            constexpr int ng = part ? GY : 2, W = GATED ? 64 : 32 * ng, CW = GATED ? 32 : W;
            const int64_t c0 = cur.n0 + (GATED ? wn * 64 + part * 32 : part * kHalf + wn * W);
            auto with = [&](auto WHOLE) {
                constexpr bool whole = decltype(WHOLE)::value;
                Residual<CW, 32> res[4];
                if (e.residual) {
                    #pragma unroll
                    for (int i = 0; i < 4; i++) res[i].template load<whole>(e, ln, first + i * 32, M, c0, N);
                }
                Columns<GATED, W> cols;
                cols.template load<whole>(e, ln, c0, N);
                #pragma unroll
                for (int i = 0; i < 4; i++) {
                    #pragma unroll
                    for (int f = 0; f < W / 32; f++)
                        #pragma unroll
                        for (int b = 0; b < 4; b++)
                            *reinterpret_cast<v4f*>(stage + staged<W>(er, f * 8 + eg * 4 + b)) =
                                quad(acc[i][GATED ? 2 * f + part : 2 * part + f], b, sm[i]);
                    store_staged<GATED, ACT, W, 32, whole>(stage, e, cols, res[i], ln, first + i * 32, M, c0, N);
                }
            };
            if (first + 128 <= M && c0 + CW <= N) with(std::true_type{});
            else with(std::false_type{});
        };
        finish(I0);
        finish(I1);
        if (t_next < 0) break;
        t = t_next;
        cur = nxt;
    }
    wait_loads<0>();
}

// f(gated, activation form) with both as types
template <class F>
void for_kind(bool gated, int act, F&& f) {
    auto with = [&](auto G) {
        if (act == kErf) f(G, std::integral_constant<int, kErf>{});
        else if (act == kTanh) f(G, std::integral_constant<int, kTanh>{});
        else if (act == kSilu) f(G, std::integral_constant<int, kSilu>{});
        else f(G, std::integral_constant<int, kClip>{});
    };
    if (gated) with(std::true_type{}); else with(std::false_type{});
}

// Checks the sizes and makes the plan (0.1 to 0.8 us for more than 16 rows);
// without a device, for one of 256 CUs.  M = 0 needs none.
int checked_plan(int64_t M, int64_t R, int64_t C, int32_t gated, int cus, Plan* p) {
    if (M < 0 || R < 1 || M > INT32_MAX || R > kMaxRows || (gated && R % 2))
        return fail(TANS_EINVAL, "linear: need M >= 0 below 2^31 and R in 1 .. 2^27, even if gated");
    if (C < 16 || C % 16 || C > kMaxCols)
        return fail(TANS_EINVAL, "linear: C must be a multiple of 16, 16 .. 2^22");
    *p = M ? plan(M, gated ? R / 2 : R, C, gated, cus > 0 ? cus : 256) : Plan{};
    return TANS_OK;
}

}  // namespace

extern "C" {

int tans_fp8_linear_workspace(int64_t M, int64_t R, int64_t C, int32_t gated, int64_t* bytes) {
    if (!bytes) return fail(TANS_EINVAL, "linear: null pointer");
    Plan p;
    const int rc = checked_plan(M, R, C, gated, tans_internal_cu_count(), &p);
    if (rc == TANS_OK) *bytes = p.bytes;
    return rc;
}

int tans_fp8_linear(const void* a, const float* a_scale, const void* w, const float* w_scale,
                    float scale, const void* bias, const void* residual, int32_t activation,
                    int32_t gated, int64_t M, int64_t R, int64_t C, void* workspace,
                    int64_t workspace_bytes, void* y, void* stream) {
    const int cus = tans_internal_cu_count();
    Plan p;
    const int rc = checked_plan(M, R, C, gated, cus, &p);
    if (rc != TANS_OK) return rc;
    if (activation < 0 || activation > TANS_ACT_GELU_TANH)
        return fail(TANS_EINVAL, "linear: activation must be 0 .. 4");
    if (M == 0) return TANS_OK;
    if (!a || !w || !y) return fail(TANS_EINVAL, "linear: null pointer");
    // (bias and residual are read as rows of y are, which start anywhere if N is odd)
    if (!aligned(a, 16) || !aligned(w, 16) || !aligned(y, 16) || !aligned(residual, 2) ||
        !aligned(bias, 2) || !aligned(a_scale, 4) || !aligned(w_scale, 4))
        return fail(TANS_EINVAL,
                    "linear: misaligned buffer (scales 4, bias and residual 2, others 16 bytes)");
    if (p.bytes > 0 && (!workspace || !aligned(workspace, 16) || workspace_bytes < p.bytes))
        return fail(TANS_EINVAL, "linear: workspace too small, null or misaligned (16 bytes)");
    const int64_t N = gated ? R / 2 : R;
    if (cus <= 0) return fail(TANS_EHIP, "linear: cannot query the device's CU count");
    const Epilogue e = {a_scale, w_scale, (const uint16_t*)bias, (const uint16_t*)residual,
                        (uint16_t*)y, scale,
                        activation == TANS_ACT_RELU ? 0.0f : -INFINITY};
    const int act = activation == TANS_ACT_GELU ? kErf
                    : activation == TANS_ACT_GELU_TANH ? kTanh
                    : activation == TANS_ACT_SILU ? kSilu : kClip;
    const uint8_t *a8 = (const uint8_t*)a, *w8 = (const uint8_t*)w;
    const hipStream_t st = (hipStream_t)stream;
    auto launch = [&](auto kernel, int64_t blocks, int threads, auto... args) {
        if (blocks > INT32_MAX / threads) return fail(TANS_EINVAL, "linear: too many outputs for one call");
        hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(threads), 0, st, args...);
        return hip_check(hipGetLastError(), "linear kernel launch");
    };
    int out = TANS_OK;
    for_kind(gated, act, [&](auto G, auto A) {
        constexpr bool g = decltype(G)::value;
        constexpr int ac = decltype(A)::value;
        auto stream_rows = [&](auto MA) {
            constexpr int ma = decltype(MA)::value;
            const int64_t wide = (N + (g ? 16 : 32) - 1) / (g ? 16 : 32);
            if constexpr (!g) {
                if (p.few) {
                    out = launch(linear_stream_kernel<g, ac, ma, 1, 4, 4>, (N + 15) / 16, 256, a8, w8, M, N, C, e);
                    return;
                }
            }
            out = launch(linear_stream_kernel<g, ac, ma, 2, 4, 2>, wide, 256, a8, w8, M, N, C, e);
        };
        if (p.kind == kStream) {
            if (M <= 8) stream_rows(kInt<1>);
            else if (M <= 16) stream_rows(kInt<2>);
            else stream_rows(kInt<4>);
        } else if (p.kind == kMid) {
            const MidMap map = {(int)p.tiles_m, (int)p.tiles_n, p.splits, p.Np, (float*)workspace};
            const int64_t blocks = p.tiles_m * p.tiles_n * p.splits;
            if (blocks > INT32_MAX) {
                out = fail(TANS_EINVAL, "linear: too many outputs for one call");
                return;
            }
            auto mid = [&](auto MI, auto NW) {
                constexpr int mi = decltype(MI)::value, nw = decltype(NW)::value;
                constexpr int kib = (4 * mi + nw - 1) / nw * nw + 4 * nw;   // of a step
                constexpr int pipe = 4 * kib <= 160 ? 4 : 3;
                if (p.mi == mi && p.nw == nw)
                    out = launch(linear_mid_kernel<g, ac, mi, nw, pipe>, blocks, nw * kLanes, a8, w8, M, N, C, map, e);
            };
            if (p.pairs) {
                out = launch(linear_mid_kernel<g, ac, 4, 4, 2>, blocks, 4 * kLanes, a8, w8, M, N, C, map, e);
                return;
            }
            mid(kInt<1>, kInt<2>);
            mid(kInt<1>, kInt<4>);
            mid(kInt<2>, kInt<4>);
            mid(kInt<2>, kInt<5>);
            mid(kInt<3>, kInt<4>);
            mid(kInt<4>, kInt<4>);
            mid(kInt<4>, kInt<5>);
            mid(kInt<4>, kInt<6>);
            mid(kInt<4>, kInt<8>);
            mid(kInt<6>, kInt<5>);
            if (out == TANS_OK && p.splits > 1)
                out = launch(linear_join_kernel<g, ac>, (M * (p.Np / 4) + 255) / 256, 256, map, M, N, e);
        } else {
            if (p.tiles_m > INT32_MAX / p.tiles_n) {
                out = fail(TANS_EINVAL, "linear: too many outputs for one call");
                return;
            }
            const TileMap map = {(int)p.tiles_m, (int)p.tiles_n};
            const int64_t blocks = tile_blocks(p.tiles_m * p.tiles_n, cus);
            if constexpr (!g) {
                if (p.nw == 6) {
                    out = launch(linear_tile_kernel<g, ac, 1>, blocks, 256, a8, w8, M, N, C, map, e);
                    return;
                }
            }
            out = launch(linear_tile_kernel<g, ac, 2>, blocks, 256, a8, w8, M, N, C, map, e);
        }
    });
    return out;
}

}  // extern "C"
