// Matrix product of FP8 rows with FP8 weights, its epilogue included
// (gfx950).  No counterpart in the reference.
//
//   v[m][n] = a_scale[m] * w_scale[n] * scale * sum_k a[m][k] w[n][k] + bias[n]
//   y[m][n] = act(v[m][n]) + residual[m][n]
//   gated: y[m][j] = act(v[m][j]) * v[m][F + j] + residual[m][j], F = R / 2
//
// a and w hold E4M3FN bytes; the products of v_mfma_f32_16x16x128_f8f6f4 are
// exact and summed in 32 bits; y is rounded once, to bf16.
#include <math.h>

#include <algorithm>
#include <type_traits>

#include "launch.h"
#include "layer.h"

namespace {

typedef int v8i __attribute__((ext_vector_type(8)));

constexpr int64_t kMaxCols = int64_t(1) << 22;   // a tile's rows stay below 2^32 bytes

constexpr float kLog2e = 1.44269504f;

struct Epilogue {
    const float* a_scale;        // [M] or null (1)
    const float* w_scale;        // [R] or null (1)
    const uint16_t* bias;        // bf16 [R] or null
    const uint16_t* residual;    // bf16 [M, N] or null
    uint16_t* y;                 // bf16 [M, N]
    float scale;
    float lo;                    // kClip: the least value
    float c1, c3;                // kSigmoid: of the sigmoid's argument, times log2 e
};

// The activations in three forms, each a kernel of its own:
//   kClip     max(v, lo): none (lo = -infinity) and ReLU (a NaN stays one)
//   kSigmoid  v * sigmoid(b1 v + b3 v^3): SiLU (b1 = 1, b3 = 0) and GELU's tanh
//             form, (1 + tanh(u)) / 2 = sigmoid(2 u)
//   kErf      v Phi(v), erfc by Abramowitz and Stegun 7.1.26 (absolute error
//             below 1.5e-7)
enum Act { kClip, kSigmoid, kErf };

template <int ACT>
__device__ __forceinline__ float activate(float v, const Epilogue& e) {
    if constexpr (ACT == kClip) {
        return v < e.lo ? e.lo : v;
    } else if constexpr (ACT == kSigmoid) {
        // the square is kept finite, for b3 = 0 times it
        const float sq = __builtin_fminf(v * v, 1e30f);
        const float x = v * __builtin_fmaf(e.c3, sq, e.c1);
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

// A wave computes 16 rows of a times 16 outputs; 4 waves of a workgroup take
// consecutive groups of 16 outputs.  Operands go from memory straight to
// registers: lane l holds row l % 16 of either and, of each 128 columns,
// columns 32 (l / 16) .. + 31.  Of the 16 x 16 products, lane l gets those of
// a's row l % 16 with weight rows 4 (l / 16) .. + 3.
template <bool GATED, int ACT>
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
        float v = activate<ACT>(scaled(acc[i], c), e);
        if (GATED) v *= scaled(up[i], N + c);
        if (e.residual) v += bf16_lo(e.residual[m * N + c]);
        e.y[m * N + c] = (uint16_t)bf16_pack(v, 0.0f);
    }
}


// Scale and bias of w's rows first + c .. first + c + CN - 1, of which those
// with c + i < N exist (the others are repeats of the last).
template <int CN>
__device__ __forceinline__ void columns(const Epilogue& e, int64_t first, int64_t c, int64_t N,
                                        float (&ws)[CN], float (&bs)[CN]) {
    #pragma unroll
    for (int i = 0; i < CN; i++) {
        ws[i] = 1.0f;
        bs[i] = 0.0f;
    }
    uint16_t b[CN];
    if (c + CN <= N) {
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
// Tiles of 256 rows of a by 256 rows of w, for products with many rows.
// ---------------------------------------------------------------------
constexpr int kTile = 256;          // rows of either operand
constexpr int kHalf = 128;          // w's rows come in two halves (gated: gate and value)
constexpr int kStep = 128;          // columns (bytes) of a step
constexpr int kUnit = kHalf * kStep;
constexpr int kTileWaves = 4;
// An offset past every tile's bytes (kTile * kMaxCols = 2^30), also with a
// tile's row offset added
constexpr uint32_t kOut = 0x80000000u;

// 16 bytes a lane from memory to LDS, lane l's to lds + 16 l; zeros from
// offsets out of range.
__device__ __forceinline__ void load_lds(const Rsrc& src, uint8_t* lds, uint32_t offset) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(src, (__attribute__((address_space(3))) void*)lds, 16,
                                             (int)offset, 0, 0, 0);
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

__device__ __forceinline__ v8i join(const v4u& lo, const v4u& hi) {
    return v8i{(int)lo.x, (int)lo.y, (int)lo.z, (int)lo.w,
               (int)hi.x, (int)hi.y, (int)hi.z, (int)hi.w};
}

typedef float v16f __attribute__((ext_vector_type(16)));

__device__ __forceinline__ v16f mfma(const v8i& w, const v8i& a, const v16f& c) {
    return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(w, a, c, 0, 0, 0, 0, 0, 0);
}

// Where a workgroup's tiles lie: the tile sequence takes groups of kGroupM
// tiles of a's rows, in each of them w's tiles in order and the group's row
// tiles innermost; an eighth of the sequence goes to each of the 8 XCDs
// (workgroup b runs on XCD b % 8), so that the tiles an XCD works on at a time
// share their rows of a and w in its L2.
constexpr int kXcds = 8;
constexpr int kGroupM = 8;

struct TileMap {
    int tiles_m, tiles_n;
    __device__ __forceinline__ int count() const { return tiles_m * tiles_n; }
    // the i-th tile of workgroup b of `blocks`, or -1
    __device__ __forceinline__ int at(int i, int b, int blocks) const {
        const int xcd = b % kXcds, T = count();
        const int per = T / kXcds, more = T % kXcds;
        const int first = xcd * per + (xcd < more ? xcd : more);
        const int n = per + (xcd < more ? 1 : 0);
        const int peers = (blocks - xcd + kXcds - 1) / kXcds;
        const int k = i * peers + b / kXcds;
        return k < n ? first + k : -1;
    }
    __device__ __forceinline__ void place(int t, int& tm, int& tn) const {
        const int group = t / (kGroupM * tiles_n);
        const int m_first = group * kGroupM;
        const int gm = tiles_m - m_first < kGroupM ? tiles_m - m_first : kGroupM;
        const int in = t - group * kGroupM * tiles_n;
        tm = m_first + in % gm;
        tn = in / gm;
    }
};

template <bool GATED, int ACT>
__global__ __launch_bounds__(kTileWaves * kLanes, 1) void linear_tile_kernel(
    const uint8_t* __restrict__ a, const uint8_t* __restrict__ w, int64_t M, int64_t N, int64_t C,
    TileMap map, Epilogue e) {
    // Two steps' operands, each in units of its own (128 rows, 16 KiB; the
    // compiler tells loads into different arrays apart, and waits for none
    // that a read does not need): s<operand><half><step % 2>
    __shared__ __attribute__((aligned(1024))) uint8_t sa00[kUnit], sa10[kUnit], sw00[kUnit], sw10[kUnit];
    __shared__ __attribute__((aligned(1024))) uint8_t sa01[kUnit], sa11[kUnit], sw01[kUnit], sw11[kUnit];
    const int lane = threadIdx.x & (kLanes - 1);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kLanes);
    const int wm = wave >> 1, wn = wave & 1;
    const int r = lane & 31, g = lane >> 5;
    const uint32_t row_bytes = (uint32_t)C;
    const int steps = (int)((C + 2 * kStep - 1) / (2 * kStep)) * 2;   // even

    // Of the 32 x 32 products of an instruction lane (g, r) gets those of a's
    // row r with w's rows 8 i + 4 g + c (i, c = 0 .. 3) of the operand; w's row
    // 16 g + 4 i + c is put there, so that a lane's 16 outputs are consecutive.
    const int wrow = ((r >> 2) & 1) * 16 + (r >> 3) * 4 + (r & 3);

    // Loads: one instruction brings 8 rows of 128 bytes, lane l the 16 bytes
    // that belong at position l % 8 of row l / 8.  A row's 16-byte pieces are
    // permuted by an exclusive or with a key of the row, see `frag`.
    const int lrow = wave * 8 + (lane >> 3), lpos = lane & 7;
    const int akey = ((lane >> 4) & 3) | ((wave & 1) << 2);
    const int wkey = ((lane >> 4) & 1) | ((wave >> 1) << 1) | ((lane >> 5) << 2);
    const uint32_t acol = (uint32_t)(lpos ^ akey) * 16, wcol = (uint32_t)(lpos ^ wkey) * 16;
    const uint32_t lbase = (uint32_t)lrow * row_bytes;

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
        s.n0 = (int64_t)tn * (GATED ? kHalf : kTile);
        auto rows = [&](int64_t have, int most) {
            return (uint32_t)(have < 0 ? 0 : have < most ? have : most) * row_bytes;
        };
        s.a = rsrc(a + s.m0 * C, rows(M - s.m0, kTile));
        s.w0 = rsrc(w + s.n0 * C, rows(N - s.n0, kHalf));
        const int64_t second = GATED ? N + s.n0 : s.n0 + kHalf;
        const uint32_t bytes1 = rows(GATED ? N - s.n0 : N - second, kHalf);
        s.w1 = rsrc(bytes1 ? w + second * C : w, bytes1);
        return s;
    };
    // Half h of a's or w's rows of step k into a unit, in 4 loads (j) of each
    // wave; columns past C come as zeros.  a's half h is rows 64 h .. of each
    // 128, w's half h rows 128 h ...
    auto fetch_a = [&](const Src& s, int k, int h, uint8_t* unit, int j) {
        const uint32_t c = (uint32_t)k * kStep + acol;
        load_lds(s.a, unit + opaque_s(wave * 1024) + j * 4096,
                 (c < row_bytes ? lbase + c : kOut) +
                     (uint32_t)((j >> 1) * 128 + h * 64 + (j & 1) * 32) * row_bytes);
    };
    auto fetch_w = [&](const Src& s, int k, int h, uint8_t* unit, int j) {
        const uint32_t c = (uint32_t)k * kStep + wcol;
        load_lds(h ? s.w1 : s.w0, unit + opaque_s(wave * 1024) + j * 4096,
                 (c < row_bytes ? lbase + c : kOut) + (uint32_t)j * 32 * row_bytes);
    };

    // Fragments: of each group of 32 rows lane (g, r) takes the 16-byte pieces
    // g, 2 + g, 4 + g and 6 + g of one, two for each of two products.
    const int key = (r >> 1) & 7;
    uint32_t abase[4], wbase[4];
    #pragma unroll
    for (int q = 0; q < 4; q++) {
        const uint32_t piece = (uint32_t)((2 * q + g) ^ key) * 16;
        abase[q] = opaque_v((wm * 64 + r) * 128 + piece);
        wbase[q] = opaque_v((wn * 64 + wrow) * 128 + piece);
    }
    v8i fa[4][2], fw[4][2];     // [2 h + group of 32 rows][product]: half h
    v16f acc[4][4];
    auto zero = [&]() {
        #pragma unroll
        for (int i = 0; i < 4; i++)
            #pragma unroll
            for (int j = 0; j < 4; j++)
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
        set(fw[2 * h + s / 4][s % 4 / 2], s % 2, *reinterpret_cast<const v4u*>(unit + s / 4 * 4096 + wbase[s % 4]));
    };
    // The 8 products of halves HA and HW, each with what `with` issues before
    // it (LDS reads for the next phase, loads).
    auto multiply = [&](auto HA, auto HW, auto&& with) {
        constexpr int ha = decltype(HA)::value, hw = decltype(HW)::value;
        #pragma unroll
        for (int s = 0; s < 8; s++) {
            with(s);
            v16f& c = acc[2 * ha + s % 4 / 2][2 * hw + s % 2];
            c = mfma(fw[2 * hw + s % 2][s / 4], fa[2 * ha + s % 4 / 2][s / 4], c);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    constexpr std::integral_constant<int, 0> I0{};
    constexpr std::integral_constant<int, 1> I1{};
    // A barrier for which all but each wave's last LEFT loads into LDS have
    // arrived, and its LDS reads (the compiler's own waits cover a wave's own
    // loads only; __syncthreads would wait for all of them).
    auto arrive = [](auto LEFT) {
        constexpr int n = decltype(LEFT)::value;
        __builtin_amdgcn_sched_barrier(0);
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_waitcnt((n & 15) | (n >> 4) << 14 | 0x070);   // vmcnt(n), lgkmcnt(0)
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
    };
    constexpr std::integral_constant<int, 16> LEFT2{};   // the loads of two half steps
    constexpr std::integral_constant<int, 24> LEFT3{};
    // A step in two halves, on its units a0, a1, x, y (w's halves X and Y) and
    // the next step's a0n, yn; a's half 0 and w's half X are in registers.  Each
    // half reads two units and refills the two that the half before has read
    // with the step after the next (k2 of s2), so that a load has two to three
    // half steps to arrive in.  Leaves a's half 0 and w's half Y of the next step
    // in registers.
    auto step = [&](auto X, auto Y, uint8_t* a0, uint8_t* a1, uint8_t* x, uint8_t* y, uint8_t* a0n,
                    uint8_t* yn, const Src& s2, int k2) {
        constexpr int hx = decltype(X)::value, hy = decltype(Y)::value;
        arrive(LEFT2);
        multiply(I0, X, [&](int s) {
            read_w(hy, y, s);
            if (s % 2) fetch_a(s2, k2, 0, a0, s / 2);
        });
        multiply(I0, Y, [&](int s) {
            read_a(1, a1, s);
            if (s % 2) fetch_w(s2, k2, hx, x, s / 2);
        });
        arrive(LEFT2);
        multiply(I1, Y, [&](int s) {
            read_a(0, a0n, s);
            if (s % 2) fetch_w(s2, k2, hy, y, s / 2);
        });
        multiply(I1, X, [&](int s) {
            read_w(hy, yn, s);
            if (s % 2) fetch_a(s2, k2, 1, a1, s / 2);
        });
    };

    int i = 0;
    int t = map.at(0, blockIdx.x, gridDim.x);
    if (t < 0) return;
    cur = source(t);
    auto fetch = [&](auto&& load) {
        #pragma unroll
        for (int j = 0; j < 4; j++) load(j);
    };
    // in the order in which they are read
    fetch([&](int j) { fetch_a(cur, 0, 0, sa00, j); });
    fetch([&](int j) { fetch_w(cur, 0, 0, sw00, j); });
    fetch([&](int j) { fetch_w(cur, 0, 1, sw10, j); });
    fetch([&](int j) { fetch_a(cur, 0, 1, sa10, j); });
    fetch([&](int j) { fetch_a(cur, 1, 0, sa01, j); });
    fetch([&](int j) { fetch_w(cur, 1, 1, sw11, j); });
    fetch([&](int j) { fetch_w(cur, 1, 0, sw01, j); });
    fetch([&](int j) { fetch_a(cur, 1, 1, sa11, j); });
    arrive(LEFT3);
    while (true) {
        const int t_next = map.at(++i, blockIdx.x, gridDim.x);
        nxt = source(t_next);
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

        const bool vec = N % 8 == 0;
        #pragma unroll
        for (int f = 0; f < (GATED ? 2 : 4); f++) {
            // 16 consecutive outputs of each of 4 rows
            const int64_t col = cur.n0 + f / 2 * kHalf + wn * 64 + f % 2 * 32 + g * 16;
            float ws[16], bs[16], wu[16], bu[16];
            columns(e, 0, col, N, ws, bs);
            if (GATED) columns(e, N, col, N, wu, bu);
            #pragma unroll
            for (int i = 0; i < 4; i++) {
                const int64_t m = cur.m0 + wm * 128 + i * 32 + r;
                if (m >= M) break;
                const float sm = e.a_scale ? e.a_scale[m] : 1.0f;
                float v[16];
                #pragma unroll
                for (int c = 0; c < 16; c++) {
                    v[c] = activate<ACT>(acc[i][f][c] * sm * ws[c] + bs[c], e);
                    if (GATED) v[c] *= acc[i][2 + f % 2][c] * sm * wu[c] + bu[c];
                }
                const int64_t o = m * N + col;
                if (vec && col + 16 <= N) {
                    #pragma unroll
                    for (int b = 0; b < 2; b++) {
                        if (e.residual) {
                            const v4u u = *reinterpret_cast<const v4u*>(e.residual + o + 8 * b);
                            #pragma unroll
                            for (int c = 0; c < 4; c++) {
                                v[8 * b + 2 * c] += bf16_lo(u[c]);
                                v[8 * b + 2 * c + 1] += bf16_hi(u[c]);
                            }
                        }
                        v4u u;
                        #pragma unroll
                        for (int c = 0; c < 4; c++) u[c] = bf16_pack(v[8 * b + 2 * c], v[8 * b + 2 * c + 1]);
                        *reinterpret_cast<v4u*>(e.y + o + 8 * b) = u;
                    }
                } else {
                    #pragma unroll
                    for (int c = 0; c < 16; c++) {
                        if (col + c >= N) break;
                        if (e.residual) v[c] += bf16_lo(e.residual[o + c]);
                        e.y[o + c] = (uint16_t)bf16_pack(v[c], 0.0f);
                    }
                }
            }
        }
        if (t_next < 0) break;
        t = t_next;
        cur = nxt;
    }
}

// f(gated, activation form) with both as types
template <class F>
void for_kind(bool gated, int act, F&& f) {
    auto with = [&](auto G) {
        if (act == kErf) f(G, std::integral_constant<int, kErf>{});
        else if (act == kSigmoid) f(G, std::integral_constant<int, kSigmoid>{});
        else f(G, std::integral_constant<int, kClip>{});
    };
    if (gated) with(std::true_type{}); else with(std::false_type{});
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
    const float tanh_c1 = 2.0f * 0.79788456f * kLog2e;   // 2 sqrt(2 / pi)
    const bool tanh_form = activation == TANS_ACT_GELU_TANH;
    const Epilogue e = {a_scale, w_scale, (const uint16_t*)bias, (const uint16_t*)residual,
                        (uint16_t*)y, scale,
                        activation == TANS_ACT_RELU ? 0.0f : -INFINITY,
                        tanh_form ? tanh_c1 : kLog2e, tanh_form ? 0.044715f * tanh_c1 : 0.0f};
    const int act = activation == TANS_ACT_GELU ? kErf
                    : activation == TANS_ACT_SILU || tanh_form ? kSigmoid : kClip;
    if (M > 128) {
        const TileMap map = {(int)((M + kTile - 1) / kTile), (int)((N + (gated ? kHalf : kTile) - 1) / (gated ? kHalf : kTile))};
        const int64_t tiles = (int64_t)map.tiles_m * map.tiles_n;
        const int cus = tans_internal_cu_count();
        auto launch = [&](auto kernel) {
            hipLaunchKernelGGL(kernel, dim3((unsigned)std::min<int64_t>(tiles, cus)), dim3(256), 0,
                               (hipStream_t)stream, (const uint8_t*)a, (const uint8_t*)w, M, N, C, map, e);
        };
        for_kind(gated, act, [&](auto G, auto A) {
            launch(linear_tile_kernel<decltype(G)::value, decltype(A)::value>);
        });
        return hip_check(hipGetLastError(), "linear_tile_kernel launch");
    }
    const int64_t blocks = (N + 63) / 64 * ((M + 15) / 16);
    if (blocks > UINT32_MAX / 256) return fail(TANS_EINVAL, "linear: too many outputs for one call");
    const dim3 grid((unsigned)blocks);
    auto launch = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, grid, dim3(256), 0, (hipStream_t)stream, (const uint8_t*)a,
                           (const uint8_t*)w, M, N, C, e);
    };
    for_kind(gated, act, [&](auto G, auto A) {
        launch(linear_kernel<decltype(G)::value, decltype(A)::value>);
    });
    return hip_check(hipGetLastError(), "linear_kernel launch");
}

}  // extern "C"
