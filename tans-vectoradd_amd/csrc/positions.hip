// Rotary positions, alone and with the writing of keys and values into a paged cache
// (gfx950).  No counterpart in the reference.
//
//   a = position * frequency[i], for the pair i of a head
//   u' = magnitude (u cos a - v sin a), v' = magnitude (u sin a + v cos a)
//   (half layout: u = x[i], v = x[i + rot / 2]; interleaved: x[2 i], x[2 i + 1])
//
// and x'[d] = x[d] for d >= rot.
//
// An angle is a fraction of a turn in 64-bit fixed point: the frequency as a number
// of turns without its whole ones, times 2^64, times the position, modulo 2^64.  The
// product is exact, so a position of 2^20 or 2^30 has the error of the frequency's
// own last bit times the position and no more, where a product in 32 bits would be
// off by 2^-24 of the angle, some 0.06 radians at 2^20.  Sine and cosine come from
// Taylor polynomials on an eighth of a turn either way (the first terms left out are
// below 2^-28 of the value).  One rounding, to bf16; a row that goes to an 8-bit
// cache is rounded to 8 bits from 32, with a scale of its own.
#include <algorithm>

#include "cache.h"
#include "launch.h"

namespace {

struct Angle { float cos, sin; };

// cos and sin of f * position
__device__ __forceinline__ Angle angle_of(double f, int32_t position, float sign, float magnitude) {
    double turns = f * 0.15915494309189533577;   // 1 / (2 pi)
    turns = (turns - floor(turns)) * 4294967296.0;
    const uint32_t hi = (uint32_t)turns, lo = (uint32_t)((turns - (double)hi) * 4294967296.0);
    const uint32_t p = (uint32_t)position;
    uint32_t a = p * hi + __umulhi(p, lo);
    if (position < 0) a -= lo;   // (p is 2^32 more than the position)
    // a quarter turn's number and what is left, an eighth of a turn at most
    const uint32_t quarter = (a + 0x20000000u) >> 30;
    const float x = (float)(int32_t)(a - (quarter << 30)) * 1.4629180792671596e-9f;   // 2 pi / 2^32
    const float z = x * x;
    float s = __builtin_fmaf(z, 2.7557319e-6f, -1.9841270e-4f);
    s = __builtin_fmaf(z, s, 8.3333333e-3f);
    s = __builtin_fmaf(z, s, -1.6666667e-1f);
    s = __builtin_fmaf(z * s, x, x);
    float c = __builtin_fmaf(z, -2.7557319e-7f, 2.4801587e-5f);
    c = __builtin_fmaf(z, c, -1.3888889e-3f);
    c = __builtin_fmaf(z, c, 4.1666667e-2f);
    c = __builtin_fmaf(z, c, -0.5f);
    c = __builtin_fmaf(z, c, 1.0f);
    float cos = quarter & 1 ? s : c, sin = quarter & 1 ? c : s;
    if ((quarter + 1) & 2) cos = -cos;
    if (quarter & 2) sin = -sin;
    return {cos * magnitude, sin * sign * magnitude};
}

struct Rotation {
    const int32_t* positions;   // [N]
    const double* frequencies;  // [rot / 2]
    int rot, D;
    float magnitude, sign;      // sign: -1 for the inverse
};

// One head's 16 elements of a thread: chunk c of 16 of them, as two runs of 8.  Those
// of the rotated part hold whole pairs: half layout, the c-th 8 u's and their v's.
template <bool INTER>
struct Chunk {
    int at[2];
    bool turned;
    Angle a[kVec];
    __device__ __forceinline__ void set(const Rotation& r, int c, int token) {
        turned = c < r.rot / 16;
        at[0] = !INTER && turned ? 8 * c : 16 * c;
        at[1] = !INTER && turned ? r.rot / 2 + 8 * c : 16 * c + 8;
        if (turned) {
            const int32_t p = r.positions[token];
            #pragma unroll
            for (int i = 0; i < kVec; i++) a[i] = angle_of(r.frequencies[8 * c + i], p, r.sign, r.magnitude);
        }
    }
    __device__ __forceinline__ void turn(float (&u)[kVec], float (&v)[kVec]) const {
        if (!turned) return;
        #pragma unroll
        for (int i = 0; i < kVec; i++) {
            float& x = INTER ? (i < 4 ? u[2 * i] : v[2 * i - 8]) : u[i];
            float& y = INTER ? (i < 4 ? u[2 * i + 1] : v[2 * i - 7]) : v[i];
            const float t = x * a[i].cos - y * a[i].sin;
            y = x * a[i].sin + y * a[i].cos;
            x = t;
        }
    }
};

__device__ __forceinline__ v4u pack8(const float (&f)[kVec]) {
    return v4u{bf16_pack(f[0], f[1]), bf16_pack(f[2], f[3]), bf16_pack(f[4], f[5]), bf16_pack(f[6], f[7])};
}

// Threads: `waves` waves share a token, each thread has one chunk of every `step`-th
// head, so that its angles are computed once for all of them.
struct Share {
    int token, head, chunk, step;
    __device__ __forceinline__ bool set(int waves, int chunks, int N) {
        const int team = waves * kLanes, t = threadIdx.x % team;
        token = (int)blockIdx.x * ((int)blockDim.x / team) + threadIdx.x / team;
        step = team / chunks;
        head = t / chunks;
        chunk = t % chunks;
        return token < N && head < step;
    }
};

constexpr int kThreads = 256;
constexpr int kAhead = 4;   // heads whose loads are under way at a time

// Memory bounds it: 8192 tokens of 48 heads of 128 read and written once, 201 MB, in 41 us
// (4.9 TB/s, a large copy's rate); the sines of a token are computed once for all its
// heads.  One token takes 2.9 us, a launch and two dependent loads.

template <bool INTER>
__global__ __launch_bounds__(kThreads) void rotary_kernel(const uint16_t* x, int64_t x_stride, Rotation r,
                                                          int N, int H, int waves, uint16_t* out,
                                                          int64_t out_stride) {
    Share s;
    if (!s.set(waves, r.D / 16, N)) return;
    Chunk<INTER> c;
    c.set(r, s.chunk, s.token);
    const uint16_t* from = x + s.token * x_stride;
    uint16_t* to = out + s.token * out_stride;
    for (int h0 = s.head; h0 < H; h0 += kAhead * s.step) {
        v4u in[kAhead][2];
        #pragma unroll
        for (int i = 0; i < kAhead; i++) {
            const int h = h0 + i * s.step < H ? h0 + i * s.step : h0;
            #pragma unroll
            for (int j = 0; j < 2; j++) in[i][j] = *reinterpret_cast<const v4u*>(from + h * r.D + c.at[j]);
        }
        #pragma unroll
        for (int i = 0; i < kAhead; i++) {
            const int h = h0 + i * s.step;
            if (h >= H) break;
            float u[kVec], v[kVec];
            unpack(in[i][0], u);
            unpack(in[i][1], v);
            c.turn(u, v);
            *reinterpret_cast<v4u*>(to + h * r.D + c.at[0]) = pack8(u);
            *reinterpret_cast<v4u*>(to + h * r.D + c.at[1]) = pack8(v);
        }
    }
}

struct Rows { const uint16_t* p; int64_t stride; };
struct Caches { void *k, *v; float *k_scale, *v_scale; };

// The q heads, then k's, then v's as one sequence of heads.  4 x 2048 tokens of 40 + 8 + 8
// heads of 128 into an 8-bit cache, 151 MB, take 34 us (4.5 TB/s); 61 trees of 7 to 25
// tokens 7 us, of which the search for the token's sequence and its slot's page are three
// dependent loads.
template <bool INTER, bool FP8>
__global__ __launch_bounds__(kThreads) void append_kernel(Rows q, Rows k, Rows v, Rotation r, Batch batch,
                                                          Caches cache, int Hq, int waves,
                                                          uint16_t* q_out) {
    Share s;
    if (!s.set(waves, r.D / 16, batch.N)) return;   // (whole waves: D / 16 divides 64)
    const int b = find_sequence(batch, s.token);
    if (!batch.owns(b, s.token)) return;
    Chunk<INTER> c;
    c.set(r, s.chunk, s.token);
    uint32_t slot;
    const bool fits = batch.slot_of(b, s.token, slot);
    const int Hkv = (int)batch.heads, H = Hq + 2 * Hkv;
    auto place = [&](int h) {
        return h < Hq ? q.p + s.token * q.stride + h * r.D
               : h < Hq + Hkv ? k.p + s.token * k.stride + (h - Hq) * r.D
                              : v.p + s.token * v.stride + (h - Hq - Hkv) * r.D;
    };
    for (int h0 = s.head; h0 < H; h0 += kAhead * s.step) {
        v4u in[kAhead][2];
        #pragma unroll
        for (int i = 0; i < kAhead; i++) {
            const uint16_t* from = place(h0 + i * s.step < H ? h0 + i * s.step : h0);
            #pragma unroll
            for (int j = 0; j < 2; j++) in[i][j] = *reinterpret_cast<const v4u*>(from + c.at[j]);
        }
        #pragma unroll
        for (int i = 0; i < kAhead; i++) {
            const int h = h0 + i * s.step;
            float x[2][kVec];
            unpack(in[i][0], x[0]);
            unpack(in[i][1], x[1]);
            if (h < Hq + Hkv) c.turn(x[0], x[1]);
            float scale = 1.0f, inv = 1.0f;
            if (FP8) {   // (a head's lanes are neighbours, of which all or none have a head)
                float top = amax8(x[1], amax8(x[0], __builtin_bit_cast(float, kAmaxMinBits)));
                top = dpp_join<Max, 0xB1>(top);    // lane ^ 1
                top = dpp_join<Max, 0x4E>(top);    // lane ^ 2
                if (r.D >= 128) top = dpp_join<Max, 0x141>(top);   // mirrored in halves of 16
                if (r.D >= 256) top = dpp_join<Max, 0x140>(top);   // mirrored in 16
                scale = top / kFp8Max;
                inv = 1.0f / scale;
            }
            if (h >= H) continue;
            if (h < Hq) {
                uint16_t* to = q_out + ((int64_t)s.token * Hq + h) * r.D;
                *reinterpret_cast<v4u*>(to + c.at[0]) = pack8(x[0]);
                *reinterpret_cast<v4u*>(to + c.at[1]) = pack8(x[1]);
                continue;
            }
            const bool key = h < Hq + Hkv;
            uint32_t row;
            if (!fits || !batch.row(b, slot, (uint32_t)(h - Hq - (key ? 0 : Hkv)), row)) continue;
            void* to = key ? cache.k : cache.v;
            if constexpr (FP8) {
                uint8_t* p = (uint8_t*)to + (int64_t)row * r.D;
                *reinterpret_cast<v2u*>(p + c.at[0]) = to_fp8(x[0], scale, inv);
                *reinterpret_cast<v2u*>(p + c.at[1]) = to_fp8(x[1], scale, inv);
                if (s.chunk == 0) (key ? cache.k_scale : cache.v_scale)[row] = scale;
            } else {
                uint16_t* p = (uint16_t*)to + (int64_t)row * r.D;
                *reinterpret_cast<v4u*>(p + c.at[0]) = pack8(x[0]);
                *reinterpret_cast<v4u*>(p + c.at[1]) = pack8(x[1]);
            }
        }
    }
}

constexpr int kMaxDim = 1024;   // a head's chunks are at most a wave's lanes

int rotation_check(const std::string& op, const void* positions, const void* frequencies, int64_t rot,
                   int64_t D) {
    if (rot < 16 || rot % 16 || rot > D)
        return fail(TANS_EINVAL, op + ": the rotated part must be a multiple of 16, 16 .. D");
    if (!positions || !frequencies) return fail(TANS_EINVAL, op + ": null pointer");
    if (!aligned(positions, 4) || !aligned(frequencies, 8))
        return fail(TANS_EINVAL, op + ": misaligned buffer (positions 4, frequencies 8 bytes)");
    return TANS_OK;
}

// Waves that share a token: one, or as many as bring the heads into one round while
// that leaves CUs without a workgroup.
int token_waves(int64_t N, int64_t tasks, int cus) {
    int waves = 1;
    while (waves < kThreads / kLanes && N * waves < 4 * (int64_t)cus && tasks > waves * kLanes) waves *= 2;
    return waves;
}

}  // namespace

extern "C" {

int tans_rotary(const void* x, int64_t x_stride, const int32_t* positions, const double* frequencies,
                int64_t N, int64_t H, int64_t D, int64_t rot, int32_t interleaved, int32_t inverse,
                float magnitude, void* out, int64_t out_stride, void* stream) {
    const std::string op = "rotary";
    if (N < 0 || N > INT32_MAX / 2) return fail(TANS_EINVAL, op + ": N must be 0 .. 2^30 - 1");
    if (H < 1 || H > 65535) return fail(TANS_EINVAL, op + ": H must be 1 .. 65535");
    if (D < 16 || D % 16 || D > kMaxDim)
        return fail(TANS_EINVAL, op + ": D must be a multiple of 16, 16 .. 1024");
    if (N == 0) return TANS_OK;
    if (!x || !out) return fail(TANS_EINVAL, op + ": null pointer");
    int rc = rotation_check(op, positions, frequencies, rot, D);
    if (rc == TANS_OK) rc = stride_check(op, "x", x, x_stride, H * D);
    if (rc == TANS_OK) rc = stride_check(op, "out", out, out_stride, H * D);
    if (rc != TANS_OK) return rc;
    const int waves = token_waves(N, H * (D / 16), tans_internal_cu_count());
    const int tokens = kThreads / kLanes / waves;   // of a workgroup
    const Rotation r = {positions, frequencies, (int)rot, (int)D, magnitude, inverse ? -1.0f : 1.0f};
    auto launch = [&](auto kernel) {
        // (a launch has fewer than 2^32 threads: 2^23 workgroups at a time)
        for (int64_t n = 0; n < N; n += (int64_t(1) << 23) * tokens) {
            const int64_t some = std::min<int64_t>(N - n, (int64_t(1) << 23) * tokens);
            Rotation rn = r;
            rn.positions += n;
            hipLaunchKernelGGL(kernel, dim3((unsigned)((some + tokens - 1) / tokens)), dim3(kThreads), 0,
                               (hipStream_t)stream, (const uint16_t*)x + n * x_stride, x_stride, rn,
                               (int)some, (int)H, waves, (uint16_t*)out + n * out_stride, out_stride);
        }
        return hip_check(hipGetLastError(), "rotary_kernel launch");
    };
    return interleaved ? launch(rotary_kernel<true>) : launch(rotary_kernel<false>);
}

int tans_rotary_append(const void* q, int64_t q_stride, const void* k, int64_t k_stride, const void* v,
                       int64_t v_stride, const int32_t* positions, const double* frequencies,
                       int64_t rot, int32_t interleaved, float magnitude, void* k_cache, void* v_cache,
                       float* k_scale, float* v_scale, int64_t pages, int64_t heads, int64_t page,
                       int64_t dim, const int32_t* table, int64_t per, const int32_t* starts,
                       const int32_t* lens, int64_t B, int64_t N, int64_t q_heads, void* q_out,
                       void* stream) {
    const std::string op = "rotary_append";
    int rc = batch_check(op, k_cache, v_cache, k_scale, v_scale, pages, heads, page, dim, table, per,
                         starts, lens, B, N, q_heads);
    if (rc != TANS_OK || N == 0 || B == 0) return rc;
    if (!q || !k || !v || !q_out) return fail(TANS_EINVAL, op + ": null pointer");
    rc = rotation_check(op, positions, frequencies, rot, dim);
    if (rc == TANS_OK) rc = stride_check(op, "q", q, q_stride, q_heads * dim);
    if (rc == TANS_OK) rc = stride_check(op, "k", k, k_stride, heads * dim);
    if (rc == TANS_OK) rc = stride_check(op, "v", v, v_stride, heads * dim);
    if (rc == TANS_OK && !aligned(q_out, 16)) rc = fail(TANS_EINVAL, op + ": q_out is misaligned (16 bytes)");
    if (rc != TANS_OK) return rc;
    const int waves = token_waves(N, (q_heads + 2 * heads) * (dim / 16), tans_internal_cu_count());
    const int tokens = kThreads / kLanes / waves;
    if ((N + tokens - 1) / tokens > (1 << 23)) return fail(TANS_EINVAL, op + ": too many tokens for one call");
    const Rotation r = {positions, frequencies, (int)rot, (int)dim, magnitude, 1.0f};
    const Batch batch = make_batch(table, starts, lens, B, per, N, pages, heads, page);
    auto launch = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, dim3((unsigned)((N + tokens - 1) / tokens)), dim3(kThreads), 0,
                           (hipStream_t)stream, Rows{(const uint16_t*)q, q_stride},
                           Rows{(const uint16_t*)k, k_stride}, Rows{(const uint16_t*)v, v_stride}, r, batch,
                           Caches{k_cache, v_cache, k_scale, v_scale}, (int)q_heads, waves, (uint16_t*)q_out);
        return hip_check(hipGetLastError(), "append_kernel launch");
    };
    if (k_scale) return interleaved ? launch(append_kernel<true, true>) : launch(append_kernel<false, true>);
    return interleaved ? launch(append_kernel<true, false>) : launch(append_kernel<false, false>);
}

}  // extern "C"
