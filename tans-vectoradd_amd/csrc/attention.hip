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

#include <algorithm>

#include "attention_plan.h"
#include "cache.h"
#include "launch.h"

namespace {

using namespace tans_attention;

typedef int v2i __attribute__((ext_vector_type(2)));
typedef short v4s __attribute__((ext_vector_type(4)));
typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef float v16f __attribute__((ext_vector_type(16)));

constexpr float kLog2e = 1.44269504f;
constexpr float kNone = -INFINITY;   // the maximum of nothing

struct Args {
    Batch batch;
    const uint16_t* q;
    int64_t q_stride;
    const uint8_t *k, *v;
    const float *k_scale, *v_scale;
    const uint8_t* mask;   // [N][W] or null
    int W, Hq, G;          // G: query heads of a cache head
    float c;               // scale / ln 2
    uint16_t* out;
    Work work;
    float* parts;          // of split items: [workgroups][2][rows][D], then [workgroups][2][rows][2]
};

// A sequence's part in the work: its row tiles and the slots' units.
struct Seq {
    int start, tokens, context, slots;   // slots: the context's and the new tokens'
    int tiles, units;
};

__device__ __forceinline__ Seq sequence(const Args& a, int b) {
    Seq s;
    s.start = a.batch.start(b);
    s.tokens = a.batch.tokens(b);
    s.context = a.batch.context(b);
    const int64_t all = (int64_t)s.context + s.tokens;
    s.slots = (int)(all < a.batch.capacity() ? all : a.batch.capacity());
    s.tiles = row_tiles(s.tokens, a.G, a.work.rows);
    s.units = slot_units(s.slots);
    return s;
}

__device__ __forceinline__ int64_t cost(const Args& a, int b) {
    if (b >= a.batch.B) return 0;
    const Seq s = sequence(a, b);
    return (int64_t)a.batch.heads * s.tiles * (a.work.whole ? 1 : s.units + a.work.item);
}

__device__ __forceinline__ int64_t uniform(int64_t v) {
    return (int64_t)((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)v) |
                     (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(v >> 32)) << 32);
}

// The work of all sequences, and that of those before b.
__device__ __forceinline__ void total_cost(const Args& a, int b, int64_t& all, int64_t& before) {
    const int lane = threadIdx.x & (kLanes - 1);
    all = before = 0;
    if (a.batch.B == 1) {
        all = uniform(cost(a, 0));
        return;
    }
    for (int i = lane; i < a.batch.B; i += kLanes) {
        const int64_t c = cost(a, i);
        all += c;
        before += i < b ? c : 0;
    }
    #pragma unroll
    for (int i = 1; i < kLanes; i *= 2) {
        all += __shfl_xor(all, i);
        before += __shfl_xor(before, i);
    }
    all = uniform(all);
    before = uniform(before);
}

// The sequence that piece `at` < all of the work belongs to; at becomes the piece's
// number within it.
__device__ __forceinline__ int find_piece(const Args& a, int64_t& at) {
    if (a.batch.B == 1) return 0;
    const int lane = threadIdx.x & (kLanes - 1);
    int64_t before = 0;
    for (int first = 0; first < a.batch.B; first += kLanes) {
        const int64_t mine = cost(a, first + lane);
        int64_t sum = mine;
        #pragma unroll
        for (int i = 1; i < kLanes; i *= 2) {
            const int64_t other = __shfl_up(sum, i);
            if (lane >= i) sum += other;
        }
        const uint64_t past = __builtin_amdgcn_ballot_w64(before + sum > at);
        if (past) {
            const int l = __ffsll((unsigned long long)past) - 1;
            at = uniform(at - before - __shfl(sum - mine, l));
            return first + l;
        }
        before += __shfl(sum, kLanes - 1);
    }
    return a.batch.B - 1;   // (not reached)
}

// 16 or 4 bytes a lane from memory to LDS, lane l's to lds + 16 l or 4 l.
template <int BYTES>
__device__ __forceinline__ void load_lds(const void* from, uint8_t* to) {
    const auto* p = (const __attribute__((address_space(1))) void*)from;
    auto* lds = (__attribute__((address_space(3))) void*)to;
    if constexpr (BYTES == 16) __builtin_amdgcn_global_load_lds(p, lds, 16, 0, 0);
    else __builtin_amdgcn_global_load_lds(p, lds, 4, 0, 0);
}

// Waits until at most N of the wave's loads are under way.
template <int N>
__device__ __forceinline__ void wait_loads() {
    static_assert(N < 64, "a 6-bit counter");
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt((N & 15) | (N >> 4) << 14 | 0xF70);
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
}

// A barrier for which all but each wave's last N loads into LDS have arrived, and its
// LDS reads.
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

__device__ __forceinline__ uint32_t opaque_v(uint32_t x) {
    asm volatile("" : "+v"(x));
    return x;
}

// A lane's value and that of lane ^ 32, in one order for both: the swap of a register
// with itself.  Read through a 64-bit cast: as a vector of floats that are cast back to
// numbers the compiler has lost one of them.
__device__ __forceinline__ uint64_t halves(uint32_t u) {
    return __builtin_bit_cast(uint64_t, __builtin_amdgcn_permlane32_swap(u, u, false, false));
}
__device__ __forceinline__ uint32_t all_bits(uint32_t u) {
    const uint64_t p = halves(u);
    return (uint32_t)p | (uint32_t)(p >> 32);
}
__device__ __forceinline__ float larger(float v) {
    const uint64_t p = halves(__builtin_bit_cast(uint32_t, v));
    return fmaxf(__builtin_bit_cast(float, (uint32_t)p), __builtin_bit_cast(float, (uint32_t)(p >> 32)));
}
__device__ __forceinline__ float sum_of(float v) {
    const uint64_t p = halves(__builtin_bit_cast(uint32_t, v));
    return __builtin_bit_cast(float, (uint32_t)p) + __builtin_bit_cast(float, (uint32_t)(p >> 32));
}

__device__ __forceinline__ v16f mfma(const v8bf& a, const v8bf& b, const v16f& c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}

// 8 E4M3FN bytes as bf16, which holds them exactly
__device__ __forceinline__ v8bf from_fp8(uint32_t lo, uint32_t hi) {
    const v4u u = {__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, false)),
                   __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, true)),
                   __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, false)),
                   __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, true))};
    return __builtin_bit_cast(v8bf, u);
}

// Infinities and NaN among the values of a 32-bit word: join() gathers words, any() says
// whether one of them held any, drop() puts zero in their place.
template <bool FP8> struct Odd;
template <> struct Odd<false> {
    typedef uint16_t v2h __attribute__((ext_vector_type(2)));
    static __device__ __forceinline__ uint32_t join(uint32_t most, uint32_t x) {
        return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(v2h, most),
                                                                      __builtin_bit_cast(v2h, x & 0x7FFF7FFFu)));
    }
    static __device__ __forceinline__ bool any(uint32_t most) {
        return (most & 0xFFFFu) >= 0x7F80u || most >= 0x7F800000u;
    }
    static __device__ __forceinline__ uint32_t drop(uint32_t x) {
        return x & (((x & 0x7F80u) == 0x7F80u ? 0u : 0xFFFFu) | ((x & 0x7F800000u) == 0x7F800000u ? 0u : 0xFFFF0000u));
    }
};
template <> struct Odd<true> {   // (the bytes 7F and FF are NaN: 7F + 1 has the top bit)
    static __device__ __forceinline__ uint32_t join(uint32_t most, uint32_t x) {
        return most | ((x & 0x7F7F7F7Fu) + 0x01010101u);
    }
    static __device__ __forceinline__ bool any(uint32_t most) { return most & 0x80808080u; }
    static __device__ __forceinline__ uint32_t drop(uint32_t x) {
        const uint32_t top = ((x & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u;
        return x & ~(top | (top - (top >> 7)));
    }
};

// The n lowest bits, all of them or none.
__device__ __forceinline__ uint32_t first_bits(int n) {
    return n <= 0 ? 0u : n >= 32 ? 0xFFFFFFFFu : (1u << n) - 1;
}

// Where a unit's rows lie in LDS: 32 rows of RB bytes, whose 16-byte pieces are
// permuted by an exclusive or with a key of the row so that the reads touch all banks.
template <int D, bool FP8>
struct Tile {
    static constexpr int RB = FP8 ? D : 2 * D;
    static constexpr int pieces = RB / 16, bytes = kUnit * RB;
    static constexpr int loads = bytes / 1024;         // of 64 lanes and 16 bytes
    static constexpr int per_load = 1024 / RB;         // rows
    static __device__ __forceinline__ uint32_t key_of_k(uint32_t row) {
        return RB == 64 ? (row >> 1) & 3 : row & 7;
    }
    static __device__ __forceinline__ uint32_t key_of_v(uint32_t row) {
        return !FP8 ? 2 * (row & 3)
               : RB == 64 ? ((row >> 1) & 1) | ((row >> 3) & 1) << 1 : (row & 3) | ((row >> 3) & 1) << 2;
    }
};

// 32 slots at a time.  S^T = K Q^T by 32 x 32 x 16 products: lane (g, r), lane 32 g +
// r, gets query row r's scores with the slots 8 i + 4 g + c (i, c = 0 .. 3), so that a
// row's maximum and sum are one lane's and its other half's.  Those 16 are, rounded to
// bf16, the operand of O^T = V^T P^T as they lie there, if the slots are taken in that
// order; V's operand, 8 slots of one dimension, comes from LDS by transposing reads.
template <int D, bool FP8, int RT, bool SHARED, int NW, int STAGES>
__global__ __launch_bounds__(NW * kLanes, 1) void attend_kernel(Args a) {
    using T = Tile<D, FP8>;
    constexpr int kRows = 32 * RT * (SHARED ? NW : 1);
    constexpr int kShare = SHARED ? NW : 1;               // waves that share a tile
    constexpr int kLoads = 2 * T::loads / kShare;         // of a wave and unit
    static_assert(2 * T::loads % kShare == 0, "loads");
    constexpr int kIssue = kLoads + (FP8 ? 1 : 0);        // with the scales'
    constexpr int kScales = FP8 ? 256 : 0;
    constexpr int kStage = 2 * T::bytes + kScales * (SHARED ? NW : 1);
    constexpr int kRing = kStage * (SHARED ? 1 : NW);
    __shared__ __attribute__((aligned(1024))) uint8_t ring0[kRing], ring1[kRing],
        ring2[STAGES > 2 ? kRing : 16], ring3[STAGES > 3 ? kRing : 16];
    __shared__ float stat[SHARED ? 1 : NW][kRows][2];
    const int lane = threadIdx.x & (kLanes - 1);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kLanes);
    const int r = lane & 31, g = lane >> 5;

    int64_t all, none;
    total_cost(a, 0, all, none);
    const int groups = a.work.whole ? 0 : work_groups(a.work, all);
    if (a.work.whole ? (int64_t)blockIdx.x >= all : (int)blockIdx.x >= groups) return;
    int64_t at = a.work.whole ? (int64_t)blockIdx.x : range_start(all, groups, blockIdx.x);
    int64_t left = a.work.whole ? 1 : range_start(all, groups, blockIdx.x + 1) - at;
    int64_t in = at;   // the piece's number in its sequence
    int b = find_piece(a, in);
    Seq s = sequence(a, b);

    // addresses in a stage, of K's and V's operands
    const uint32_t mine = SHARED ? 0 : wave * kStage;
    uint32_t kbase[4], vbase[4];
    #pragma unroll
    for (int i = 0; i < 4; i++) {
        kbase[i] = opaque_v(mine + r * T::RB + (((2 * i + g) ^ T::key_of_k(r)) % T::pieces) * 16);
        const int l = lane & 15, half = (lane >> 4) & 1;
        if constexpr (FP8) {
            const uint32_t row = l / 2 < 4 ? 4 * g + l / 2 : 4 + 4 * g + l / 2;
            vbase[i] = opaque_v(mine + T::bytes + row * T::RB +
                                (((2 * i + half) ^ T::key_of_v(row)) % T::pieces) * 16 + l % 2 * 8);
        } else {
            const uint32_t row = 4 * g + l / 4;
            vbase[i] = opaque_v(mine + T::bytes + row * T::RB +
                                (((4 * (i & 1) + 2 * half + l % 4 / 2) ^ T::key_of_v(row)) % T::pieces) * 16 +
                                l % 2 * 8);
        }
    }
    // pieces of a row that the keys permute: 8, or 4
    constexpr int kTurn = T::pieces < 8 ? 4 : 8;

    while (left > 0) {
        // the item: row tile `tile` of cache head h, units first .. end - 1 of it
        int h, tile, first, end;
        bool is_whole;
        bool cut;    // it began in another workgroup's run
        if (a.work.whole) {
            h = (int)(in % a.batch.heads);
            tile = s.tiles - 1 - (int)(in / a.batch.heads);
            first = 0;
            end = s.units;
            is_whole = true;
            cut = false;
            left = 0;
        } else {
            const int pieces = s.units + a.work.item;
            const int64_t item = in / pieces;
            const int from = (int)(in - item * pieces);
            h = (int)(item / s.tiles);
            tile = (int)(item - (int64_t)h * s.tiles);
            const int to = (int)(from + left < pieces ? from + left : pieces);
            first = max(0, from - a.work.item);
            end = to - a.work.item;   // (none of its units if not above first)
            is_whole = first == 0 && end == s.units;
            cut = first > 0;
            left -= to - from;
            in += to - from;
        }
        if (end > first) {
        const int rows = s.tokens * a.G, row0 = tile * kRows + (SHARED ? wave * 32 * RT : 0);
        // without a mask no row of the tile sees a slot past its last token's
        int seen = s.units;
        if (!a.mask) {
            const int last = min(s.tokens - 1, (tile * kRows + kRows - 1) / a.G);
            seen = slot_units((int)min((int64_t)s.slots, (int64_t)s.context + last + 1));
        }
        const int stop = end < seen ? end : seen;

        v8bf q[RT][D / 16];
        int token[RT];
        #pragma unroll
        for (int t = 0; t < RT; t++) {
            const int row = row0 + 32 * t + r;
            token[t] = row < rows ? row / a.G : -1;
            const uint16_t* p = a.q + (int64_t)(s.start + token[t]) * a.q_stride +
                                (int64_t)(h * a.G + row % a.G) * D;
            #pragma unroll
            for (int j = 0; j < D / 16; j++) {
                v4u u = {0, 0, 0, 0};
                if (row < rows)
                    u = *reinterpret_cast<const v4u*>(p + (FP8 ? j / 2 * 32 + 16 * g + j % 2 * 8 : 16 * j + 8 * g));
                q[t][j] = __builtin_bit_cast(v8bf, u);
            }
        }
        v16f acc[RT][D / 32];
        float m[RT], l[RT];
        auto clear = [&]() {
            #pragma unroll
            for (int t = 0; t < RT; t++) {
                m[t] = kNone;
                l[t] = 0.0f;
                #pragma unroll
                for (int n = 0; n < D / 32; n++)
                    #pragma unroll
                    for (int c = 0; c < 16; c++) acc[t][n][c] = 0.0f;
            }
        };
        clear();

        // The rows of unit u: looked up in the table two units before they are loaded.
        struct Lookup { uint32_t entry, off; bool in; };
        auto look_up = [&](int u) {
            const uint32_t slot = (uint32_t)u * kUnit + r;
            Lookup o;
            o.in = u < stop && slot < (uint32_t)s.slots;
            const uint32_t i = o.in ? slot / a.batch.page : 0;
            o.off = slot - i * a.batch.page;
            o.entry = s.slots > 0 ? (uint32_t)a.batch.table[(int64_t)b * a.batch.per + i] : 0;
            return o;
        };
        // loads unit's rows (of nothing: row 0's, which no lane sees); the slots that exist
        auto issue = [&](const Lookup& o, uint8_t* stage) {
            const bool valid = o.in && o.entry < a.batch.pages;
            const uint32_t row = valid ? (o.entry * a.batch.heads + h) * a.batch.page + o.off : 0;
            const uint32_t exists = (uint32_t)__builtin_amdgcn_ballot_w64(valid);
            // K's loads, then V's; the rows that a lane loads come from their lanes
            auto of = [&](int i) { return (SHARED ? (wave * kLoads + i) % T::loads : i) * T::per_load + lane / T::pieces; };
            constexpr int kDistinct = SHARED ? kLoads : T::loads;
            uint32_t from[kDistinct];
            #pragma unroll
            for (int i = 0; i < kDistinct; i++) from[i] = __shfl(row, of(i));
            #pragma unroll
            for (int i = 0; i < kLoads; i++) {
                const int n = SHARED ? wave * kLoads + i : i;
                const bool is_v = n >= T::loads;
                const uint32_t at = of(i % kDistinct), key = is_v ? T::key_of_v(at) : T::key_of_k(at);
                load_lds<16>((is_v ? a.v : a.k) + (int64_t)from[i % kDistinct] * T::RB + ((lane % T::pieces) ^ key) * 16,
                             stage + mine + n * 1024);
            }
            if constexpr (FP8)
                load_lds<4>((g ? a.v_scale : a.k_scale) + row,
                            stage + mine + 2 * T::bytes + (SHARED ? wave * kScales : 0));
            return exists;
        };

        auto compute = [&](auto MASKED, int u, uint32_t exists, const uint8_t* stage) {
            constexpr bool masked = decltype(MASKED)::value;
            v16f sc[RT];
            #pragma unroll
            for (int t = 0; t < RT; t++)
                #pragma unroll
                for (int c = 0; c < 16; c++) sc[t][c] = 0.0f;
            constexpr int kStep = FP8 ? 2 : 1;   // products of a read
            constexpr int kReads = D / 16 / kStep;
            v4u kr[kReads];
            #pragma unroll
            for (int j = 0; j < kReads; j++)
                kr[j] = *reinterpret_cast<const v4u*>(stage + kbase[j % (kTurn / 2)] + j / (kTurn / 2) * (16 * kTurn));
            __builtin_amdgcn_sched_barrier(0);
            #pragma unroll
            for (int j = 0; j < kReads; j++) {
                #pragma unroll
                for (int e = 0; e < kStep; e++) {
                    const v8bf kf = FP8 ? from_fp8(kr[j][2 * e], kr[j][2 * e + 1]) : __builtin_bit_cast(v8bf, kr[j]);
                    #pragma unroll
                    for (int t = 0; t < RT; t++) sc[t] = mfma(kf, q[t][kStep * j + e], sc[t]);
                }
            }
            // V's operands, under way during the exponentials
            v2u vr[D / 32][2][FP8 ? 1 : 2];
            #pragma unroll
            for (int n = 0; n < D / 32; n++)
                #pragma unroll
                for (int k = 0; k < 2; k++) {
                    if constexpr (FP8) {
                        typedef __attribute__((address_space(3))) v2i* P;
                        vr[n][k][0] = __builtin_bit_cast(v2u, __builtin_amdgcn_ds_read_tr8_b64_v2i32(
                            (P)(stage + vbase[n % (kTurn / 2)] + n / (kTurn / 2) * (16 * kTurn) + k * 16 * T::RB)));
                    } else {
                        typedef __attribute__((address_space(3))) v4s* P;
                        const uint8_t* from = stage + vbase[n % 2] + n / 2 * 128 + k * 16 * T::RB;
                        vr[n][k][0] = __builtin_bit_cast(v2u, __builtin_amdgcn_ds_read_tr16_b64_v4i16((P)from));
                        vr[n][k][1] = __builtin_bit_cast(v2u, __builtin_amdgcn_ds_read_tr16_b64_v4i16((P)(from + 8 * T::RB)));
                    }
                }
            __builtin_amdgcn_sched_barrier(0);
            float vs[FP8 ? 16 : 1];
            if constexpr (FP8) {
                const uint8_t* scales = stage + mine + 2 * T::bytes + (SHARED ? wave * kScales : 0);
                #pragma unroll
                for (int i = 0; i < 4; i++) {
                    const v4f ks = *reinterpret_cast<const v4f*>(scales + (8 * i + 4 * g) * 4);
                    const v4f vi = *reinterpret_cast<const v4f*>(scales + 128 + (8 * i + 4 * g) * 4);
                    #pragma unroll
                    for (int c = 0; c < 4; c++) {
                        vs[4 * i + c] = vi[c];
                        #pragma unroll
                        for (int t = 0; t < RT; t++) sc[t][4 * i + c] *= ks[c];
                    }
                }
            }
            uint32_t sees[RT];   // the unit's slots that a row sees
            if constexpr (masked) {
                const int before = s.context - u * kUnit;   // slots of the context
                #pragma unroll
                for (int t = 0; t < RT; t++) {
                    sees[t] = first_bits(a.mask ? before : before + token[t] + 1);
                    if (a.mask && before < kUnit) {
                        // (a row's first column where the tile has none of its own)
                        const uint8_t* row = a.mask + (int64_t)(s.start + max(token[t], 0)) * a.W;
                        uint32_t bits = 0;
                        #pragma unroll
                        for (int i = 0; i < 16; i++) {
                            const int key = i / 4 * 8 + 4 * g + i % 4, j = key - before;
                            const uint32_t bit = row[j < 0 ? 0 : j < a.W ? j : a.W - 1];
                            bits |= (j >= 0 && j < a.W ? bit : 0) << key;
                        }
                        sees[t] |= all_bits(bits);
                    }
                    sees[t] = token[t] >= 0 ? sees[t] & exists : 0;
                    const uint32_t mine = sees[t] >> 4 * g;
                    #pragma unroll
                    for (int i = 0; i < 16; i++)
                        if (!(mine >> (i / 4 * 8 + i % 4) & 1)) sc[t][i] = kNone;
                }
            }
            v8bf p[RT][2];
            #pragma unroll
            for (int t = 0; t < RT; t++) {
                float top = sc[t][0];
                #pragma unroll
                for (int i = 1; i < 16; i++) top = fmaxf(top, sc[t][i]);
                top = larger(top);
                if (__builtin_amdgcn_ballot_w64(top > m[t])) {
                    const float next = fmaxf(m[t], top);
                    const float by = next == kNone ? 0.0f : __builtin_amdgcn_exp2f((m[t] - next) * a.c);
                    m[t] = next;
                    l[t] *= by;
                    #pragma unroll
                    for (int n = 0; n < D / 32; n++)
                        #pragma unroll
                        for (int c = 0; c < 16; c++) acc[t][n][c] *= by;
                }
                const float mc = m[t] == kNone ? 0.0f : m[t] * a.c;
                float e[16];
                #pragma unroll
                for (int i = 0; i < 16; i++) {
                    e[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[t][i], a.c, -mc));
                    l[t] += e[i];
                    // (what is not seen may have any scale)
                    if constexpr (FP8) e[i] = masked && e[i] == 0.0f ? 0.0f : e[i] * vs[i];
                }
                #pragma unroll
                for (int k = 0; k < 2; k++)
                    p[t][k] = __builtin_bit_cast(v8bf, v4u{bf16_pack(e[8 * k], e[8 * k + 1]),
                                                          bf16_pack(e[8 * k + 2], e[8 * k + 3]),
                                                          bf16_pack(e[8 * k + 4], e[8 * k + 5]),
                                                          bf16_pack(e[8 * k + 6], e[8 * k + 7])});
            }
            // A value that is infinite or NaN reaches the rows that see its slot, and by the
            // matrix product it would reach the others as well (0 times it is NaN): it is
            // left out there, and added below.
            uint64_t odd = 0;
            if constexpr (masked) {
                uint32_t most = 0;
                #pragma unroll
                for (int n = 0; n < D / 32; n++)
                    #pragma unroll
                    for (int k = 0; k < 2; k++)
                        #pragma unroll
                        for (int w = 0; w < (FP8 ? 2 : 4); w++) most = Odd<FP8>::join(most, vr[n][k][w / 2][w % 2]);
                odd = __builtin_amdgcn_ballot_w64(Odd<FP8>::any(most));
                if (odd) {
                    #pragma unroll
                    for (int n = 0; n < D / 32; n++)
                        #pragma unroll
                        for (int k = 0; k < 2; k++)
                            #pragma unroll
                            for (int w = 0; w < (FP8 ? 2 : 4); w++) vr[n][k][w / 2][w % 2] = Odd<FP8>::drop(vr[n][k][w / 2][w % 2]);
                }
            }
            #pragma unroll
            for (int n = 0; n < D / 32; n++) {
                #pragma unroll
                for (int k = 0; k < 2; k++) {
                    const v2u* x = vr[n][k];
                    const v8bf vf = FP8 ? from_fp8(x[0][0], x[0][1])
                                  : __builtin_bit_cast(v8bf, v4u{x[0][0], x[0][1], x[FP8 ? 0 : 1][0], x[FP8 ? 0 : 1][1]});
                    #pragma unroll
                    for (int t = 0; t < RT; t++) acc[t][n] = mfma(vf, p[t][k], acc[t][n]);
                }
            }
            if constexpr (masked) {
                if (odd) {
                    for (uint32_t key = 0; key < kUnit; key++) {
                        const uint8_t* row = stage + mine + T::bytes + key * T::RB + g * (FP8 ? 4 : 8);
                        const uint32_t by = T::key_of_v(key);
                        #pragma unroll
                        for (int i = 0; i < D / 8; i++) {   // 4 dimensions of 8
                            float x[4];
                            if constexpr (FP8) {
                                const uint32_t u = *reinterpret_cast<const uint32_t*>(row + ((i / 2) ^ by) * 16 + i % 2 * 8);
                                #pragma unroll
                                for (int c = 0; c < 4; c++)   // (the bytes 7F and FF are NaN)
                                    x[c] = (u >> 8 * c & 0x7F) == 0x7F ? __builtin_nanf("") : 0.0f;
                            } else {
                                const v2u u = *reinterpret_cast<const v2u*>(row + (i ^ by) * 16);
                                #pragma unroll
                                for (int c = 0; c < 4; c++) {
                                    x[c] = c % 2 ? bf16_hi(u[c / 2]) : bf16_lo(u[c / 2]);
                                    if (__builtin_isfinite(x[c])) x[c] = 0.0f;
                                }
                            }
                            #pragma unroll
                            for (int t = 0; t < RT; t++)
                                if (sees[t] >> key & 1)
                                    #pragma unroll
                                    for (int c = 0; c < 4; c++) acc[t][i / 4][i % 4 * 4 + c] += x[c];
                        }
                    }
                }
            }
        };


        // A wave's units: every one, or the NW-th from its own on.  Below `plain` every row
        // sees all of a unit's slots, if they exist.
        constexpr int kBy = SHARED ? 1 : NW;
        const int plain = min(stop, (int)(((int64_t)s.context + (a.mask ? 0 : tile * kRows / a.G + 1)) / kUnit));
        const int u0 = first + (SHARED ? 0 : wave);
        uint8_t* const rings[4] = {ring0, ring1, ring2, ring3};
        uint32_t exists[STAGES];
        Lookup la, lb;
        auto fetch = [&](int v, int i) {   // unit v, whose lookup is la, into stage i
            const Lookup l = la;
            la = lb;
            lb = look_up(v + 2 * kBy);
            exists[i] = issue(l, rings[i]);
        };
        constexpr int kAhead = SHARED ? STAGES - 1 : STAGES;   // units under way
        auto begin = [&](int v) {
            la = look_up(v);
            lb = look_up(v + kBy);
            #pragma unroll
            for (int i = 0; i < kAhead; i++) fetch(v + i * kBy, i);
        };
        begin(u0);
        // Plain units, a round of the stages at a time (an exit between two stages would
        // make the compiler wait for all loads in each).
        int u = u0;
        uint32_t whole = 0xFFFFFFFFu;
        while (u + (STAGES - 1) * kBy < plain) {
            #pragma unroll
            for (int i = 0; i < STAGES; i++) {
                if constexpr (SHARED) {
                    arrive<(kAhead - 1) * kIssue>();
                    whole &= exists[i];
                    // (the stage that all waves have read before the barrier)
                    fetch(u + kAhead, (i + kAhead) % STAGES);
                    compute(std::false_type{}, u, 0, rings[i]);
                } else {
                    wait_loads<(kAhead - 1) * kIssue>();
                    whole &= exists[i];
                    compute(std::false_type{}, u, 0, rings[i]);
                    // (the reads of this stage have come: the products have used them)
                    __builtin_amdgcn_sched_barrier(0);
                    asm volatile("" ::: "memory");
                    fetch(u + STAGES * kBy, i);
                    __builtin_amdgcn_sched_barrier(0);
                }
                u += kBy;
            }
        }
        if (__builtin_amdgcn_readfirstlane(whole) != 0xFFFFFFFFu) {
            // some of them were of pages that do not exist: all over again, slot by slot
            if constexpr (SHARED) arrive<0>(); else wait_loads<0>();
            clear();
            u = u0;
            begin(u);
        }
        // The others: kAhead units lie in the stages from the first on.
        while (true) {
            if constexpr (SHARED) arrive<0>(); else wait_loads<0>();
            for (int i = 0; i < kAhead && u < stop; i++, u += kBy) {
                const uint8_t* stage = i == 0 ? ring0 : i == 1 ? ring1 : i == 2 ? ring2 : ring3;
                uint32_t e = exists[0];
                #pragma unroll
                for (int k = 1; k < kAhead; k++) e = i == k ? exists[k] : e;
                compute(std::true_type{}, u, e, stage);
            }
            if (u >= stop) break;
            if constexpr (SHARED) arrive<0>();
            __builtin_amdgcn_sched_barrier(0);
            asm volatile("" ::: "memory");
            #pragma unroll
            for (int i = 0; i < kAhead; i++) fetch(u + i * kBy, i);
        }
        if constexpr (SHARED) arrive<0>();   // (before the ring is filled again)

        #pragma unroll
        for (int t = 0; t < RT; t++) l[t] = sum_of(l[t]);
        const bool to_parts = !is_whole;
        const int64_t slot = (int64_t)blockIdx.x * 2 + (cut ? 0 : 1);
        float* part_o = a.parts + slot * kRows * D;
        float* part_s = a.parts + ((int64_t)a.work.groups * 2 * kRows * D) + slot * kRows * 2;
        auto out_row = [&](int row) {   // of q's rows, out
            return a.out + ((int64_t)(s.start + row / a.G) * a.Hq + h * a.G + row % a.G) * D;
        };
        if constexpr (SHARED) {
            #pragma unroll
            for (int t = 0; t < RT; t++) {
                const int row = row0 + 32 * t + r, local = row - tile * kRows;
                if (row >= rows) continue;
                const float by = l[t] == 0.0f ? 0.0f : 1.0f / l[t];
                if (to_parts && g == 0) {
                    part_s[local * 2] = m[t];
                    part_s[local * 2 + 1] = l[t];
                }
                uint16_t* o = out_row(row);
                #pragma unroll
                for (int n = 0; n < D / 32; n++)
                    #pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const int d = 32 * n + 8 * i + 4 * g;
                        const v4f x = {acc[t][n][4 * i], acc[t][n][4 * i + 1], acc[t][n][4 * i + 2], acc[t][n][4 * i + 3]};
                        if (to_parts) {
                            *reinterpret_cast<v4f*>(part_o + local * D + d) = x;
                        } else {
                            *reinterpret_cast<v2u*>(o + d) = v2u{bf16_pack(x[0] * by, x[1] * by), bf16_pack(x[2] * by, x[3] * by)};
                        }
                    }
            }
        } else {
            // The waves' sums are added in wave order, brought to the largest of their maxima.
            #pragma unroll
            for (int t = 0; t < RT; t++)
                if (g == 0) {
                    stat[wave][32 * t + r][0] = m[t];
                    stat[wave][32 * t + r][1] = l[t];
                }
            __syncthreads();   // (all waves' loads into the ring have come, and their reads)
            constexpr int kHold = 32 * RT * D * 4;   // bytes of a wave's sums
            auto held = [&](int w) {   // (rings of whole waves' sums)
                constexpr int kPer = kRing / kHold;
                static_assert(kPer >= 1 && kPer * STAGES >= NW, "the rings hold the sums");
                uint8_t* ring = w / kPer == 0 ? ring0 : w / kPer == 1 ? ring1 : w / kPer == 2 ? ring2 : ring3;
                return (float*)(ring + w % kPer * kHold);
            };
            float* hold = held(wave);
            #pragma unroll
            for (int t = 0; t < RT; t++) {
                float top = kNone;
                #pragma unroll
                for (int w = 0; w < NW; w++) top = fmaxf(top, stat[w][32 * t + r][0]);
                const float by = m[t] == kNone ? 0.0f : __builtin_amdgcn_exp2f((m[t] - top) * a.c);
                #pragma unroll
                for (int n = 0; n < D / 32; n++)
                    #pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const int row = 32 * t + r, piece = 8 * n + 2 * i + g;
                        *reinterpret_cast<v4f*>(hold + row * D + (piece ^ (row & 15)) * 4) =
                            v4f{acc[t][n][4 * i] * by, acc[t][n][4 * i + 1] * by, acc[t][n][4 * i + 2] * by,
                                acc[t][n][4 * i + 3] * by};
                    }
            }
            __syncthreads();
            const int valid = min(kRows, rows - tile * kRows);
            for (int x = threadIdx.x; x < valid * (D / 4); x += NW * kLanes) {
                const int row = x / (D / 4), piece = x % (D / 4);
                float top = kNone, sum = 0.0f;
                #pragma unroll
                for (int w = 0; w < NW; w++) top = fmaxf(top, stat[w][row][0]);
                v4f o = {0, 0, 0, 0};
                #pragma unroll
                for (int w = 0; w < NW; w++) {
                    const float mw = stat[w][row][0];
                    sum += mw == kNone ? 0.0f : stat[w][row][1] * __builtin_amdgcn_exp2f((mw - top) * a.c);
                    o += *reinterpret_cast<const v4f*>(held(w) + row * D + (piece ^ (row & 15)) * 4);
                }
                if (to_parts) {
                    *reinterpret_cast<v4f*>(part_o + row * D + piece * 4) = o;
                    if (piece == 0) {
                        part_s[row * 2] = top;
                        part_s[row * 2 + 1] = sum;
                    }
                } else {
                    const float by = sum == 0.0f ? 0.0f : 1.0f / sum;
                    *reinterpret_cast<v2u*>(out_row(tile * kRows + row) + piece * 4) =
                        v2u{bf16_pack(o[0] * by, o[1] * by), bf16_pack(o[2] * by, o[3] * by)};
                }
            }
            if (left > 0) __syncthreads();   // (before the ring is filled again)
        }
        }
        // the next item's sequence
        if (left > 0 && in == (int64_t)a.batch.heads * s.tiles * (s.units + a.work.item)) {
            in = 0;
            do {
                if (++b == a.batch.B) return;   // (not reached while nobody writes to the batch)
                s = sequence(a, b);
            } while (s.tiles == 0);
        }
    }
}

// The rows of items that several workgroups share, from their parts in the order of
// the slots.  A wave takes a row.
template <int D>
__global__ __launch_bounds__(256) void join_kernel(Args a) {
    const int lane = threadIdx.x & (kLanes - 1);
    const int64_t id = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x / kLanes);
    const int n = (int)(id / a.Hq), hq = (int)(id % a.Hq);
    if (n >= a.batch.N) return;
    const int b = find_sequence(a.batch, n);
    if (b < 0 || n >= a.batch.start(b + 1)) return;
    const Seq s = sequence(a, b);
    int64_t all, before;
    total_cost(a, b, all, before);
    const int groups = work_groups(a.work, all);
    const int h = hq / a.G, row = (n - s.start) * a.G + hq % a.G;
    const int tile = row / a.work.rows, local = row % a.work.rows;
    const int64_t from = before + ((int64_t)h * s.tiles + tile) * (s.units + a.work.item) + a.work.item,
                  to = from + s.units;
    const int w0 = range_of(all, groups, from), w1 = range_of(all, groups, to - 1);
    if (w0 == w1) return;   // (one workgroup had the whole item)
    constexpr int E = D / kLanes;
    const float* stats = a.parts + (int64_t)a.work.groups * 2 * a.work.rows * D;
    auto slot = [&](int w) { return ((int64_t)w * 2 + (from < range_start(all, groups, w) ? 0 : 1)) * a.work.rows + local; };
    float top = kNone;
    for (int w = w0; w <= w1; w++) top = fmaxf(top, stats[slot(w) * 2]);
    float sum = 0.0f, o[E] = {};
    for (int w = w0; w <= w1; w++) {
        const float m = stats[slot(w) * 2];
        const float by = m == kNone ? 0.0f : __builtin_amdgcn_exp2f((m - top) * a.c);
        sum += stats[slot(w) * 2 + 1] * by;
        #pragma unroll
        for (int i = 0; i < E; i++) o[i] += a.parts[slot(w) * D + lane * E + i] * by;
    }
    const float by = sum == 0.0f ? 0.0f : 1.0f / sum;
    uint16_t* out = a.out + ((int64_t)n * a.Hq + hq) * D + lane * E;
    #pragma unroll
    for (int i = 0; i < E; i++) out[i] = (uint16_t)bf16_pack(o[i] * by, 0.0f);
}

}  // namespace

extern "C" {

int tans_tree_attention_workspace(int64_t N, int64_t B, int64_t q_heads, int64_t heads, int64_t dim,
                                  int64_t slots, int64_t max_tokens, int64_t* bytes) {
    if (!bytes) return fail(TANS_EINVAL, "tree_attention: null pointer");
    if (N < 0 || B < 0 || heads < 1 || q_heads < heads || q_heads % heads || q_heads > 65535 ||
        (dim != 64 && dim != 128 && dim != 256) || slots < 0 || slots > INT32_MAX || max_tokens < 0 ||
        N > INT32_MAX / 2 || B >= INT32_MAX)
        return fail(TANS_EINVAL, "tree_attention: sizes out of range");
    const int cus = tans_internal_cu_count();
    *bytes = N && B ? plan(N, B, q_heads, heads, dim, slots, max_tokens, cus > 0 ? cus : 256).bytes : 0;
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
    if (!(scale > 0.0f) || scale > 1.0e38f) return fail(TANS_EINVAL, op + ": scale must be positive and finite");
    if (max_tokens < 0) return fail(TANS_EINVAL, op + ": max_tokens must not be negative");
    if (N == 0 || B == 0) return TANS_OK;
    if (!q || !out) return fail(TANS_EINVAL, op + ": null pointer");
    rc = stride_check(op, "q", q, q_stride, q_heads * dim);
    if (rc == TANS_OK && !aligned(out, 16)) rc = fail(TANS_EINVAL, op + ": out is misaligned (16 bytes)");
    if (rc != TANS_OK) return rc;
    const int cus = tans_internal_cu_count();
    if (cus <= 0) return fail(TANS_EHIP, op + ": cannot query the device's CU count");
    const Plan p = plan(N, B, q_heads, heads, dim, per * page, max_tokens, cus);
    if (p.bytes > 0 && (!workspace || !aligned(workspace, 16) || workspace_bytes < p.bytes))
        return fail(TANS_EINVAL, op + ": workspace too small, null or misaligned (16 bytes)");
    if (p.blocks > INT32_MAX / 256) return fail(TANS_EINVAL, op + ": too many tokens for one call");
    Args a = {};
    a.batch = {table, starts, lens, (int)B, (int)per, (int)N, (uint32_t)pages, (uint32_t)heads, (uint32_t)page};
    a.q = (const uint16_t*)q;
    a.q_stride = q_stride;
    a.k = (const uint8_t*)k_cache;
    a.v = (const uint8_t*)v_cache;
    a.k_scale = k_scale;
    a.v_scale = v_scale;
    a.mask = (const uint8_t*)mask;
    a.W = (int)mask_cols;
    a.Hq = (int)q_heads;
    a.G = (int)(q_heads / heads);
    a.c = scale * kLog2e;
    a.out = (uint16_t*)out;
    a.work = p.work;
    a.parts = (float*)workspace;
    auto launch = [&](auto kernel, int threads) {
        hipLaunchKernelGGL(kernel, dim3((unsigned)p.blocks), dim3(threads), 0, (hipStream_t)stream, a);
        return hip_check(hipGetLastError(), "attend_kernel launch");
    };
    auto with = [&](auto DIM, auto EIGHT) {
        constexpr int D = decltype(DIM)::value;
        constexpr bool f8 = decltype(EIGHT)::value;
        constexpr int nw = D == 256 && !f8 ? 2 : 4;
        constexpr int stage = (2 * Tile<D, f8>::bytes + (f8 ? 256 : 0)) * nw;
        constexpr int stages = 4 * stage <= (132 << 10) ? 4 : 2;
        int rc;
        if (p.kind == kFew) rc = launch(attend_kernel<D, f8, 1, false, nw, stages>, nw * kLanes);
        else if (p.kind == kMany) rc = launch(attend_kernel<D, f8, 1, true, 4, 3>, 4 * kLanes);
        else {
            if constexpr (D < 256) {
                if (p.kind == kSome) rc = launch(attend_kernel<D, f8, 2, false, nw, stages>, nw * kLanes);
                else rc = launch(attend_kernel<D, f8, 2, true, 4, 3>, 4 * kLanes);
            } else {
                rc = fail(TANS_EINVAL, "tree_attention: no such kernel");   // (not reached: plan())
            }
        }
        if (rc == TANS_OK && !p.work.whole) {
            hipLaunchKernelGGL((join_kernel<D>), dim3((unsigned)((N * q_heads + 3) / 4)), dim3(256), 0,
                               (hipStream_t)stream, a);
            rc = hip_check(hipGetLastError(), "join_kernel launch");
        }
        return rc;
    };
    auto types = [&](auto DIM) {
        return k_scale ? with(DIM, std::true_type{}) : with(DIM, std::false_type{});
    };
    if (dim == 64) return types(std::integral_constant<int, 64>{});
    if (dim == 128) return types(std::integral_constant<int, 128>{});
    return types(std::integral_constant<int, 256>{});
}

}  // extern "C"
