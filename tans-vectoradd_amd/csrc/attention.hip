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

// The item that a workgroup's run ends in, if it begins there too and others go on with it.
struct Cut { int start, rows, tile, h, last; };   // last: the workgroup that has its end, or -1

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
    Cut* cuts;             // [workgroups]
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
    return pieces_of(a.work, a.batch.heads, s.tiles, s.units);
}

__device__ __forceinline__ int64_t uniform(int64_t v) {
    return (int64_t)((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)v) |
                     (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(v >> 32)) << 32);
}

// The work of all sequences.
__device__ __forceinline__ int64_t total_cost(const Args& a) {
    if (a.batch.B == 1) return uniform(add_pieces(a.work, 0, cost(a, 0)));
    int64_t all = 0;
    for (int i = threadIdx.x & (kLanes - 1); i < a.batch.B; i += kLanes) all = add_pieces(a.work, all, cost(a, i));
    #pragma unroll
    for (int i = 1; i < kLanes; i *= 2) all = add_pieces(a.work, all, __shfl_xor(all, i));
    return uniform(all);
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

// LDS is addressed by pointers of its own address space: a plain pointer to it that the
// compiler keeps in a table and loads from there it takes for one to memory.
#define TANS_LDS __attribute__((address_space(3)))
typedef TANS_LDS uint8_t* Lds;
template <class V>
__device__ __forceinline__ V lds_read(Lds from) { return *(const TANS_LDS V*)from; }

// 16 or 4 bytes a lane from memory to LDS, lane l's to lds + 16 l or 4 l.
template <int BYTES>
__device__ __forceinline__ void load_lds(const void* from, Lds to) {
    const auto* p = (const __attribute__((address_space(1))) void*)from;
    auto* lds = (TANS_LDS void*)to;
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

// Two probabilities as bf16, and what a bf16 cut off leaves of one: 2^-15 of it is lost by
// both together.  (Never zero of what is not, since an infinite value times it would be NaN.)
__device__ __forceinline__ uint32_t bf16_cut(float a, float b) {
    return __builtin_amdgcn_perm(__builtin_bit_cast(uint32_t, b), __builtin_bit_cast(uint32_t, a), 0x07060302u);
}
__device__ __forceinline__ float rest_of(float x, float cut) { return fmaxf(x - cut, x * 7.6293945e-6f); }   // 2^-17

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

// Where a lane finds its operands in a stage: K's (slots x dimensions) and V's.
template <int D, bool FP8>
struct Places {
    using T = Tile<D, FP8>;
    static constexpr int turn = T::pieces < 8 ? 4 : 8;   // pieces of a row that the keys permute
    uint32_t k[4], v[4];
    __device__ __forceinline__ void set(int lane) {
        const int r = lane & 31, g = lane >> 5, l = lane & 15, half = (lane >> 4) & 1;
        #pragma unroll
        for (int i = 0; i < 4; i++) {
            k[i] = opaque_v(r * T::RB + (((2 * i + g) ^ T::key_of_k(r)) % T::pieces) * 16);
            if constexpr (FP8) {
                const uint32_t row = l / 2 < 4 ? 4 * g + l / 2 : 4 + 4 * g + l / 2;
                v[i] = opaque_v(T::bytes + row * T::RB + (((2 * i + half) ^ T::key_of_v(row)) % T::pieces) * 16 + l % 2 * 8);
            } else {
                const uint32_t row = 4 * g + l / 4;
                v[i] = opaque_v(T::bytes + row * T::RB +
                                (((4 * (i & 1) + 2 * half + l % 4 / 2) ^ T::key_of_v(row)) % T::pieces) * 16 + l % 2 * 8);
            }
        }
    }
    // operand j of K: 8 dimensions of slot r, those that load_query gives product j (of 8
    // bits j and j + 1, j even)
    __device__ __forceinline__ v4u read_k(Lds stage, int j) const {
        const int i = FP8 ? j / 2 : j;
        return lds_read<v4u>(stage + k[i % (turn / 2)] + i / (turn / 2) * (16 * turn));
    }
    // operand of V for dimensions 32 n .. 32 n + 31 and half h of the slots
    __device__ __forceinline__ v4u read_v(Lds stage, int n, int h) const {
        if constexpr (FP8) {
            typedef TANS_LDS v2i* P;
            const v2u x = __builtin_bit_cast(v2u, __builtin_amdgcn_ds_read_tr8_b64_v2i32(
                (P)(stage + v[n % (turn / 2)] + n / (turn / 2) * (16 * turn) + h * 16 * T::RB)));
            return v4u{x[0], x[1], 0, 0};
        } else {
            typedef TANS_LDS v4s* P;
            const Lds from = stage + v[n % 2] + n / 2 * 128 + h * 16 * T::RB;
            const v2u x = __builtin_bit_cast(v2u, __builtin_amdgcn_ds_read_tr16_b64_v4i16((P)from));
            const v2u y = __builtin_bit_cast(v2u, __builtin_amdgcn_ds_read_tr16_b64_v4i16((P)(from + 8 * T::RB)));
            return v4u{x[0], x[1], y[0], y[1]};
        }
    }
};

// A tile's 32 rows of q, lane (g, r) holding row r's operands.
template <int D, bool FP8>
__device__ __forceinline__ void load_query(const uint16_t* p, bool exists, v8bf (&q)[D / 16]) {
    const int g = (threadIdx.x & (kLanes - 1)) >> 5;
    #pragma unroll
    for (int j = 0; j < D / 16; j++) {
        v4u u = {0, 0, 0, 0};
        if (exists) u = *reinterpret_cast<const v4u*>(p + (FP8 ? j / 2 * 32 + 16 * g + j % 2 * 8 : 16 * j + 8 * g));
        q[j] = __builtin_bit_cast(v8bf, u);
    }
}

// The running sums of 32 rows: lane (g, r) has row r's dimensions 32 n + 8 i + 4 g + c in
// acc[n][4 i + c], its maximum, and of its sum the part of its own slots.
//
// The maximum is one that exponents refer to, not the largest score: it is raised, and
// the sums brought to it, when a score exceeds it by more than 2^kLoose in the
// probability.  That keeps the factor of D values out of all but a few units, and costs
// no bits: probabilities are rounded to bf16 whatever their exponent, sums are 32 bits'.
constexpr float kLoose = 8.0f;
template <int D>
struct Sums {
    v16f acc[D / 32];
    float m, l;
    __device__ __forceinline__ void clear() {
        m = kNone;
        l = 0.0f;
        #pragma unroll
        for (int n = 0; n < D / 32; n++)
            #pragma unroll
            for (int c = 0; c < 16; c++) acc[n][c] = 0.0f;
    }
    // Admits a unit's scores; returns what to take from score * c in the exponent.
    __device__ __forceinline__ float admit(const v16f& sc, float c) {
        float top = sc[0];
        #pragma unroll
        for (int i = 1; i < 16; i++) top = fmaxf(top, sc[i]);
        top = larger(top);
        // (where m is kNone any score but that one exceeds it; NaN has no part in top)
        if (__builtin_amdgcn_ballot_w64((top - m) * c > kLoose)) {
            const float next = fmaxf(m, top);
            const float by = next == kNone ? 0.0f : __builtin_amdgcn_exp2f((m - next) * c);
            m = next;
            l *= by;
            #pragma unroll
            for (int n = 0; n < D / 32; n++)
                #pragma unroll
                for (int i = 0; i < 16; i++) acc[n][i] *= by;
        }
        return m == kNone ? 0.0f : m * c;
    }
};

// The scales of a lane's 16 slots: 8 i + 4 g + c for value 4 i + c.
__device__ __forceinline__ void read_scales(Lds from, float (&f)[16]) {
    const int g = (threadIdx.x & (kLanes - 1)) >> 5;
    #pragma unroll
    for (int i = 0; i < 4; i++) {
        const v4f x = lds_read<v4f>(from + (8 * i + 4 * g) * 4);
        #pragma unroll
        for (int c = 0; c < 4; c++) f[4 * i + c] = x[c];
    }
}

// A unit for 32 rows.  S^T = K Q^T by 32 x 32 x 16 products: lane (g, r), lane 32 g + r,
// gets query row r's scores with the slots 8 i + 4 g + c (i, c = 0 .. 3), so that a row's
// maximum and sum are one lane's and its other half's.  Those 16 are, rounded to bf16,
// the operand of O^T = V^T P^T as they lie there, if the slots are taken in that order;
// V's operand, 8 slots of one dimension, comes from LDS by transposing reads.
//
// Rounded to bf16, a probability loses 2^-8 of itself at most, and the result's error against
// 64 bits becomes about 1.4 times that of its own rounding (1.0 to 1.6 for single rows).  It is
// the type in which the matrix cores multiply by bf16 values without a loss of theirs.  SPLIT
// holds 16 bits, as the sum of two bf16 that are each multiplied: for shared items of 32 rows of
// a bf16 cache, whose products wait for memory (one token of 262144 slots 192.0 -> 192.6 us, 7 of
// 4000 33.1 / 33.1, 256 of 512 128.3 -> 131.4).  Elsewhere it costs too much: one token of 700
// slots 12.7 -> 13.9, 8 bits 262144 slots 110 -> 114, 17 trees 39.7 -> 44.6, a tree of 8 with 64
// rows 47 -> 51; and tiles of 128 or 256 rows are bound by their products.
struct Mask {
    int token;         // the lane's row's, in its sequence, or -1
    int start;         // the sequence's first row of q
    int before;        // slots of the context from the unit's first on, 32 at most
    uint32_t exists;   // of the unit's slots
};
template <int D, bool FP8, bool MASKED, bool SPLIT>
__device__ __forceinline__ void attend_unit(const Args& a, const Places<D, FP8>& at, Lds stage, Lds scales,
                                            const v8bf (&q)[D / 16], Sums<D>& sums,
                                            const Mask& mask) {
    using T = Tile<D, FP8>;
    const int lane = threadIdx.x & (kLanes - 1), g = lane >> 5;
    v16f sc;
    #pragma unroll
    for (int c = 0; c < 16; c++) sc[c] = 0.0f;
    constexpr int kStep = FP8 ? 2 : 1;   // products of a read
    v4u kr[D / 16 / kStep];
    #pragma unroll
    for (int j = 0; j < D / 16; j += kStep) kr[j / kStep] = at.read_k(stage, j);
    __builtin_amdgcn_sched_barrier(0);
    #pragma unroll
    for (int j = 0; j < D / 16; j++) {
        const v4u& x = kr[j / kStep];
        sc = mfma(FP8 ? from_fp8(x[2 * (j % 2)], x[2 * (j % 2) + 1]) : __builtin_bit_cast(v8bf, x), q[j], sc);
    }
    // V's operands, under way during the exponentials
    v4u vr[D / 32][2];
    #pragma unroll
    for (int n = 0; n < D / 32; n++)
        #pragma unroll
        for (int k = 0; k < 2; k++) vr[n][k] = at.read_v(stage, n, k);
    __builtin_amdgcn_sched_barrier(0);
    float vs[16];
    if constexpr (FP8) {
        float ks[16];
        read_scales(scales, ks);
        read_scales(scales + 128, vs);
        #pragma unroll
        for (int i = 0; i < 16; i++) sc[i] *= ks[i];
    }
    uint32_t sees = 0xFFFFFFFFu;   // the unit's slots that the row sees
    if constexpr (MASKED) {
        sees = first_bits(a.mask ? mask.before : mask.before + mask.token + 1);
        if (a.mask && mask.before < kUnit) {
            // (a row's first column where the tile has none of its own)
            const uint8_t* row = a.mask + (int64_t)(mask.start + max(mask.token, 0)) * a.W;
            uint32_t bits = 0;
            #pragma unroll
            for (int i = 0; i < 16; i++) {
                const int key = i / 4 * 8 + 4 * g + i % 4, j = key - mask.before;
                const uint32_t bit = row[j < 0 ? 0 : j < a.W ? j : a.W - 1];
                bits |= (j >= 0 && j < a.W ? bit : 0) << key;
            }
            sees |= all_bits(bits);
        }
        sees = mask.token >= 0 ? sees & mask.exists : 0;
        const uint32_t mine = sees >> 4 * g;
        #pragma unroll
        for (int i = 0; i < 16; i++)
            if (!(mine >> (i / 4 * 8 + i % 4) & 1)) sc[i] = kNone;
    }
    const float mc = sums.admit(sc, a.c);
    v8bf p[2], rest[2];
    float e[16];
    #pragma unroll
    for (int i = 0; i < 16; i++) {
        e[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[i], a.c, -mc));
        sums.l += e[i];
        // (what is not seen may have any scale)
        if constexpr (FP8) e[i] = MASKED && e[i] == 0.0f ? 0.0f : e[i] * vs[i];
    }
    #pragma unroll
    for (int k = 0; k < 2; k++) {
        v4u high, low = {0, 0, 0, 0};
        #pragma unroll
        for (int i = 0; i < 4; i++) {
            const float x = e[8 * k + 2 * i], y = e[8 * k + 2 * i + 1];
            high[i] = SPLIT ? bf16_cut(x, y) : bf16_pack(x, y);
            if constexpr (SPLIT) low[i] = bf16_pack(rest_of(x, bf16_lo(high[i])), rest_of(y, bf16_hi(high[i])));
        }
        p[k] = __builtin_bit_cast(v8bf, high);
        rest[k] = __builtin_bit_cast(v8bf, low);
    }
    // A value that is infinite or NaN reaches the rows that see its slot, and by the
    // matrix product it would reach the others as well (0 times it is NaN): it is left out
    // there, and added below.
    uint64_t odd = 0;
    if constexpr (MASKED) {
        uint32_t most = 0;
        #pragma unroll
        for (int n = 0; n < D / 32; n++)
            #pragma unroll
            for (int k = 0; k < 2; k++)
                #pragma unroll
                for (int w = 0; w < (FP8 ? 2 : 4); w++) most = Odd<FP8>::join(most, vr[n][k][w]);
        odd = __builtin_amdgcn_ballot_w64(Odd<FP8>::any(most));
        if (odd) {
            #pragma unroll
            for (int n = 0; n < D / 32; n++)
                #pragma unroll
                for (int k = 0; k < 2; k++)
                    #pragma unroll
                    for (int w = 0; w < (FP8 ? 2 : 4); w++) vr[n][k][w] = Odd<FP8>::drop(vr[n][k][w]);
        }
    }
    #pragma unroll
    for (int n = 0; n < D / 32; n++)
        #pragma unroll
        for (int k = 0; k < 2; k++) {
            const v8bf v = FP8 ? from_fp8(vr[n][k][0], vr[n][k][1]) : __builtin_bit_cast(v8bf, vr[n][k]);
            sums.acc[n] = mfma(v, p[k], sums.acc[n]);
            if constexpr (SPLIT) sums.acc[n] = mfma(v, rest[k], sums.acc[n]);
        }
    if constexpr (MASKED) {
        if (odd) {
            for (uint32_t key = 0; key < kUnit; key++) {
                const Lds row = stage + T::bytes + key * T::RB + g * (FP8 ? 4 : 8);
                const uint32_t by = T::key_of_v(key);
                #pragma unroll
                for (int i = 0; i < D / 8; i++) {   // 4 dimensions of 8
                    float x[4];
                    if constexpr (FP8) {
                        const uint32_t u = lds_read<uint32_t>(row + ((i / 2) ^ by) * 16 + i % 2 * 8);
                        #pragma unroll
                        for (int c = 0; c < 4; c++)   // (the bytes 7F and FF are NaN)
                            x[c] = (u >> 8 * c & 0x7F) == 0x7F ? __builtin_nanf("") : 0.0f;
                    } else {
                        const v2u u = lds_read<v2u>(row + (i ^ by) * 16);
                        #pragma unroll
                        for (int c = 0; c < 4; c++) {
                            x[c] = c % 2 ? bf16_hi(u[c / 2]) : bf16_lo(u[c / 2]);
                            if (__builtin_isfinite(x[c])) x[c] = 0.0f;
                        }
                    }
                    if (sees >> key & 1)
                        #pragma unroll
                        for (int c = 0; c < 4; c++) sums.acc[i / 4][i % 4 * 4 + c] += x[c];
                }
            }
        }
    }
}

// A workgroup's run of the work, item by item.
struct Item {
    int h, tile, first, end;   // row tile `tile` of cache head h, units first .. end - 1 of it
    bool whole;                // all of its units
    bool cut;                  // it began in another workgroup's run
};
struct Run {
    int64_t left, in;   // pieces; the next one's number in its sequence
    int64_t all, at;    // all of the work; the next piece
    int b, groups, index;   // index: the run's number
    Seq s;
    __device__ __forceinline__ bool begin(const Args& a) {
        all = total_cost(a);
        groups = a.work.whole ? 0 : work_groups(a.work, all);
        // Runs that follow each other go to one XCD, where a head's row tiles read the same rows
        // through one L2 (2048 tokens of a prompt 678 us without).
        index = groups == (int)gridDim.x ? run_of(blockIdx.x, groups) : blockIdx.x;
        if (!a.work.whole && threadIdx.x == 0) a.cuts[index].last = -1;
        if (a.work.whole ? index >= all : index >= groups) return false;
        in = at = a.work.whole ? index : range_start(all, groups, index);
        left = a.work.whole ? 1 : range_start(all, groups, index + 1) - in;
        b = find_piece(a, in);
        s = sequence(a, b);
        return true;
    }
    __device__ __forceinline__ Item take(const Args& a) {
        Item o;
        if (a.work.whole) {
            o.h = (int)(in % a.batch.heads);
            o.tile = s.tiles - 1 - (int)(in / a.batch.heads);
            o.first = 0;
            o.end = s.units;
            o.whole = true;
            o.cut = false;
            left = 0;
            return o;
        }
        const int pieces = s.units + a.work.item;
        const int64_t item = in / pieces;
        const int from = (int)(in - item * pieces);
        o.h = (int)(item / s.tiles);
        o.tile = (int)(item - (int64_t)o.h * s.tiles);
        const int to = (int)(from + left < pieces ? from + left : pieces);
        o.first = max(0, from - a.work.item);
        o.end = to - a.work.item;   // (none of its units if not above first)
        o.whole = o.first == 0 && o.end == s.units;
        o.cut = o.first > 0;
        if (!o.cut && o.end > 0 && !o.whole && threadIdx.x == 0)
            a.cuts[index] = {s.start, s.tokens * a.G, o.tile, o.h, range_of(all, groups, at - from + pieces - 1)};
        left -= to - from;
        in += to - from;
        at += to - from;
        return o;
    }
    // The next item's sequence; false if there is none.
    __device__ __forceinline__ bool go_on(const Args& a) {
        if (left <= 0) return false;
        if (in == (int64_t)a.batch.heads * s.tiles * (s.units + a.work.item)) {
            in = 0;
            do {
                if (++b == a.batch.B) return false;   // (not reached while nobody writes to the batch)
                s = sequence(a, b);
            } while (s.tiles == 0);
        }
        return true;
    }
    __device__ __forceinline__ int stop(const Args& a, const Item& o, int rows) const {
        return tile_stop(a.mask, s.context, s.tokens, s.slots, o.tile, rows, a.G, o.end);
    }
    __device__ __forceinline__ int plain(const Args& a, const Item& o, int rows, int stop) const {
        return tile_plain(a.mask, s.context, s.slots, o.tile, rows, a.G, stop);
    }
};

// The rows of a unit of the item's slots, looked up in the table well before they are
// loaded: lane (g, r) has slot r's.
struct Lookup { uint32_t entry, off; bool in; };
__device__ __forceinline__ Lookup look_up(const Args& a, const Run& run, int u, int stop) {
    const uint32_t slot = (uint32_t)u * kUnit + (threadIdx.x & 31);
    Lookup o;
    o.in = u < stop && slot < (uint32_t)run.s.slots;
    const uint32_t i = o.in ? a.batch.page_of(slot) : 0;
    o.off = slot - i * a.batch.page;
    o.entry = run.s.slots > 0 ? (uint32_t)a.batch.table[(int64_t)run.b * a.batch.per + i] : 0;
    return o;
}

// Loads a unit's rows (of nothing: row 0's, which no lane sees) into a stage, or where NW
// waves share it a wave's part of them.  find() says which rows a lane's loads take and
// returns the slots that exist; it goes through LDS, so the loads come later.
template <int D, bool FP8, int NW>
struct Loads {
    using T = Tile<D, FP8>;
    // (units of fewer loads than waves: two waves load the same)
    static constexpr int kLoads = 2 * T::loads > NW ? 2 * T::loads / NW : 1;
    static constexpr int kDistinct = kLoads < T::loads ? kLoads : T::loads;
    static constexpr int kIssue = kLoads + (FP8 ? 1 : 0);   // with the scales'
    static_assert(kLoads == 1 || 2 * T::loads % NW == 0, "loads");
    uint32_t from[kDistinct], mine;
    // the i-th load's number in the stage, K's and then V's
    static __device__ __forceinline__ int number(int i) {
        const int wave = NW > 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x / kLanes) : 0;
        return (wave * kLoads + i) % (2 * T::loads);
    }
    static __device__ __forceinline__ int row_of(int i) {
        return number(i) % T::loads * T::per_load + (threadIdx.x & (kLanes - 1)) / T::pieces;
    }
    __device__ __forceinline__ uint32_t find(const Args& a, const Lookup& o, int h) {
        const bool valid = o.in && o.entry < a.batch.pages;
        mine = valid ? (o.entry * a.batch.heads + h) * a.batch.page + o.off : 0;
        #pragma unroll
        for (int i = 0; i < kDistinct; i++) from[i] = __shfl(mine, row_of(i));
        return (uint32_t)__builtin_amdgcn_ballot_w64(valid);
    }
    __device__ __forceinline__ void issue(const Args& a, Lds stage, Lds scales) const {
        const int lane = threadIdx.x & (kLanes - 1);
        #pragma unroll
        for (int i = 0; i < kLoads; i++) {
            const int n = number(i);
            const bool is_v = n >= T::loads;
            const uint32_t at = row_of(i), key = is_v ? T::key_of_v(at) : T::key_of_k(at);
            load_lds<16>((is_v ? a.v : a.k) + (int64_t)from[i % kDistinct] * T::RB + ((lane % T::pieces) ^ key) * 16,
                         stage + n * 1024);
        }
        if constexpr (FP8) load_lds<4>((lane >> 5 ? a.v_scale : a.k_scale) + mine, scales);
    }
};

// The same where pages are multiples of 16 rows, so that each half of a unit, and with it
// each load, lies in one page: pages are looked up and addresses computed once a wave, by
// scalar instructions, and lanes add a constant.  For D = 256, whose waves have 8 loads a
// unit (2048 tokens of a prompt 645 us through lanes' lookups, 593 so); with D = 128 and 2 loads
// the scalar chain behind the barrier costs more than it saves (683 / 709), D = 64 442 / 512.
template <int D, bool FP8, int NW>
struct PagedLoads {
    using T = Tile<D, FP8>;
    using L = Loads<D, FP8, NW>;
    uint32_t offset[L::kLoads];   // a lane's, from the first row of a load
    uint32_t entry[2], off[2];    // the next unit's halves
    bool in[2];
    __device__ __forceinline__ void set() {
        const int lane = threadIdx.x & (kLanes - 1);
        #pragma unroll
        for (int i = 0; i < L::kLoads; i++) {
            const uint32_t at = L::row_of(i), key = L::number(i) >= T::loads ? T::key_of_v(at) : T::key_of_k(at);
            offset[i] = lane / T::pieces * T::RB + ((lane % T::pieces) ^ key) * 16;
        }
    }
    // (the table through the scalar cache: nothing writes to it meanwhile; it has an entry,
    // since this runs beside plain units, whose slots the sequence has)
    __device__ __forceinline__ void look_up(const Args& a, const Run& run, int u, int stop) {
        const auto* table = (const __attribute__((address_space(4))) int32_t*)a.batch.table + (int64_t)run.b * a.batch.per;
        #pragma unroll
        for (int k = 0; k < 2; k++) {
            const uint32_t slot = (uint32_t)u * kUnit + 16 * k;
            in[k] = u < stop && slot < (uint32_t)run.s.slots;
            const uint32_t i = in[k] ? a.batch.page_of(slot) : 0;
            off[k] = in[k] ? slot - i * a.batch.page : 0;
            entry[k] = (uint32_t)table[i];
        }
    }
    // Loads the unit that was looked up; whether all of its slots exist.
    __device__ __forceinline__ bool issue(const Args& a, int h, Lds stage, Lds scales) const {
        const int lane = threadIdx.x & (kLanes - 1);
        uint32_t row[2];
        bool all = true;
        #pragma unroll
        for (int k = 0; k < 2; k++) {
            const bool valid = in[k] && entry[k] < a.batch.pages;
            row[k] = valid ? (entry[k] * a.batch.heads + h) * a.batch.page + off[k] : 0;
            all = all && valid;
        }
        #pragma unroll
        for (int i = 0; i < L::kLoads; i++) {
            const int n = L::number(i), first = n % T::loads * T::per_load;
            const uint32_t from = (first >= 16 ? row[1] : row[0]) + first % 16;
            load_lds<16>((n >= T::loads ? a.v : a.k) + (int64_t)from * T::RB + offset[i], stage + n * 1024);
        }
        if constexpr (FP8) load_lds<4>((lane >> 5 ? a.v_scale : a.k_scale) + (lane & 16 ? row[1] : row[0]) + (lane & 15), scales);
        return all;
    }
};

// Where an item's sums go: to `out`, or to its part.
struct Target {
    uint16_t* out;
    float *part_o, *part_s;
    bool parts;
};
template <int D>
__device__ __forceinline__ Target target(const Args& a, const Run& run, const Item& o, int rows) {
    const int64_t slot = (int64_t)run.index * 2 + (o.cut ? 0 : 1);
    return {a.out, a.parts + slot * rows * D,
            a.parts + ((int64_t)a.work.groups * 2 * rows * D) + slot * rows * 2, !o.whole};
}
__device__ __forceinline__ int64_t out_row(const Args& a, const Run& run, const Item& o, int row) {
    return (int64_t)(run.s.start + row / a.G) * a.Hq + o.h * a.G + row % a.G;
}

// Few rows: every wave takes all 32 RT rows of the tile and every NW-th unit, through a
// ring of its own in LDS that loads write without a register between; the waves' sums are
// added at the end.  Nothing makes the waves wait for each other, so that each keeps its
// ring's loads under way.  Memory bounds it: one token of 262144 slots, 8 heads, D = 128,
// 193 us (1.07 GB at 5.6 TB/s); 96 tokens over 100 .. 16000 slots in 8 bits 138 us (648 MB at
// 4.7 TB/s); D = 256 reaches 4.1-4.4 TB/s, with two waves' rings of 32 KB a unit.  (Some spill
// registers, up to 45 with D = 256: stored and loaded again at an item's begin and end, not in
// the loops over its units.)
template <int D, bool FP8, int RT, int NW, int STAGES, int WAVES, bool SPLIT>
__global__ __launch_bounds__(NW * kLanes, WAVES) void attend_kernel(Args a) {
    using T = Tile<D, FP8>;
    constexpr int kRows = 32 * RT;
    constexpr int kIssue = Loads<D, FP8, 1>::kIssue;
    constexpr int kStage = 2 * T::bytes + (FP8 ? 256 : 0);
    constexpr int kRing = kStage * NW;
    __shared__ __attribute__((aligned(1024))) uint8_t ring0[kRing], ring1[kRing],
        ring2[STAGES > 2 ? kRing : 16], ring3[STAGES > 3 ? kRing : 16];
    __shared__ float stat[NW][kRows][2];
    const int lane = threadIdx.x & (kLanes - 1);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kLanes);
    const int r = lane & 31, g = lane >> 5;
    const uint32_t mine = wave * kStage;
    Run run;
    if (!run.begin(a)) return;
    Places<D, FP8> at;
    at.set(lane);

    do {
        const Item o = run.take(a);
        if (o.end <= o.first) continue;
        const Seq& s = run.s;
        const int rows = s.tokens * a.G, stop = run.stop(a, o, kRows), plain = run.plain(a, o, kRows, stop);
        v8bf q[RT][D / 16];
        Mask mask[RT];
        Sums<D> sums[RT];
        #pragma unroll
        for (int t = 0; t < RT; t++) {
            const int row = o.tile * kRows + 32 * t + r;
            mask[t].token = row < rows ? row / a.G : -1;
            mask[t].start = s.start;
            load_query<D, FP8>(a.q + (int64_t)(s.start + mask[t].token) * a.q_stride + (int64_t)(o.h * a.G + row % a.G) * D,
                               row < rows, q[t]);
            sums[t].clear();
        }
        auto compute = [&](auto MASKED, int u, uint32_t exists, Lds stage) {
            #pragma unroll
            for (int t = 0; t < RT; t++) {
                mask[t].before = min(s.context - u * kUnit, kUnit);
                mask[t].exists = exists;
                attend_unit<D, FP8, decltype(MASKED)::value, SPLIT>(a, at, stage + mine, stage + mine + 2 * T::bytes, q[t], sums[t], mask[t]);
                // (the second tile reads the stage again: its operands in registers from one
                // tile to the next would be more than there are)
                __builtin_amdgcn_sched_barrier(0);
                asm volatile("" ::: "memory");
            }
        };

        const Lds rings[4] = {(Lds)ring0, (Lds)ring1, (Lds)ring2, (Lds)ring3};
        uint32_t exists[STAGES];
        Lookup la, lb;
        auto fetch = [&](int v, int i) {   // unit v, whose lookup is la, into stage i
            const Lookup l = la;
            la = lb;
            lb = look_up(a, run, v + 2 * NW, stop);
            Loads<D, FP8, 1> loads;
            exists[i] = loads.find(a, l, o.h);
            loads.issue(a, rings[i] + mine, rings[i] + mine + 2 * T::bytes);
        };
        auto begin = [&](int v) {
            la = look_up(a, run, v, stop);
            lb = look_up(a, run, v + NW, stop);
            #pragma unroll
            for (int i = 0; i < STAGES; i++) fetch(v + i * NW, i);
        };
        const int u0 = o.first + wave;
        int u = u0;
        begin(u0);
        // Plain units, a round of the stages at a time (an exit between two stages would
        // make the compiler wait for all loads in each).
        uint32_t whole = 0xFFFFFFFFu;
        while (u + (STAGES - 1) * NW < plain) {
            #pragma unroll
            for (int i = 0; i < STAGES; i++) {
                wait_loads<(STAGES - 1) * kIssue>();
                whole &= exists[i];
                compute(std::false_type{}, u, 0, rings[i]);
                // (the reads of this stage have come: the products have used them)
                fetch(u + STAGES * NW, i);
                __builtin_amdgcn_sched_barrier(0);
                u += NW;
            }
        }
        if (__builtin_amdgcn_readfirstlane(whole) != 0xFFFFFFFFu) {
            // some of them were of pages that do not exist: all over again, slot by slot
            wait_loads<0>();
            #pragma unroll
            for (int t = 0; t < RT; t++) sums[t].clear();
            u = u0;
            begin(u);
        }
        // The others: they lie in the stages from the first on.
        while (true) {
            wait_loads<0>();
            for (int i = 0; i < STAGES && u < stop; i++, u += NW) {
                const Lds stage = i == 0 ? rings[0] : i == 1 ? rings[1] : i == 2 ? rings[2] : rings[3];
                uint32_t e = exists[0];
                #pragma unroll
                for (int k = 1; k < STAGES; k++) e = i == k ? exists[k] : e;
                compute(std::true_type{}, u, e, stage);
            }
            if (u >= stop) break;
            #pragma unroll
            for (int i = 0; i < STAGES; i++) fetch(u + i * NW, i);
        }

        // The waves' sums are added in wave order, brought to the largest of their maxima.
        const Target to = target<D>(a, run, o, kRows);
        #pragma unroll
        for (int t = 0; t < RT; t++) {
            sums[t].l = sum_of(sums[t].l);
            if (g == 0) {
                stat[wave][32 * t + r][0] = sums[t].m;
                stat[wave][32 * t + r][1] = sums[t].l;
            }
        }
        __syncthreads();   // (all waves' loads into the ring have come, and their reads)
        constexpr int kHold = 32 * RT * D * 4;   // bytes of a wave's sums
        auto held = [&](int w) {   // (rings of whole waves' sums)
            constexpr int kPer = kRing / kHold;
            static_assert(kPer >= 1 && kPer * STAGES >= NW, "the rings hold the sums");
            const int i = w / kPer;
            return (i == 0 ? rings[0] : i == 1 ? rings[1] : i == 2 ? rings[2] : rings[3]) + w % kPer * kHold;
        };
        const Lds hold = held(wave);
        #pragma unroll
        for (int t = 0; t < RT; t++) {
            float top = kNone;
            #pragma unroll
            for (int w = 0; w < NW; w++) top = fmaxf(top, stat[w][32 * t + r][0]);
            const float by = sums[t].m == kNone ? 0.0f : __builtin_amdgcn_exp2f((sums[t].m - top) * a.c);
            #pragma unroll
            for (int n = 0; n < D / 32; n++)
                #pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int row = 32 * t + r, piece = 8 * n + 2 * i + g;
                    const v16f& x = sums[t].acc[n];
                    *(TANS_LDS v4f*)(hold + row * D * 4 + (piece ^ (row & 15)) * 16) =
                        v4f{x[4 * i] * by, x[4 * i + 1] * by, x[4 * i + 2] * by, x[4 * i + 3] * by};
                }
        }
        __syncthreads();
        const int valid = min(kRows, rows - o.tile * kRows);
        for (int x = threadIdx.x; x < valid * (D / 4); x += NW * kLanes) {
            const int row = x / (D / 4), piece = x % (D / 4);
            float top = kNone, sum = 0.0f;
            #pragma unroll
            for (int w = 0; w < NW; w++) top = fmaxf(top, stat[w][row][0]);
            v4f f = {0, 0, 0, 0};
            #pragma unroll
            for (int w = 0; w < NW; w++) {
                const float mw = stat[w][row][0];
                sum += mw == kNone ? 0.0f : stat[w][row][1] * __builtin_amdgcn_exp2f((mw - top) * a.c);
                f += lds_read<v4f>(held(w) + row * D * 4 + (piece ^ (row & 15)) * 16);
            }
            if (to.parts) {
                *reinterpret_cast<v4f*>(to.part_o + row * D + piece * 4) = f;
                if (piece == 0) {
                    to.part_s[row * 2] = top;
                    to.part_s[row * 2 + 1] = sum;
                }
            } else {
                const float by = sum == 0.0f ? 0.0f : 1.0f / sum;
                *reinterpret_cast<v2u*>(to.out + out_row(a, run, o, o.tile * kRows + row) * D + piece * 4) =
                    v2u{bf16_pack(f[0] * by, f[1] * by), bf16_pack(f[2] * by, f[3] * by)};
            }
        }
        if (run.left > 0) __syncthreads();   // (before the ring is filled again)
    } while (run.go_on(a));
}

// Many rows: each of NW waves takes 32 rows of the tile and all units, which pass through
// LDS once for all of them.  A unit's products with K run beside the exponentials of the
// one before in the same wave's instructions, step by step (a step is a matrix instruction
// and what goes beside it), and where the registers hold it (WAVES) two waves a SIMD fill
// each other's gaps.  2048 tokens of 40 heads over 14000 slots and themselves, D = 128: 672 us,
// 938 TFLOP/s (D = 64 440 us, D = 256 with 16 heads 605, 8 bits 758).  The matrix cores are busy
// 43% of the cycles; a quarter of the waves' time is waits (the unit's barrier and LDS), a
// third waits for its turn to issue.  Two tiles of 32 rows a wave and one wave a SIMD, which
// reads LDS half as often, took 893 us.
template <int D, bool FP8, int NW, int WAVES, bool PAGED>
__global__ __launch_bounds__(NW * kLanes, WAVES) void attend_rows_kernel(Args a) {
    using T = Tile<D, FP8>;
    constexpr int STAGES = 4;
    constexpr int kRows = 32 * NW;
    constexpr int kIssue = Loads<D, FP8, NW>::kIssue;
    constexpr int kStage = 2 * T::bytes + (FP8 ? 256 * NW : 0);
    constexpr int kSteps = D / 16;   // products with K, and with V, of a unit and 32 rows
    __shared__ __attribute__((aligned(1024))) uint8_t ring0[kStage], ring1[kStage], ring2[kStage], ring3[kStage];
    const Lds rings[4] = {(Lds)ring0, (Lds)ring1, (Lds)ring2, (Lds)ring3};
    const int lane = threadIdx.x & (kLanes - 1);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kLanes);
    const int r = lane & 31, g = lane >> 5;
    const uint32_t my_scales = 2 * T::bytes + wave * 256;
    Run run;
    if (!run.begin(a)) return;
    Places<D, FP8> at;
    at.set(lane);

    do {
        const Item o = run.take(a);
        if (o.end <= o.first) continue;
        const Seq& s = run.s;
        const int rows = s.tokens * a.G, row = o.tile * kRows + wave * 32 + r;
        const int stop = run.stop(a, o, kRows), plain = run.plain(a, o, kRows, stop);
        v8bf q[D / 16];
        Mask mask;
        Sums<D> sums;
        mask.token = row < rows ? row / a.G : -1;
        mask.start = s.start;
        load_query<D, FP8>(a.q + (int64_t)(s.start + mask.token) * a.q_stride + (int64_t)(o.h * a.G + row % a.G) * D,
                           row < rows, q);
        sums.clear();
        uint32_t exists[STAGES];
        Lookup la, lb;
        Loads<D, FP8, NW> loads;
        auto find = [&](int v, int i) {   // unit v, whose lookup is la, into stage i
            const Lookup l = la;
            la = lb;
            lb = look_up(a, run, v + 2, stop);
            exists[i] = loads.find(a, l, o.h);
        };
        auto issue = [&](int i) { loads.issue(a, rings[i], rings[i] + my_scales); };
        auto begin = [&](int v) {
            la = look_up(a, run, v, stop);
            lb = look_up(a, run, v + 1, stop);
            #pragma unroll
            for (int i = 0; i < STAGES; i++) {
                find(v + i, i);
                issue(i);
            }
        };
        int u = o.first;
        if (u < stop) begin(u);

        // Plain units: the first, and then rounds of the stages.
        uint32_t whole = 0xFFFFFFFFu;
        if (plain > u) {
            v16f sc[2];
            v4u kr[kSteps], vr[kSteps];   // operands (8 bits: as they were read)
            float ks[FP8 ? 16 : 1], vs[FP8 ? 16 : 1], e[16], mc = 0.0f;
            uint32_t p[8];
            auto read_k = [&](Lds stage, int j) {
                if (!FP8 || j % 2 == 0) kr[j] = at.read_k(stage, j);
            };
            auto read_v = [&](Lds stage, int x) { vr[x] = at.read_v(stage, x % (D / 32), x / (D / 32)); };
            auto with_k = [&](v16f& to, int j) {
                const v4u& x = kr[FP8 ? j / 2 * 2 : j];
                v16f zero = {};
                to = mfma(FP8 ? from_fp8(x[2 * (j % 2)], x[2 * (j % 2) + 1]) : __builtin_bit_cast(v8bf, x), q[j],
                          j == 0 ? zero : to);
            };
            auto with_v = [&](int x) {
                const uint32_t* w = p + x / (D / 32) * 4;
                v16f& to = sums.acc[x % (D / 32)];
                to = mfma(FP8 ? from_fp8(vr[x][0], vr[x][1]) : __builtin_bit_cast(v8bf, vr[x]),
                          __builtin_bit_cast(v8bf, v4u{w[0], w[1], w[2], w[3]}), to);
            };
            auto step = [] {
                __builtin_amdgcn_sched_barrier(0);
                asm volatile("" ::: "memory");
            };
            // The exponentials of a unit's scores: the first half in steps 0 .. kSteps - 1, beside the
            // next unit's products with K, the others in half as many, beside the first half's
            // products with V.
            auto exponential = [&](v16f& x, int c) {
                e[c] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[c], a.c, -mc));
                sums.l += e[c];
                if constexpr (FP8) e[c] *= vs[c];
                if (c % 2) p[c / 2] = bf16_pack(e[c - 1], e[c]);
            };
            auto first_half = [&](v16f& x, int i) {
                if (i == 0) {
                    if constexpr (FP8)
                        #pragma unroll
                        for (int c = 0; c < 16; c++) x[c] *= ks[c];
                    mc = sums.admit(x, a.c);
                } else {
                    #pragma unroll
                    for (int c = 8 * (i - 1) / (kSteps - 1); c < 8 * i / (kSteps - 1); c++) exponential(x, c);
                }
            };
            auto second_half = [&](v16f& x, int i) {
                constexpr int n = kSteps / 2;
                if (i < n)
                    #pragma unroll
                    for (int c = 8 + 8 * i / n; c < 8 + 8 * (i + 1) / n; c++) exponential(x, c);
            };
            auto scales = [&](Lds stage) {
                if constexpr (FP8) {
                    read_scales(stage + my_scales, ks);
                    read_scales(stage + my_scales + 128, vs);
                }
            };

            arrive<2 * kIssue>();   // the first two units
            #pragma unroll
            for (int j = 0; j < kSteps; j++) read_k(rings[0], j);
            scales(rings[0]);
            #pragma unroll
            for (int j = 0; j < kSteps; j++) with_k(sc[0], j);
            whole &= exists[0];
            #pragma unroll
            for (int j = 0; j < kSteps; j++) read_k(rings[1], j);
            PagedLoads<D, FP8, NW> pages;
            if constexpr (PAGED) {
                pages.set();
                pages.look_up(a, run, u + STAGES, stop);
            }
            for (int n = (plain - u - 1) / STAGES; n > 0; n--) {
                #pragma unroll
                for (int i = 0; i < STAGES; i++, u++) {   // unit u, in stage i
                    whole &= exists[(i + 1) % STAGES];
                    #pragma unroll
                    for (int j = 0; j < kSteps; j++) {
                        with_k(sc[(i + 1) % 2], j);
                        first_half(sc[i % 2], j);
                        // (LDS answers in order: find() after K's reads, before V's)
                        constexpr int kAt = kSteps / 4;
                        if (!PAGED && j == kAt) find(u + STAGES, i);
                        if (j > kAt && 2 * (j - kAt - 1) < kSteps) {
                            read_v(rings[i], 2 * (j - kAt - 1));
                            read_v(rings[i], 2 * (j - kAt - 1) + 1);
                        }
                        step();
                    }
                    arrive<kIssue>();   // unit u + 2; unit u has been read
                    if constexpr (PAGED) {
                        exists[i] = pages.issue(a, o.h, rings[i], rings[i] + my_scales) ? 0xFFFFFFFFu : 0;
                        pages.look_up(a, run, u + STAGES + 1, stop);
                    } else {
                        issue(i);
                    }
                    #pragma unroll
                    for (int j = 0; j < kSteps; j++) {
                        with_v(j);
                        second_half(sc[i % 2], j);
                        read_k(rings[(i + 2) % STAGES], j);
                        if (j == kSteps - 1) scales(rings[(i + 1) % STAGES]);
                        step();
                    }
                }
            }
            // the last one's rest
            #pragma unroll
            for (int x = 0; x < kSteps; x++) read_v(rings[0], x);
            #pragma unroll
            for (int i = 0; i < kSteps; i++) first_half(sc[0], i);
            #pragma unroll
            for (int i = 0; i < kSteps; i++) second_half(sc[0], i);
            #pragma unroll
            for (int x = 0; x < kSteps; x++) with_v(x);
            u++;
            arrive<0>();   // (before the ring is filled again)
            if (__builtin_amdgcn_readfirstlane(whole) != 0xFFFFFFFFu) {
                // some of them were of pages that do not exist: all over again, slot by slot
                sums.clear();
                u = o.first;
            }
            if (u < stop) begin(u);
        }
        // The others: they lie in the stages from the first on.
        while (u < stop) {
            arrive<0>();
            for (int i = 0; i < STAGES && u < stop; i++, u++) {
                const Lds stage = i == 0 ? rings[0] : i == 1 ? rings[1] : i == 2 ? rings[2] : rings[3];
                mask.before = min(s.context - u * kUnit, kUnit);
                mask.exists = exists[0];
                #pragma unroll
                for (int k = 1; k < STAGES; k++) mask.exists = i == k ? exists[k] : mask.exists;
                attend_unit<D, FP8, true, false>(a, at, stage, stage + my_scales, q, sums, mask);
            }
            arrive<0>();   // (before the ring is filled again)
            if (u < stop) {
                #pragma unroll
                for (int i = 0; i < STAGES; i++) {
                    find(u + i, i);
                    issue(i);
                }
            }
        }

        const Target to = target<D>(a, run, o, kRows);
        const float l = sum_of(sums.l);
        const int local = row - o.tile * kRows;
        if (row < rows) {
            const float by = l == 0.0f ? 0.0f : 1.0f / l;
            if (to.parts && g == 0) {
                to.part_s[local * 2] = sums.m;
                to.part_s[local * 2 + 1] = l;
            }
            uint16_t* out = to.out + out_row(a, run, o, row) * D;
            #pragma unroll
            for (int n = 0; n < D / 32; n++)
                #pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int d = 32 * n + 8 * i + 4 * g;
                    const v16f& c = sums.acc[n];
                    const v4f x = {c[4 * i], c[4 * i + 1], c[4 * i + 2], c[4 * i + 3]};
                    if (to.parts)
                        *reinterpret_cast<v4f*>(to.part_o + local * D + d) = x;
                    else
                        *reinterpret_cast<v2u*>(out + d) = v2u{bf16_pack(x[0] * by, x[1] * by), bf16_pack(x[2] * by, x[3] * by)};
                }
        }
    } while (run.go_on(a));
}

// The rows of items that several workgroups share, from their parts in the order of the
// slots: a workgroup for ROWS rows (y) of each run that could be the first of several (x).
// A thread has 4 dimensions of a row's parts; threads that the rows leave share the parts.
template <int D, int ROWS>
__global__ __launch_bounds__(256) void join_kernel(Args a) {
    const Cut cut = a.cuts[blockIdx.x];
    const int first = (int)blockIdx.y * ROWS;
    const int end = min(min(a.work.rows, cut.rows - cut.tile * a.work.rows), first + ROWS);
    if (cut.last < 0 || first >= end) return;
    constexpr int T = D / 4, kTeams = 256 / T;   // threads of a row's part
    __shared__ __attribute__((aligned(16))) float sums[kTeams][D], total[kTeams];
    const int w0 = blockIdx.x, n = cut.last - w0 + 1;
    constexpr int share = kTeams > ROWS ? kTeams / ROWS : 1;   // teams that share a row
    const float* stats = a.parts + (int64_t)a.work.groups * 2 * a.work.rows * D;
    const int team = threadIdx.x / T, t = threadIdx.x % T, mine = team % share;
    for (int row0 = first; row0 < end; row0 += kTeams / share) {
        const int local = row0 + team / share;
        if (local < end) {
            // (a run's first item is its part 0 if it began in another's, its last one part 1)
            auto slot = [&](int i) { return ((int64_t)(w0 + i) * 2 + (i ? 0 : 1)) * a.work.rows + local; };
            float top = kNone;
            #pragma unroll 8
            for (int i = 0; i < n; i++) top = fmaxf(top, stats[slot(i) * 2]);
            float sum = 0.0f;
            v4f o = {0, 0, 0, 0};
            #pragma unroll 8
            for (int i = mine; i < n; i += share) {
                const float m = stats[slot(i) * 2];
                const float by = m == kNone ? 0.0f : __builtin_amdgcn_exp2f((m - top) * a.c);
                sum += stats[slot(i) * 2 + 1] * by;
                o += *reinterpret_cast<const v4f*>(a.parts + slot(i) * D + t * 4) * by;
            }
            *reinterpret_cast<v4f*>(&sums[team][t * 4]) = o;
            if (t == 0) total[team] = sum;
        }
        __syncthreads();
        if (local < end && mine == 0) {
            float sum = 0.0f;
            v4f o = {0, 0, 0, 0};
            for (int i = 0; i < share; i++) {
                sum += total[team + i];
                o += *reinterpret_cast<const v4f*>(&sums[team + i][t * 4]);
            }
            const float by = sum == 0.0f ? 0.0f : 1.0f / sum;
            const int row = cut.tile * a.work.rows + local;
            uint16_t* out = a.out + ((int64_t)(cut.start + row / a.G) * a.Hq + cut.h * a.G + row % a.G) * D + t * 4;
            *reinterpret_cast<v2u*>(out) = v2u{bf16_pack(o[0] * by, o[1] * by), bf16_pack(o[2] * by, o[3] * by)};
        }
        __syncthreads();
    }
}

}  // namespace

extern "C" {

int tans_tree_attention_workspace(int64_t N, int64_t B, int64_t q_heads, int64_t heads, int64_t dim,
                                  int64_t slots, int64_t max_tokens, int64_t* bytes) {
    if (!bytes) return fail(TANS_EINVAL, "tree_attention: null pointer");
    if (N < 0 || B < 0 || heads < 1 || q_heads < heads || q_heads % heads || q_heads > 65535 ||
        (dim != 64 && dim != 128 && dim != 256) || slots < 0 || slots > INT32_MAX || max_tokens < 0 ||
        N > INT32_MAX / 2 || N > INT32_MAX / q_heads || B >= INT32_MAX)
        return fail(TANS_EINVAL, "tree_attention: sizes out of range");
    const int cus = tans_internal_cu_count();
    // (an 8-bit cache takes no less)
    *bytes = N && B ? plan(N, B, q_heads, heads, dim, true, slots, max_tokens, cus > 0 ? cus : 256).bytes : 0;
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
    if (mask && (mask_cols < 1 || mask_cols > INT32_MAX))
        return fail(TANS_EINVAL, op + ": the mask must have 1 .. 2^31 - 1 columns");
    if (!(scale > 0.0f) || scale > 1.0e38f) return fail(TANS_EINVAL, op + ": scale must be positive and finite");
    if (max_tokens < 0) return fail(TANS_EINVAL, op + ": max_tokens must not be negative");
    if (N > INT32_MAX / q_heads) return fail(TANS_EINVAL, op + ": N times the query heads must be below 2^31");
    if (N == 0 || B == 0) return TANS_OK;
    if (!q || !out) return fail(TANS_EINVAL, op + ": null pointer");
    rc = stride_check(op, "q", q, q_stride, q_heads * dim);
    if (rc == TANS_OK && !aligned(out, 16)) rc = fail(TANS_EINVAL, op + ": out is misaligned (16 bytes)");
    if (rc != TANS_OK) return rc;
    const int cus = tans_internal_cu_count();
    if (cus <= 0) return fail(TANS_EHIP, op + ": cannot query the device's CU count");
    const Plan p = plan(N, B, q_heads, heads, dim, k_scale != nullptr, per * page, max_tokens, cus);
    if (p.bytes > 0 && (!workspace || !aligned(workspace, 16) || workspace_bytes < p.bytes))
        return fail(TANS_EINVAL, op + ": workspace too small, null or misaligned (16 bytes)");
    if (p.blocks > INT32_MAX / 256) return fail(TANS_EINVAL, op + ": too many tokens for one call");
    Args a = {};
    a.batch = make_batch(table, starts, lens, B, per, N, pages, heads, page);
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
    a.cuts = (Cut*)((char*)workspace + p.parts_bytes);
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
        constexpr int pair_stages = 2 * stages * stage <= (160 << 10) ? stages : 2;
        int rc;
        if (p.kind == kFew) {
            rc = TANS_EINVAL;
            if constexpr (few_pairs(D, f8))
                if (p.pairs) rc = launch(attend_kernel<D, f8, 1, nw, pair_stages, 2, !f8>, nw * kLanes);
            if (!p.pairs)
                rc = p.work.whole ? launch(attend_kernel<D, f8, 1, nw, stages, 1, false>, nw * kLanes)
                                  : launch(attend_kernel<D, f8, 1, nw, stages, 1, !f8>, nw * kLanes);
        } else if (p.kind == kMany) {
            if constexpr (D == 256)
                rc = page % 16 == 0 ? launch(attend_rows_kernel<D, f8, 4, 1, true>, 4 * kLanes)
                                    : launch(attend_rows_kernel<D, f8, 4, 1, false>, 4 * kLanes);
            else
                rc = launch(attend_rows_kernel<D, f8, 4, 2, false>, 4 * kLanes);
        } else {
            if constexpr (D < 256) {
                if (p.kind == kSome) rc = launch(attend_kernel<D, f8, 2, nw, stages, 1, false>, nw * kLanes);
                else rc = launch(attend_rows_kernel<D, f8, 8, 2, false>, 8 * kLanes);
            } else {
                rc = fail(TANS_EINVAL, "tree_attention: no such kernel");   // (not reached: plan())
            }
        }
        if (rc == TANS_OK && !p.work.whole && p.work.groups > 1) {
            auto join = [&](auto kernel, int rows) {
                hipLaunchKernelGGL(kernel, dim3(p.work.groups - 1, p.work.rows / rows), dim3(256), 0, (hipStream_t)stream, a);
            };
            if (p.work.rows <= 64) join(join_kernel<D, 4>, 4);
            else join(join_kernel<D, 8>, 8);
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
