// The paged cache of keys and values and the packed batch that reads and writes it:
// what positions.hip and attention.hip share.
//
// The cache holds `pages` pages of `page` rows for each of `heads` heads:
// [pages][heads][page][dim], bf16, or E4M3FN bytes with a float scale per row.  A
// page's rows of one head are contiguous, so that a head's workgroup reads runs of
// whole pages.
//
// Slot s of sequence b is row s % page of page table[b][s / page].  A batch's tokens
// are packed: rows starts[b] .. starts[b + 1] - 1 are sequence b's, and token t of
// them has slot lens[b] + t.  These numbers lie in device memory, where the host does
// not see them, so the kernels bound each of them: no value makes an access leave
// the buffers.
#ifndef TANS_CACHE_H
#define TANS_CACHE_H

#include <stdint.h>

#include <string>

#include "layer.h"

namespace {

struct Batch {
    const int32_t* table;    // [B][per]: pages
    const int32_t* starts;   // [B + 1]
    const int32_t* lens;     // [B]
    int B, per, N;           // N: rows of q
    uint32_t pages, heads, page;

    __device__ __forceinline__ int64_t capacity() const { return (int64_t)per * page; }
    __device__ __forceinline__ int start(int b) const {
        const int s = starts[b];
        return s < 0 ? 0 : s < N ? s : N;
    }
    // tokens and slots before them (neither is negative; the slots within the table's)
    __device__ __forceinline__ int tokens(int b) const {
        const int n = start(b + 1) - start(b);
        return n > 0 ? n : 0;
    }
    __device__ __forceinline__ int context(int b) const {
        const int64_t c = lens[b];
        return (int)(c < 0 ? 0 : c < capacity() ? c : capacity());
    }
    // Row of the cache (of all heads' and pages') of slot s < capacity() and head h;
    // false if the table's entry is no page.
    __device__ __forceinline__ bool row(int b, uint32_t s, uint32_t h, uint32_t& r) const {
        const uint32_t i = s / page, p = (uint32_t)table[(int64_t)b * per + i];
        r = (p * heads + h) * page + (s - i * page);
        return p < pages;
    }
};

// The last sequence that starts at or before row n, or -1: 64 starts are compared
// at a time, by the lanes of a wave.
__device__ __forceinline__ int find_sequence(const Batch& batch, int n) {
    const int lane = threadIdx.x & (kLanes - 1);
    int lo = 0, hi = batch.B;   // lo of them start at or before n, those from hi on do not
    while (lo < hi) {
        const int step = (hi - lo + kLanes - 1) / kLanes;
        const int i = lo + (lane + 1) * step - 1;
        const bool before = i < hi && batch.starts[i] <= n;
        const int k = __popcll(__builtin_amdgcn_ballot_w64(before));
        const int next = lo + k * step + step - 1;   // the first probe that is not
        lo += k * step;
        hi = next < hi ? next : hi;
    }
    return lo - 1;
}

// Host side ---------------------------------------------------------------

// The batch's sizes and pointers, alike for both operators.
inline int batch_check(const std::string& op, const void* k, const void* v, const void* k_scale,
                       const void* v_scale, int64_t pages, int64_t heads, int64_t page, int64_t dim,
                       const void* table, int64_t per, const void* starts, const void* lens, int64_t B,
                       int64_t N, int64_t q_heads) {
    if (dim != 64 && dim != 128 && dim != 256)
        return fail(TANS_EINVAL, op + ": the heads' dimension must be 64, 128 or 256");
    if (heads < 1 || heads > 65535 || q_heads < heads || q_heads > 65535 || q_heads % heads)
        return fail(TANS_EINVAL, op + ": the query heads must be a multiple of the cache's heads, at most 65535");
    if (pages < 1 || page < 1 || page > (1 << 20) || pages > INT32_MAX ||
        pages * page >= (int64_t(1) << 32) / heads)
        return fail(TANS_EINVAL, op + ": need pages, rows of a page (at most 2^20) and fewer than 2^32 rows in all");
    if (B < 0 || B >= INT32_MAX || per < 0 || per > INT32_MAX / page)
        return fail(TANS_EINVAL, op + ": need B >= 0 and fewer than 2^31 slots a sequence");
    if (N < 0 || N > INT32_MAX / 2) return fail(TANS_EINVAL, op + ": N must be 0 .. 2^30 - 1");
    if (N == 0 || B == 0) return TANS_OK;
    if (!k || !v || !starts || !lens || (per && !table)) return fail(TANS_EINVAL, op + ": null pointer");
    if (!k_scale != !v_scale)
        return fail(TANS_EINVAL, op + ": an 8-bit cache has scales of keys and of values");
    if (!aligned(k, 16) || !aligned(v, 16) || !aligned(k_scale, 4) || !aligned(v_scale, 4) ||
        !aligned(table, 4) || !aligned(starts, 4) || !aligned(lens, 4))
        return fail(TANS_EINVAL, op + ": misaligned buffer (cache 16, others 4 bytes)");
    return TANS_OK;
}

inline int stride_check(const std::string& op, const char* name, const void* p, int64_t stride,
                        int64_t row) {
    if (stride < row || stride % 8 || stride > (int64_t(1) << 40))
        return fail(TANS_EINVAL, op + ": the stride of " + name +
                                     " must be a multiple of 8 elements, at least a row");
    if (!aligned(p, 16)) return fail(TANS_EINVAL, op + ": " + name + " is misaligned (16 bytes)");
    return TANS_OK;
}

}  // namespace

#endif  // TANS_CACHE_H
