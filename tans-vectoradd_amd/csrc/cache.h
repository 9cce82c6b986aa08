// The paged cache of keys and values and the packed batch that reads and writes it:
// what positions.hip and attention.hip share.  (Which row is whose: cache_rows.h.)
#ifndef TANS_CACHE_H
#define TANS_CACHE_H

#include <stdint.h>

#include <string>

#include "cache_rows.h"
#include "layer.h"

namespace {

using tans_cache::Batch;

// The last sequence that starts at or before row n, or -1.
__device__ __forceinline__ int find_sequence(const Batch& batch, int n) {
    const int lane = threadIdx.x & (kLanes - 1);
    return tans_cache::find_sequence(batch.B, [&](int lo, int step, int hi) {
        const int64_t i = lo + (int64_t)(lane + 1) * step - 1;
        return (int)__popcll(__builtin_amdgcn_ballot_w64(i < hi && batch.starts[i] <= n));
    });
}

// Host side ---------------------------------------------------------------

inline Batch make_batch(const int32_t* table, const int32_t* starts, const int32_t* lens, int64_t B,
                        int64_t per, int64_t N, int64_t pages, int64_t heads, int64_t page) {
    Batch b = {};
    b.table = table;
    b.starts = starts;
    b.lens = lens;
    b.B = (int)B;
    b.per = (int)per;
    b.N = (int)N;
    b.pages = (uint32_t)pages;
    b.heads = (uint32_t)heads;
    b.set_page((uint32_t)page);
    return b;
}

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
