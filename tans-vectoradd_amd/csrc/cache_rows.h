// The paged cache of keys and values and the packed batch that reads and writes it:
// which row is whose, in plain C++.
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
#ifndef TANS_CACHE_ROWS_H
#define TANS_CACHE_ROWS_H

#include <stdint.h>

#ifdef __HIPCC__
#define TANS_BOTH __host__ __device__ inline __attribute__((always_inline))
#else
#define TANS_BOTH inline
#endif

namespace tans_cache {

struct Batch {
    const int32_t* table;    // [B][per]: pages
    const int32_t* starts;   // [B + 1]
    const int32_t* lens;     // [B]
    int B, per, N;           // N: rows of q
    uint32_t pages, heads, page;
    // slot / page = (slot * inverse) >> (31 + shift) for slots below 2^31: inverse is 2^(31 +
    // shift) / page rounded up, with 2^shift >= page, so it is too large by less than 1, and the
    // quotient by less than 2^31 / 2^(31 + shift) <= 1 / page
    uint32_t inverse;
    int shift;

    inline void set_page(uint32_t rows) {
        page = rows;
        shift = 0;
        while ((uint32_t(1) << shift) < rows) shift++;
        inverse = (uint32_t)(((uint64_t(1) << (31 + shift)) + rows - 1) / rows);
    }
    TANS_BOTH uint32_t page_of(uint32_t slot) const {
        return (uint32_t)((uint64_t)(2 * slot) * inverse >> 32) >> shift;
    }
    TANS_BOTH int64_t capacity() const { return (int64_t)per * page; }
    TANS_BOTH int start(int b) const {
        const int s = starts[b];
        return s < 0 ? 0 : s < N ? s : N;
    }
    // tokens and slots before them (neither is negative; the slots within the table's)
    TANS_BOTH int tokens(int b) const {
        const int n = start(b + 1) - start(b);
        return n > 0 ? n : 0;
    }
    TANS_BOTH int context(int b) const {
        const int64_t c = lens[b];
        return (int)(c < 0 ? 0 : c < capacity() ? c : capacity());
    }
    // Whether row n is one of sequence b's tokens, for the b that find_sequence gives: -1
    // before the first, and where starts go back maybe one that begins behind the row.
    TANS_BOTH bool owns(int b, int n) const { return b >= 0 && n >= start(b) && n < start(b + 1); }
    // The slot of row n, which sequence b owns; false if it lies past the table's.
    TANS_BOTH bool slot_of(int b, int n, uint32_t& s) const {
        const int64_t i = (int64_t)context(b) + (n - start(b));
        s = (uint32_t)i;
        return i < capacity();
    }
    // Row of the cache (of all heads' and pages') of slot s < capacity() and head h;
    // false if the table's entry is no page.
    TANS_BOTH bool row(int b, uint32_t s, uint32_t h, uint32_t& r) const {
        const uint32_t i = page_of(s), p = (uint32_t)table[(int64_t)b * per + i];
        r = (p * heads + h) * page + (s - i * page);
        return p < pages;
    }
};

// The last sequence that starts at or before row n, or -1.  `before(lo, step, hi)` says
// how many of the starts lo + step - 1, lo + 2 step - 1, .. (64 of them, those below hi)
// are at or before n; the lanes of a wave look at them together.
template <class Before>
TANS_BOTH int find_sequence(int B, Before before) {
    int lo = 0, hi = B;   // lo of them are at or before n, those from hi on are not
    while (lo < hi) {
        const int step = (int)(((int64_t)hi - lo + 63) / 64);
        const int k = before(lo, step, hi);
        const int64_t next = lo + (int64_t)(k + 1) * step - 1;   // the first that is not
        lo += k * step;
        hi = next < hi ? (int)next : hi;
    }
    return lo - 1;
}

}  // namespace tans_cache

#endif  // TANS_CACHE_ROWS_H
