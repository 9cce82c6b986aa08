// How the attention of attention.hip is computed, chosen by sizes and the device's CU
// count, and which workgroup takes which part of the work; plain C++.
//
// The rows of an item are a row tile of one sequence and cache head: the new tokens'
// query heads that read it, token by token.  A unit is 32 slots.  The work is a line of
// pieces: sequence by sequence, in it head by head, tile by tile, unit by unit.  Split:
// every workgroup takes an equal run of the pieces, at whose ends an item may be cut;
// the parts of a cut item are joined by a second kernel.  Whole: a workgroup an item.
#ifndef TANS_ATTENTION_PLAN_H
#define TANS_ATTENTION_PLAN_H

#include <stdint.h>

#include <algorithm>

#include "cache_rows.h"   // TANS_BOTH

namespace tans_attention {

constexpr int kUnit = 32;   // slots of a unit

struct Work {
    int rows;      // of a tile
    int groups;    // workgroups, of which as many work as have `least` pieces
    int least;
    int item;      // pieces that an item counts besides its units
    int whole;
    // pieces that no batch exceeds, unless its starts go back: sequences that overlap could hold
    // any number, so they are counted up to here only (what lies behind is not computed)
    int64_t most;
};
constexpr int64_t kMostPieces = int64_t(1) << 50;   // (weeks of work)

TANS_BOTH int row_tiles(int64_t tokens, int64_t G, int rows) {
    return (int)((tokens * G + rows - 1) / rows);
}

// (one at least, so that a row that sees nothing is written)
TANS_BOTH int slot_units(int slots) {
    return slots > 0 ? (int)(((int64_t)slots + kUnit - 1) / kUnit) : 1;
}

// Of row tile `tile` (rows of G query heads a token, token by token) of a sequence of
// `tokens` new ones, `context` slots before them and `slots` in all: the units that are
// computed end at stop, with a mask at `end`, without one behind the slot of the tile's last
// token; below plain, at most stop, all of a unit's slots are the sequence's and every row of
// the tile sees them.
TANS_BOTH int tile_stop(bool masked, int context, int tokens, int slots, int tile, int rows, int G, int end) {
    if (masked) return end;
    const int last = std::min(tokens - 1, (tile * rows + rows - 1) / G);
    return std::min(end, slot_units((int)std::min((int64_t)slots, (int64_t)context + last + 1)));
}
TANS_BOTH int tile_plain(bool masked, int context, int slots, int tile, int rows, int G, int stop) {
    const int64_t seen = (int64_t)context + (masked ? 0 : tile * rows / G + 1);
    return std::min(stop, (int)(std::min((int64_t)slots, seen) / kUnit));
}

// Pieces of a sequence, and of several.
TANS_BOTH int64_t pieces_of(const Work& w, int64_t heads, int tiles, int units) {
    return heads * tiles * (w.whole ? 1 : units + w.item);
}
TANS_BOTH int64_t add_pieces(const Work& w, int64_t all, int64_t more) { return std::min(all + more, w.most); }

// Workgroups that share `all` pieces.
TANS_BOTH int work_groups(const Work& w, int64_t all) {
    const int64_t most = (all + w.least - 1) / w.least;
    return (int)(most < w.groups ? most : w.groups);
}

// First piece of workgroup i < groups, and the workgroup of piece `at`: the last one
// that starts at or before it.  (all is at most kMostPieces, groups are below 2^12; an item
// that is not counted to its end has pieces from all on, which are the last workgroup's.)
TANS_BOTH int64_t range_start(int64_t all, int groups, int i) { return all * i / groups; }
TANS_BOTH int range_of(int64_t all, int groups, int64_t at) {
    // all i / groups <= at, so i < (at + 1) groups / all
    return at < all ? (int)(((at + 1) * groups - 1) / all) : groups - 1;
}

// The run of workgroup i of `groups`: workgroups go to the 8 XCDs in turn, and XCD x takes
// the x-th eighth of the runs (all of them one by one where they do not divide).
constexpr int kXcds = 8;
TANS_BOTH int run_of(int i, int groups) { return groups % kXcds ? i : i % kXcds * (groups / kXcds) + i / kXcds; }

// Rows of q of a tile: 32 or 64, of which each wave takes all and the waves share the
// slots, or 128 or 256, of which each of 4 or 8 waves takes 32 and the slots pass through
// LDS once for all.  256 rows read K and V half as often; below 1024 rows an odd number of
// 128s is taken as such, where the last tile of 256 would be half empty (a tree of 61
// tokens, 305 rows, over 32771 slots: 97 us, 102 with tiles of 256; in 8 bits 88 / 111).
// D = 256 has the registers for 32 rows a wave and one wave a SIMD only.
enum Kind { kFew, kSome, kMany, kMost };
struct Plan {
    Kind kind;
    Work work;
    bool pairs;              // two workgroups a CU
    int64_t blocks, parts_bytes, bytes;   // workgroups; of the parts; of the workspace
};

// Whether a CU's LDS holds the rings of two workgroups of the kernel for few rows.
constexpr bool few_pairs(int64_t dim, bool eight) { return dim * (eight ? 1 : 2) <= 128; }

inline Plan plan(int64_t N, int64_t B, int64_t q_heads, int64_t heads, int64_t dim, bool eight,
                 int64_t slots, int64_t max_tokens, int cus) {
    // (any number of tokens may be given: no sequence has more than INT32_MAX)
    const int64_t G = q_heads / heads, rows = std::min<int64_t>(max_tokens, INT32_MAX) * G;
    Plan p = {};
    const bool odd = (rows + 127) / 128 % 2 == 1 && rows < 1024;
    p.kind = rows <= 32 ? kFew : rows <= 64 && dim < 256 ? kSome
             : rows <= 128 || dim == 256 || odd ? kMany : kMost;
    p.work.rows = 32 << p.kind;
    // no more items than this
    const int64_t items = (N * G / p.work.rows + std::min(N, B)) * heads;
    p.work.least = 8;
    p.work.item = p.kind >= kMany ? 8 : (int)(196608 / (2 * kUnit * dim * (eight ? 1 : 2)));
    // An item a workgroup, without a second kernel that joins parts: few slots, up to 24 units
    // where the items are few as well (one token of 760 slots 12.8 us, shared 15.3; of 800 13.8 / 15.3,
    // 1024 15.8 / 15.3; 32 sequences of 512 18.7 / 20.9; but 256 of them 158 / 131, and D = 256, 700
    // slots 27.9 / 22.3), or so many items that they fill the CUs evenly.  (slots are the table's:
    // the host does not know the sequences', and a wider table takes the shared path.)
    p.work.whole = slots <= 8 * kUnit ||
                   (p.kind < kMany && dim < 256 && slots <= 24 * kUnit && items <= 2 * (int64_t)cus) ||
                   (p.kind >= kMany && items >= 4 * (int64_t)cus);
    p.work.most = std::min(p.work.whole ? items : items * (slot_units((int)slots) + p.work.item), kMostPieces);
    if (p.work.whole) {
        p.blocks = items;
        return p;
    }
    // Two workgroups a CU, of which one streams while the other begins or ends an item, but
    // for items that are longer than a run.  D = 128 in 8 bits, two against one: 256 sequences
    // of 512 slots 84 / 119 us, 96 of 100 .. 16000 140 / 137, one of 262144 120 / 110.
    p.pairs = p.kind == kFew && few_pairs(dim, eight) && items > cus;
    p.work.groups = p.pairs || (p.kind == kMany && dim < 256) ? 2 * cus : cus;
    p.blocks = p.work.groups;
    p.parts_bytes = (int64_t)p.work.groups * 2 * p.work.rows * (dim + 2) * 4;
    p.bytes = p.parts_bytes + (int64_t)p.work.groups * 5 * 4;
    return p;
}

}  // namespace tans_attention

#endif  // TANS_ATTENTION_PLAN_H
