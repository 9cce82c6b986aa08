// How the FP8 product of linear.hip is computed, chosen by sizes and the
// device's CU count, and which workgroup takes which tile; plain C++.
#ifndef TANS_LINEAR_PLAN_H
#define TANS_LINEAR_PLAN_H

#include <stdint.h>

#include <algorithm>

namespace tans_linear {

constexpr int kStep = 128;   // columns (bytes) of a step

// How a product is computed.
enum Kind { kStream, kMid, kTiles };
struct Plan {
    Kind kind;
    bool few;       // kStream: few rows of w, one group of 16 a workgroup
    int mi, nw;     // kMid: 32 mi rows of a by 32 nw rows of w
    int splits;     // kMid
    bool pairs;     // kMid: two workgroups a CU
    int64_t tiles_m, tiles_n, Np;
    int64_t bytes;  // of partial sums
};

// Tiles by their rows, with what a step of 128 columns and a round of tiles on
// all CUs take besides, in us: least squares over 1,300 timings of 130 products
// of random sizes (17 .. 4096 rows of a, w up to 178 MB from memory) on 256
// CUs.  The choice that these figures give is on average 3% slower than the
// fastest of all that were timed (at most 29%), any single tile 25% and more.
struct Tile { int mi, nw; float step, round; };
constexpr Tile kMids[] = {
    {1, 2, 0.29f, 0.4f}, {1, 4, 0.50f, 0.2f}, {2, 4, 0.56f, 1.4f}, {2, 5, 0.70f, 1.7f},
    {3, 4, 0.65f, 2.0f}, {4, 4, 0.72f, 3.0f}, {4, 5, 0.88f, 3.7f}, {4, 6, 0.97f, 2.8f},
    {4, 8, 1.21f, 2.2f}, {6, 5, 1.22f, 4.3f}};
// The large tiles: 256 rows of a by 256, or not gated 192, rows of w.  Down
// 5120 x 17408: 2048 rows of a 172 / 156 us, 4096 350 / 305; 3000 by 5120 x
// 5120 80 / 106, 1500 70 / 55.
// A gated tile's epilogue takes longer (512 rows by 34816 x 5120: two rounds of
// these 134 us, three of 128 x 192 119).
constexpr Tile kBig = {8, 8, 1.15f, 12.0f}, kBigGated = {8, 8, 1.15f, 18.0f},
               kBig192 = {8, 6, 1.05f, 4.0f};
constexpr float kLaunch = 4.0f, kJoin = 2.9f;        // us: a call; the second kernel
constexpr float kReadRate = 5.9e6f;                  // bytes of w a us
constexpr float kSumRate = 4.6e6f;                   // bytes of partial sums a us
constexpr int kMaxSplits = 16;

inline Plan plan(int64_t M, int64_t N, int64_t C, bool gated, int cus) {
    auto parts = [](int64_t n, int64_t of) { return (n + of - 1) / of; };
    const int64_t halves = gated ? 2 : 1, w_bytes = N * halves * C;
    Plan p = {};
    p.splits = 1;
    // Up to 16 rows, the instruction's; up to 32 while w is small: 24 rows by
    // 6806 x 5232 (gated) 12.6 us against 15.5 by tiles, by 34816 x 5120 38.0
    // against 31.6.
    if (M <= 16 || (M <= 32 && w_bytes <= (int64_t(40) << 20))) {
        p.kind = kStream;
        // 16 rows a workgroup, its loads twice as deep, while 32 would leave
        // half of the CUs idle: one row by 1024 x 8192 5.4 us against 8.1, by
        // 4096 x 4096 6.1 against 6.0, by 7000 x 4096 8.3 against 7.3.
        p.few = !gated && 2 * parts(N, 32) <= cus;
        return p;
    }
    const int64_t steps = parts(C, kStep);
    // Few steps and many tiles: tiles of 128 x 128, two to a CU, if they are
    // mostly filled.  Of 27 random products of 1 to 6 steps 10% faster on
    // average than the choice below (at most 30%: 1101 rows by 15045 x 528 with
    // residual 44.8 us against 63.5; 4591 by 15173 x 272 132 against 157), 18%
    // slower at worst; of 8 and more steps slower.
    const int64_t m4 = parts(M, 128), n4 = parts(N, 128 / halves);
    if (steps <= 6 && m4 * n4 >= 2 * cus && 4 * M >= 3 * 128 * m4 && m4 * n4 <= INT32_MAX / 256) {
        p.kind = kMid;
        p.pairs = true;
        p.mi = p.nw = 4;
        p.tiles_m = m4;
        p.tiles_n = n4;
        return p;
    }
    float best = 0.0f;
    auto consider = [&](Kind kind, const Tile& t, int splits) {
        const int64_t tm = parts(M, 32 * t.mi), tn = parts(N, 32 * t.nw / halves);
        // (a launch has fewer than 2^31 threads; the large tiles' stay)
        if (kind == kMid && tm * tn * splits > INT32_MAX / (64 * t.nw)) return;
        const float rounds = (float)parts(tm * tn * splits, cus);
        float us = kLaunch + rounds * (t.round + (float)parts(steps, splits) * t.step);
        us = std::max(us, kLaunch + 1.0f + (float)w_bytes / kReadRate);
        if (splits > 1) us += kJoin + (float)splits * (float)(M * N * halves) * 8.0f / kSumRate;
        if (best > 0.0f && us >= best) return;
        best = us;
        p.kind = kind;
        p.mi = t.mi;
        p.nw = t.nw;
        p.splits = splits;
        p.tiles_m = tm;
        p.tiles_n = tn;
    };
    consider(kTiles, gated ? kBigGated : kBig, 1);
    if (!gated) consider(kTiles, kBig192, 1);
    for (const Tile& t : kMids) {
        for (int s = 1; s <= kMaxSplits && (s == 1 || steps >= 3 * s); s++) consider(kMid, t, s);
    }
    if (p.kind == kMid && p.splits > 1) {
        p.Np = parts(N, 16) * 16;
        p.bytes = p.splits * M * halves * p.Np * 4;
    }
    return p;
}

// Workgroups run on XCD (block % 8): a permutation of the blocks that gives each
// XCD a run of neighbours.
constexpr int kXcds = 8;
constexpr int xcd_order(int block, int blocks) {
    const int xcd = block % kXcds, per = blocks / kXcds, more = blocks % kXcds;
    return xcd * per + (xcd < more ? xcd : more) + block / kXcds;
}

// Where a persistent workgroup's tiles lie: the tile sequence takes groups of
// kGroupM tiles of a's rows, in each of them w's tiles in order and the group's
// row tiles innermost; an eighth of the sequence goes to each of the 8 XCDs
// (workgroup b runs on XCD b % 8), so that the tiles an XCD works on at a time
// share their rows of a and w in its L2.
constexpr int kGroupM = 8;

struct TileMap {
    int tiles_m, tiles_n;
    constexpr int count() const { return tiles_m * tiles_n; }
    // the i-th tile of workgroup b of `blocks`, or -1
    constexpr int at(int i, int b, int blocks) const {
        const int xcd = b % kXcds, T = count();
        const int per = T / kXcds, more = T % kXcds;
        const int first = xcd * per + (xcd < more ? xcd : more);
        const int n = per + (xcd < more ? 1 : 0);
        const int peers = (blocks - xcd + kXcds - 1) / kXcds;
        const int k = i * peers + b / kXcds;
        return k < n ? first + k : -1;
    }
    constexpr void place(int t, int& tm, int& tn) const {
        const int group = t / (kGroupM * tiles_n);
        const int m_first = group * kGroupM;
        const int gm = tiles_m - m_first < kGroupM ? tiles_m - m_first : kGroupM;
        const int in = t - group * kGroupM * tiles_n;
        tm = m_first + in % gm;
        tn = in / gm;
    }
};

// Persistent workgroups: one a CU, and one for each eighth of the sequence that
// holds a tile (no other workgroup takes those) on a device of fewer than 8 CUs.
constexpr int64_t tile_blocks(int64_t tiles, int cus) {
    return std::min<int64_t>(tiles, std::max(cus, kXcds));
}

}  // namespace tans_linear

#endif  // TANS_LINEAR_PLAN_H
