// decode_cut.cuh -- the work list of a decode attention call and its cut into block
// ranges: what decode_attn.cu's kernels walk through, and the launch's plan.  Plain
// arithmetic that also compiles for the host, where the tests run it.
#pragma once
#include <climits>
#include <cstdint>

#include "velo_cuda.h"

#ifdef __CUDACC__
#define VELO_HD __host__ __device__ __forceinline__
#else
#define VELO_HD inline
#endif

namespace velo {

constexpr int kMinUnits = 4;  // units per block at least: one per warp

// Resident blocks per SM: INT8 pages with at most 8 query heads per KV head need
// the third (12 warps) to cover the latency of their conversions.
constexpr int blocks_per_sm(int kv, int R) { return kv == VELO_KV_INT8 && R <= 1 ? 3 : 2; }
// Query heads of an item: 8 R, or 4 for R = 0, where the tile's columns 4 .. 7 repeat
// heads 0 .. 3 and carry the remainders of their weights.
constexpr int rows_of(int R) { return R ? 8 * R : 4; }
// tiles of 8 query heads per item: f32 items hold 8 heads, the others 4 (half the MMAs
// for P V), 8 or up to 16
constexpr int row_tiles(int group, int kv) { return kv == VELO_KV_F32 ? 1 : group > 8 ? 2 : group > 4 ? 1 : 0; }

constexpr int tokens_of(int kv) { return kv == VELO_KV_F16 ? 16 : kv == VELO_KV_INT8 ? 32 : 8; }

// What the join costs, in units of a block's time: items are only cut where whole ones would
// make some block later by more.  Items of at most this, or of a quarter of a block's range, are
// never cut.
constexpr int join_units(int kv, int D) { return (kv == VELO_KV_F16 ? 24 : kv == VELO_KV_INT8 ? 10 : 12) * (128 / D); }

struct Plan {
    int main, blocks;  // resident blocks; with the tail's, the grid
    int group;    // query heads per KV head
    int tiles;    // query-head tiles per KV head
};

// a / b, a >= 0 and b > 0: below 2^22 the f32 quotient is within one of it, which the
// remainder settles (a third of an integer division's latency; a block starts with a
// chain of these).
VELO_HD int quotient(int a, int b) {
#ifdef __CUDA_ARCH__
    if (a >= 1 << 22) return a / b;
    const int q = (int)__fdividef((float)a, (float)b), r = a - q * b;
    return q + (r >= b) - (r < 0);
#else
    return a / b;
#endif
}

// The largest b with pre[b] <= u.
VELO_HD int find_sequence(const int* pre, int B, int u) {
    int lo = 0, hi = B;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (pre[mid] <= u)
            lo = mid;
        else
            hi = mid;
    }
    return lo;
}

struct Item {
    int b, it, start, units;  // sequence, item of the sequence, first unit, units
};
template <int kTok>
VELO_HD Item item_of(const int* pre, const int* lens, int B, int u) {
    Item x;
    x.b = find_sequence(pre, B, u);
    x.units = (lens[x.b] + kTok - 1) / kTok;
    x.it = quotient(u - pre[x.b], x.units);
    x.start = pre[x.b] + x.it * x.units;
    return x;
}

// The cut of the list.  `main` blocks, resident from the start, have equal ranges.
// SMs do not advance alike (range ends of one launch were 30 % apart), so when a
// range is long the last twelfth of the list is left to short ranges in
// blocks that start as the first ones end (ragged INT8 batch of 128: 227 -> 207 us at
// full clock, 236 -> 234 under the power cap; 64 x 4096 f16: 173.7 -> 171).
constexpr int kTailPerMain = 1, kTailShare = 12;  // blocks; part of the list
constexpr int kTailUnits = 64;                   // least large range
constexpr int kTailStates = 24;                  // most short ranges of an item: its join reads that many states
// n units in k ranges: the first n % k have one unit more.
struct Share {
    int n, k, q, r;
    VELO_HD Share(int n_, int k_) : n(n_), k(k_), q(k_ ? quotient(n_, k_) : 0), r(n_ - q * k_) {}
    VELO_HD int at(int c) const { return c * q + (c < r ? c : r); }  // first unit of range c
    VELO_HD int range_of(int u) const {
        return u < r * (q + 1) ? quotient(u, q + 1) : r + quotient(u - r * (q + 1), q);
    }
};
struct Cut {
    Share big, tail;  // the large ranges, then the short ones
    bool uncut;       // no item is cut
    VELO_HD int blocks() const { return big.k + tail.k; }
    VELO_HD int total() const { return big.n + tail.n; }
    VELO_HD int at(int c) const { return c <= big.k ? big.at(c) : big.n + tail.at(c - big.k); }
    VELO_HD int block_of(int u) const {
        return u < big.n ? big.range_of(u) : big.k + tail.range_of(u - big.n);
    }
    // Items up to this length are not cut by the start of block c (never more in the tail, so
    // that moving a cut to an item's start keeps the cuts in order).
    VELO_HD int whole(int c, int least) const {
        const int quarter = (c <= big.k ? big.q : tail.q) / 4;
        return uncut ? INT_MAX : quarter > least ? quarter : least;
    }
};
// items: how many there are, longest: units of the longest.
VELO_HD Cut cut_list(const Plan& plan, int total, int items, int longest, int join_units) {
    const int tail = plan.blocks - plan.main, most = (total + kMinUnits - 1) / kMinUnits;
    const int blocks = most < plan.main ? most : plan.main;
    const Share even(total, blocks);
    // Whole items make the fullest block per * longest - q longer than an equal share at most, and with
    // several to a block half of the longest on average.  Cutting costs the join and each block an
    // item's start and end more (128 x 100-600 tokens INT8 48.8 us cut, 45.1 uncut; where blocks would
    // idle, 16 x 400-800, 15.5 against 17.3).
    const int per = blocks ? quotient(items + blocks - 1, blocks) : 0;
    const bool uncut = total > 0 && (2 * ((long long)per * longest - even.q) <= 3 * join_units ||
                                     (per > 1 && longest <= 2 * join_units));
    if (tail > 0 && quotient(total, plan.main) >= kTailUnits &&
        longest <= kTailStates * quotient(total / kTailShare, tail)) {
        const int n = total / kTailShare;
        return Cut{Share(total - n, plan.main), Share(n, tail), uncut};
    }
    return Cut{even, Share(0, 0), uncut};
}

// First unit of block c: moved to the start of the item it falls into when that is short.
template <int kTok>
VELO_HD int cut_at(const int* pre, const int* lens, int B, const Cut& k, int join_units, int c) {
    const int u = c < k.blocks() ? k.at(c) : k.total();
    if (c == 0 || u >= k.total()) return u;
    const Item x = item_of<kTok>(pre, lens, B, u);
    return x.units <= k.whole(c, join_units) ? x.start : u;
}


// Units that an item of this page type can have in a table of max_pages (of 16 tokens).
VELO_HD int most_units(int kv, int max_pages) {
    return (int)(((int64_t)max_pages * 16 + tokens_of(kv) - 1) / tokens_of(kv));
}
inline int main_blocks(int kv, int R, int sm_count) { return blocks_per_sm(kv, R) * sm_count; }
inline int all_blocks(int kv, int R, int sm_count) { return main_blocks(kv, R, sm_count) * (1 + kTailPerMain); }

inline Plan make_plan(int kv, int group, int n_kv, int B, int max_pages, int sm_count) {
    const int R = row_tiles(group, kv);
    Plan p;
    p.main = main_blocks(kv, R, sm_count);
    p.blocks = all_blocks(kv, R, sm_count);
    p.group = group;
    p.tiles = (group + rows_of(R) - 1) / rows_of(R);
    // the tail's blocks only where cut_list can come to use them: enough work in this table,
    // and enough items that the longest is not above kTailStates short ranges
    const int most = most_units(kv, max_pages);
    const long long items = (long long)B * n_kv * p.tiles;
    if (items * most < (long long)kTailUnits * p.main ||
        items * kTailStates < (long long)kTailShare * (p.blocks - p.main))
        p.blocks = p.main;
    return p;
}

}  // namespace velo
