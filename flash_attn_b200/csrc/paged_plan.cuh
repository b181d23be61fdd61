// What the parts of a launch over a paged cache are worked out from on the device (paged_parts.cuh): the lengths are known there only,
// and a captured launch is replayed on others.
//
// A sequence's rows (new tokens x query heads of a K/V head) are cut into blocks of plan.rows; block, K/V head and sequence are an
// item, whose keys are walked in tiles of 128.  The parts of an item leave their rows un-normalised in the workspace, and the CTA
// that comes last puts them together.
#pragma once
#include "fa_internal.h"
#include "fa_paged.h"

namespace fa {

struct PagedPlan {
    SeqTable seq;
    int heads_k, group;
    int table_keys;       // keys that the page table has room for
    int rows;             // rows of a block
    int block_tokens;     // tokens that a block may reach into
    FastDiv div_rows;
    int is_causal, window_left, window_right;
    int slots;            // CTAs that the device runs at once
    int min_share;        // tiles that a part is worth starting for
    int long_share;       // of launches of more than one wave: parts are no shorter than this
    int waves;            // and shares no shorter than this part of a slot's tiles
    int one_wave;         // tiles a slot up to which all parts are to run at once
    int most_parts;       // of an item: as many as the table's width gives (a length may be beyond it)
    int partials;         // parts of split items that there is room for (0: nothing is split)
    int grid;             // parts that there are CTAs for
};

#ifdef __CUDACC__

// Keys that rows at positions [p0, p1] see: [lo, hi), within the keys there are.  (Keys, rows and windows are below 2^30.)
__device__ __forceinline__ void visible_keys(const PagedPlan& p, int keys, int p0, int p1, int* lo, int* hi) {
    int l = 0, h = keys;
    if (p.window_left >= 0) l = max(l, p0 - p.window_left);
    if (p.window_right >= 0) h = min(h, p1 + p.window_right + 1);
    if (p.is_causal) h = min(h, p1 + 1);
    *hi = max(h, 0);
    *lo = min(l, *hi);
}
// And of these the ones to walk: of keys beyond the page table one is kept, by which their rows are known to be without a page (for a
// length of 2^30 in a table of one page a CTA would walk eight million tiles of nothing).
__device__ __forceinline__ void walked_keys(const PagedPlan& p, int keys, int p0, int p1, int* lo, int* hi) {
    visible_keys(p, keys, p0, p1, lo, hi);
    *hi = min(*hi, max(*lo, p.table_keys) + 1);
}

// Blocks of a sequence, and the most tiles that one of them walks.
__device__ __forceinline__ int2 blocks_and_tiles(const PagedPlan& p, const SeqSpan& s) {
    const int n = s.end - s.first;
    if (n <= 0) return make_int2(0, 0);
    const unsigned rows = static_cast<unsigned>(n) * static_cast<unsigned>(p.group);  // (tokens * heads < 2^30)
    const int blocks = static_cast<int>(fast_div(p.div_rows, rows + p.rows - 1));
    int lo, hi;
    walked_keys(p, s.keys, s.keys - n, s.keys - 1, &lo, &hi);
    int keys = hi - lo;
    const int right = p.is_causal ? 0 : p.window_right;
    bool cut = false;
    if (p.window_left >= 0 && right >= 0) {
        const int most = p.window_left + right + min(p.block_tokens, n);
        cut = most < keys;
        if (cut) keys = most;
    }
    return make_int2(blocks, (keys + kTile - 1) / kTile + (keys > 0 && (cut || lo > 0) ? 1 : 0));
}

// Part `part` of `parts` of n tiles: [lo, hi).
__device__ __forceinline__ void part_of(int n, int part, int parts, int* lo, int* hi) {
    const int each = static_cast<int>(static_cast<unsigned>(n) / static_cast<unsigned>(parts)), more = n - each * parts;
    *lo = part * each + min(part, more);
    *hi = *lo + each + (part < more ? 1 : 0);
}

__device__ __forceinline__ int parts_of(const PagedPlan& p, int tiles, int share) {
    if (p.partials == 0 || tiles <= share) return 1;
    return min(static_cast<int>(static_cast<unsigned>(tiles + share - 1) / static_cast<unsigned>(share)), p.most_parts);
}
// ---- the end of a split item ---------------------------------------------------------------------------------------------------------
// Each part leaves its rows, un-normalised, with their maxima (log2 units) and sums; then it counts itself in, and the last puts the
// rows together: O = sum_j 2^(m_j - m) O_j / l, l = sum_j 2^(m_j - m) l_j, in the order of the parts whoever is last.
//
// A count needs no clearing before the launch: that c have come is the word kCountMark + c kCountStep, and whatever else lies there (a
// workspace that was never used, or that something else has been written to) counts as none come yet.  The last of the parts leaves
// none come for the next launch.  The step is odd, so that it has an inverse modulo 2^64 and each word stands for one c, of which those
// below 2^16 are counts: one word of 2^48, and none that differs from a count in one of its four 16-bit pieces (kCountStep^-1 times
// such a difference is 2^47 or more off zero).
constexpr unsigned long long kCountMark = 0x9d3f6ba817c50000ull, kCountStep = 0x0fd630f1f29d0da9ull, kCountUnstep = 0xd7da0cbaef15e699ull;
static_assert(kCountStep * kCountUnstep == 1ull, "inverse modulo 2^64");
__device__ __forceinline__ unsigned long long come(unsigned long long word) { return (word - kCountMark) * kCountUnstep; }
constexpr unsigned long long kMostCome = 0xffffull;

// Whether this CTA is the last of its item (one thread, to whom the CTA's partial rows are visible; they are to the others' after).
__device__ __forceinline__ bool count_in(unsigned long long* count, int parts) {
    __threadfence();
    unsigned long long was = atomicAdd(count, kCountStep);
    while (come(was) > kMostCome) {  // not a count: whoever makes it one is the first to come, the others add themselves again
        const unsigned long long seen = *reinterpret_cast<volatile unsigned long long*>(count);
        if (come(seen) <= kMostCome) was = atomicAdd(count, kCountStep);
        else if (atomicCAS(count, seen, kCountMark + kCountStep) == seen) was = kCountMark;  // (ends: a failed exchange is another part's doing)
    }
    const bool last = static_cast<int>(come(was)) + 1 == parts;
    if (last) {
        *reinterpret_cast<volatile unsigned long long*>(count) = kCountMark;
        __threadfence();
    }
    return last;
}
#endif

}  // namespace fa
