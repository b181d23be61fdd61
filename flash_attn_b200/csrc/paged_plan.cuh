// How a launch over a paged cache is shared out among its CTAs, worked out on the device: the lengths are known there only (and a
// captured launch is replayed on others).
//
// A sequence's rows (new tokens x query heads of a K/V head) are cut into blocks of plan.rows; block, K/V head and sequence are an
// item, whose keys are walked in tiles of 128.  Every CTA reads all lengths and works out the same plan, a block of threads a
// chunk of sequences: the sum of all items' tiles, from it the tiles that a CTA should take, from that each sequence's parts, and the
// running sum of the CTAs, in which its own index names its sequence, item and part.  That costs a launch about a microsecond
// before its first load, and no launch of its own.
//
// The share.  One wave of equal parts is the shortest launch where the device holds that many CTAs at once: the smallest share
// with which the parts of all items fit, found by bisection.  Where items alone are more than that, or the parts are long, several waves
// of smaller parts even out what the waves leave (`waves`).
#pragma once
#include "fa_internal.h"
#include "fa_paged.h"

namespace fa {

struct PagedPlan {
    SeqTable seq;
    int heads_k, group;
    int rows;             // rows of a block
    int is_causal, window_left, window_right;
    int slots;            // CTAs that the device runs at once
    int min_share;        // tiles that a part is worth starting for
    int long_share;       // a share above this is cut into waves
    int partials;         // blocks of partial results that there is room for (0: nothing is split)
};

constexpr int kPagedWaves = 3;
constexpr int kPlanSeqs = 128;  // sequences up to which the share is searched for (the same in every kernel that works the plan out)

// Blocks of partial results that a plan can need: parts of split items are at most twice the shares there are.
inline long long most_partials(int slots) { return 2LL * kPagedWaves * slots; }

#ifdef __CUDACC__

// What a CTA does: part `part` of `parts` of block `blk` of K/V head `head` of sequence `b`.
struct PagedWork {
    int b, head, blk, part, parts;
    int slot;             // where part 0 leaves its partial result
    int first, n, keys;   // rows of the sequence: first row, new tokens, keys
};

// Keys that rows at positions [p0, p1] see: [lo, hi), within the keys there are.
__device__ __forceinline__ void visible_keys(const PagedPlan& p, int keys, int p0, int p1, int* lo, int* hi) {
    long long l = 0, h = keys;
    if (p.window_left >= 0) l = max(l, static_cast<long long>(p0) - p.window_left);
    if (p.window_right >= 0) h = min(h, static_cast<long long>(p1) + p.window_right + 1);
    if (p.is_causal) h = min(h, static_cast<long long>(p1) + 1);
    h = max(h, 0LL);
    l = min(l, h);
    *lo = static_cast<int>(l);
    *hi = static_cast<int>(h);
}

// Blocks of a sequence and the most tiles that one of them walks.
__device__ __forceinline__ int2 blocks_and_tiles(const PagedPlan& p, const SeqSpan& s) {
    const int n = s.end - s.first;
    if (n <= 0) return make_int2(0, 0);
    const int blocks = static_cast<int>((static_cast<long long>(n) * p.group + p.rows - 1) / p.rows);
    int lo, hi;
    visible_keys(p, s.keys, s.keys - n, s.keys - 1, &lo, &hi);
    long long keys = hi - lo;
    const long long right = p.is_causal ? 0 : p.window_right;
    const int tokens = min((p.rows + p.group - 1) / p.group + 1, n);  // (a block may begin and end inside a token)
    if (p.window_left >= 0 && right >= 0) keys = min(keys, p.window_left + right + tokens);
    return make_int2(blocks, static_cast<int>((keys + kTile - 1) / kTile + (keys > 0 && lo > 0 ? 1 : 0) + (keys < hi - lo ? 1 : 0)));
}

template <int kThreads>
struct PlanScratch {
    static_assert(kThreads >= kPlanSeqs, "a thread keeps one of them");
    int2 seq[kPlanSeqs];                      // blocks and tiles of the sequences, where they are few
    unsigned long long sum[kThreads / 32];
    int items[kThreads / 32];
    int3 scan[kThreads / 32];
    PagedWork found;
    int have;
};

__device__ __forceinline__ int parts_of(const PagedPlan& p, int tiles, int share) {
    return p.partials > 0 ? max(1, (tiles + share - 1) / share) : 1;
}

// The work of CTA `want` (by_split: of the `want`-th split item, part 0), by all kThreads threads; false where there is none.
template <int kThreads>
__device__ __forceinline__ bool find_work(const PagedPlan& p, PlanScratch<kThreads>& sm, int want, bool by_split, PagedWork* work) {
    constexpr int kWarps = kThreads / 32;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int batch = p.seq.batch;
    const bool few = batch <= kPlanSeqs;
    // ---- tiles of all items
    SeqSpan span = {0, 0, 0};
    int2 mine = make_int2(0, 0);
    unsigned long long tiles = 0;
    int items = 0;
    for (int b = threadIdx.x; b < batch; b += kThreads) {
        span = seq_span(p.seq, b);
        mine = blocks_and_tiles(p, span);
        tiles += static_cast<unsigned long long>(mine.x) * mine.y;
        items += mine.x;
    }
    if (few && threadIdx.x < kPlanSeqs) sm.seq[threadIdx.x] = mine;
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        tiles += __shfl_xor_sync(0xffffffffu, tiles, o);
        items += __shfl_xor_sync(0xffffffffu, items, o);
    }
    if (lane == 0) {
        sm.sum[warp] = tiles;
        sm.items[warp] = items;
    }
    if (threadIdx.x == 0) sm.have = 0;
    __syncthreads();
    tiles = 0;
    items = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
        tiles += sm.sum[w];
        items += sm.items[w];
    }
    // ---- the share
    const long long all = static_cast<long long>(tiles) * p.heads_k;
    const long long per = (all + p.slots - 1) / p.slots;
    int share = static_cast<int>(min(max(per, static_cast<long long>(p.min_share)), 0x7fffffffLL));
    if (p.partials > 0) {
        if (share > p.long_share || !few || static_cast<long long>(items) * p.heads_k > p.slots) {
            share = static_cast<int>(min(max((all + kPagedWaves * p.slots - 1) / (kPagedWaves * p.slots), static_cast<long long>(min(share, p.long_share))),
                                         0x7fffffffLL));
        } else {
            // (every warp for itself: lanes over the sequences)
            int lo = share, hi = share;
            auto fits = [&](int s) {
                int ctas = 0;
                for (int b = lane; b < batch; b += 32) {
                    const int2 x = sm.seq[b];
                    ctas += x.x * parts_of(p, x.y, s);
                }
                return static_cast<long long>(__reduce_add_sync(0xffffffffu, ctas)) * p.heads_k <= p.slots;
            };
            if (!fits(share)) {
                // (with all tiles of a sequence in one part the items fit; a quarter more at a time gets there in a few steps)
                do {
                    lo = hi;
                    hi += (hi >> 2) + 1;
                } while (!fits(hi));
                while (hi - lo > 1) {
                    const int mid = (lo + hi) >> 1;
                    if (fits(mid)) hi = mid; else lo = mid;
                }
                share = hi;
            }
        }
    }
    // ---- running sums: CTAs, split items, their partial results
    int3 carry = make_int3(0, 0, 0);
    for (int b0 = 0; b0 < batch; b0 += kThreads) {
        const int b = b0 + static_cast<int>(threadIdx.x);
        if (!few) {
            mine = make_int2(0, 0);
            if (b < batch) {
                span = seq_span(p.seq, b);
                mine = blocks_and_tiles(p, span);
            }
        }
        const int parts = parts_of(p, mine.y, share);
        const int n = mine.x * p.heads_k;
        const int3 own = make_int3(n * parts, parts > 1 ? n : 0, parts > 1 ? n * parts : 0);
        int3 run = own;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int x = __shfl_up_sync(0xffffffffu, run.x, o), y = __shfl_up_sync(0xffffffffu, run.y, o), z = __shfl_up_sync(0xffffffffu, run.z, o);
            if (lane >= o) {
                run.x += x;
                run.y += y;
                run.z += z;
            }
        }
        if (lane == 31) sm.scan[warp] = run;
        __syncthreads();
        int3 before = carry;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            const int3 x = sm.scan[w];
            if (w < warp) {
                before.x += x.x;
                before.y += x.y;
                before.z += x.z;
            }
            carry.x += x.x;
            carry.y += x.y;
            carry.z += x.z;
        }
        before.x += run.x - own.x;
        before.y += run.y - own.y;
        before.z += run.z - own.z;
        const int at = want - (by_split ? before.y : before.x);
        if (at >= 0 && at < (by_split ? own.y : own.x)) {
            // (a sequence whose partial results have no room is not split: its part 0 does it all)
            const bool room = before.z + own.z <= p.partials;
            PagedWork w;
            w.b = b;
            w.first = span.first;
            w.n = span.end - span.first;
            w.keys = span.keys;
            w.parts = parts;
            const int item_parts = by_split ? 1 : parts;
            // part by part of a head, its blocks side by side: CTAs of neighbouring index read the same keys
            const int per_part = mine.x;
            const int outer = at / per_part;
            w.blk = at - outer * per_part;
            if (p.is_causal) w.blk = per_part - 1 - w.blk;  // (the longest first)
            w.head = outer / item_parts;
            w.part = outer - w.head * item_parts;
            w.slot = before.z + (w.head * mine.x + w.blk) * parts;
            if (!room) w.parts = 1;
            sm.found = w;
            sm.have = parts == 1 || room || (!by_split && w.part == 0) ? 1 : 0;
        }
        __syncthreads();
    }
    *work = sm.found;
    return sm.have != 0;
}
#endif

}  // namespace fa
