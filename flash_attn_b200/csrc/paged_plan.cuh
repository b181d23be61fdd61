// How a launch over a paged cache is shared out among its CTAs, worked out on the device: the lengths are known there only (and a
// captured launch is replayed on others).
//
// A sequence's rows (new tokens x query heads of a K/V head) are cut into blocks of plan.rows; block, K/V head and sequence are an
// item, whose keys are walked in tiles of 128.  Every CTA reads all lengths and works out the same plan: the sum of all items'
// tiles, from it the tiles that a part should take (the share), from that each sequence's parts, and the running sum of the CTAs, in
// which its own index names its sequence, item and part.  Up to kPlanSeqs sequences each warp does that for itself, four sequences a
// lane and nothing but shuffles between them; more go through shared memory, a sequence a thread at a time.
//
// The parts of an item leave their rows un-normalised in the workspace, and the CTA that comes last puts them together.
#pragma once
#include "fa_internal.h"
#include "fa_paged.h"

namespace fa {

struct PagedPlan {
    SeqTable seq;
    int heads_k, group;
    int rows;             // rows of a block
    int block_tokens;     // tokens that a block may reach into
    int rows_over, rows_upto;  // sequences of more rows than the one and no more than the other are this launch's
    FastDiv div_rows;
    int is_causal, window_left, window_right;
    int slots;            // CTAs that the device runs at once
    int min_share;        // tiles that a part is worth starting for
    int long_share;       // of launches of more than one wave: parts are no shorter than this
    int waves;            // and shares no shorter than this part of a slot's tiles
    int one_wave;         // decode kernel: tiles a slot up to which all parts are to run at once
    int most_parts;       // of an item: as many as the table's width gives (a length may be beyond it)
    int partials;         // parts of split items that there is room for (0: nothing is split)
};

constexpr int kPlanSeqs = 128;

#ifdef __CUDACC__

// What a CTA does: part `part` of `parts` of block `blk` of K/V head `head` of sequence `b`.
struct PagedWork {
    int b, head, blk, part, parts;
    int slot;             // where part 0 of the item leaves its rows
    int first, n, keys;   // the sequence's first row, new tokens, keys
};

// Keys that rows at positions [p0, p1] see: [lo, hi), within the keys there are.  (Keys, rows and windows are below 2^30.)
__device__ __forceinline__ void visible_keys(const PagedPlan& p, int keys, int p0, int p1, int* lo, int* hi) {
    int l = 0, h = keys;
    if (p.window_left >= 0) l = max(l, p0 - p.window_left);
    if (p.window_right >= 0) h = min(h, p1 + p.window_right + 1);
    if (p.is_causal) h = min(h, p1 + 1);
    *hi = max(h, 0);
    *lo = min(l, *hi);
}

// Blocks of a sequence, and the most tiles that one of them walks.
__device__ __forceinline__ int2 blocks_and_tiles(const PagedPlan& p, const SeqSpan& s) {
    const int n = s.end - s.first;
    if (n <= 0) return make_int2(0, 0);
    const unsigned rows = static_cast<unsigned>(n) * static_cast<unsigned>(p.group);  // (tokens * heads < 2^30)
    if (static_cast<int>(rows) <= p.rows_over || static_cast<int>(rows) > p.rows_upto) return make_int2(0, 0);
    const int blocks = static_cast<int>(fast_div(p.div_rows, rows + p.rows - 1));
    int lo, hi;
    visible_keys(p, s.keys, s.keys - n, s.keys - 1, &lo, &hi);
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

struct PlanScratch {
    unsigned long long sum[16];
    int items[16];
    int2 scan[16];
    PagedWork found;
    int have;
};

__device__ __forceinline__ int parts_of(const PagedPlan& p, int tiles, int share) {
    if (p.partials == 0 || tiles <= share) return 1;
    return min(static_cast<int>(static_cast<unsigned>(tiles + share - 1) / static_cast<unsigned>(share)), p.most_parts);
}
__device__ __forceinline__ long long ceil_div(unsigned long long x, int d) {
    if (x <= 0xffffffffull - d) return static_cast<long long>((static_cast<unsigned>(x) + d - 1) / static_cast<unsigned>(d));  // (the long division takes twice as long)
    return static_cast<long long>((x + d - 1) / d);
}
// The share of a launch of several waves.
__device__ __forceinline__ int long_share_of(const PagedPlan& p, unsigned long long tiles) {
    return static_cast<int>(min(max(ceil_div(tiles, p.waves * p.slots), static_cast<long long>(p.long_share)), 0x3fffffffLL));
}

// Item and part of the `at`-th CTA of a sequence of `blocks` blocks, whose first is `slot` parts into the workspace.
__device__ __forceinline__ bool item_of(const PagedPlan& p, int at, int blocks, int parts, int slot, PagedWork* w) {
    // part by part of a head, its blocks side by side: CTAs of neighbouring index read the same keys
    const int outer = static_cast<int>(static_cast<unsigned>(at) / static_cast<unsigned>(blocks));
    w->blk = at - outer * blocks;
    if (p.is_causal) w->blk = blocks - 1 - w->blk;  // (the longest first)
    w->head = static_cast<int>(static_cast<unsigned>(outer) / static_cast<unsigned>(parts));
    w->part = outer - w->head * parts;
    w->parts = parts;
    w->slot = slot + (w->head * blocks + w->blk) * parts;
    if (parts > 1 && slot + blocks * p.heads_k * parts > p.partials) {  // no room for the sequence's partial rows: part 0 does it all
        w->parts = 1;
        return w->part == 0;
    }
    return true;
}

// The work of CTA `want`; false where there is none.  By all kThreads threads.
template <int kThreads>
__device__ __forceinline__ bool find_work(const PagedPlan& p, PlanScratch& sm, int want, PagedWork* work) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int batch = p.seq.batch;
    if (batch <= kPlanSeqs) {
        // ---- every warp for itself: lane l has sequences 4 l .. 4 l + 3
        SeqSpan span[4];
        int2 own[4];
        unsigned long long tiles = 0;
        int items = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int b = lane * 4 + i;
            span[i] = {0, 0, 0};
            if (b < batch) span[i] = seq_span(p.seq, b);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            own[i] = blocks_and_tiles(p, span[i]);
            tiles += static_cast<unsigned long long>(own[i].x) * own[i].y;
            items += own[i].x;
        }
        int share = 1;
        if (p.partials > 0) {
            const unsigned low = __reduce_add_sync(0xffffffffu, static_cast<unsigned>(tiles) & 0xfffffu);
            const unsigned high = __reduce_add_sync(0xffffffffu, static_cast<unsigned>(tiles >> 20));
            tiles = (static_cast<unsigned long long>(high) << 20) + low;
            items = __reduce_add_sync(0xffffffffu, items);
            tiles *= p.heads_k;
            const long long per = ceil_div(tiles, p.slots);
            if (per > p.long_share || static_cast<long long>(items) * p.heads_k > p.slots) {
                share = long_share_of(p, tiles);
            } else {
                // one wave: the smallest share with which all parts run at once
                auto fits = [&](int s) {
                    int ctas = 0;
#pragma unroll
                    for (int i = 0; i < 4; ++i) ctas += own[i].x * parts_of(p, own[i].y, s);
                    return __reduce_add_sync(0xffffffffu, ctas) * static_cast<long long>(p.heads_k) <= p.slots;
                };
                int hi = max(static_cast<int>(per), p.min_share), lo = hi;
                if (!fits(hi)) {
                    do {
                        lo = hi;
                        hi += (hi >> 2) + 1;
                    } while (!fits(hi));  // (ends: with a part an item they fit)
                    while (hi - lo > 1) {
                        const int mid = (lo + hi) >> 1;
                        if (fits(mid)) hi = mid; else lo = mid;
                    }
                }
                share = hi;
            }
        }
        int parts[4];
        int2 run = make_int2(0, 0);  // CTAs, parts of split items
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            parts[i] = parts_of(p, own[i].y, share);
            const int ctas = own[i].x * p.heads_k * parts[i];
            run.x += ctas;
            run.y += parts[i] > 1 ? ctas : 0;
        }
        const int2 mine = run;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int x = __shfl_up_sync(0xffffffffu, run.x, o), y = __shfl_up_sync(0xffffffffu, run.y, o);
            if (lane >= o) {
                run.x += x;
                run.y += y;
            }
        }
        run.x -= mine.x;
        run.y -= mine.y;
        const unsigned owner = __ballot_sync(0xffffffffu, want >= run.x && want < run.x + mine.x);
        if (owner == 0) return false;
        int at = want - run.x, slot = run.y, b = lane * 4, blocks = 0, n_parts = 1;
        SeqSpan s = {0, 0, 0};
        bool found = false;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int ctas = own[i].x * p.heads_k * parts[i];
            if (!found) {
                if (at < ctas) {
                    found = true;
                    b += i;
                    blocks = own[i].x;
                    n_parts = parts[i];
                    s = span[i];
                } else {
                    at -= ctas;
                    slot += parts[i] > 1 ? ctas : 0;
                }
            }
        }
        const int src = __ffs(owner) - 1;
        at = __shfl_sync(0xffffffffu, at, src);
        slot = __shfl_sync(0xffffffffu, slot, src);
        blocks = __shfl_sync(0xffffffffu, blocks, src);
        n_parts = __shfl_sync(0xffffffffu, n_parts, src);
        work->b = __shfl_sync(0xffffffffu, b, src);
        work->first = __shfl_sync(0xffffffffu, s.first, src);
        work->n = __shfl_sync(0xffffffffu, s.end - s.first, src);
        work->keys = __shfl_sync(0xffffffffu, s.keys, src);
        return item_of(p, at, blocks, n_parts, slot, work);
    }
    // ---- many sequences: through shared memory
    constexpr int kWarps = kThreads / 32;
    unsigned long long tiles = 0;
    if (threadIdx.x == 0) sm.have = 0;
    if (p.partials > 0) {
        for (int b = threadIdx.x; b < batch; b += kThreads) {
            const int2 x = blocks_and_tiles(p, seq_span(p.seq, b));
            tiles += static_cast<unsigned long long>(x.x) * x.y;
        }
#pragma unroll
        for (int o = 16; o; o >>= 1) tiles += __shfl_xor_sync(0xffffffffu, tiles, o);
        if (lane == 0) sm.sum[warp] = tiles;
    }
    __syncthreads();
    int share = 1;
    if (p.partials > 0) {
        tiles = 0;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) tiles += sm.sum[w];
        share = long_share_of(p, tiles * p.heads_k);
    }
    int2 carry = make_int2(0, 0);
    for (int b0 = 0; b0 < batch; b0 += kThreads) {
        const int b = b0 + static_cast<int>(threadIdx.x);
        SeqSpan s = {0, 0, 0};
        if (b < batch) s = seq_span(p.seq, b);
        const int2 x = blocks_and_tiles(p, s);
        const int parts = parts_of(p, x.y, share), ctas = x.x * p.heads_k * parts;
        const int2 mine = make_int2(ctas, parts > 1 ? ctas : 0);
        int2 run = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int u = __shfl_up_sync(0xffffffffu, run.x, o), v = __shfl_up_sync(0xffffffffu, run.y, o);
            if (lane >= o) {
                run.x += u;
                run.y += v;
            }
        }
        if (lane == 31) sm.scan[warp] = run;
        __syncthreads();
        run.x += carry.x - mine.x;
        run.y += carry.y - mine.y;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            const int2 y = sm.scan[w];
            if (w < warp) {
                run.x += y.x;
                run.y += y.y;
            }
            carry.x += y.x;
            carry.y += y.y;
        }
        if (want >= run.x && want < run.x + mine.x) {
            PagedWork w;
            w.b = b;
            w.first = s.first;
            w.n = s.end - s.first;
            w.keys = s.keys;
            sm.have = item_of(p, want - run.x, x.x, parts, run.y, &w) ? 1 : 0;
            sm.found = w;
        }
        __syncthreads();
    }
    *work = sm.found;
    return sm.have != 0;
}

// ---- the end of a split item ---------------------------------------------------------------------------------------------------------
// Each part leaves its rows, un-normalised, with their maxima (log2 units) and sums; then it counts itself in, and the last puts the
// rows together: O = sum_j 2^(m_j - m) O_j / l, l = sum_j 2^(m_j - m) l_j, in the order of the parts whoever is last.
//
// A count needs no clearing before the launch: its upper 48 bits say that it is one.  Whatever else lies there (a workspace that
// was never used) counts as none come yet, and the last of the parts leaves none come for the next launch.
constexpr unsigned long long kCountMark = 0x9d3f6ba817c5ull << 16;

// Whether this CTA is the last of its item (one thread, to whom the CTA's partial rows are visible; they are to the others' after).
__device__ __forceinline__ bool count_in(unsigned long long* count, int parts) {
    __threadfence();
    unsigned long long was = atomicAdd(count, 1ull);
    while ((was & ~0xffffull) != kCountMark) {  // not a count: whoever makes it one is the first to come, the others add themselves again
        const unsigned long long seen = *reinterpret_cast<volatile unsigned long long*>(count);
        if ((seen & ~0xffffull) == kCountMark) was = atomicAdd(count, 1ull);
        else if (atomicCAS(count, seen, kCountMark | 1ull) == seen) was = kCountMark;  // (ends: a failed exchange is another part's doing)
    }
    const bool last = static_cast<int>(was & 0xffffull) + 1 == parts;
    if (last) {
        *reinterpret_cast<volatile unsigned long long*>(count) = kCountMark;
        __threadfence();
    }
    return last;
}
#endif

}  // namespace fa
