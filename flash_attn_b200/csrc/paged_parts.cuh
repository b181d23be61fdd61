// How the kernels over a paged cache share a launch out.
//
// An item (a block of rows of a sequence and K/V head; paged_plan.cuh) is cut into equal parts of at most `share` tiles, and the parts of
// all items are numbered.  The grid is as large as their number can be; CTA i begins with part i, and while it works on one its
// producer warp takes the next from the CTAs that have not started yet (cluster launch control): setting up, the first loads and the
// last rows of a CTA take ten microseconds, and what the grid has too many of are taken without starting.  Nothing is dealt out
// beforehand, since CTAs differ in speed by a tenth.  (64 sequences of 100 .. 8192 keys, 8 K/V heads of 128 columns: 82 us; a CTA a part
// 86; the same length for each of 296 CTAs 84, and 24 sequences of 500 .. 4000 keys, 16 heads of 64 columns, 57 to 65 instead of 49.)
//
// Long parts have the lower numbers, so that the short ones fill what the long ones leave at the end.
//
// The lengths of all sequences are read by one warp, which knows where the parts of each begin from a scan over them, 32 sequences at a
// time; a later part is looked for from the one before on, an earlier one (nothing says in which order CTAs are taken) from the start.
#pragma once
#include "paged_kernels.h"

namespace fa {

// Tiles [lo, lo + n_tiles) of an item, as the warps of a CTA hand it to each other.
struct alignas(16) PagedSeg {
    int b, head, first, n;        // sequence, K/V head, the sequence's first row, new tokens
    int keys, row0, n_rows, part; // keys; rows of the block, inside the sequence (n_rows = 0: there is no other part); part of
    int parts, slot, lo, n_tiles; // the item's parts, and where part 0 leaves its rows
    int vis_lo, vis_hi, pad[2];   // keys that any of the rows sees (and the table's room, or a key more)
};

constexpr int kSizes = 3;       // of parts: more than half a share, more than a quarter, less
constexpr int kWarpSeqs = 256;  // sequences up to which one warp adds their tiles up

#ifdef __CUDACC__

__device__ __forceinline__ long long divide(long long x, long long d) {
    if (((x | d) >> 32) == 0) return static_cast<unsigned>(x) / static_cast<unsigned>(d);
    return x / d;
}
__device__ __forceinline__ long long scan_add(long long v, int lane) {  // inclusive, over the lanes of a warp
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long x = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += x;
    }
    return v;
}
__device__ __forceinline__ long long sum_all(long long v) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
__device__ __forceinline__ void prefetch_l1(const void* p) { asm volatile("prefetch.global.L1 [%0];" ::"l"(p)); }

// Parts are counted in 36 bits: 32 sequences of 2^30 blocks each, which cu_seqlens_q that go back and forth can come to.
constexpr int kPartBits = 36;
__device__ __forceinline__ long long part_count(long long x) { return x & ((1LL << kPartBits) - 1); }

// The parts of a launch, by one warp.
struct PartLine {
    int share;
    // sequences b0 + lane
    int b0, pass, passes, parts;
    SeqSpan s;
    int2 x;                  // blocks, tiles
    long long own, upto;     // parts of the lane's sequence (and above kPartBits those of split items), and of the lanes up to it
    long long base;          // of the sequences before b0

    __device__ __forceinline__ void read(const PagedPlan& p, int b) {
        s = {0, 0, 0};
        if (b < p.seq.batch) s = seq_span(p.seq, b);
        x = blocks_and_tiles(p, s);
    }
    __device__ __forceinline__ void count(const PagedPlan& p, int lane) {
        parts = parts_of(p, x.y, share);
        int size = 0;
        if (passes > 1) {
            const int longest = static_cast<int>(static_cast<unsigned>(x.y + parts - 1) / static_cast<unsigned>(parts));
            size = longest * 2 > share ? 0 : longest * 4 > share ? 1 : kSizes - 1;
        }
        own = size == pass ? static_cast<long long>(x.x) * p.heads_k * parts : 0;
        if (parts > 1) own |= own << kPartBits;  // (fewer than 2 waves * slots of all)
        upto = scan_add(own, lane);
    }
    // tiles: of all sequences and K/V heads, where the block has added them up (more than kWarpSeqs sequences).
    __device__ __forceinline__ void start(const PagedPlan& p, int lane, long long tiles) {
        const int batch = p.seq.batch;
        if (batch <= kWarpSeqs) {
            if (batch > 32 && lane * 32 < batch) {
                prefetch_l1(p.seq.seqlens_k + lane * 32);
                if (p.seq.cu_seqlens_q) prefetch_l1(p.seq.cu_seqlens_q + lane * 32);
            }
            long long sum = 0;
#pragma unroll 1
            for (int b = (batch - 1) / 32 * 32; b >= 0; b -= 32) {
                read(p, b + lane);
                sum += static_cast<long long>(x.x) * x.y;
            }
            tiles = sum_all(sum) * p.heads_k;
        } else {
            read(p, lane);
        }
        const long long per = divide(tiles + p.slots - 1, p.slots);
        share = static_cast<int>(min(max(divide(tiles + static_cast<long long>(p.waves) * p.slots - 1, static_cast<long long>(p.waves) * p.slots),
                                         static_cast<long long>(p.long_share)), 0x3fffffffLL));
        passes = kSizes;
        if (batch <= 32 && per <= p.one_wave) {
            auto ctas_with = [&](int y) { return __reduce_add_sync(0xffffffffu, static_cast<unsigned>(x.x * p.heads_k * parts_of(p, x.y, y))); };
            if (static_cast<long long>(ctas_with(0x3fffffff)) <= p.slots) {  // the smallest share with which all parts run at once
                int one = max(static_cast<int>(per), p.min_share);
                while (static_cast<long long>(ctas_with(one)) > p.slots) one += (one >> 3) + 1;  // (ends: with a part an item they fit)
                if (one <= max(static_cast<int>(per + (per >> 2)), 4 * p.min_share)) {  // (else a few long parts would be waited for)
                    share = one;
                    passes = 1;
                }
            }
        }
        b0 = 0;
        pass = 0;
        base = 0;
        count(p, lane);
    }
    // Part `nth` of all; false: there are not so many, or it belongs to an item that the launch has no CTAs or no room for.  (Rows that
    // several sequences claim are more than the launch was made for: such an item is left out with all of its parts.)
    __device__ __forceinline__ bool find(const PagedPlan& p, const FastDiv& div_group, int nth, int lane, PagedSeg* g) {
        bool again = nth < part_count(base);  // (of sequences that the scan has left behind)
        if (nth >= p.grid || (!again && pass >= passes)) return false;  // (at the end of the scan, base: of all)
        for (;;) {
            if (again) {
                base = 0;
                b0 = pass = 0;
                again = false;
            } else {
                const long long sum = __shfl_sync(0xffffffffu, upto, 31);
                if (nth < part_count(base + sum)) break;
                base += sum;
                b0 += 32;
                if (b0 >= p.seq.batch) {
                    if (++pass >= passes) return false;
                    b0 = 0;
                }
            }
            if (p.seq.batch > 32) read(p, b0 + lane);
            count(p, lane);
        }
        const long long before = base + upto - own;
        const unsigned owner = __ballot_sync(0xffffffffu, nth >= part_count(before) && nth < part_count(before + own));
        const int src = __ffs(owner) - 1;
        const int at = __shfl_sync(0xffffffffu, nth - static_cast<int>(part_count(before)), src);
        g->slot = __shfl_sync(0xffffffffu, static_cast<int>(before >> kPartBits), src) + at;
        g->b = b0 + src;
        g->first = __shfl_sync(0xffffffffu, s.first, src);
        g->n = __shfl_sync(0xffffffffu, s.end, src) - g->first;
        g->keys = __shfl_sync(0xffffffffu, s.keys, src);
        g->parts = __shfl_sync(0xffffffffu, parts, src);
        const int item = static_cast<int>(static_cast<unsigned>(at) / static_cast<unsigned>(g->parts));
        g->part = at - item * g->parts;
        g->slot -= g->part;
        if (g->parts > p.grid - (nth - g->part) || (g->parts > 1 && g->parts > p.partials - g->slot)) return false;
        const int blocks = __shfl_sync(0xffffffffu, x.x, src);
        g->head = static_cast<int>(static_cast<unsigned>(item) / static_cast<unsigned>(blocks));
        const int blk = item - g->head * blocks;
        g->row0 = (p.is_causal ? blocks - 1 - blk : blk) * p.rows;  // (the longest first)
        g->n_rows = min(p.rows, g->n * p.group - g->row0);
        const int p_first = g->keys - g->n;
        const int tok_lo = static_cast<int>(fast_div(div_group, static_cast<uint32_t>(g->row0)));
        const int tok_hi = static_cast<int>(fast_div(div_group, static_cast<uint32_t>(g->row0 + g->n_rows - 1)));
        walked_keys(p, g->keys, p_first + tok_lo, p_first + tok_hi, &g->vis_lo, &g->vis_hi);
        const int tile0 = g->vis_lo / kTile, tiles = g->vis_hi > g->vis_lo ? (g->vis_hi + kTile - 1) / kTile - tile0 : 0;
        int from, to;
        part_of(tiles, g->part, g->parts, &from, &to);
        g->lo = tile0 + from;
        g->n_tiles = to - from;
        return true;
    }
};
#endif

}  // namespace fa
