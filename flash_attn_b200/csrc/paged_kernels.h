// Arguments and launches of the attention kernels over a paged cache.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>
#include "fa_internal.h"
#include "paged_plan.cuh"
#include "sm100_ptx.cuh"

namespace fa {

// How the boxes of a pool's tensor map are told apart.  A box is the tokens of a page (128 of them at most) of one head:
//   whole rows: all 128 columns, eight tokens after eight, the first 64 columns of eight before the last 64 of them.  Its map counts the
//     pool's tokens in eights, pages and (where their stride is a number of eights) heads together: (64, 8, 2, eights, heads).
//   half rows: 64 columns, a box for each half: (columns, slots, heads, pages).  For 64-wide heads, heads that do not fill their
//     columns, and strides that the other does not reach.
// A box takes the SM about 80 cycles to issue however small it is, which is what small pages cost: 64 x 8192 keys, 8 K/V heads of 128
// columns, pages of 16 tokens: 347 us with half rows, 322 with whole ones (309 with pages of 128).
struct PageBoxes {
    int page_step, head_step;  // whole rows: eights from one page and one head to the next
    int head_coord;            // 1: heads have a coordinate of their own
    int outside;               // an eight beyond the pool
};

struct PagedArgs {
    PagedPlan plan;
    FastDiv div_group;        // query heads of a K/V head
    PageBoxes k_box, v_box;
    const void* q;
    void* o;
    float* lse;
    const int* page_table;
    long long table_stride;
    int table_width, num_pages, page_shift;
    int whole_rows;           // of K and V boxes
    int heads, head_dim;
    int tile_tokens;          // tokens of a query tile of 128 rows: 128 / group
    long long q_stride[2], o_stride[2];  // elements from one token and head to the next
    float scale_log2;
    const float* alibi_slopes;
    int o_is_fp32;
    int o_units;              // rows of the output begin at 16 bytes
    int o_tma;                // and 32 rows of a K/V head are whole tokens: they have a tensor map
    float* o_partial;         // [parts of split items][plan.rows][64 or 128], un-normalised
    float2* ml_partial;       // [parts of split items][plan.rows]: maximum (log2 units) and sum
    unsigned long long* counts;  // [parts of split items]: those of an item's first part are its count
    int* status;
#ifdef FA_TEST_SHORT_WAIT
    int leave_out;            // test build only: the first CTA loads no tile of its stream from this one on; -1: it loads them all
#endif
};

// columns: rows of a block, 1, 4, 8 or 16.
cudaError_t launch_paged_decode(const PagedArgs& a, const CUtensorMap& tk, const CUtensorMap& tv, int columns, bool bf16, unsigned grid,
                                cudaStream_t stream);
// D = 64 or 128 (head_dim rounded up), NQ query tiles a block.
template <int D, int NQ>
cudaError_t launch_paged_tiled(const PagedArgs& a, const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv, const CUtensorMap& to, bool bf16,
                               unsigned grid, cudaStream_t stream);
template <> cudaError_t launch_paged_tiled<64, 1>(const PagedArgs&, const CUtensorMap&, const CUtensorMap&, const CUtensorMap&, const CUtensorMap&, bool, unsigned, cudaStream_t);
template <> cudaError_t launch_paged_tiled<64, 2>(const PagedArgs&, const CUtensorMap&, const CUtensorMap&, const CUtensorMap&, const CUtensorMap&, bool, unsigned, cudaStream_t);
template <> cudaError_t launch_paged_tiled<128, 1>(const PagedArgs&, const CUtensorMap&, const CUtensorMap&, const CUtensorMap&, const CUtensorMap&, bool, unsigned, cudaStream_t);
template <> cudaError_t launch_paged_tiled<128, 2>(const PagedArgs&, const CUtensorMap&, const CUtensorMap&, const CUtensorMap&, const CUtensorMap&, bool, unsigned, cudaStream_t);

#ifdef __CUDACC__
// The pages of a tile of 128 keys, as the lanes of the warp that loads them have them: a box a lane.
struct PageLane {
    int page_rows, page_bytes;  // tokens and bytes of a box
    int nth;                    // page of the tile, >= 128 / page_rows: none
    int column;                 // first column of the box
    int to;                     // where it goes in the tile
};
// kHalves = 64-column halves of a row.
template <int kHalves>
__device__ __forceinline__ PageLane page_lane(const PagedArgs& a, int lane) {
    PageLane p;
    const bool whole = kHalves == 2 && a.whole_rows;
    p.page_rows = min(1 << a.page_shift, kTile);
    p.page_bytes = p.page_rows * (whole ? 256 : 128);
    p.nth = whole ? lane : lane / kHalves;
    p.column = whole ? 0 : lane % kHalves * 64;
    p.to = whole ? lane * p.page_bytes : lane % kHalves * (kTile * 128) + p.nth * p.page_bytes;
    return p;
}
// The page that this lane loads for a tile, -1: none (no row sees a key of it).  One that is not in the pool sets `bad` and gives a
// box outside of the tensor map, which lands as zeros.
__device__ __forceinline__ int page_lookup(const PagedArgs& a, const PageLane& p, const int* table, int tile, int vis_lo, int vis_hi, bool* bad) {
    const int key = tile * kTile + p.nth * p.page_rows;
    if (p.nth * p.page_rows >= kTile || key >= vis_hi || key + p.page_rows <= vis_lo) return -1;
    const int nth = key >> a.page_shift;
    const int page = nth < a.table_width ? __ldg(table + nth) : -1;
    if (page >= 0 && page < a.num_pages) return page;
    *bad = true;
    return a.num_pages;
}
template <int kHalves>
__device__ __forceinline__ void page_load(const PagedArgs& a, const PageBoxes& box, const PageLane& p, const CUtensorMap* map, uint32_t dst, uint32_t bar,
                                          int tile, int head, int page) {
    const uint32_t boxes = __popc(__ballot_sync(0xffffffffu, page >= 0));
    if ((threadIdx.x & 31) == 0) mbar_expect_tx(bar, boxes * p.page_bytes);
    __syncwarp();
    if (page < 0) return;
    const int slot = (tile * kTile) & ((1 << a.page_shift) - 1);
    if (kHalves == 2 && a.whole_rows)
        tma_load_5d(dst + p.to, map, bar, 0, 0, 0, page < a.num_pages ? page * box.page_step + head * box.head_step + (slot >> 3) : box.outside,
                    head * box.head_coord);
    else
        tma_load_4d(dst + p.to, map, bar, p.column, slot, head, page);
}
// Test build only (-DFA_TEST_SHORT_WAIT): whether tile n of the CTA's stream is not loaded, so that the bounded waits behind it run out.
__device__ __forceinline__ bool left_out(const PagedArgs& a, int n) {
#ifdef FA_TEST_SHORT_WAIT
    return blockIdx.x == 0 && a.leave_out >= 0 && n >= a.leave_out;
#else
    return false;
#endif
}
// Zeros over the rows of a tile outside [head, tail), by a warp.
template <int kHalves>
__device__ __forceinline__ void clear_rows(const PagedArgs& a, uint32_t tile, int head, int tail) {
    const bool whole = kHalves == 2 && a.whole_rows;
    for (int i = threadIdx.x & 31; i < kTile * kHalves * 8; i += 32) {
        const int row = whole ? (i >> 7) * 8 + ((i >> 3) & 7) : (i >> 3) % kTile;
        if (row < head || row >= tail) st_shared_v4(tile + i * 16, 0u, 0u, 0u, 0u);
    }
    fence_proxy_async_smem();
    __syncwarp();
}
#endif

}  // namespace fa
