// Attention of few rows a sequence over a paged K/V cache (single tokens, the check of guessed tokens): HBM-bound, each K/V byte used
// once.
//
// A CTA walks parts of the keys of blocks of rows, one behind the other (paged_parts.cuh).  The operands are swapped, as in the decode
// kernel for contiguous K/V, so that the 128 lanes of tensor memory hold KEYS:
//     S^T[128 keys x 16] = K_tile[128 x d] * Q^T[d x 16],   O^T[d x 16] += V_tile^T[d x 128 keys] * P[128 keys x 16]
// with the block's rows (a row is a token and a query head; the heads of a K/V head lie side by side) in the first kH columns.
// A tile of 128 keys is 128 / page_size pages, or a part of one: a lane of the producer warp looks a page up and issues its box, so
// that all boxes of a tile leave in one instruction and the lookup's latency hides behind the wait for a free slot.  Pages of which
// no row sees a key are not looked up.
//
// [64 x 32 heads on 8, 8192 keys each, d 128]: 322 us with pages of 16 tokens, 6.7 TB/s; 100 .. 8192 keys: 82 us, 5.4 TB/s (set-up 5 us, the
// last parts 8); one sequence of 1000 keys: 13 us.  The code is kept short on purpose: what runs once is fetched from HBM first.
// Spills at 168 registers (bytes stored): 130 and 90 with one column of D = 128 and 64, 24 with four, 8 with eight, none with sixteen.
//
// What the pool holds beyond a sequence is not known, and 0 * NaN is NaN: keys that no row sees have P = 0 by their scores, and
// their rows of a V tile are overwritten with zeros before its MMAs, on the first and last tile of a block.
#include <algorithm>
#include <atomic>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <type_traits>
#include "decode_mma.cuh"
#include "paged_kernels.h"
#include "paged_merge.cuh"
#include "paged_plan.cuh"
#include "paged_parts.cuh"
#include "sm100_ptx.cuh"

namespace fa {

namespace {

constexpr int kPThreads = 192;  // four softmax warps, producer, MMA issuer
constexpr int kSegs = 4;        // parts that the producer may have handed on before the first of them is done
constexpr float kPLog2e = 1.4426950408889634f;
constexpr float kPLn2 = 0.6931471805599453f;

// kH = columns in use of the 16: 1, 4, 8 or 16.  D = 64 or 128 (head_dim rounded up).
template <int kH, int D>
struct PCfg {
    static constexpr int kChunk = 2;                  // KV tiles of a softmax step
    static constexpr int kTmemO = 2 * kChunk * 16;    // S^T: 2 buffers of kChunk tiles x 16 columns; O^T: 16 columns behind them
    static constexpr int kTmemCols = 128;
    static constexpr int kTileBytes = kTile * D * 2;
    static constexpr int kStages = D == 64 ? 6 : 3;   // 96 KB in flight either way
    static constexpr int kQBufs = kH == 16 ? 1 : 2;   // of the next item's rows beside this one's, where there is room
    static constexpr int kNumBars = 2 * kStages + 2 + 2 + 3 + 2 * kQBufs + 2 * kSegs + 1;
    static constexpr int kHalfBytes = kH == 16 ? 2048 : 1024;  // K-major operand of 16 rows: from the first 64 elements to the second
    static constexpr int kOperandBytes = 2 * kHalfBytes;
    static constexpr int kSmemRing = 0;
    static constexpr int kSmemP = kStages * kTileBytes;  // (before that: sums of the plan)
    static constexpr int kSmemQ = kSmemP + kChunk * kOperandBytes + (kH == 16 ? 0 : 1024);  // (+ what rows 8-15 touch)
    static constexpr int kSmemBar = kSmemQ + kQBufs * kOperandBytes + (kH == 16 ? 0 : 1024);
    static constexpr int kSmemRed = (kSmemBar + 8 * kNumBars + 15) / 16 * 16;  // float[2][4][kH] maxima, float[4][kH] sums
    static constexpr int kSmemMisc = kSmemRed + 3 * 4 * kH * 4;
    static constexpr int kSmemSegs = kSmemMisc + 32 + 4 * kSegs;                // PagedSeg[kSegs + 1], a taken CTA
    static constexpr int kSmemEnd = kSmemSegs + (kSegs + 1) * static_cast<int>(sizeof(PagedSeg)) + 16;
    static constexpr int kSmemReach = kSmemP + (D == 64 ? 1024 : 0);  // V^T is an M = 128 operand: with D = 64 its upper rows read the next eight keys
    static constexpr int kSmemBytes = (kSmemEnd > kSmemReach ? kSmemEnd : kSmemReach) + 1024;
    static_assert(kSmemBytes <= 115712, "two CTAs per SM");
    
};

// Whether `ok` holds for all of the 128 threads of named barrier 1.
__device__ __forceinline__ bool all_of_128(bool ok) {
    uint32_t all;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.u32 p, %1, 0;\n\t"
        "barrier.cta.red.and.pred q, 1, 128, p;\n\t"
        "selp.u32 %0, 1, 0, q;\n\t}"
        : "=r"(all) : "r"(ok ? 1u : 0u) : "memory");
    return all != 0;
}

template <bool kBf16, int kH, int D>
__global__ void __launch_bounds__(kPThreads, 2)
paged_decode_kernel(const __grid_constant__ CUtensorMap tmap_k, const __grid_constant__ CUtensorMap tmap_v, const __grid_constant__ PagedArgs a) {
    using C = PCfg<kH, D>;
    constexpr int kChunkTiles = C::kChunk, kStages = C::kStages, kTileBytes = C::kTileBytes, kHalves = D / 64;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t* smem_gen = smem_raw + (smem_base - smem_u32(smem_raw));
    const uint32_t sRing = smem_base + C::kSmemRing, sP = smem_base + C::kSmemP, sQ = smem_base + C::kSmemQ, bar0 = smem_base + C::kSmemBar;
    const uint32_t bar_full = bar0;                        // [kStages]
    const uint32_t bar_empty = bar_full + 8 * kStages;     // [kStages]
    const uint32_t bar_s_full = bar_empty + 8 * kStages;   // [2]
    const uint32_t bar_s_free = bar_s_full + 16;           // [2]
    const uint32_t bar_p_full = bar_s_free + 16;
    const uint32_t bar_p_free = bar_p_full + 8;
    const uint32_t bar_o_done = bar_p_free + 8;
    const uint32_t bar_q_full = bar_o_done + 8;            // [kQBufs]
    const uint32_t bar_q_free = bar_q_full + 8 * C::kQBufs;  // [kQBufs]
    const uint32_t bar_seg_full = bar_q_free + 8 * C::kQBufs;  // [kSegs]
    const uint32_t bar_seg_free = bar_seg_full + 8 * kSegs;    // [kSegs]
    const uint32_t bar_taken = bar_seg_free + 8 * kSegs;
    float* red = reinterpret_cast<float*>(smem_gen + C::kSmemRed);
    volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(smem_gen + C::kSmemMisc);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(smem_gen + C::kSmemMisc + 4);
    volatile int* last_flag = reinterpret_cast<volatile int*>(smem_gen + C::kSmemMisc + 8);
    volatile int* handed_on = reinterpret_cast<volatile int*>(smem_gen + C::kSmemMisc + 12);  // parts so far
    volatile int* left_over = reinterpret_cast<volatile int*>(smem_gen + C::kSmemMisc + 16);  // 1: a part that was taken too late to be handed on
    volatile int* done = reinterpret_cast<volatile int*>(smem_gen + C::kSmemMisc + 20);       // parts that the softmax warps are done with
    volatile int* give_up = reinterpret_cast<volatile int*>(smem_gen + C::kSmemMisc + 24);    // 1: not even a taken CTA's number came
    volatile int* bad_seg = reinterpret_cast<volatile int*>(smem_gen + C::kSmemMisc + 32);    // [kSegs]: the part met a bad page
    PagedSeg* segs = reinterpret_cast<PagedSeg*>(smem_gen + C::kSmemSegs);
    const uint32_t taken = smem_base + C::kSmemSegs + (kSegs + 1) * static_cast<int>(sizeof(PagedSeg));

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    grid_dep_launch_dependents();
    if (warp == 4 && lane == 0) {
        *abort_flag = 0;
        *handed_on = 0;
        *left_over = 0;
        *give_up = 0;
        for (int i = 0; i < kSegs; ++i) {
            mbar_init(bar_seg_full + 8 * i, 1);
            mbar_init(bar_seg_free + 8 * i, 5);  // (the MMA warp and the softmax warps)
        }
        mbar_init(bar_taken, 1);
        tma_prefetch_desc(&tmap_k);
        tma_prefetch_desc(&tmap_v);
        for (int i = 0; i < C::kQBufs; ++i) {
            mbar_init(bar_q_full + 8 * i, 32);
            mbar_init(bar_q_free + 8 * i, 1);
        }
        for (int s = 0; s < kStages; ++s) {
            mbar_init(bar_full + 8 * s, 1);
            mbar_init(bar_empty + 8 * s, 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(bar_s_full + 8 * i, 1);
            mbar_init(bar_s_free + 8 * i, 4);
        }
        mbar_init(bar_p_full, 4);
        mbar_init(bar_p_free, 1);
        mbar_init(bar_o_done, 1);
        mbar_fence_init();
    }
    grid_dep_wait();  // every thread, before its first global access
    auto chunk_tiles = [](int tiles, int c) { return min(kChunkTiles, tiles - c * kChunkTiles); };

    long long tiles_in_all = 0;
    if (a.plan.seq.batch > kWarpSeqs) {
        long long sum = 0;
        for (int b = threadIdx.x; b < a.plan.seq.batch; b += kPThreads) {
            const int2 x = blocks_and_tiles(a.plan, seq_span(a.plan.seq, b));
            sum += static_cast<long long>(x.x) * x.y;
        }
        sum = sum_all(sum);
        long long* sums = reinterpret_cast<long long*>(smem_gen + C::kSmemP);
        if (lane == 0) sums[warp] = sum;
        __syncthreads();
        for (int i = 0; i < kPThreads / 32; ++i) tiles_in_all += sums[i];
        tiles_in_all *= a.plan.heads_k;
    }
    // ---- set-up.  The producer does not wait for it.
    if (warp == 5) {
        tmem_alloc(smem_u32(const_cast<uint32_t*>(tmem_slot)), C::kTmemCols);
        tmem_relinquish();
        tc_fence_before_sync();
    }
    if (warp == 4) {
        __syncwarp();
        asm volatile("bar.arrive 2, %0;" ::"n"(kPThreads) : "memory");
    } else {
        asm volatile("bar.sync 2, %0;" ::"n"(kPThreads) : "memory");
        tc_fence_after_sync();
    }
    // The rows of a part: column `lane`'s token, query head, maximum and sum, and this thread's column of all rows.  By the softmax warps.
    auto finish = [&](const PagedSeg& g, int my_tok, int my_head, float m_ref, float l_all, const uint32_t (&o_raw)[kH]) {
        const int r = threadIdx.x;
        const long long part_row = g.parts > 1 ? (static_cast<long long>(g.slot) + g.part) * kH : 0;
#pragma unroll
        for (int n = 0; n < kH; ++n) {
            const float m_n = __shfl_sync(0xffffffffu, m_ref, n), l_sum = __shfl_sync(0xffffffffu, l_all, n);
            const int tok = __shfl_sync(0xffffffffu, my_tok, n), head = __shfl_sync(0xffffffffu, my_head, n);
            if (n >= g.n_rows) continue;
            const long long token = static_cast<long long>(g.first) + tok;
            if (g.parts > 1) {  // un-normalised, for the last part to come
                if (r < D) a.o_partial[(part_row + n) * D + r] = __uint_as_float(o_raw[n]);
                if (r == 0) a.ml_partial[part_row + n] = make_float2(m_n, l_sum);
            } else {
                const long long at = token * a.o_stride[0] + head * a.o_stride[1] + r;
                const float o_val = l_sum == 0.0f ? 0.0f : __uint_as_float(o_raw[n]) * (1.0f / l_sum);
                if (r < a.head_dim) {
                    if (a.o_is_fp32) static_cast<float*>(a.o)[at] = o_val;
                    else if (kBf16) static_cast<__nv_bfloat16*>(a.o)[at] = __float2bfloat16_rn(o_val);
                    else static_cast<__half*>(a.o)[at] = __float2half_rn(o_val);
                }
                if (r == 0 && a.lse != nullptr) a.lse[token * a.heads + head] = l_sum == 0.0f ? -INFINITY : fmaf(m_n, kPLn2, logf(l_sum));
            }
        }
        if (g.parts > 1 && last_to_come<128>(a, g.slot, g.parts, last_flag))
            merge_parts<D, kBf16, 4, (kH < 4 ? 1 : kH / 4)>(a, g.slot, g.parts, g.head, g.first, g.row0, g.n_rows, warp);
    };
    int fail = 0;

    if (warp == 4) {
        // ======================= producer =======================================
        // The stream of tiles, chunk by chunk and part by part: K(0), K(1), V(0), K(2), V(1), ...
        const PageLane mine = page_lane<kHalves>(a, lane);
        // The parts: the CTA's own, then those of CTAs that have not started.
        PartLine line;
        int index = static_cast<int>(blockIdx.x), asked = 0, answered = 0;
        auto ask = [&] {
            if (asked > answered || index < 0) return;
            if (lane == 0) {
                mbar_expect_tx(bar_taken, 16);
                launch_take(taken, bar_taken);
            }
            ++asked;
        };
        auto answer = [&](volatile int* give_up) -> bool {  // to the last question: index
            if (!mbar_wait_warp_ok(bar_taken, answered & 1, give_up)) return false;
            index = launch_taken(taken);
            fence_proxy_async_smem();  // (read before the next answer is written)
            __syncwarp();
            ++answered;
            return true;
        };
        line.start(a.plan, lane, tiles_in_all);
        int nth = 0;        // parts handed on
        bool owed = false;  // `index` was taken and is not handed on yet
        auto find = [&](int at) -> int {  // part `index` into segs[at]: its tiles, -1: there is no such part
            PagedSeg g;
            const bool have = index >= 0 && line.find(a.plan, a.div_group, index, lane, &g);
            if (!have) g.n_rows = 0;
            if (lane == 0) segs[at] = g;
            __syncwarp();
            return have ? g.n_tiles : -1;
        };
        // The tiles of the next part (there may be none of them), -1: there is no other part.  false: a wait gave up.
        auto next_part = [&](int* tiles) -> bool {
            if (nth > 0) {
                ask();
                if (asked > answered && !answer(abort_flag)) return false;
            }
            owed = index >= 0;
            const int at = nth % kSegs;
            if (nth >= kSegs && !mbar_wait_warp_ok(bar_seg_free + 8 * at, (nth / kSegs - 1) & 1, abort_flag)) return false;
            for (;;) {
                *tiles = find(at);
                owed = false;
                if (*tiles >= 0 || index < 0) break;
                ask();  // a CTA behind the last part need not start; one before it may still be taken
                if (!answer(abort_flag)) return false;
            }
            if (lane == 0) {
                bad_seg[at] = 0;
                *handed_on = nth + 1;
                mbar_arrive(bar_seg_full + 8 * at);
            }
            __syncwarp();
            ++nth;
            return true;
        };
        int slot = 0;
        auto push_chunk = [&](bool of_k, int part, int tiles, int c) -> bool {
            const PagedSeg& g = segs[part % kSegs];  // (not free before its last V tile has been used)
            const int vis_lo = g.vis_lo, vis_hi = g.vis_hi, head = g.head, tile0 = g.lo + c * kChunkTiles;
            const int* table = a.page_table + g.b * a.table_stride;
            for (int t = 0; t < chunk_tiles(tiles, c); ++t) {
                const int st = slot % kStages, tile = tile0 + t;
                if (left_out(a, slot)) {
                    ++slot;
                    continue;
                }
                bool bad = false;
                const int page = page_lookup(a, mine, table, tile, vis_lo, vis_hi, &bad);
                if (__any_sync(0xffffffffu, bad) && lane == 0) {
                    bad_seg[part % kSegs] = 1;  // (before what the readers' barriers wait for)
                    if (a.status != nullptr) atomicExch(a.status, FA_STATUS_PAGE);
                }
                if (!mbar_wait_warp_ok(bar_empty + 8 * st, ((slot / kStages) & 1) ^ 1, abort_flag)) return false;
                page_load<kHalves>(a, of_k ? a.k_box : a.v_box, mine, of_k ? &tmap_k : &tmap_v, sRing + st * kTileBytes, bar_full + 8 * st, tile, head, page);
                ++slot;
            }
            return true;
        };
        // row n of the block goes to row n of the Q operand (16-byte unit u -> half u/8, unit (u%8) ^ (n%8): the 128-byte swizzle)
        auto push_q = [&](int part, int of) -> bool {
            const PagedSeg& g = segs[part % kSegs];
            const int row0 = g.row0, n_rows = g.n_rows, head0 = g.head * a.plan.group;
            const long long token0 = g.first;
            const int buf = of % C::kQBufs;
            if (of >= C::kQBufs && !mbar_wait_warp_ok(bar_q_free + 8 * buf, (of / C::kQBufs - 1) & 1, abort_flag)) return false;
            constexpr int kUnits = D / 8;
#pragma unroll
            for (int i0 = 0; i0 < kUnits * kH; i0 += 32) {
                const int i = i0 + lane, u = i % kUnits, n = i / kUnits;
                const bool take = i < kUnits * kH && n < n_rows && u * 8 < a.head_dim;
                const uint16_t* from = static_cast<const uint16_t*>(a.q);
                if (take) {
                    const int tok = static_cast<int>(fast_div(a.div_group, static_cast<uint32_t>(row0 + n)));
                    const int head = head0 + row0 + n - tok * a.plan.group;
                    from += (token0 + tok) * a.q_stride[0] + head * a.q_stride[1] + u * 8;
                }
                if (i < kUnits * kH)
                    copy16_async_if(sQ + buf * C::kOperandBytes + (u >> 3) * C::kHalfBytes + n * 128 + (((u & 7) ^ (n & 7)) << 4), from, take);
            }
            copies_arrive(bar_q_full + 8 * buf);
            return true;
        };
        // The K tiles are a chunk ahead of the V tiles: part, its tiles, chunk; K's part among those with tiles.  A part without tiles
        // takes a turn of each, in which nothing is loaded: were several handed on in one turn, the ring could be full of them while
        // the last V tiles of the part before, which its oldest place waits for, are still to be issued.
        int k_part = 0, k_tiles = 0, ck = 0, v_part = 0, v_tiles = -1, cv = 0, nk = -1;
        bool ok = true;
        while (ok && (k_tiles >= 0 || v_tiles >= 0)) {
            if (k_tiles >= 0 && ++ck * kChunkTiles >= k_tiles) {
                ok = next_part(&k_tiles);
                ck = 0;
                k_part = nth - 1;
                if (ok && k_tiles > 0) ok = push_q(k_part, ++nk);
            }
            // (the answer is here when it is needed, and a long part leaves the next to who is sooner done)
            if (ok && k_tiles >= 0 && (ck + 1) * kChunkTiles >= k_tiles) ask();
#pragma unroll 1
            for (int kv = 0; kv < 2; ++kv) {
                const bool of_k = kv == 0;
                if (ok && (of_k ? k_tiles : v_tiles) > 0) ok = push_chunk(of_k, of_k ? k_part : v_part, of_k ? k_tiles : v_tiles, of_k ? ck : cv);
            }
            if (v_tiles < 0 || ++cv * kChunkTiles >= v_tiles) {
                v_part = k_part;
                v_tiles = k_tiles;
                cv = 0;
            }
        }
        if (!ok) {  // a part may have been taken that nobody else will do
            if (asked > answered && answer(give_up)) owed = index >= 0;
            if (owed && find(kSegs) >= 0) *left_over = 1;
        }
        copies_wait_all();
        if (!ok) fail = 1;
    } else if (warp == 5) {
        // ======================= MMA issuer =====================================
        constexpr uint32_t idesc_qk = make_idesc_swapped(kBf16, false);
        constexpr uint32_t idesc_pv = make_idesc_swapped(kBf16, true);
        // bytes from eight keys of a tile to the next, and from their first 64 columns to the others
        const uint32_t eight_bytes = D == 128 && a.whole_rows ? 2048 : 1024, half_bytes = D == 64 || a.whole_rows ? 1024 : kTile * 128;
        const uint32_t tmem_base = *tmem_slot, tmem_o = tmem_base + C::kTmemO;
        int slot = 0, qk_chunks = 0, pv_chunks = 0;
        auto qk_chunk = [&](int tiles, int c, int nth) -> bool {
            const int buf = qk_chunks & 1, q_buf = nth % C::kQBufs;
            if (qk_chunks >= 2 && !mbar_wait_warp_ok(bar_s_free + 8 * buf, ((qk_chunks >> 1) - 1) & 1, abort_flag)) return false;
            if (c == 0) {
                if (!mbar_wait_warp_ok(bar_q_full + 8 * q_buf, (nth / C::kQBufs) & 1, abort_flag)) return false;
                fence_proxy_async_smem();  // (copied by threads, read by the tensor core)
            }
            const uint32_t q = sQ + q_buf * C::kOperandBytes;
            for (int t = 0; t < chunk_tiles(tiles, c); ++t) {
                const int st = slot % kStages;
                if (!mbar_wait_warp_ok(bar_full + 8 * st, (slot / kStages) & 1, abort_flag)) return false;
                tc_fence_after_sync();
                const uint32_t kt = sRing + st * kTileBytes;
                if (lane == 0) {
#pragma unroll
                    for (int ks = 0; ks < D / 16; ++ks) {
                        const uint32_t off = (ks / 4) * half_bytes + (ks % 4) * 32;
                        const uint32_t qoff = (ks / 4) * C::kHalfBytes + (ks % 4) * 32;
                        umma_ss(tmem_base + buf * (kChunkTiles * 16) + t * 16, make_smem_desc(kt + off, 0, eight_bytes), make_smem_desc(q + qoff, 0, 1024), idesc_qk,
                                ks > 0 ? 1u : 0u);
                    }
                    umma_commit(bar_empty + 8 * st);
                }
                ++slot;
            }
            if (lane == 0) {
                umma_commit(bar_s_full + 8 * buf);
                if ((c + 1) * kChunkTiles >= tiles) umma_commit(bar_q_free + 8 * q_buf);
            }
            ++qk_chunks;
            return true;
        };
        auto pv_chunk = [&](int part, int tiles, int c) -> bool {
            const PagedSeg& g = segs[part % kSegs];
            const int vis_lo = g.vis_lo, vis_hi = g.vis_hi, tile0 = g.lo + c * kChunkTiles;
            if (!mbar_wait_warp_ok(bar_p_full, pv_chunks & 1, abort_flag)) return false;
            tc_fence_after_sync();
            for (int t = 0; t < chunk_tiles(tiles, c); ++t) {
                const int st = slot % kStages;
                if (!mbar_wait_warp_ok(bar_full + 8 * st, (slot / kStages) & 1, abort_flag)) return false;
                tc_fence_after_sync();
                const uint32_t vt = sRing + st * kTileBytes;
                const int key0 = (tile0 + t) * kTile;
                if (key0 < vis_lo || key0 + kTile > vis_hi) {
                    // rows that no query row sees may hold anything
                    clear_rows<kHalves>(a, vt, max(vis_lo - key0, 0), min(max(vis_hi - key0, 0), kTile));
                }
                if (lane == 0) {
#pragma unroll
                    for (int ks = 0; ks < 8; ++ks) {
                        // A = V^T: 16 keys a step
                        const uint32_t poff = t * C::kOperandBytes + (ks / 4) * C::kHalfBytes + (ks % 4) * 32;
                        umma_ss(tmem_o, make_smem_desc(vt + ks * 2 * eight_bytes, half_bytes, eight_bytes), make_smem_desc(sP + poff, 0, 1024), idesc_pv,
                                (c > 0 || t > 0 || ks > 0) ? 1u : 0u);
                    }
                    umma_commit(bar_empty + 8 * st);
                }
                ++slot;
            }
            if (lane == 0) {
                umma_commit(bar_p_free);
                if ((c + 1) * kChunkTiles >= tiles) umma_commit(bar_o_done);
            }
            ++pv_chunks;
            return true;
        };
        auto free_part = [&](int part) {
            __syncwarp();
            if (lane == 0) mbar_arrive(bar_seg_free + 8 * (part % kSegs));
        };
        int k_part = -1, k_tiles = 0, ck = 0, v_part = 0, v_tiles = -1, cv = 0, nk = -1;
        bool ok = true;
        while (ok && (k_tiles >= 0 || v_tiles >= 0)) {
            if (k_tiles >= 0 && ++ck * kChunkTiles >= k_tiles) {
                ++k_part;
                ok = mbar_wait_warp_ok(bar_seg_full + 8 * (k_part % kSegs), (k_part / kSegs) & 1, abort_flag);
                if (ok) k_tiles = segs[k_part % kSegs].n_rows > 0 ? segs[k_part % kSegs].n_tiles : -1;
                ck = 0;
                if (k_tiles > 0) ++nk;
            }
            if (ok && k_tiles > 0) ok = qk_chunk(k_tiles, ck, nk);
            if (ok && v_tiles > 0) ok = pv_chunk(v_part, v_tiles, cv);
            if (v_tiles < 0 || ++cv * kChunkTiles >= v_tiles) {
                if (v_tiles >= 0) free_part(v_part);
                v_part = k_part;
                v_tiles = k_tiles;
                cv = 0;
            }
        }
        if (!ok) fail = 2;
    } else {
        // ======================= softmax over keys / epilogue ===================
        // (A wait that gives up does not end the walk: every part writes its rows, as NaN, and counts itself in.)
        const uint32_t tmem_base = *tmem_slot, tmem_o = tmem_base + C::kTmemO;
        const int r = threadIdx.x;  // key inside a tile; output column in the epilogue
        const uint32_t lane_base = static_cast<uint32_t>(warp * 32) << 16;
        // scores stay unscaled and the scale is folded into the exponent's FMA, except with ALiBi
        const bool alibi = a.alibi_slopes != nullptr;
        const float scale2 = a.scale_log2, exp_scale = alibi ? 1.0f : a.scale_log2;
        // this key's element of column n in the P operand: row n, 128-byte swizzled
        uint8_t* p_half = smem_gen + C::kSmemP + (r >> 6) * C::kHalfBytes + (r & 7) * 2;
        const uint32_t p_unit = static_cast<uint32_t>((r & 63) >> 3);
        PagedSeg g;
        int chunks = 0;      // of all parts so far
        int with_tiles = 0;  // parts so far that had tiles
        int nth = 0;
        for (;; ++nth) {
            // (all four warps go on, or none: the producer may hand a part on while a wait gives up)
            if (!all_of_128(mbar_wait_warp_ok(bar_seg_full + 8 * (nth % kSegs), (nth / kSegs) & 1, abort_flag))) {
                fail = 6;
                break;
            }
            g = segs[nth % kSegs];
            if (g.n_rows == 0) break;
            const int p_first = g.keys - g.n;  // position of the sequence's first new token
            const int nc = g.n_rows;           // columns in use
            // column `lane`: its token and query head, its ALiBi slope; handed round
            const int my_tok = static_cast<int>(fast_div(a.div_group, static_cast<uint32_t>(g.row0 + lane)));
            const int my_head = g.head * a.plan.group + g.row0 + lane - my_tok * a.plan.group;
            // tiles [full_lo, full_hi) need no mask: every row sees all of their keys
            int full_lo, full_hi;
            {
                int l0, h0, l1, h1;
                const int tok_lo = __shfl_sync(0xffffffffu, my_tok, 0), tok_hi = __shfl_sync(0xffffffffu, my_tok, nc - 1);
                visible_keys(a.plan, g.keys, p_first + tok_lo, p_first + tok_lo, &l0, &h0);
                visible_keys(a.plan, g.keys, p_first + tok_hi, p_first + tok_hi, &l1, &h1);
                full_lo = (max(l0, l1) + kTile - 1) / kTile;
                full_hi = min(h0, h1) / kTile;
            }
            float slope = 0.0f;
            if (alibi && lane < nc) slope = a.alibi_slopes[my_head] * kPLog2e;
            float m_ref = -INFINITY;  // CTA-wide running max of column `lane` (lanes < kH of every warp), log2 units
            float l_part[kH];         // this thread's share of each column's row sum
#pragma unroll
            for (int n = 0; n < kH; ++n) l_part[n] = 0.0f;

            const int n_chunks = (g.n_tiles + kChunkTiles - 1) / kChunkTiles;
            for (int c = 0; c < n_chunks; ++c, ++chunks) {
                const int buf = chunks & 1;
                const int nt = chunk_tiles(g.n_tiles, c);
                const int tile0 = g.lo + c * kChunkTiles;
                if (!mbar_wait_warp_ok(bar_s_full + 8 * buf, (chunks >> 1) & 1, abort_flag)) fail = 3;
                tc_fence_after_sync();
                uint32_t raw[kChunkTiles][kH];
#pragma unroll
                for (int t = 0; t < kChunkTiles; ++t) {
                    if (t < nt) {
                        tmem_ld_heads<kH>(tmem_base + lane_base + buf * (kChunkTiles * 16) + t * 16, raw[t]);
                    } else {
#pragma unroll
                        for (int n = 0; n < kH; ++n) raw[t][n] = 0xff800000u;  // -inf
                    }
                }
                tmem_wait_ld();
                tc_fence_before_sync();
                __syncwarp();
                if (lane == 0) mbar_arrive(bar_s_free + 8 * buf);
                float v[kChunkTiles][kH];
#pragma unroll
                for (int t = 0; t < kChunkTiles; ++t) {
#pragma unroll
                    for (int n = 0; n < kH; ++n) v[t][n] = __uint_as_float(raw[t][n]);
                }
                if (alibi || tile0 < full_lo || tile0 + nt > full_hi) {
                    // keys relative to the sequence's first new token
                    int rel[kChunkTiles];
                    bool in_range[kChunkTiles];
#pragma unroll
                    for (int t = 0; t < kChunkTiles; ++t) {
                        const int key = (tile0 + t) * kTile + r;
                        in_range[t] = t < nt && key < g.keys;
                        rel[t] = key - p_first;
                    }
#pragma unroll
                    for (int n = 0; n < kH; ++n) {
                        const float slope_n = alibi ? __shfl_sync(0xffffffffu, slope, n) : 0.0f;
                        const int tok = __shfl_sync(0xffffffffu, my_tok, n);
#pragma unroll
                        for (int t = 0; t < kChunkTiles; ++t) {
                            const int ahead = rel[t] - tok;  // > 0: the key lies after the query
                            bool keep = in_range[t];
                            if (a.plan.is_causal && ahead > 0) keep = false;
                            if (a.plan.window_left >= 0 && -ahead > a.plan.window_left) keep = false;
                            if (a.plan.window_right >= 0 && ahead > a.plan.window_right) keep = false;
                            if (alibi) v[t][n] = fmaf(-slope_n, fabsf(static_cast<float>(ahead)), v[t][n] * scale2);
                            if (!keep) v[t][n] = -INFINITY;
                        }
                    }
                }
                float* red_c = red + buf * 4 * kH;
                {
                    float m_w[kH];
#pragma unroll
                    for (int n = 0; n < kH; ++n) {
                        float m = v[0][n];
#pragma unroll
                        for (int t = 1; t < kChunkTiles; ++t) m = fmaxf(m, v[t][n]);
                        m_w[n] = warp_max(m);
                    }
                    if (lane == 0) {
#pragma unroll
                        for (int n = 0; n < kH; ++n) red_c[warp * kH + n] = m_w[n];
                    }
                }
                named_barrier_128();

                // the previous chunk's P V must be done before P is overwritten or O rescaled
                if (chunks > 0) {
                    if (!mbar_wait_warp_ok(bar_p_free, (chunks - 1) & 1, abort_flag)) fail = 4;
                    tc_fence_after_sync();
                }
                // lane n keeps column n's running max (raised only when it grew by > 2^8) and hands it round
                float m_new = m_ref, factor = 1.0f;
                if (lane < kH) {
                    const float m_chunk = fmaxf(fmaxf(red_c[lane], red_c[kH + lane]), fmaxf(red_c[2 * kH + lane], red_c[3 * kH + lane])) * exp_scale;
                    if (m_chunk > m_ref + 8.0f || m_ref == -INFINITY) m_new = fmaxf(m_ref, m_chunk);
                    if (m_new != m_ref) factor = (m_ref == -INFINITY) ? 0.0f : ex2f(m_ref - m_new);
                }
                if (__any_sync(0xffffffffu, m_new != m_ref)) {  // CTA-uniform: every warp sees the same maxima
                    float f[kH];
#pragma unroll
                    for (int n = 0; n < kH; ++n) {
                        f[n] = __shfl_sync(0xffffffffu, factor, n);
                        l_part[n] *= f[n];
                    }
                    if (c > 0) {
                        uint32_t ov[kH];
                        tmem_ld_heads<kH>(tmem_o + lane_base, ov);
                        tmem_wait_ld();
#pragma unroll
                        for (int n = 0; n < kH; ++n) ov[n] = __float_as_uint(__uint_as_float(ov[n]) * f[n]);
                        tmem_st_heads<kH>(tmem_o + lane_base, ov);
                        tmem_wait_st();
                    }
                }
                m_ref = m_new;
                const float neg_lane = (m_new == -INFINITY) ? 0.0f : -m_new;

#pragma unroll
                for (int n = 0; n < kH; ++n) {
                    const float neg_m = __shfl_sync(0xffffffffu, neg_lane, n);
                    uint8_t* p_row = p_half + n * 128 + ((p_unit ^ (n & 7)) << 4);
#pragma unroll
                    for (int t = 0; t < kChunkTiles; t += 2) {
                        float p[2];
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            p[i] = ex2f(fmaf(v[t + i][n], exp_scale, neg_m));
                            l_part[n] += p[i];
                        }
                        uint32_t h;  // P is rounded to the inputs' type for the tensor core, two tiles' elements together; its sum is not
                        if constexpr (kBf16) {
                            const __nv_bfloat162 x = __floats2bfloat162_rn(p[0], p[1]);
                            h = *reinterpret_cast<const uint32_t*>(&x);
                        } else {
                            const __half2 x = __floats2half2_rn(p[0], p[1]);
                            h = *reinterpret_cast<const uint32_t*>(&x);
                        }
                        if (t < nt) *reinterpret_cast<uint16_t*>(p_row + t * C::kOperandBytes) = static_cast<uint16_t>(h);
                        if (t + 1 < nt) *reinterpret_cast<uint16_t*>(p_row + (t + 1) * C::kOperandBytes) = static_cast<uint16_t>(h >> 16);
                    }
                }
                fence_proxy_async_smem();
                tc_fence_before_sync();
                __syncwarp();
                if (lane == 0) mbar_arrive(bar_p_full);
            }

            // ---- epilogue ----------------------------------------------------------------
            uint32_t o_raw[kH];
#pragma unroll
            for (int n = 0; n < kH; ++n) o_raw[n] = 0u;
            float l_all = 0.0f;  // column `lane`'s sum
            if (g.n_tiles > 0) {
#pragma unroll
                for (int n = 0; n < kH; ++n) {
                    float l_warp = l_part[n];
#pragma unroll
                    for (int o = 16; o >= 1; o >>= 1) l_warp += __shfl_xor_sync(0xffffffffu, l_warp, o);
                    if (lane == 0) red[8 * kH + warp * kH + n] = l_warp;
                }
                if (mbar_wait_warp_ok(bar_o_done, with_tiles & 1, abort_flag)) {
                    tc_fence_after_sync();
                    tmem_ld_heads<kH>(tmem_o + lane_base, o_raw);
                    tmem_wait_ld();
                    tc_fence_before_sync();
                } else {
                    fail = 5;
                }
                named_barrier_128();
                // A wait gave up, or a visible page was not there (set by whoever saw it, before the last MMA could complete): none of
                // the rows may pass for a softmax.
                const float spoilt = *abort_flag != 0 || bad_seg[nth % kSegs] != 0 ? __int_as_float(0x7fc00000) : 0.0f;
                if (lane < kH) l_all = (red[8 * kH + lane] + red[9 * kH + lane]) + (red[10 * kH + lane] + red[11 * kH + lane]) + spoilt;
                ++with_tiles;
            }
            finish(g, my_tok, my_head, m_ref, l_all, o_raw);
            __syncwarp();
            if (lane == 0) mbar_arrive(bar_seg_free + 8 * (nth % kSegs));
        }
        if (r == 0) *done = nth;
    }

    if (fail != 0) {
        *abort_flag = 1;
        if (lane == 0 && a.status != nullptr) atomicExch(a.status, 300 + fail);
        const long long t0 = clock64();
        while (clock64() - t0 < 200000) { }  // (copies in flight land before the CTA's memory is another's)
    }
    tc_fence_before_sync();
    __syncthreads();
    if (*abort_flag != 0 && warp < 4) {
        // Parts that were taken and not done: their rows are NaN, and they are counted in, for the item's other parts.
        for (int i = *done, n = *handed_on + *left_over; i < n; ++i) {
            const PagedSeg g = segs[i < *handed_on ? i % kSegs : kSegs];
            if (g.n_rows == 0) continue;
            const int tok = static_cast<int>(fast_div(a.div_group, static_cast<uint32_t>(g.row0 + lane)));
            uint32_t none[kH];
#pragma unroll
            for (int n_col = 0; n_col < kH; ++n_col) none[n_col] = 0u;
            finish(g, tok, g.head * a.plan.group + g.row0 + lane - tok * a.plan.group, -INFINITY, __int_as_float(0x7fc00000), none);
        }
    }
    if (warp == 5) {
        __syncwarp();
        tc_fence_after_sync();
        tmem_dealloc(*tmem_slot, C::kTmemCols);
    }
}

}  // namespace

cudaError_t launch_paged_decode(const PagedArgs& a, const CUtensorMap& tk, const CUtensorMap& tv, int columns, bool bf16, unsigned grid,
                                cudaStream_t stream) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(kPThreads);
    cfg.stream = stream;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    auto run = [&](auto kern, int smem, std::atomic<bool>* configured) -> cudaError_t {
        if (dev < 0 || dev >= 64 || !configured[dev].load(std::memory_order_acquire)) {
            const cudaError_t err = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
            if (err != cudaSuccess) return err;
            if (dev >= 0 && dev < 64) configured[dev].store(true, std::memory_order_release);
        }
        cfg.dynamicSmemBytes = smem;
        return cudaLaunchKernelEx(&cfg, kern, tk, tv, a);
    };
    auto by_type = [&](auto h, auto wide) -> cudaError_t {
        constexpr int kH = decltype(h)::value, D = decltype(wide)::value, smem = PCfg<kH, D>::kSmemBytes;
        static std::atomic<bool> configured[2][64];
        return bf16 ? run(paged_decode_kernel<true, kH, D>, smem, configured[0]) : run(paged_decode_kernel<false, kH, D>, smem, configured[1]);
    };
    auto by_dim = [&](auto h) -> cudaError_t {
        return a.head_dim <= 64 ? by_type(h, std::integral_constant<int, 64>()) : by_type(h, std::integral_constant<int, 128>());
    };
    switch (columns) {
        case 1: return by_dim(std::integral_constant<int, 1>());
        case 4: return by_dim(std::integral_constant<int, 4>());
        case 8: return by_dim(std::integral_constant<int, 8>());
        default: return by_dim(std::integral_constant<int, 16>());
    }
}

}  // namespace fa
