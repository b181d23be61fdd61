// Attention of chunks of new tokens over a paged K/V cache: tensor-bound.
//
// A CTA walks parts of the keys of blocks of rows, one behind the other (paged_parts.cuh); a block is NQ query tiles of 128 rows.  A
// row is a token and a query head: the heads of a K/V head lie side by side in a tile (row = token * group + head, as one TMA box of Q
// lands), so that they share every K/V tile and a few tokens fill it; where the group does not divide 128 the tile's last rows are
// left over.
// The walk is the tiled kernel's for contiguous K/V: a TMA warp feeds a ring of K/V tiles, an MMA warp issues S = Q K^T into tensor
// memory, four softmax warps a query tile keep a row a thread, write P over S, and the MMA warp adds P V; two query tiles alternate
// on the tensor pipe.  A KV tile is 128 / page_size pages (or a part of one), a box each, looked up and issued by a lane each.
// KV tiles are visited from the last to the first: with a causal mask the second query tile's own diagonal tile comes first.
//
// What the pool holds beyond a sequence is not known, and 0 * NaN is NaN: rows of a V tile that no row of the block sees are
// overwritten with zeros before its MMAs (first and last tile only).
//
// 2048 tokens over 32768 keys, 32 heads on 8, d 128: twenty calls in a row 933 us each, 1.14 PFLOP/s, a thousand (under the power cap) 1042,
// 1.02; a KV tile of two query tiles 1.8 to 2.1 us (a chain of latencies of two softmax warps a scheduler).  Six prompts of 200 .. 2048
// tokens: 43 us, where parts of one to eight tiles begin and end.  Spills (bytes stored): 88 with two query tiles at D = 128, up to 16 at
// D = 64, 200 to 250 with one (128 registers at launch).
#include <algorithm>
#include <atomic>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <type_traits>
#include "paged_kernels.h"
#include "paged_merge.cuh"
#include "paged_parts.cuh"
#include "paged_plan.cuh"
#include "sm100_ptx.cuh"
#include "tiled_mma.cuh"

// (compiled once for each, side by side)
#if !defined(FA_PAGED_D) || !defined(FA_PAGED_NQ)
#error "compiled with FA_PAGED_D = 64 or 128 and FA_PAGED_NQ = 1 or 2"
#endif

namespace fa {

namespace {

constexpr float kRescaleThreshold = 8.0f;  // log2 units: rescale O only when the max grew by > 2^8
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr int kSegs = 4;  // parts that the producer may have handed on before the first of them is done

// The MMAs of one S = Q K^T tile in one asm block, so that the issuing thread does no other work between them (16-byte units: a k-step
// is 2 inside 64 columns; Q's next 64 columns lie 16 KB further, K's `k_jump` past their last step).
#define FA_PAGED_QK(qi, ki)                                                                    \
    "add.u32 qa, qa, " qi ";\n\tadd.u32 kb, kb, " ki ";\n\t"                                     \
    "mov.b64 da, {qa, %3};\n\tmov.b64 db, {kb, %4};\n\t"                                        \
    "tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %5, p1;\n\t"
template <int D>
__device__ __forceinline__ void issue_qk(uint32_t d_tmem, uint32_t q_lo, uint32_t k_lo, uint32_t q_hi, uint32_t k_hi, uint32_t k_jump, uint32_t idesc) {
#define FA_PAGED_QK_HEAD                                                                       \
    "{\n\t.reg .pred p0, p1;\n\t.reg .b32 qa, kb;\n\t.reg .b64 da, db;\n\t"                       \
    "setp.ne.b32 p0, 0, 0;\n\tsetp.eq.b32 p1, 0, 0;\n\tmov.b32 qa, %1;\n\tmov.b32 kb, %2;\n\t"      \
    "mov.b64 da, {qa, %3};\n\tmov.b64 db, {kb, %4};\n\t"                                        \
    "tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %5, p0;\n\t"
    if constexpr (D == 128) {
        asm volatile(FA_PAGED_QK_HEAD FA_PAGED_QK("2", "2") FA_PAGED_QK("2", "2") FA_PAGED_QK("2", "2") FA_PAGED_QK("1018", "%6") FA_PAGED_QK("2", "2")
                         FA_PAGED_QK("2", "2") FA_PAGED_QK("2", "2") "}"
                     ::"r"(d_tmem), "r"(q_lo), "r"(k_lo), "r"(q_hi), "r"(k_hi), "r"(idesc), "r"(k_jump)
                     : "memory");
    } else {
        asm volatile(FA_PAGED_QK_HEAD FA_PAGED_QK("2", "2") FA_PAGED_QK("2", "2") FA_PAGED_QK("2", "2") "}"
                     ::"r"(d_tmem), "r"(q_lo), "r"(k_lo), "r"(q_hi), "r"(k_hi), "r"(idesc)
                     : "memory");
    }
}
// Four MMAs of O += P V, from k-step kFrom on: P advances 8 columns of tensor memory a step, V `v_step`.
#define FA_PAGED_PV                                                                            \
    "add.u32 pa, pa, 8;\n\tadd.u32 vb, vb, %6;\n\tmov.b64 db, {vb, %3};\n\t"                       \
    "tcgen05.mma.cta_group::1.kind::f16 [%0], [pa], db, %4, p1;\n\t"
template <int kFrom>
__device__ __forceinline__ void issue_pv(uint32_t d_tmem, uint32_t p_tmem, uint32_t v_lo, uint32_t v_hi, uint32_t v_step, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p0, p1;\n\t.reg .b32 pa, vb;\n\t.reg .b64 db;\n\t"
        "setp.ne.b32 p0, %5, 0;\n\tsetp.eq.b32 p1, 0, 0;\n\tmov.b32 pa, %1;\n\tmov.b32 vb, %2;\n\tmov.b64 db, {vb, %3};\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [pa], db, %4, p0;\n\t" FA_PAGED_PV FA_PAGED_PV FA_PAGED_PV "}"
        ::"r"(d_tmem), "r"(p_tmem + kFrom * 8), "r"(v_lo + kFrom * v_step), "r"(v_hi), "r"(idesc), "r"(accumulate), "r"(v_step)
        : "memory");
}

template <int D, int NQ>
struct TCfg {
    static constexpr int kThreads = NQ == 2 ? 384 : 256;
    // Registers: the CTA owns kThreads * kRegsLaunch from launch on (168 a thread under __launch_bounds__(384, 1), 128 under (256, 2));
    // an increase that asks for more than the helper warps released would wait for ever.
    static constexpr int kRegsLaunch = NQ == 2 ? 168 : 128;
    static constexpr int kRegsHelper = NQ == 2 ? 72 : 48;
    static constexpr int kRegsSoftmax = NQ == 2 ? 216 : 208;
    static_assert(NQ * 128 * kRegsSoftmax + 128 * kRegsHelper <= kThreads * kRegsLaunch, "register hand-over exceeds the CTA's allocation");
    static constexpr int kProducerWarp = NQ * 4, kMmaWarp = NQ * 4 + 1;
    static constexpr int kStages = (D == 64) ? (NQ == 2 ? 3 : 2) : (NQ == 2 ? 2 : 1);
    static constexpr int kBoxes = D / 64;
    static constexpr int kTileBytes = kTile * D * 2;
    static constexpr int kTmemCols = NQ == 2 ? 512 : 256;  // S_i at i * 128 (P_i over its first half), O_i behind them
    static constexpr int kTmemO = NQ * kTile;
    static constexpr int kSmemQ = 0;
    static constexpr int kSmemK = NQ * kTileBytes;
    static constexpr int kSmemV = kSmemK + kStages * kTileBytes;
    static constexpr int kStageBytes = NQ == 2 || D == 64 ? 4096 : 2048;          // of its output rows that a warp has in shared memory at once
    static constexpr int kSmemRows = kSmemV + kStages * kTileBytes;
    static constexpr int kSmemBar = kSmemRows + NQ * 4 * kStageBytes;
    static constexpr int kNumBars = 2 + 2 * NQ + 4 * kStages + 2 * kSegs + 1;
    static constexpr int kSmemMisc = (kSmemBar + 8 * kNumBars + 15) / 16 * 16;  // tensor-memory address, abort flag, last part's flag
    static constexpr int kSmemSegs = kSmemMisc + 16 + 4 * kSegs;                // (which parts met a bad page;) PagedSeg[kSegs], a taken CTA
    static constexpr int kSmemBytes = kSmemSegs + kSegs * static_cast<int>(sizeof(PagedSeg)) + 16 + 1024;  // + alignment slack
    static_assert(kSmemBytes <= (NQ == 2 ? 232448 : 115712), "one or two CTAs per SM");
};

template <int D, int NQ, bool kBf16, bool kAlibi>
__global__ void __launch_bounds__(TCfg<D, NQ>::kThreads, NQ == 1 ? 2 : 1)
paged_tiled_kernel(const __grid_constant__ CUtensorMap tmap_q, const __grid_constant__ CUtensorMap tmap_k,
                   const __grid_constant__ CUtensorMap tmap_v, const __grid_constant__ CUtensorMap tmap_o, const __grid_constant__ PagedArgs a) {
    using C = TCfg<D, NQ>;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t* smem_gen = smem_raw + (smem_base - smem_u32(smem_raw));
    const uint32_t sQ = smem_base + C::kSmemQ, sK = smem_base + C::kSmemK, sV = smem_base + C::kSmemV, bar0 = smem_base + C::kSmemBar;
    const uint32_t bar_q_full = bar0;
    const uint32_t bar_s_full = bar0 + 8;                      // [NQ]
    const uint32_t bar_o_full = bar_s_full + 8 * NQ;           // [NQ]
    const uint32_t bar_k_full = bar_o_full + 8 * NQ;           // [kStages]
    const uint32_t bar_k_empty = bar_k_full + 8 * C::kStages;  // [kStages]
    const uint32_t bar_v_full = bar_k_empty + 8 * C::kStages;  // [kStages]
    const uint32_t bar_v_empty = bar_v_full + 8 * C::kStages;  // [kStages]
    const uint32_t bar_q_free = bar_v_empty + 8 * C::kStages;
    const uint32_t bar_taken = bar_q_free + 8;
    const uint32_t bar_seg_full = bar_taken + 8;               // [kSegs]
    const uint32_t bar_seg_free = bar_seg_full + 8 * kSegs;    // [kSegs]
    volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(smem_gen + C::kSmemMisc);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(smem_gen + C::kSmemMisc + 4);
    volatile int* last_flag = reinterpret_cast<volatile int*>(smem_gen + C::kSmemMisc + 8);
    volatile int* bad_seg = reinterpret_cast<volatile int*>(smem_gen + C::kSmemMisc + 16);  // [kSegs]: the part met a bad page
    PagedSeg* segs = reinterpret_cast<PagedSeg*>(smem_gen + C::kSmemSegs);
    const uint32_t taken = smem_base + C::kSmemSegs + kSegs * static_cast<int>(sizeof(PagedSeg));

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    grid_dep_launch_dependents();
    if (warp == C::kProducerWarp) {
        if (lane < C::kNumBars) mbar_init(bar0 + 8 * lane, bar0 + 8 * lane >= bar_seg_free ? 1 + NQ * 4 : 1);
        if (lane == 0) {
            *abort_flag = 0;
            tma_prefetch_desc(&tmap_q);
            tma_prefetch_desc(&tmap_k);
            tma_prefetch_desc(&tmap_v);
        }
        __syncwarp();
        if (lane == 0) mbar_fence_init();
    }
    grid_dep_wait();  // every thread, before its first global access
    long long tiles_in_all = 0;
    if (a.plan.seq.batch > kWarpSeqs) {
        long long sum = 0;
        for (int b = threadIdx.x; b < a.plan.seq.batch; b += C::kThreads) {
            const int2 x = blocks_and_tiles(a.plan, seq_span(a.plan.seq, b));
            sum += static_cast<long long>(x.x) * x.y;
        }
        sum = sum_all(sum);
        long long* sums = reinterpret_cast<long long*>(smem_gen + C::kSmemRows);
        if (lane == 0) sums[warp] = sum;
        __syncthreads();
        for (int i = 0; i < C::kThreads / 32; ++i) tiles_in_all += sums[i];
        tiles_in_all *= a.plan.heads_k;
    }
    const int tile_tokens = a.tile_tokens, tile_rows = tile_tokens * a.plan.group;
    // The tiles of a part that query tile i walks: [lo, hi).
    struct Range { int lo, hi; };
    auto range_of = [&](const PagedSeg& g, int token0, int i) -> Range {
        const int t0 = token0 + i * tile_tokens, t1 = min(t0 + tile_tokens, g.n) - 1;
        int l = 0, h = 0;
        if (t1 >= t0) visible_keys(a.plan, g.keys, g.keys - g.n + t0, g.keys - g.n + t1, &l, &h);
        const int lo = max(h > l ? l / kTile : g.lo, g.lo);
        return {lo, max(min(h > l ? (h + kTile - 1) / kTile : lo, g.lo + g.n_tiles), lo)};
    };
    auto token_of = [&](const PagedSeg& g) { return static_cast<int>(fast_div(a.div_group, static_cast<uint32_t>(g.row0))); };
    // Parts are handed on and freed whatever else gives up: every warp walks all parts of the CTA, so that each is counted in.  (No flag ends these waits; each is bounded all the same.)
    auto wait_part = [&](uint32_t bar, uint32_t parity) -> bool {
        for (int i = 0; i < 8; ++i) {
            volatile int own = 0;
            if (mbar_wait_warp(bar, parity, &own)) return true;
        }
        return false;
    };

    // ---- set-up: tensor memory
    if (warp == C::kMmaWarp) {
        tmem_alloc(smem_u32(const_cast<uint32_t*>(tmem_slot)), C::kTmemCols);
        tmem_relinquish();
    }
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    const uint32_t tmem_base = *tmem_slot;

    int fail = 0;
    if (warp >= NQ * 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::kRegsHelper));
        if (warp == C::kProducerWarp) {
            // ======================= producer =======================================
            const PageLane page_box = page_lane<C::kBoxes>(a, lane);
            PartLine line;
            line.start(a.plan, lane, tiles_in_all);
            int index = static_cast<int>(blockIdx.x), asked = 0, answered = 0;  // the CTA whose part is next; -1: there is none
            auto ask = [&] {
                if (asked > answered || index < 0 || fail != 0) return;
                if (lane == 0) {
                    mbar_expect_tx(bar_taken, 16);
                    launch_take(taken, bar_taken);
                }
                ++asked;
            };
            auto answer = [&] {
                index = -1;
                if (asked == answered) return;  // (not asked: something gave up)
                if (!wait_part(bar_taken, answered & 1)) return;
                index = launch_taken(taken);
                fence_proxy_async_smem();  // (read before the next answer is written)
                __syncwarp();
                ++answered;
            };
            int tt = 0, parts_with_tiles = 0;
            bool first = true;
            for (int nth = 0;;) {
                if (fail == 0 && __any_sync(0xffffffffu, *abort_flag != 0)) fail = 1;  // (no more than what was taken)
                if (!first) {
                    ask();
                    answer();
                }
                first = false;
                const int at = nth % kSegs;
                if (nth >= kSegs && !wait_part(bar_seg_free + 8 * at, (nth / kSegs - 1) & 1)) { fail = 3; break; }
                PagedSeg g;
                const bool have = index >= 0 && line.find(a.plan, a.div_group, index, lane, &g);
                if (!have && index >= 0) continue;  // (a CTA behind the last part need not start; one before it may still be taken)
                if (!have) g.n_rows = 0;
                if (lane == 0) {
                    segs[at] = g;
                    bad_seg[at] = 0;
                    mbar_arrive(bar_seg_full + 8 * at);
                }
                __syncwarp();
                ++nth;
                if (!have) break;
                if (g.n_tiles == 0) continue;
                const int* table = a.page_table + g.b * a.table_stride;
                bool met_bad = false;
                auto lookup = [&](int tile) { return page_lookup(a, page_box, table, tile, g.vis_lo, g.vis_hi, &met_bad); };
                auto load = [&](bool of_k, uint32_t dst, uint32_t bar, int tile, int page) {
                    page_load<C::kBoxes>(a, of_k ? a.k_box : a.v_box, page_box, of_k ? &tmap_k : &tmap_v, dst, bar, tile, g.head, page);
                };
                const int token0 = token_of(g), hi = g.lo + g.n_tiles;
                for (int t = 0; t < g.n_tiles && fail == 0; ++t, ++tt) {  // KV tiles are walked from the last to the first
                    if (left_out(a, tt)) continue;
                    const int st = tt % C::kStages;
                    const uint32_t ph = (tt / C::kStages) & 1;
                    const int tile = hi - 1 - t, page = lookup(tile);
                    if (__any_sync(0xffffffffu, met_bad) && lane == 0) bad_seg[at] = 1;  // (before what the readers' barriers wait for)
                    if (!mbar_wait_warp(bar_k_empty + 8 * st, ph ^ 1, abort_flag)) { fail = 1; break; }
                    load(true, sK + st * C::kTileBytes, bar_k_full + 8 * st, tile, page);
                    if (t == 0) {
                        if (parts_with_tiles > 0 && !mbar_wait_warp(bar_q_free, (parts_with_tiles - 1) & 1, abort_flag)) { fail = 1; break; }
                        ++parts_with_tiles;
                        int q_tiles = 0;
#pragma unroll
                        for (int i = 0; i < NQ; ++i) q_tiles += token0 + i * tile_tokens < g.n ? 1 : 0;
                        if (lane == 0) mbar_expect_tx(bar_q_full, q_tiles * C::kBoxes * tile_rows * 128);
                        __syncwarp();
                        if (lane < q_tiles * C::kBoxes) {
                            const int i = lane / C::kBoxes, b = lane % C::kBoxes;
                            tma_load_4d(sQ + i * C::kTileBytes + b * (kTile * 128), &tmap_q, bar_q_full, b * 64, 0, g.head, g.first + token0 + i * tile_tokens);
                        }
                    }
                    if (t + 1 == g.n_tiles) ask();  // (the answer is here when it is needed)
                    if (!mbar_wait_warp(bar_v_empty + 8 * st, ph ^ 1, abort_flag)) { fail = 2; break; }
                    load(false, sV + st * C::kTileBytes, bar_v_full + 8 * st, tile, page);
                }
                if (__any_sync(0xffffffffu, met_bad) && lane == 0 && a.status != nullptr) atomicExch(a.status, FA_STATUS_PAGE);
                if (fail != 0 && lane == 0) *abort_flag = 1;
                __syncwarp();
            }
        } else if (warp == C::kMmaWarp) {
            // ======================= MMA issuer =====================================
            const bool leader = elect_one();
            constexpr uint32_t idesc_qk = make_idesc_f16(kTile, kTile, kBf16, false);
            constexpr uint32_t idesc_pv = make_idesc_f16(kTile, D, kBf16, true);
            // bytes from eight keys of a tile to the next, and from their first 64 columns to the others
            const uint32_t eight_bytes = D == 128 && a.whole_rows ? 2048 : 1024, half_bytes = D == 128 && a.whole_rows ? 1024 : kTile * 128;
            const uint64_t dq = make_smem_desc(0, 0, 1024), dk = make_smem_desc(0, 0, eight_bytes), dv = make_smem_desc(0, half_bytes, eight_bytes);
            const uint32_t q_hi = static_cast<uint32_t>(dq >> 32), kv_hi = static_cast<uint32_t>(dk >> 32);
            const uint32_t q_lo = static_cast<uint32_t>(dq) | (sQ >> 4), k_lo = static_cast<uint32_t>(dk) | (sK >> 4), v_lo = static_cast<uint32_t>(dv) | (sV >> 4);
            const uint32_t k_jump = half_bytes / 16 - 6, v_step = eight_bytes / 8;
            auto issue_s = [&](int i, int st) {
                issue_qk<D>(tmem_base + i * kTile, q_lo + ((i * C::kTileBytes) >> 4), k_lo + ((st * C::kTileBytes) >> 4), q_hi, kv_hi, k_jump, idesc_qk);
                umma_commit(bar_s_full + 8 * i);
            };
            // After a wait gave up, here or elsewhere: nothing more is issued, and the named barriers are not met any more (the softmax
            // warps, which post their arrivals without waiting, may be tiles ahead by then).
            auto ready = [&](uint32_t bar, uint32_t parity, int code) {
                if (fail == 0 && !mbar_wait_warp(bar, parity, abort_flag)) fail = code;
            };
            auto meet = [&](int barrier) {
                if (__any_sync(0xffffffffu, *abort_flag != 0)) fail = fail != 0 ? fail : 8;
                if (fail == 0) named_sync(barrier);
                tc_fence_after_sync();
            };
            int tt = 0, parts_with_tiles = 0;
            for (int nth = 0;; ++nth) {
                const int at = nth % kSegs;
                if (!wait_part(bar_seg_full + 8 * at, (nth / kSegs) & 1)) { fail = 3; break; }
                const PagedSeg& g = segs[at];
                if (g.n_rows == 0) break;
                const int n_union = g.n_tiles, hi = g.lo + g.n_tiles, vis_lo = g.vis_lo, vis_hi = g.vis_hi;
                Range range[NQ];
#pragma unroll
                for (int i = 0; i < NQ; ++i) range[i] = range_of(g, token_of(g), i);
                auto active = [&](int i, int tile) { return tile >= range[i].lo && tile < range[i].hi; };
                if (n_union > 0) {
                    ready(bar_q_full, parts_with_tiles & 1, 4);
                    ++parts_with_tiles;
                    ready(bar_k_full + 8 * (tt % C::kStages), (tt / C::kStages) & 1, 5);
                    tc_fence_after_sync();
                    if (leader && fail == 0) {
#pragma unroll
                        for (int i = 0; i < NQ; ++i)
                            if (active(i, hi - 1)) issue_s(i, tt % C::kStages);
                        umma_commit(bar_k_empty + 8 * (tt % C::kStages));
                        if (n_union == 1) umma_commit(bar_q_free);
                    }
                }
                for (int t = 0; t < n_union; ++t, ++tt) {
                    const int tile = hi - 1 - t;
                    const int st = tt % C::kStages;
                    const uint32_t ph = (tt / C::kStages) & 1;
                    const int st1 = (tt + 1) % C::kStages;
                    const uint32_t ph1 = ((tt + 1) / C::kStages) & 1;
                    const bool more = t + 1 < n_union;
                    ready(bar_v_full + 8 * st, ph, 6);
                    // keys that no row of the block sees: their rows of V may hold anything
                    if (tile * kTile < vis_lo || tile * kTile + kTile > vis_hi)
                        clear_rows<C::kBoxes>(a, sV + st * C::kTileBytes, max(vis_lo - tile * kTile, 0), min(vis_hi - tile * kTile, kTile));
                    if (more) ready(bar_k_full + 8 * st1, ph1, 7);
#pragma unroll
                    for (int i = 0; i < NQ; ++i) {
                        if (active(i, tile)) {
                            // P V starts on the first half of P while the second half is exponentiated
                            meet(1 + 2 * i);
                            if (leader && fail == 0)
                                issue_pv<0>(tmem_base + C::kTmemO + i * D, tmem_base + i * kTile, v_lo + ((st * C::kTileBytes) >> 4), kv_hi, v_step, idesc_pv,
                                            tile < range[i].hi - 1 ? 1u : 0u);
                            meet(2 + 2 * i);
                            if (leader && fail == 0) {
                                issue_pv<kSplitSteps>(tmem_base + C::kTmemO + i * D, tmem_base + i * kTile, v_lo + ((st * C::kTileBytes) >> 4), kv_hi, v_step,
                                                      idesc_pv, 1u);
                                if (tile == range[i].lo) umma_commit(bar_o_full + 8 * i);
                            }
                        }
                        if (more && active(i, tile - 1) && leader && fail == 0) issue_s(i, st1);
                    }
                    if (leader && fail == 0) {
                        umma_commit(bar_v_empty + 8 * st);
                        if (more) umma_commit(bar_k_empty + 8 * st1);
                        if (t + 2 == n_union) umma_commit(bar_q_free);
                    }
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(bar_seg_free + 8 * at);
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(C::kRegsSoftmax));
        // ======================= softmax / epilogue =============================
        const int qi = warp >> 2;           // which query tile of the CTA
        const int r = threadIdx.x & 127;    // row inside the tile
        const int r_tok = static_cast<int>(fast_div(a.div_group, static_cast<uint32_t>(r)));
        const uint32_t lane_base = static_cast<uint32_t>((warp & 3) * 32) << 16;
        const uint32_t tmem_s = tmem_base + qi * kTile;          // S, 128 fp32 columns; P (16-bit, two per column) over the first half
        const uint32_t tmem_o = tmem_base + C::kTmemO + qi * D;  // O, D fp32 columns
        const uint32_t my_s_full = bar_s_full + 8 * qi, my_o_full = bar_o_full + 8 * qi;
        const float scale2 = a.scale_log2;
        uint32_t s_phase = 0, o_phase = 0;
        for (int nth = 0;; ++nth) {
            const int at = nth % kSegs;
            if (!wait_part(bar_seg_full + 8 * at, (nth / kSegs) & 1)) { fail = 10; break; }
            const PagedSeg& g = segs[at];
            if (g.n_rows == 0) break;
            const int token0 = token_of(g), keys = g.keys;
            const int tok = token0 + qi * tile_tokens + r_tok;                 // token inside the sequence
            const int head = g.head * a.plan.group + r - r_tok * a.plan.group;  // query head
            const bool mine = r_tok < tile_tokens && tok < g.n;                // (rows left over are walked too; nobody reads them)
            const int qpos = keys - g.n + tok;
            const Range range = range_of(g, token0, qi);
            const int t_lo = range.lo, n_tiles = range.hi - t_lo;
            float m_ref = -INFINITY;  // running max in log2 units (scaled, biased)
            float l_sum = 0.0f;
            float slope2 = 0.0f;
            if constexpr (kAlibi) slope2 = mine ? a.alibi_slopes[head] * kLog2e : 0.0f;

            for (int j = 0; j < n_tiles; ++j) {
                const int cb = t_lo + n_tiles - 1 - j;  // from the last KV tile of this query tile to the first
                const int kbase = cb * kTile;
                // columns this row may attend to inside the tile: [c_lo, c_hi] (worked out before S arrives)
                int c_lo = 0, c_hi = kTile - 1;
                if (mine) {
                    c_hi = min(c_hi, keys - 1 - cb * kTile);
                    if (a.plan.is_causal) c_hi = min(c_hi, qpos - kbase);
                    if (a.plan.window_right >= 0) c_hi = min(c_hi, qpos + a.plan.window_right - kbase);
                    if (a.plan.window_left >= 0) c_lo = max(0, min(qpos - a.plan.window_left - kbase, kTile));
                }
                const bool tile_masked = __any_sync(0xffffffffu, c_lo > 0 || c_hi < kTile - 1);
                if (fail != 0 || !mbar_wait_warp(my_s_full, (s_phase + j) & 1, abort_flag)) {
                    // a wait gave up: keep the barrier protocol alive (the MMA warp counts on two arrivals per tile) and do nothing else
                    fail = 8;
                    named_arrive(1 + 2 * qi);
                    named_arrive(2 + 2 * qi);
                    continue;
                }
                tc_fence_after_sync();

                float s[128];
                {
                    uint32_t tmp[4][32];
#pragma unroll
                    for (int c = 0; c < 4; ++c) tmem_ld32(tmem_s + lane_base + c * 32, tmp[c]);
                    tmem_wait_ld();
#pragma unroll
                    for (int c = 0; c < 128; ++c) s[c] = __uint_as_float(tmp[c / 32][c % 32]);
                }
                if (tile_masked) {
                    // (two passes: a causal diagonal, the common case, needs only the upper bound)
                    if (__any_sync(0xffffffffu, c_hi < kTile - 1)) {
#pragma unroll
                        for (int c = 0; c < 128; ++c)
                            if (c > c_hi) s[c] = -INFINITY;
                    }
                    if (__any_sync(0xffffffffu, c_lo > 0)) {
#pragma unroll
                        for (int c = 0; c < 128; ++c)
                            if (c < c_lo) s[c] = -INFINITY;
                    }
                }
                if constexpr (kAlibi) {
                    const float dist0 = static_cast<float>(qpos - kbase);
#pragma unroll
                    for (int c = 0; c < 128; ++c) s[c] = fmaf(-slope2, fabsf(dist0 - static_cast<float>(c)), s[c] * scale2);
                }
                // tile max in log2 units; without ALiBi it is taken over the raw scores and the scale folded into the exponent's FMA
                float m_tile;
                {
                    float mx[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
                    for (int c = 4; c < 128; c += 8) {
                        mx[0] = max3(mx[0], s[c], s[c + 1]);
                        mx[1] = max3(mx[1], s[c + 2], s[c + 3]);
                        if (c + 4 < 128) {
                            mx[2] = max3(mx[2], s[c + 4], s[c + 5]);
                            mx[3] = max3(mx[3], s[c + 6], s[c + 7]);
                        }
                    }
                    m_tile = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
                    if constexpr (!kAlibi) m_tile *= scale2;
                }
                // lazy rescale: keep the old reference max unless the new one is much larger
                float m_new = m_ref, factor = 1.0f;
                if (m_tile > m_ref + kRescaleThreshold || m_ref == -INFINITY) {
                    m_new = fmaxf(m_ref, m_tile);
                    factor = (m_ref == -INFINITY) ? 0.0f : fast_exp2(m_ref - m_new);
                }
                const bool rescale = (j > 0) && (m_new != m_ref);
                if (__any_sync(0xffffffffu, rescale)) {
                    // P V of the previous tile has completed (its commit precedes s_full), so O is stable.  A row that has seen no key yet
                    // starts from zero, whatever the values of keys that it does not see have left.
                    const float f = rescale ? factor : 1.0f;
                    const uint32_t seen = rescale && m_ref == -INFINITY ? 0u : 0xffffffffu;
#pragma unroll
                    for (int c = 0; c < D / 32; ++c) {
                        uint32_t orow[32];
                        tmem_ld32(tmem_o + lane_base + c * 32, orow);
                        tmem_wait_ld();
#pragma unroll
                        for (int i = 0; i < 32; ++i) orow[i] = __float_as_uint(__uint_as_float(orow[i] & seen) * f);
                        tmem_st32(tmem_o + lane_base + c * 32, orow);
                    }
                }
                l_sum *= (m_new != m_ref) ? factor : 1.0f;
                m_ref = m_new;
                const float neg_m = (m_ref == -INFINITY) ? 0.0f : -m_ref;

                // P = exp2(s * scale - m), rounded to the inputs' type for the tensor core; its sum is not
                float2 acc[4] = {{0.f, 0.f}, {0.f, 0.f}, {0.f, 0.f}, {0.f, 0.f}};
                const float2 neg_m2 = make_float2(neg_m, neg_m);
                const float2 scale22 = kAlibi ? make_float2(1.0f, 1.0f) : make_float2(scale2, scale2);
                // (All by the special function unit: the cubic that the kernel for contiguous K/V takes for a quarter of them is off by 7.5e-5,
                // which the LSE shows, and it gains nothing here: 935 us with none of 2048 new tokens over 32768 keys, 978 with a quarter.)
#pragma unroll
                for (int c = 0; c < 4; ++c) {  // quarters of 32 columns
                    uint32_t pr[16];
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const int col = c * 32 + i * 2;
                        const float2 x = __ffma2_rn(make_float2(s[col], s[col + 1]), scale22, neg_m2);
                        const float2 p = make_float2(fast_exp2(x.x), fast_exp2(x.y));
                        acc[i & 3] = __fadd2_rn(acc[i & 3], p);
                        pr[i] = pack2<kBf16>(p.x, p.y);
                    }
                    tmem_st16(tmem_s + lane_base + c * 16, pr);
                    if (c == (kSplitSteps * 16) / 32 - 1) {
                        // the first kSplitSteps*16 columns are stored: let the MMA warp start P V on them
                        tmem_wait_st();
                        tc_fence_before_sync();
                        named_arrive(1 + 2 * qi);
                    }
                }
                l_sum += (acc[0].x + acc[0].y) + (acc[1].x + acc[1].y) + (acc[2].x + acc[2].y) + (acc[3].x + acc[3].y);
                tmem_wait_st();
                tc_fence_before_sync();
                named_arrive(2 + 2 * qi);
            }

            s_phase += n_tiles;
            // ---- epilogue: rows of any place, a few at a time through this warp's room in shared memory --------------------------------
            bool have_o = false;
            if (n_tiles > 0) {
                if (fail == 0 && mbar_wait_warp(my_o_full, o_phase, abort_flag)) { tc_fence_after_sync(); have_o = true; }
                else if (fail == 0) fail = 9;
                o_phase ^= 1;
            }
            // A wait gave up, or a visible page was not there: none of the rows may pass for a softmax.
            if (g.n_tiles > 0 && (*abort_flag != 0 || bad_seg[at] != 0)) l_sum = __int_as_float(0x7fc00000);
            float o[D];
#pragma unroll
            for (int c = 0; c < D; c += 32) {
                uint32_t orow[32];
#pragma unroll
                for (int i = 0; i < 32; ++i) orow[i] = 0u;
                if (have_o) tmem_ld32(tmem_o + lane_base + c, orow);
#pragma unroll
                for (int i = 0; i < 32; ++i) o[c + i] = __uint_as_float(orow[i]);
            }
            if (have_o) tmem_wait_ld();
            bool last = true;
            if (g.parts > 1) {
                // A part's rows lie column group by column group, so that the threads, a row each, write and read side by side.
                const long long step = a.plan.rows;
                const long long row0 = static_cast<long long>(g.slot) * step + qi * tile_rows + r;  // part 0's
                auto row_of = [&](int part) { return reinterpret_cast<float4*>(a.o_partial) + (g.slot + static_cast<long long>(part)) * step * (D / 4) + qi * tile_rows + r; };
                if (mine) {
                    float4* to = row_of(g.part);
#pragma unroll
                    for (int c = 0; c < D / 4; ++c) to[c * step] = make_float4(o[4 * c], o[4 * c + 1], o[4 * c + 2], o[4 * c + 3]);
                    a.ml_partial[row0 + g.part * step] = make_float2(m_ref, l_sum);
                }
                last = last_to_come<NQ * 128>(a, g.slot, g.parts, last_flag);
                if (last) {
                    // O = sum_j 2^(m_j - m) O_j, l = sum_j 2^(m_j - m) l_j, in the order of the parts whoever is last
#pragma unroll
                    for (int c = 0; c < D; ++c) o[c] = 0.0f;
                    m_ref = -INFINITY;
                    l_sum = 0.0f;
                    if (mine) {
#pragma unroll 4
                        for (int j = 0; j < g.parts; ++j) m_ref = fmaxf(m_ref, __ldcg(a.ml_partial + row0 + j * step).x);
                        const float base = m_ref == -INFINITY ? 0.0f : m_ref;
#pragma unroll 1
                        for (int j = 0; j < g.parts; ++j) {
                            const float2 x = __ldcg(a.ml_partial + row0 + j * step);
                            const float f = exp2f(x.x - base);
                            l_sum += x.x == -INFINITY ? x.y : f * x.y;  // (a part that saw no key: 0; one that saw only NaN: NaN)
                            const float4* from = row_of(j);
                            if (f == 0.0f) continue;  // (nothing, or what masked values made of it)
#pragma unroll
                            for (int c = 0; c < D / 4; ++c) {
                                const float4 v = __ldcg(from + c * step);
                                o[4 * c] = fmaf(f, v.x, o[4 * c]);
                                o[4 * c + 1] = fmaf(f, v.y, o[4 * c + 1]);
                                o[4 * c + 2] = fmaf(f, v.z, o[4 * c + 2]);
                                o[4 * c + 3] = fmaf(f, v.w, o[4 * c + 3]);
                            }
                        }
                    }
                }
            }
            const long long first_row = static_cast<long long>(g.first) + token0 + qi * tile_tokens;  // (of Q)
            // of this warp's 32 (a part that others will put together: none)
            const int rows_left = last ? min(tile_rows, g.n_rows - qi * tile_rows) - (warp & 3) * 32 : 0;
            if (last && mine && a.lse != nullptr) a.lse[(first_row + r_tok) * a.heads + head] = l_sum == 0.0f ? -INFINITY : fmaf(m_ref, kLn2, logf(l_sum));
            if (__any_sync(0xffffffffu, l_sum == 0.0f)) {  // (a row without keys is 0, whatever the values of keys that it does not see have left)
#pragma unroll
                for (int c = 0; c < D; ++c) o[c] = l_sum == 0.0f ? 0.0f : o[c];
            }
            const float inv = l_sum == 0.0f ? 0.0f : 1.0f / l_sum;  // (NaN stays)
#pragma unroll
            for (int c = 0; c < D; ++c) o[c] *= inv;
            const uint32_t rows = smem_base + C::kSmemRows + warp * C::kStageBytes;
            if (lane == 0) tma_store_wait_read();  // (what the part before has left there)
            __syncwarp();
            // kRows rows of the warp in turn: laid out in shared memory by their threads, 16-byte units swizzled over eight rows, and
            // written by the whole warp, 16 bytes a lane.
            const int head0 = g.head * a.plan.group;
            auto place = [&](int k) -> long long {  // element of row k of the warp in the output
                const int row = (warp & 3) * 32 + k, k_tok = static_cast<int>(fast_div(a.div_group, static_cast<uint32_t>(row)));
                return (first_row + k_tok) * a.o_stride[0] + (head0 + row - k_tok * a.plan.group) * a.o_stride[1];
            };
            if (rows_left > 0 && a.o_is_fp32) {
                constexpr int kRows = C::kStageBytes / (D * 4), kUnits = D / 4, kPerWarp = 32 / kUnits;
#pragma unroll 1
                for (int h = 0; h < 32; h += kRows) {
                    if (lane / kRows == h / kRows) {
#pragma unroll
                        for (int i = 0; i < kUnits; ++i)
                            st_shared_v4(rows + (lane % kRows) * (D * 4) + (i ^ (lane & 7)) * 16, __float_as_uint(o[4 * i]), __float_as_uint(o[4 * i + 1]),
                                         __float_as_uint(o[4 * i + 2]), __float_as_uint(o[4 * i + 3]));
                    }
                    __syncwarp();
#pragma unroll
                    for (int k0 = 0; k0 < kRows; k0 += kPerWarp) {
                        const int k = h + k0 + lane / kUnits, u = lane % kUnits;
                        if (k >= rows_left || u * 4 >= a.head_dim) continue;
                        const float4 v = ld_shared_f32x4(rows + (k % kRows) * (D * 4) + (u ^ (k & 7)) * 16);
                        *reinterpret_cast<float4*>(static_cast<float*>(a.o) + place(k) + u * 4) = v;
                    }
                    __syncwarp();
                }
            } else if (rows_left > 0) {
                constexpr int kRows = C::kStageBytes / (D * 2), kUnits = D / 8, kPerWarp = 32 / kUnits;
                uint32_t packed[D / 2];
#pragma unroll
                for (int c = 0; c < D / 2; ++c) packed[c] = pack2<kBf16>(o[2 * c], o[2 * c + 1]);
                const bool whole = C::kStageBytes == 4096 && a.o_tma && rows_left >= 32;
                if (whole) {  // all 32 rows of the warp: by TMA, 64 columns at a time (prompts of six requests: 45.4 us, by hand 50.5)
#pragma unroll
                    for (int half = 0; half < D / 64; ++half) {
                        if (half > 0) {
                            if (lane == 0) tma_store_wait_read();
                            __syncwarp();
                        }
#pragma unroll
                        for (int u = 0; u < 8; ++u)
                            st_shared_v4(rows + lane * 128 + ((u ^ (lane & 7)) << 4), packed[half * 32 + 4 * u], packed[half * 32 + 4 * u + 1],
                                         packed[half * 32 + 4 * u + 2], packed[half * 32 + 4 * u + 3]);
                        fence_proxy_async_smem();
                        __syncwarp();
                        if (lane == 0) {
                            tma_store_4d(&tmap_o, rows, half * 64, 0, g.head,
                                         static_cast<int>(first_row) + static_cast<int>(fast_div(a.div_group, static_cast<uint32_t>((warp & 3) * 32))));
                            tma_store_commit();
                        }
                    }
                }
#pragma unroll 1
                for (int h = whole ? 32 : 0; h < 32; h += kRows) {
                    if (lane / kRows == h / kRows) {
#pragma unroll
                        for (int i = 0; i < kUnits; ++i)
                            st_shared_v4(rows + (lane % kRows) * (D * 2) + (i ^ (lane & 7)) * 16, packed[4 * i], packed[4 * i + 1], packed[4 * i + 2], packed[4 * i + 3]);
                    }
                    __syncwarp();
#pragma unroll
                    for (int k0 = 0; k0 < kRows; k0 += kPerWarp) {
                        const int k = h + k0 + lane / kUnits, u = lane % kUnits;
                        if (k >= rows_left || u * 8 >= a.head_dim) continue;
                        const float4 v = ld_shared_f32x4(rows + (k % kRows) * (D * 2) + (u ^ (k & 7)) * 16);
                        uint16_t* to = static_cast<uint16_t*>(a.o) + place(k) + u * 8;
                        if (a.o_units) {
                            *reinterpret_cast<float4*>(to) = v;
                        } else {
                            *reinterpret_cast<float2*>(to) = make_float2(v.x, v.y);
                            *reinterpret_cast<float2*>(to + 4) = make_float2(v.z, v.w);
                        }
                    }
                    __syncwarp();
                }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(bar_seg_free + 8 * at);
        }
        if (lane == 0) tma_store_wait_read();
    }

    if (fail != 0) {
        *abort_flag = 1;
        if (lane == 0 && a.status != nullptr) atomicExch(a.status, 310 + fail);
        const long long t0 = clock64();
        while (clock64() - t0 < 200000) { }
    }
    tc_fence_before_sync();
    __syncthreads();
    if (warp == C::kMmaWarp) {
        __syncwarp();
        tc_fence_after_sync();
        tmem_dealloc(tmem_base, C::kTmemCols);
    }
}

}  // namespace

template <>
cudaError_t launch_paged_tiled<FA_PAGED_D, FA_PAGED_NQ>(const PagedArgs& a, const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv, const CUtensorMap& to, bool bf16,
                                                        unsigned grid, cudaStream_t stream) {
    using C = TCfg<FA_PAGED_D, FA_PAGED_NQ>;
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(C::kThreads);
    cfg.dynamicSmemBytes = C::kSmemBytes;
    cfg.stream = stream;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    static std::atomic<bool> configured[4][64];
    auto run = [&](auto kern, std::atomic<bool>* done) -> cudaError_t {
        if (dev < 0 || dev >= 64 || !done[dev].load(std::memory_order_acquire)) {
            const cudaError_t err = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmemBytes);
            if (err != cudaSuccess) return err;
            if (dev >= 0 && dev < 64) done[dev].store(true, std::memory_order_release);
        }
        return cudaLaunchKernelEx(&cfg, kern, tq, tk, tv, to, a);
    };
    if (a.alibi_slopes != nullptr)
        return bf16 ? run(paged_tiled_kernel<FA_PAGED_D, FA_PAGED_NQ, true, true>, configured[0])
                    : run(paged_tiled_kernel<FA_PAGED_D, FA_PAGED_NQ, false, true>, configured[1]);
    return bf16 ? run(paged_tiled_kernel<FA_PAGED_D, FA_PAGED_NQ, true, false>, configured[2])
                : run(paged_tiled_kernel<FA_PAGED_D, FA_PAGED_NQ, false, false>, configured[3]);
}

}  // namespace fa
