// Attention of few rows a sequence over a paged K/V cache (single tokens, the check of guessed tokens): HBM-bound, each K/V byte used
// once.
//
// One CTA = one part of the keys of one block of rows (paged_plan.cuh).  The operands are swapped, as in the decode kernel for
// contiguous K/V, so that the 128 lanes of tensor memory hold KEYS:
//     S^T[128 keys x 16] = K_tile[128 x d] * Q^T[d x 16],   O^T[d x 16] += V_tile^T[d x 128 keys] * P[128 keys x 16]
// with the block's rows (a row is a token and a query head; the heads of a K/V head lie side by side) in the first kH columns.
// A tile of 128 keys is 128 / page_size pages, or a part of one: a lane of the producer warp looks a page up and issues its box, so
// that all boxes of a tile leave in one instruction and the lookup's latency hides behind the wait for a free slot.  Pages of which
// no row sees a key are not looked up.
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
#include "sm100_ptx.cuh"

namespace fa {

namespace {

constexpr int kPThreads = 192;  // four softmax warps, producer, MMA issuer
constexpr int kPTmemCols = 256; // S^T: 2 buffers x up to 4 tiles x 16 columns; O^T: 16 columns at 128
constexpr float kPLog2e = 1.4426950408889634f;
constexpr float kPLn2 = 0.6931471805599453f;

// kH = columns in use of the 16: 1, 4, 8 or 16.  D = 64 or 128 (head_dim rounded up).
template <int kH, int D>
struct PCfg {
    static constexpr int kChunk = kH == 16 ? 2 : 4;   // KV tiles of a softmax step
    static constexpr int kTileBytes = kTile * D * 2;
    static constexpr int kStages = D == 64 ? 6 : 3;   // 96 KB in flight either way
    static constexpr int kNumBars = 2 * kStages + 2 + 2 + 3;
    static constexpr int kHalfBytes = kH == 16 ? 2048 : 1024;  // K-major operand of 16 rows: from the first 64 elements to the second
    static constexpr int kOperandBytes = 2 * kHalfBytes;
    static constexpr int kSmemRing = 0;
    static constexpr int kSmemP = kStages * kTileBytes;  // (before that: the plan's scratch)
    static constexpr int kSmemQ = kSmemP + kChunk * kOperandBytes + (kH == 16 ? 0 : 1024);  // (+ what rows 8-15 touch)
    static constexpr int kSmemBar = kSmemQ + kOperandBytes + (kH == 16 ? 0 : 1024);
    static constexpr int kSmemRed = (kSmemBar + 8 * kNumBars + 15) / 16 * 16;  // float[2][4][kH] maxima, float[4][kH] sums
    static constexpr int kSmemMisc = kSmemRed + 3 * 4 * kH * 4;
    static constexpr int kSmemEnd = kSmemMisc + 16;
    static constexpr int kSmemReach = kSmemP + (D == 64 ? kTile * 128 : 0);  // V^T is an M = 128 operand: with D = 64 its upper rows read on
    static constexpr int kSmemBytes = (kSmemEnd > kSmemReach ? kSmemEnd : kSmemReach) + 1024;
    static_assert(kSmemBytes <= 115712, "two CTAs per SM");
    static_assert(sizeof(PlanScratch) <= kChunk * kOperandBytes, "the plan's scratch lies where P will be");
};

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
    float* red = reinterpret_cast<float*>(smem_gen + C::kSmemRed);
    volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(smem_gen + C::kSmemMisc);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(smem_gen + C::kSmemMisc + 4);
    volatile int* bad_page = reinterpret_cast<volatile int*>(smem_gen + C::kSmemMisc + 8);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    grid_dep_launch_dependents();
    if (warp == 4 && lane == 0) {
        *abort_flag = 0;
        *bad_page = 0;
        tma_prefetch_desc(&tmap_k);
        tma_prefetch_desc(&tmap_v);
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
    PagedWork w;
    if (!find_work<kPThreads>(a.plan, *reinterpret_cast<PlanScratch*>(smem_gen + C::kSmemP), static_cast<int>(blockIdx.x), &w)) return;

    // ---- the block's rows and the tiles of this part
    const int row0 = w.blk * kH;                                  // first row: token row0 / group, query head row0 % group of the K/V head
    const int nc = min(kH, w.n * a.plan.group - row0);            // columns in use
    const int p_first = w.keys - w.n;                             // position of the sequence's first new token
    const int tok_lo = static_cast<int>(fast_div(a.div_group, static_cast<uint32_t>(row0)));
    const int tok_hi = static_cast<int>(fast_div(a.div_group, static_cast<uint32_t>(row0 + nc - 1)));
    int vis_lo, vis_hi;
    visible_keys(a.plan, w.keys, p_first + tok_lo, p_first + tok_hi, &vis_lo, &vis_hi);
    const int t_first = vis_lo / kTile, t_all = vis_hi > vis_lo ? (vis_hi + kTile - 1) / kTile - t_first : 0;
    int lo, hi;
    part_of(t_all, w.part, w.parts, &lo, &hi);
    lo += t_first;
    const int n_tiles = hi + t_first - lo;
    // tiles [full_lo, full_hi) need no mask: every row sees all of their keys
    int full_lo, full_hi;
    {
        int l0, h0, l1, h1;
        visible_keys(a.plan, w.keys, p_first + tok_lo, p_first + tok_lo, &l0, &h0);
        visible_keys(a.plan, w.keys, p_first + tok_hi, p_first + tok_hi, &l1, &h1);
        full_lo = (max(l0, l1) + kTile - 1) / kTile;
        full_hi = min(h0, h1) / kTile;
    }
    const int n_chunks = (n_tiles + kChunkTiles - 1) / kChunkTiles;
    auto chunk_tiles = [&](int c) { return min(kChunkTiles, n_tiles - c * kChunkTiles); };

    if (warp == 5 && n_tiles > 0) {
        tmem_alloc(smem_u32(const_cast<uint32_t*>(tmem_slot)), kPTmemCols);
        tmem_relinquish();
    }
    // ---- producer
    const PageLane mine = page_lane<kHalves>(a, lane);
    const int* table = a.page_table + w.b * a.table_stride;
    bool met_bad = false;
    auto lookup = [&](int tile) { return page_lookup(a, mine, table, tile, vis_lo, vis_hi, &met_bad); };
    auto load = [&](bool of_k, int st, int tile, int page) {
        if (__any_sync(0xffffffffu, met_bad) && lane == 0) *bad_page = 1;  // (before what the readers' barriers wait for)
        page_load<kHalves>(a, of_k ? a.k_box : a.v_box, mine, of_k ? &tmap_k : &tmap_v, sRing + st * kTileBytes, bar_full + 8 * st, tile, w.head, page);
    };
    int pushed = 0;  // tiles whose loads have been issued (producer warp only)
    if (warp == 4) {
        // the first K tiles are put in flight before the CTA-wide sync: their latency overlaps Q's
        const int first = min(min(kStages, kChunkTiles), n_tiles);
        int page[kStages < kChunkTiles ? kStages : kChunkTiles];
#pragma unroll
        for (int i = 0; i < (kStages < kChunkTiles ? kStages : kChunkTiles); ++i) page[i] = i < first ? lookup(lo + i) : -1;
#pragma unroll
        for (int i = 0; i < (kStages < kChunkTiles ? kStages : kChunkTiles); ++i)
            if (i < first) load(true, i, lo + i, page[i]);
        pushed = first;
    }
    const long long token0 = w.first;
    if (n_tiles > 0) {
        // row n of the block goes to row n of the Q operand (16-byte unit u -> half u/8, unit (u%8) ^ (n%8): the 128-byte swizzle)
        constexpr int kUnits = D / 8;
        for (int i = threadIdx.x; i < kUnits * kH; i += kPThreads) {
            const int u = i % kUnits, n = i / kUnits;
            uint4 val = make_uint4(0u, 0u, 0u, 0u);
            if (n < nc && u * 8 < a.head_dim) {
                const int tok = static_cast<int>(fast_div(a.div_group, static_cast<uint32_t>(row0 + n)));
                const int head = w.head * a.plan.group + row0 + n - tok * a.plan.group;
                val = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.q) + (token0 + tok) * a.q_stride[0] + head * a.q_stride[1] + u * 8);
            }
            *reinterpret_cast<uint4*>(smem_gen + C::kSmemQ + (u >> 3) * C::kHalfBytes + n * 128 + (((u & 7) ^ (n & 7)) << 4)) = val;
        }
        fence_proxy_async_smem();
    }
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    const uint32_t tmem_base = (n_tiles > 0) ? *tmem_slot : 0u;
    const uint32_t tmem_o = tmem_base + 128;

    int fail = 0;

    if (n_tiles > 0 && warp == 4) {
        // ======================= TMA producer ===================================
        int slot = 0;  // running count of tiles in stream order: K(0), K(1), V(0), K(2), V(1), ... (chunks)
        auto push = [&](bool of_k, int tile) -> bool {
            if (slot < pushed) { ++slot; return true; }  // issued during set-up
            const int st = slot % kStages;
            const uint32_t ph = (slot / kStages) & 1;
            const int page = lookup(tile);
            if (!mbar_wait_warp_ok(bar_empty + 8 * st, ph ^ 1, abort_flag)) return false;
            load(of_k, st, tile, page);
            ++slot;
            return true;
        };
        auto push_chunk = [&](bool of_k, int c) -> bool {
            for (int t = 0; t < chunk_tiles(c); ++t)
                if (!push(of_k, lo + c * kChunkTiles + t)) return false;
            return true;
        };
        bool ok = push_chunk(true, 0);
        for (int c = 0; ok && c < n_chunks; ++c) {
            if (c + 1 < n_chunks) ok = push_chunk(true, c + 1);
            if (ok) ok = push_chunk(false, c);
        }
        if (!ok) fail = 1;
        if (__any_sync(0xffffffffu, met_bad) && lane == 0 && a.status != nullptr) atomicExch(a.status, FA_STATUS_PAGE);
    } else if (n_tiles > 0 && warp == 5) {
        // ======================= MMA issuer =====================================
        constexpr uint32_t idesc_qk = make_idesc_swapped(kBf16, false);
        constexpr uint32_t idesc_pv = make_idesc_swapped(kBf16, true);
        // bytes from eight keys of a tile to the next, and from their first 64 columns to the others
        const uint32_t eight_bytes = D == 128 && a.whole_rows ? 2048 : 1024, half_bytes = D == 128 && a.whole_rows ? 1024 : kTile * 128;
        int slot = 0;
        auto qk_chunk = [&](int c) -> bool {
            const int buf = c & 1;
            if (c >= 2 && !mbar_wait_warp_ok(bar_s_free + 8 * buf, ((c >> 1) - 1) & 1, abort_flag)) return false;
            tc_fence_after_sync();
            for (int t = 0; t < chunk_tiles(c); ++t) {
                const int st = slot % kStages;
                if (!mbar_wait_warp_ok(bar_full + 8 * st, (slot / kStages) & 1, abort_flag)) return false;
                tc_fence_after_sync();
                const uint32_t kt = sRing + st * kTileBytes;
                if (lane == 0) {
#pragma unroll
                    for (int ks = 0; ks < D / 16; ++ks) {
                        const uint32_t off = (ks / 4) * half_bytes + (ks % 4) * 32;
                        const uint32_t qoff = (ks / 4) * C::kHalfBytes + (ks % 4) * 32;
                        umma_ss(tmem_base + buf * 64 + t * 16, make_smem_desc(kt + off, 0, eight_bytes), make_smem_desc(sQ + qoff, 0, 1024), idesc_qk,
                                ks > 0 ? 1u : 0u);
                    }
                    umma_commit(bar_empty + 8 * st);
                }
                ++slot;
            }
            if (lane == 0) umma_commit(bar_s_full + 8 * buf);
            return true;
        };
        auto pv_chunk = [&](int c) -> bool {
            if (!mbar_wait_warp_ok(bar_p_full, c & 1, abort_flag)) return false;
            tc_fence_after_sync();
            for (int t = 0; t < chunk_tiles(c); ++t) {
                const int st = slot % kStages;
                if (!mbar_wait_warp_ok(bar_full + 8 * st, (slot / kStages) & 1, abort_flag)) return false;
                tc_fence_after_sync();
                const uint32_t vt = sRing + st * kTileBytes;
                const int key0 = (lo + c * kChunkTiles + t) * kTile;
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
            if (lane == 0) umma_commit(bar_p_free);
            return true;
        };
        bool ok = qk_chunk(0);
        for (int c = 0; ok && c < n_chunks; ++c) {
            if (c + 1 < n_chunks) ok = qk_chunk(c + 1);
            if (ok) ok = pv_chunk(c);
        }
        if (ok && lane == 0) umma_commit(bar_o_done);
        if (!ok) fail = 2;
    } else if (warp < 4) {
        // ======================= softmax over keys / epilogue ===================
        const int r = threadIdx.x;  // key inside a tile; output column in the epilogue
        const uint32_t lane_base = static_cast<uint32_t>(warp * 32) << 16;
        // scores stay unscaled and the scale is folded into the exponent's FMA, except with ALiBi
        const bool alibi = a.alibi_slopes != nullptr;
        const float scale2 = a.scale_log2, exp_scale = alibi ? 1.0f : a.scale_log2;
        // column `lane`: its token and query head, its ALiBi slope; handed round
        const int my_tok = static_cast<int>(fast_div(a.div_group, static_cast<uint32_t>(row0 + lane)));
        const int my_head = w.head * a.plan.group + row0 + lane - my_tok * a.plan.group;
        float slope = 0.0f;
        if (alibi && lane < nc) slope = a.alibi_slopes[my_head] * kPLog2e;
        float m_ref = -INFINITY;  // CTA-wide running max of column `lane` (lanes < kH of every warp), log2 units
        float l_part[kH];         // this thread's share of each column's row sum
#pragma unroll
        for (int n = 0; n < kH; ++n) l_part[n] = 0.0f;
        // this key's element of column n in the P operand: row n, 128-byte swizzled
        uint8_t* p_half = smem_gen + C::kSmemP + (r >> 6) * C::kHalfBytes + (r & 7) * 2;
        const uint32_t p_unit = static_cast<uint32_t>((r & 63) >> 3);

        for (int c = 0; c < n_chunks; ++c) {
            const int buf = c & 1;
            const int nt = chunk_tiles(c);
            const int tile0 = lo + c * kChunkTiles;
            if (!mbar_wait_warp_ok(bar_s_full + 8 * buf, (c >> 1) & 1, abort_flag)) fail = 3;
            tc_fence_after_sync();
            uint32_t raw[kChunkTiles][kH];
#pragma unroll
            for (int t = 0; t < kChunkTiles; ++t) {
                if (t < nt) {
                    tmem_ld_heads<kH>(tmem_base + lane_base + buf * 64 + t * 16, raw[t]);
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
                    in_range[t] = t < nt && key < w.keys;
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
            if (c > 0) {
                if (!mbar_wait_warp_ok(bar_p_free, (c - 1) & 1, abort_flag)) fail = 4;
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
#pragma unroll
        for (int n = 0; n < kH; ++n) {
            float l_warp = l_part[n];
#pragma unroll
            for (int o = 16; o >= 1; o >>= 1) l_warp += __shfl_xor_sync(0xffffffffu, l_warp, o);
            if (lane == 0) red[8 * kH + warp * kH + n] = l_warp;
        }
        uint32_t o_raw[kH];
#pragma unroll
        for (int n = 0; n < kH; ++n) o_raw[n] = 0u;
        if (n_tiles > 0 && fail == 0) {
            if (mbar_wait_warp_ok(bar_o_done, 0, abort_flag)) {
                tc_fence_after_sync();
                tmem_ld_heads<kH>(tmem_o + lane_base, o_raw);
                tmem_wait_ld();
            } else {
                fail = 5;
            }
        }
        named_barrier_128();
        // A wait gave up, or a visible page was not there (set by whoever saw it, before the last MMA could complete): none of the
        // rows may pass for a softmax.
        const float spoilt = *abort_flag != 0 || *bad_page != 0 ? __int_as_float(0x7fc00000) : 0.0f;
#pragma unroll
        for (int n = 0; n < kH; ++n) {
            const float m_n = __shfl_sync(0xffffffffu, m_ref, n);
            const int tok = __shfl_sync(0xffffffffu, my_tok, n), head = __shfl_sync(0xffffffffu, my_head, n);
            if (n >= nc) continue;
            const float l_sum = (red[8 * kH + n] + red[9 * kH + n]) + (red[10 * kH + n] + red[11 * kH + n]) + spoilt;
            if (w.parts > 1) {  // un-normalised, for the last part to come
                const long long at = static_cast<long long>(w.slot + w.part) * kH + n;
                if (r < D) a.o_partial[at * D + r] = __uint_as_float(o_raw[n]);
                if (r == 0) a.ml_partial[at] = make_float2(m_n, l_sum);
            } else {
                const long long at = (token0 + tok) * a.o_stride[0] + head * a.o_stride[1] + r;
                const float o_val = l_sum == 0.0f ? 0.0f : __uint_as_float(o_raw[n]) * (1.0f / l_sum);
                if (r < a.head_dim) {
                    if (a.o_is_fp32) static_cast<float*>(a.o)[at] = o_val;
                    else if (kBf16) static_cast<__nv_bfloat16*>(a.o)[at] = __float2bfloat16_rn(o_val);
                    else static_cast<__half*>(a.o)[at] = __float2half_rn(o_val);
                }
                if (r == 0 && a.lse != nullptr)
                    a.lse[(token0 + tok) * a.heads + head] = l_sum == 0.0f ? -INFINITY : fmaf(m_n, kPLn2, logf(l_sum));
            }
        }
        if (w.parts > 1 && last_to_come<128>(a, w, reinterpret_cast<volatile int*>(smem_gen + C::kSmemMisc + 12)))
            merge_parts<D, kBf16, 4>(a, w, row0, nc, warp);
    }

    if (fail != 0) {
        *abort_flag = 1;
        if (lane == 0 && a.status != nullptr) atomicExch(a.status, 300 + fail);
        const long long t0 = clock64();
        while (clock64() - t0 < 200000) { }  // (copies in flight land before the CTA's memory is another's)
    }
    tc_fence_before_sync();
    __syncthreads();
    if (warp == 5 && n_tiles > 0) {
        __syncwarp();
        tc_fence_after_sync();
        tmem_dealloc(tmem_base, kPTmemCols);
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
