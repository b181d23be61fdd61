// Attention of new tokens over a paged K/V cache: the C entry point, its checks and tensor maps, and the kernel that puts the parts of
// split rows together.
#include <algorithm>
#include <atomic>
#include <cmath>
#include <cstring>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include "fa_internal.h"
#include "fa_paged.h"
#include "paged_kernels.h"
#include "paged_plan.cuh"
#include "sm100_ptx.cuh"

namespace fa {

namespace {

// A part is not worth starting for fewer tiles than this, and shares above kLongShare are cut into waves.
constexpr int kMinShare = 4, kLongShare = 24;
constexpr int kCThreads = 128;
constexpr int kCRows = 16;  // rows of a CTA of the combine kernel

// One warp per row: O = sum_j 2^(m_j - m) O_j / l, l = sum_j 2^(m_j - m) l_j over the row's parts.  A CTA works the launch's plan out as
// the kernel before it did, to find its item; it is resident and waiting when that kernel ends.
template <int D, bool kBf16>
__global__ void __launch_bounds__(kCThreads) paged_combine_kernel(const __grid_constant__ PagedArgs a) {
    __shared__ PlanScratch<kCThreads> sm;
    grid_dep_launch_dependents();
    grid_dep_wait();
    PagedWork w;
    if (!find_work<kCThreads>(a.plan, sm, static_cast<int>(blockIdx.x), true, &w) || w.parts == 1) return;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int row0 = w.blk * a.plan.rows;
    const int n_rows = min(min(a.plan.rows, w.n * a.plan.group - row0), static_cast<int>(blockIdx.y + 1) * kCRows);
    const bool mine = lane * 4 < D;
    for (int n = blockIdx.y * kCRows + warp; n < n_rows; n += kCThreads / 32) {
        const long long at0 = static_cast<long long>(w.slot) * a.plan.rows + n;  // part j's: + j * plan.rows
        float m = -INFINITY, l = 0.0f;
        for (int j = lane; j < w.parts; j += 32) m = fmaxf(m, a.ml_partial[at0 + static_cast<long long>(j) * a.plan.rows].x);
#pragma unroll
        for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        const float base = m == -INFINITY ? 0.0f : m;
        float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        for (int j0 = 0; j0 < w.parts; j0 += 32) {
            float wt = 0.0f;
            if (j0 + lane < w.parts) {
                const float2 ml = a.ml_partial[at0 + static_cast<long long>(j0 + lane) * a.plan.rows];
                wt = exp2f(ml.x - base);
                l += ml.x == -INFINITY ? ml.y : wt * ml.y;  // (no key: l = 0; nothing but NaN: NaN)
            }
            const int n_parts = min(32, w.parts - j0);
            for (int j = 0; j < n_parts; j += 8) {
                float4 v[8];
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (mine && j + i < n_parts)
                        v[i] = *reinterpret_cast<const float4*>(a.o_partial + (at0 + static_cast<long long>(j0 + j + i) * a.plan.rows) * D + lane * 4);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float x = __shfl_sync(0xffffffffu, wt, (j + i) & 31);
                    if (mine && j + i < n_parts && x != 0.0f) {
                        acc.x = fmaf(x, v[i].x, acc.x);
                        acc.y = fmaf(x, v[i].y, acc.y);
                        acc.z = fmaf(x, v[i].z, acc.z);
                        acc.w = fmaf(x, v[i].w, acc.w);
                    }
                }
            }
        }
#pragma unroll
        for (int o = 16; o; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;  // (NaN stays)
        const int tok = static_cast<int>(fast_div(a.div_group, static_cast<uint32_t>(row0 + n)));
        const int head = w.head * a.plan.group + row0 + n - tok * a.plan.group;
        const long long token = w.first + tok;
        if (lane * 4 < a.head_dim) {
            const long long at = token * a.o_stride[0] + head * a.o_stride[1] + lane * 4;
            const float4 o = make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv);
            if (a.o_is_fp32) {
                *reinterpret_cast<float4*>(static_cast<float*>(a.o) + at) = o;
            } else if (kBf16) {
                const __nv_bfloat162 x = __floats2bfloat162_rn(o.x, o.y), y = __floats2bfloat162_rn(o.z, o.w);
                *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.o) + at) = make_uint2(*reinterpret_cast<const uint32_t*>(&x), *reinterpret_cast<const uint32_t*>(&y));
            } else {
                const __half2 x = __floats2half2_rn(o.x, o.y), y = __floats2half2_rn(o.z, o.w);
                *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.o) + at) = make_uint2(*reinterpret_cast<const uint32_t*>(&x), *reinterpret_cast<const uint32_t*>(&y));
            }
        }
        if (lane == 0 && a.lse != nullptr) a.lse[token * a.heads + head] = l == 0.0f ? -INFINITY : fmaf(m, 0.6931471805599453f, logf(l));
    }
}

int check_fwd(const fa_paged_fwd_params* p) {
    if (!p || !p->q || !p->o) return FA_ERR_INVALID_ARG;
    const fa_paged_kv& c = p->cache;
    int rc = check_cache(c, p->tokens);
    if (rc != FA_OK) return rc;
    if (p->o_dtype != c.dtype && p->o_dtype != FA_DTYPE_FP32) return FA_ERR_UNSUPPORTED;
    if (p->heads < 1 || p->heads % c.heads != 0) return FA_ERR_INVALID_ARG;
    if (p->heads / c.heads > kTile) return FA_ERR_UNSUPPORTED;
    if (!(p->softmax_scale > 0.0f) || !std::isfinite(p->softmax_scale)) return FA_ERR_INVALID_ARG;
    if (p->window_left < -1 || p->window_right < -1 || p->max_seqlen_q < 1) return FA_ERR_INVALID_ARG;
    if ((reinterpret_cast<uintptr_t>(p->q) | reinterpret_cast<uintptr_t>(p->o)) & 15u) return FA_ERR_INVALID_ARG;
    if ((reinterpret_cast<uintptr_t>(p->lse) | reinterpret_cast<uintptr_t>(p->alibi_slopes) | reinterpret_cast<uintptr_t>(p->status)) & 3u)
        return FA_ERR_INVALID_ARG;
    const int64_t counts[2] = {p->tokens, p->heads};
    for (int i = 0; i < 2; ++i) {
        if (counts[i] == 1) continue;
        if (p->q_stride[i] % 8 != 0 || p->q_stride[i] < 0 || p->o_stride[i] % 4 != 0) return FA_ERR_INVALID_ARG;
        if (p->q_stride[i] >= (1LL << 39)) return FA_ERR_TOO_LARGE;
    }
    if (!rows_apart(counts, p->o_stride, 2, c.head_dim)) return FA_ERR_INVALID_ARG;
    if (p->tokens * p->heads > 0x3fffffffLL) return FA_ERR_TOO_LARGE;
    return FA_OK;
}


// What the sizes of a call say about its launch; the lengths, which say the rest, are on the device.
struct PagedLaunch {
    int columns;               // decode kernel: rows of a block; 0: the tiled kernel
    int query_tiles;           // tiled kernel: of a block
    int rows;                  // of a block
    int slots;                 // CTAs that run at once
    int wide;                  // columns of a partial row: head_dim rounded up
    long long items;           // at most so many blocks of rows there are, over all K/V heads
    long long grid, split_items, partials;
    size_t o_bytes, bytes;     // workspace: partial rows, and all
};

PagedLaunch plan_launch(const fa_paged_fwd_params* p, int sms) {
    const fa_paged_kv& c = p->cache;
    PagedLaunch l = {};
    const int group = p->heads / c.heads;
    const long long rows = static_cast<long long>(std::min<int64_t>(p->max_seqlen_q, p->tokens)) * group;
    const int tile_rows = kTile / group * group;
    l.columns = rows == 1 ? 1 : rows <= 4 ? 4 : rows <= 8 ? 8 : rows <= 16 ? 16 : 0;
    l.query_tiles = l.columns ? 0 : rows <= tile_rows ? 1 : 2;
    l.rows = l.columns ? l.columns : l.query_tiles * tile_rows;
    l.slots = (l.query_tiles == 2 ? 1 : 2) * sms;
    l.wide = c.head_dim <= 64 ? 64 : 128;
    l.items = c.heads * (c.cu_seqlens_q ? (p->tokens * group + static_cast<long long>(c.batch) * (l.rows - 1)) / l.rows
                                        : static_cast<long long>(c.batch) * ((group + l.rows - 1) / l.rows));
    const long long slots = l.slots;
    const long long tiles = (static_cast<long long>(c.table_width) * c.page_size + kTile - 1) / kTile;
    const long long parts = (tiles + kMinShare - 1) / kMinShare;  // of one item
    if (parts > 1) {
        l.partials = std::min(most_partials(static_cast<int>(slots)), l.items * parts);
        l.split_items = std::min(l.items, kPagedWaves * slots);
    }
    l.grid = l.items + (parts > 1 ? std::min(kPagedWaves * slots, l.items * (parts - 1)) : 0);
    l.o_bytes = (static_cast<size_t>(l.partials) * l.rows * l.wide * sizeof(float) + 255) & ~static_cast<size_t>(255);
    l.bytes = l.o_bytes + ((static_cast<size_t>(l.partials) * l.rows * sizeof(float2) + 255) & ~static_cast<size_t>(255));
    return l;
}

// A 4-D tensor map: dims and strides (elements; of a dimension of one any will do) outermost last.  The last ones are kept per host
// thread, being a function of these arguments alone.
int map_of(CUtensorMap* m, int dtype, const void* base, const int64_t (&dims)[4], const int64_t (&strides)[3], const int (&box)[4]) {
    struct Entry {
        const void* base;
        int64_t dims[4], strides[3];
        int box[4], dtype;
        bool valid;
        CUtensorMap map;
    };
    constexpr int kEntries = 12;
    thread_local Entry cache[kEntries] = {};
    thread_local int next_victim = 0;
    for (const Entry& e : cache) {
        if (e.valid && e.base == base && e.dtype == dtype && std::equal(dims, dims + 4, e.dims) && std::equal(strides, strides + 3, e.strides) &&
            std::equal(box, box + 4, e.box)) {
            *m = e.map;
            return FA_OK;
        }
    }
    cuuint64_t d[4], s[3];
    cuuint32_t b[4];
    for (int i = 0; i < 4; ++i) {
        d[i] = static_cast<cuuint64_t>(dims[i]);
        b[i] = static_cast<cuuint32_t>(box[i]);
        if (i > 0) s[i - 1] = dims[i] > 1 ? static_cast<cuuint64_t>(strides[i - 1]) * 2 : 256;
    }
    const int rc = encode_map(m, dtype, 4, base, d, s, b);
    if (rc != FA_OK) return rc;
    Entry& e = cache[next_victim];
    next_victim = (next_victim + 1) % kEntries;
    e.base = base;
    std::copy(dims, dims + 4, e.dims);
    std::copy(strides, strides + 3, e.strides);
    std::copy(box, box + 4, e.box);
    e.dtype = dtype;
    e.map = *m;
    e.valid = true;
    return FA_OK;
}

// Pages: a box is 64 columns of the tokens of a page (of 128 of them at most) of one head.
int page_map(CUtensorMap* m, const fa_paged_kv& c, const void* base, const int64_t* stride) {
    return map_of(m, c.dtype, base, {c.head_dim, c.page_size, c.heads, c.num_pages}, {stride[2], stride[1], stride[0]},
                  {64, std::min(c.page_size, kTile), 1, 1});
}

// Q: a box is 64 columns of the rows of a query tile, the heads of one K/V head side by side.
int query_map(CUtensorMap* m, const fa_paged_fwd_params* p) {
    const int group = p->heads / p->cache.heads;
    return map_of(m, p->cache.dtype, p->q, {p->cache.head_dim, group, p->cache.heads, p->tokens}, {p->q_stride[1], p->q_stride[1] * group, p->q_stride[0]},
                  {64, group, 1, kTile / group});
}

}  // namespace

cudaError_t launch_paged_combine(const PagedArgs& a, bool bf16, unsigned items, cudaStream_t stream) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(items, static_cast<unsigned>((a.plan.rows + kCRows - 1) / kCRows));
    cfg.blockDim = dim3(kCThreads);
    cfg.stream = stream;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    if (a.head_dim <= 64) return cudaLaunchKernelEx(&cfg, bf16 ? paged_combine_kernel<64, true> : paged_combine_kernel<64, false>, a);
    return cudaLaunchKernelEx(&cfg, bf16 ? paged_combine_kernel<128, true> : paged_combine_kernel<128, false>, a);
}

}  // namespace fa

using namespace fa;

extern "C" {

size_t fa_paged_fwd_workspace_bytes(const fa_paged_fwd_params* p) {
    if (check_fwd(p) != FA_OK) return 0;
    int sms = 148, major = 10;
    if (current_device(&sms, &major) != FA_OK) sms = 148;
    return plan_launch(p, sms).bytes;
}

int fa_paged_fwd(const fa_paged_fwd_params* p) {
    int rc = check_fwd(p);
    if (rc != FA_OK) return rc;
    int sms = 0, major = 0;
    if ((rc = current_device(&sms, &major)) != FA_OK) return rc;
    if (major != 10) return FA_ERR_NOT_SM100;
    const PagedLaunch l = plan_launch(p, sms);
    if (l.grid > 0x7fffffffLL) return FA_ERR_TOO_LARGE;
    if (l.bytes > 0 && (!p->workspace || p->workspace_bytes < l.bytes)) return FA_ERR_WORKSPACE;
    if (l.bytes > 0 && (reinterpret_cast<uintptr_t>(p->workspace) & 15u)) return FA_ERR_INVALID_ARG;
    const fa_paged_kv& c = p->cache;
    PagedArgs a = {};
    a.plan.seq = {c.seqlens_k, c.cu_seqlens_q, c.batch, static_cast<int>(p->tokens)};
    a.plan.heads_k = c.heads;
    a.plan.group = p->heads / c.heads;
    a.plan.rows = l.rows;
    a.plan.is_causal = p->is_causal ? 1 : 0;
    a.plan.window_left = p->window_left;
    a.plan.window_right = p->window_right;
    a.plan.slots = l.slots;
    a.plan.min_share = kMinShare;
    a.plan.long_share = kLongShare;
    a.plan.partials = static_cast<int>(l.partials);
    a.div_group = make_fastdiv(static_cast<uint32_t>(a.plan.group));
    a.q = p->q;
    a.o = p->o;
    a.lse = p->lse;
    a.page_table = c.page_table;
    a.table_stride = c.table_stride;
    a.table_width = c.table_width;
    a.num_pages = c.num_pages;
    while ((1 << a.page_shift) < c.page_size) ++a.page_shift;
    a.heads = p->heads;
    a.head_dim = c.head_dim;
    a.tile_tokens = kTile / a.plan.group;
    std::copy(p->q_stride, p->q_stride + 2, a.q_stride);
    std::copy(p->o_stride, p->o_stride + 2, a.o_stride);
    a.scale_log2 = p->softmax_scale * 1.4426950408889634f;
    a.alibi_slopes = p->alibi_slopes;
    a.o_is_fp32 = p->o_dtype == FA_DTYPE_FP32;
    a.status = p->status;
    if (l.bytes > 0) {
        a.o_partial = static_cast<float*>(p->workspace);
        a.ml_partial = reinterpret_cast<float2*>(static_cast<char*>(p->workspace) + l.o_bytes);
    }
    CUtensorMap tk, tv;
    if ((rc = page_map(&tk, c, c.k, c.k_stride)) != FA_OK) return rc;
    if ((rc = page_map(&tv, c, c.v, c.v_stride)) != FA_OK) return rc;
    cudaStream_t stream = static_cast<cudaStream_t>(p->stream);
    const bool bf16 = c.dtype == FA_DTYPE_BF16;
    const unsigned grid = static_cast<unsigned>(l.grid);
    cudaError_t e;
    if (l.columns) {
        e = launch_paged_decode(a, tk, tv, l.columns, bf16, grid, stream);
    } else {
        CUtensorMap tq;
        if ((rc = query_map(&tq, p)) != FA_OK) return rc;
        if (l.wide == 64) e = l.query_tiles == 1 ? launch_paged_tiled<64, 1>(a, tq, tk, tv, bf16, grid, stream) : launch_paged_tiled<64, 2>(a, tq, tk, tv, bf16, grid, stream);
        else e = l.query_tiles == 1 ? launch_paged_tiled<128, 1>(a, tq, tk, tv, bf16, grid, stream) : launch_paged_tiled<128, 2>(a, tq, tk, tv, bf16, grid, stream);
    }
    if (e != cudaSuccess) return FA_ERR_CUDA;
    if (l.partials > 0 && launch_paged_combine(a, bf16, static_cast<unsigned>(l.split_items), stream) != cudaSuccess) return FA_ERR_CUDA;
    return FA_OK;
}

}  // extern "C"
