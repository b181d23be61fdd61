// Attention of new tokens over a paged K/V cache: the C entry point, its checks, the launch and its tensor maps.
#include <algorithm>
#include <cmath>
#include "fa_internal.h"
#include "fa_paged.h"
#include "paged_kernels.h"
#include "paged_plan.cuh"
#ifdef FA_TEST_SHORT_WAIT
#include "paged_parts.cuh"
#endif

namespace fa {

namespace {

// A part is not worth starting for fewer tiles than min_share; launches of more than one wave are cut into `waves` of parts, which are no
// shorter than long_share.  (Of 14 batches of chunks two took a sixth longer with
// parts of 4 tiles and more, none less with 16 and more.)
constexpr int kMinShare = 8, kLongShare = 16, kPagedWaves = 3, kOneWave = 24;
// The decode kernel's: a megabyte of K and V at least (kDecodeLongShare tiles of 128 columns; 64 sequences of 100 .. 8192 keys, 8 K/V
// heads of 128 columns: 82 us, with 8 tiles 84, with 24 tiles 88; 24 sequences of 500 .. 4000 keys, 16 heads of 64 columns: 49 us with
// 32 tiles, 54 with 16), and the tiles a CTA up to which a launch is one wave (4 sequences of 98304 .. 131072 keys: 298 us, in waves 309).
constexpr int kDecodeMinShare = 2, kDecodeLongShare = 16, kDecodeWaves = 4, kDecodeOneWave = 128;

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
    int min_share, long_share, waves, most_parts;
    int wide;                  // columns of a partial row: head_dim rounded up
    long long items;           // at most so many blocks of rows there are, over all K/V heads
    long long grid, partials;
    size_t count_bytes, ml_bytes, o_bytes, bytes;  // workspace: counts of parts, maxima and sums of partial rows, the rows, and all
};

// (A launch of each kernel where single tokens stand beside chunks was slower in six of eight such batches, by up to a half: what the two
// have to set up and the end of the one are not overlapped.)
PagedLaunch plan_launch(const fa_paged_fwd_params* p, int sms) {
    const fa_paged_kv& c = p->cache;
    PagedLaunch l = {};
    const int group = p->heads / c.heads;
    const long long rows = static_cast<long long>(std::min<int64_t>(p->max_seqlen_q, p->tokens)) * group;
    const int tile_rows = kTile / group * group;
    // Up to 16 rows, a block of the few-rows kernel, go there.  (32 heads on 8 of 128 columns, 16 rows: 24 sequences of 500 .. 8000 keys 67 us,
    // with one query tile 90, two 81; 4 of 30000 .. 60000 keys 119, 262, 261.  Two of its blocks, 32 rows: 89, 90, 75; and 150, 257, 257.
    // Four, 64 rows: 154, 91, 76; and 319, 262, 203.)
    l.columns = rows == 1 ? 1 : rows <= 4 ? 4 : rows <= 8 ? 8 : rows <= 16 ? 16 : 0;
    // One query tile, two CTAs an SM, where a sequence's rows fill no second one; above that two tiles share each K/V tile.  (Many short
    // sequences, one tile and two: 256 of 20 new tokens, 32 heads on 8 of 128 columns: 77 and 117 us; 64 of 128, 32 heads of 64: 46 and 66.
    // 192 rows in the 24 sequences above: 125 and 90.  Few blocks or long caches would be the faster for the second's one CTA an SM and
    // two K/V stages below that, too: the 24 sequences with 128 rows 93 and 77.)
    l.query_tiles = l.columns ? 0 : rows <= tile_rows ? 1 : 2;
    l.rows = l.columns ? l.columns : l.query_tiles * tile_rows;
    l.wide = c.head_dim <= 64 ? 64 : 128;
    l.slots = (l.query_tiles == 2 ? 1 : 2) * sms;
    l.items = c.heads * (c.cu_seqlens_q ? (p->tokens * group + static_cast<long long>(c.batch) * (l.rows - 1)) / l.rows
                                        : static_cast<long long>(c.batch) * ((group + l.rows - 1) / l.rows));
    const long long slots = l.slots;
    const long long tiles = (static_cast<long long>(c.table_width) * c.page_size + kTile - 1) / kTile;
    l.min_share = l.columns ? kDecodeMinShare : kMinShare;
    l.long_share = l.columns ? kDecodeLongShare * (128 / l.wide) : kLongShare;
    l.waves = l.columns ? kDecodeWaves : kPagedWaves;
    const long long parts = (tiles + l.min_share - 1) / l.min_share;  // of one item
    l.most_parts = static_cast<int>(parts);
    // (items longer than the share are cut into less than twice what the shares are)
    if (parts > 1) l.partials = std::min(2LL * l.waves * slots, l.items * parts);
    l.grid = l.items + std::min(l.waves * slots, l.items * (parts - 1));
    auto room = [](size_t bytes) { return (bytes + 255) & ~static_cast<size_t>(255); };
    // (the counts lie in the same place whatever the call: no count of one may be a partial row of another)
    l.count_bytes = room(2 * std::max(kPagedWaves, kDecodeWaves) * 2 * sms * sizeof(unsigned long long));
    l.ml_bytes = room(static_cast<size_t>(l.partials) * l.rows * sizeof(float2));
    l.o_bytes = room(static_cast<size_t>(l.partials) * l.rows * l.wide * sizeof(float));
    if (l.partials > 0) l.bytes = l.count_bytes + l.ml_bytes + l.o_bytes;
    return l;
}

PagedPlan plan_of(const fa_paged_fwd_params* p, const PagedLaunch& l) {
    const fa_paged_kv& c = p->cache;
    PagedPlan x = {};
    x.seq = {c.seqlens_k, c.cu_seqlens_q, c.batch, static_cast<int>(p->tokens)};
    x.heads_k = c.heads;
    x.group = p->heads / c.heads;
    x.table_keys = c.table_width * c.page_size;  // (below kMostKeys)
    x.rows = l.rows;
    x.block_tokens = l.rows / x.group + 2;  // (it may begin and end inside a token)
    x.div_rows = make_fastdiv(static_cast<uint32_t>(l.rows));
    x.is_causal = p->is_causal ? 1 : 0;
    // (a window of 2^29 or more hides nothing that the cache could hold)
    x.window_left = p->window_left < kMostKeys / 2 ? p->window_left : -1;
    x.window_right = p->window_right < kMostKeys / 2 ? p->window_right : -1;
    x.slots = l.slots;
    x.min_share = l.min_share;
    x.long_share = l.long_share;
    x.waves = l.waves;
    x.one_wave = l.columns ? kDecodeOneWave : kOneWave;
    x.most_parts = l.most_parts;
    x.partials = static_cast<int>(l.partials);
    x.grid = static_cast<int>(std::min(l.grid, 0x7fffffffLL));  // (a larger one is refused)
    return x;
}

// A tensor map: extents, strides (elements; of a dimension of one any will do) and box, innermost first.  The last ones are kept per
// host thread, being a function of these arguments alone.
struct MapShape {
    const void* base;
    int dtype, rank;
    int64_t dims[5], strides[5];  // strides[0]: 1
    int box[5];
    bool operator==(const MapShape& o) const {
        return base == o.base && dtype == o.dtype && rank == o.rank && std::equal(dims, dims + 5, o.dims) && std::equal(strides, strides + 5, o.strides) &&
               std::equal(box, box + 5, o.box);
    }
};

int map_of(CUtensorMap* m, const MapShape& shape) {
    struct Entry {
        MapShape shape;
        CUtensorMap map;
    };
    constexpr int kEntries = 12;
    thread_local Entry cache[kEntries] = {};
    thread_local int next_victim = 0;
    for (const Entry& e : cache) {
        if (e.shape.rank != 0 && e.shape == shape) {
            *m = e.map;
            return FA_OK;
        }
    }
    cuuint64_t d[5], s[4];
    cuuint32_t b[5];
    for (int i = 0; i < shape.rank; ++i) {
        d[i] = static_cast<cuuint64_t>(shape.dims[i]);
        b[i] = static_cast<cuuint32_t>(shape.box[i]);
        if (i > 0) s[i - 1] = shape.dims[i] > 1 ? static_cast<cuuint64_t>(shape.strides[i]) * 2 : 256;
    }
    const int rc = encode_map(m, shape.dtype, shape.rank, shape.base, d, s, b);
    if (rc != FA_OK) return rc;
    Entry& e = cache[next_victim];
    next_victim = (next_victim + 1) % kEntries;
    e.shape = shape;
    e.map = *m;
    return FA_OK;
}

// The whole-row map of a pool (paged_kernels.h), where its strides allow it.
bool whole_row_boxes(const fa_paged_kv& c, const void* base, const int64_t* stride, PageBoxes* x, MapShape* shape) {
    const int64_t eight = 8 * stride[2];
    if (c.head_dim != 128 || eight <= 0 || eight >= (1LL << 39)) return false;
    const int64_t page = c.num_pages > 1 ? stride[0] : 0, head = c.heads > 1 ? stride[1] : 0;
    if (page < 0 || head < 0 || page % eight != 0) return false;
    const bool apart = head % eight != 0;
    const int64_t page_step = page / eight, head_step = apart ? 0 : head / eight;
    const int64_t eights = (c.num_pages - 1) * page_step + (c.heads - 1) * head_step + c.page_size / 8;
    if (eights >= (1LL << 30)) return false;
    *x = {static_cast<int>(page_step), static_cast<int>(head_step), apart ? 1 : 0, static_cast<int>(eights)};
    *shape = {base, c.dtype, 5, {64, 8, 2, eights, apart ? c.heads : 1}, {1, stride[2], 64, eight, head}, {64, 8, 2, std::min(c.page_size, kTile) / 8, 1}};
    return true;
}

int page_maps(CUtensorMap* tk, CUtensorMap* tv, const fa_paged_kv& c, PagedArgs* a) {
    MapShape k, v;
    a->whole_rows = whole_row_boxes(c, c.k, c.k_stride, &a->k_box, &k) && whole_row_boxes(c, c.v, c.v_stride, &a->v_box, &v);
    if (!a->whole_rows) {
        const int box = std::min(c.page_size, kTile);
        k = {c.k, c.dtype, 4, {c.head_dim, c.page_size, c.heads, c.num_pages}, {1, c.k_stride[2], c.k_stride[1], c.k_stride[0]}, {64, box, 1, 1}};
        v = {c.v, c.dtype, 4, {c.head_dim, c.page_size, c.heads, c.num_pages}, {1, c.v_stride[2], c.v_stride[1], c.v_stride[0]}, {64, box, 1, 1}};
    }
    const int rc = map_of(tk, k);
    return rc != FA_OK ? rc : map_of(tv, v);
}

// Q: a box is 64 columns of the rows of a query tile, the heads of one K/V head side by side.
int query_map(CUtensorMap* m, const fa_paged_fwd_params* p) {
    const int group = p->heads / p->cache.heads;
    return map_of(m, {p->q, p->cache.dtype, 4, {p->cache.head_dim, group, p->cache.heads, p->tokens},
                      {1, p->q_stride[1], p->q_stride[1] * group, p->q_stride[0]}, {64, group, 1, kTile / group}});
}

// The output: 64 columns of the rows of a warp.
int output_map(CUtensorMap* m, const fa_paged_fwd_params* p) {
    const int group = p->heads / p->cache.heads;
    return map_of(m, {p->o, p->cache.dtype, 4, {p->cache.head_dim, group, p->cache.heads, p->tokens},
                      {1, p->o_stride[1], p->o_stride[1] * group, p->o_stride[0]}, {64, group, 1, 32 / group}});
}

}  // namespace

}  // namespace fa

using namespace fa;

#ifdef FA_TEST_SHORT_WAIT
static int test_leave_out = -1;
extern "C" int fa_test_leave_out_paged_tiles(int n) {
    test_leave_out = n;
    return 0;
}

// The parts of a call as its producers find them, asked for in any order: out[i] = part order[i], n_rows = 0 where there is none.
// Device memory both; sizes: those of the launch (numbers of parts at most, room for partial rows, SMs' worth of CTAs).
static __global__ void test_parts(const PagedPlan plan, const FastDiv div_group, const int* order, int n, PagedSeg* out) {
    const int lane = threadIdx.x;
    long long tiles = 0;
    for (int b = lane; b < plan.seq.batch; b += 32) {
        const int2 x = blocks_and_tiles(plan, seq_span(plan.seq, b));
        tiles += static_cast<long long>(x.x) * x.y;
    }
    PartLine line;
    line.start(plan, lane, sum_all(tiles) * plan.heads_k);
    for (int i = 0; i < n; ++i) {
        PagedSeg g = {};
        if (!line.find(plan, div_group, order[i], lane, &g)) g.n_rows = 0;
        if (lane == 0) out[i] = g;
        __syncwarp();
    }
}
extern "C" int fa_test_paged_parts(const fa_paged_fwd_params* p, const int* order, int n, void* out, int64_t* sizes) {
    int sms = 0, major = 0, rc = check_fwd(p);
    if (rc != FA_OK || (rc = current_device(&sms, &major)) != FA_OK) return rc;
    const PagedLaunch l = plan_launch(p, sms);
    sizes[0] = l.grid;
    sizes[1] = l.partials;
    sizes[2] = l.slots;
    if (n > 0) test_parts<<<1, 32, 0, static_cast<cudaStream_t>(p->stream)>>>(plan_of(p, l), make_fastdiv(static_cast<uint32_t>(p->heads / p->cache.heads)), order, n, static_cast<PagedSeg*>(out));
    return cudaGetLastError() == cudaSuccess ? FA_OK : FA_ERR_CUDA;
}
#endif

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
    // (the rows of a chunk come by a tensor map, whose dimensions each have a stride)
    if (!l.columns && ((p->tokens > 1 && p->q_stride[0] == 0) || (p->heads > 1 && p->q_stride[1] == 0))) return FA_ERR_INVALID_ARG;
    if (l.bytes > 0 && (!p->workspace || p->workspace_bytes < l.bytes)) return FA_ERR_WORKSPACE;
    if (l.bytes > 0 && (reinterpret_cast<uintptr_t>(p->workspace) & 15u)) return FA_ERR_INVALID_ARG;
    const fa_paged_kv& c = p->cache;
    PagedArgs a = {};
    a.plan = plan_of(p, l);
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
    a.o_units = (p->tokens == 1 || p->o_stride[0] % 8 == 0) && (p->heads == 1 || p->o_stride[1] % 8 == 0);
    a.o_tma = a.o_units && !a.o_is_fp32 && 32 % a.plan.group == 0 && p->o_stride[0] < (1LL << 39) && p->o_stride[1] * a.plan.group < (1LL << 39) &&
              p->o_stride[0] >= 0 && p->o_stride[1] >= 0;
    a.status = p->status;
#ifdef FA_TEST_SHORT_WAIT
    a.leave_out = test_leave_out;
#endif
    cudaStream_t stream = static_cast<cudaStream_t>(p->stream);
    const bool bf16 = c.dtype == FA_DTYPE_BF16;
    CUtensorMap tq, tk, tv, to = {};
    if ((rc = page_maps(&tk, &tv, c, &a)) != FA_OK) return rc;
    if (l.bytes > 0) {
        char* room = static_cast<char*>(p->workspace);
        a.counts = reinterpret_cast<unsigned long long*>(room);
        a.ml_partial = reinterpret_cast<float2*>(room + l.count_bytes);
        a.o_partial = reinterpret_cast<float*>(room + l.count_bytes + l.ml_bytes);
    }
    const unsigned grid = static_cast<unsigned>(l.grid);
    cudaError_t e;
    if (l.columns) {
        e = launch_paged_decode(a, tk, tv, l.columns, bf16, grid, stream);
    } else {
        if ((rc = query_map(&tq, p)) != FA_OK) return rc;
        if (a.o_tma && (rc = output_map(&to, p)) != FA_OK) return rc;
        if (l.wide == 64) e = l.query_tiles == 1 ? launch_paged_tiled<64, 1>(a, tq, tk, tv, to, bf16, grid, stream) : launch_paged_tiled<64, 2>(a, tq, tk, tv, to, bf16, grid, stream);
        else e = l.query_tiles == 1 ? launch_paged_tiled<128, 1>(a, tq, tk, tv, to, bf16, grid, stream) : launch_paged_tiled<128, 2>(a, tq, tk, tv, to, bf16, grid, stream);
    }
    return e == cudaSuccess ? FA_OK : FA_ERR_CUDA;
}

}  // extern "C"
