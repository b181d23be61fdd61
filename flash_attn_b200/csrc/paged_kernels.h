// Arguments and launches of the attention kernels over a paged cache.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>
#include "fa_internal.h"
#include "paged_plan.cuh"

namespace fa {

struct PagedArgs {
    PagedPlan plan;
    FastDiv div_group;        // query heads of a K/V head
    const void* q;
    void* o;
    float* lse;
    const int* page_table;
    long long table_stride;
    int table_width, num_pages, page_shift;
    int heads, head_dim;
    int tile_tokens;          // tokens of a query tile of 128 rows: 128 / group
    long long q_stride[2], o_stride[2];  // elements from one token and head to the next
    float scale_log2;
    const float* alibi_slopes;
    int o_is_fp32;
    float* o_partial;         // [parts of split items][plan.rows][64 or 128], un-normalised
    float2* ml_partial;       // [parts of split items][plan.rows]: maximum (log2 units) and sum
    int* status;
};

// columns: rows of a block, 1, 4, 8 or 16.
cudaError_t launch_paged_decode(const PagedArgs& a, const CUtensorMap& tk, const CUtensorMap& tv, int columns, bool bf16, unsigned grid,
                                cudaStream_t stream);
// D = 64 or 128 (head_dim rounded up), NQ query tiles a block.
template <int D, int NQ>
cudaError_t launch_paged_tiled(const PagedArgs& a, const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv, bool bf16, unsigned grid,
                               cudaStream_t stream);
template <> cudaError_t launch_paged_tiled<64, 1>(const PagedArgs&, const CUtensorMap&, const CUtensorMap&, const CUtensorMap&, bool, unsigned, cudaStream_t);
template <> cudaError_t launch_paged_tiled<64, 2>(const PagedArgs&, const CUtensorMap&, const CUtensorMap&, const CUtensorMap&, bool, unsigned, cudaStream_t);
template <> cudaError_t launch_paged_tiled<128, 1>(const PagedArgs&, const CUtensorMap&, const CUtensorMap&, const CUtensorMap&, bool, unsigned, cudaStream_t);
template <> cudaError_t launch_paged_tiled<128, 2>(const PagedArgs&, const CUtensorMap&, const CUtensorMap&, const CUtensorMap&, bool, unsigned, cudaStream_t);
// The split items' rows from their parts.
cudaError_t launch_paged_combine(const PagedArgs& a, bool bf16, unsigned items, cudaStream_t stream);

}  // namespace fa
