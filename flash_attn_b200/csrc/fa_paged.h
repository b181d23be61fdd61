// What the kernels around the paged K/V cache share: its device-side description, and where a new token stands.
#pragma once
#include <cstdint>
#include <cuda.h>
#include <cuda_runtime.h>
#include "../../include/fa_b200.h"

namespace fa {

// (SM count and compute capability of the current device, kept per device: fa_api.cu)
int current_device(int* sms, int* major);
// A tensor map of 16-bit elements, boxes with the 128-byte swizzle; out-of-range elements read as zero.  (fa_api.cu)
int encode_map(CUtensorMap* m, int dtype, int rank, const void* base, const cuuint64_t* dims, const cuuint64_t* strides, const cuuint32_t* box);
// Whether rows of `columns` elements with these counts and strides (of up to three dimensions) lie apart from each other, one
// dimension inside another: what is written must.
bool rows_apart(const int64_t* counts, const int64_t* strides, int n, int64_t columns);
// FA_OK, or what of the cache's description the kernels cannot follow.
int check_cache(const fa_paged_kv& c, int64_t tokens);

// Keys of a sequence; a table has room for no more (check_cache), so that a longer one is named by its missing pages.
constexpr int kMostKeys = 1 << 30;

// The sequences of a call as the device sees them.
struct SeqTable {
    const int* seqlens_k;
    const int* cu_seqlens_q;  // or null: one row a sequence
    int batch;
    int tokens;               // rows there are
};

#ifdef __CUDACC__
// Rows [first, end) of sequence b, clipped to the rows there are, and its keys.
struct SeqSpan {
    int first, end, keys;
};
__device__ __forceinline__ SeqSpan seq_span(const SeqTable& t, int b) {
    SeqSpan s;
    s.first = t.cu_seqlens_q ? __ldg(t.cu_seqlens_q + b) : b;
    s.end = t.cu_seqlens_q ? __ldg(t.cu_seqlens_q + b + 1) : b + 1;
    s.keys = min(max(__ldg(t.seqlens_k + b), 0), kMostKeys);
    s.first = min(max(s.first, 0), t.tokens);
    s.end = max(min(s.end, t.tokens), s.first);
    return s;
}
#endif

}  // namespace fa
