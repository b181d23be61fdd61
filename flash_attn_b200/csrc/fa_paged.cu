// Attention of new tokens over a paged K/V cache: the C entry point and its checks.
//
// One warp = one (row, head): 32 keys at a time, a lane each for the scores, then the lanes over the columns of V.
#include <algorithm>
#include <cmath>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include "fa_internal.h"
#include "fa_paged.h"
#include "sm100_ptx.cuh"

namespace fa {

namespace {

struct PagedArgs {
    SeqTable seq;
    const void *q, *k, *v;
    void* o;
    float* lse;
    const int* page_table;
    long long table_stride;
    int table_width, num_pages, page_shift;
    int heads, group, head_dim;
    long long qs[2], os[2], ks[3], vs[3];
    float scale;
    int is_causal, window_left, window_right;
    const float* alibi_slopes;
    int o_is_fp32;
    int* status;
};

template <typename T> __device__ __forceinline__ float to_f(T x);
template <> __device__ __forceinline__ float to_f<__half>(__half x) { return __half2float(x); }
template <> __device__ __forceinline__ float to_f<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T> __device__ __forceinline__ T from_f(float x);
template <> __device__ __forceinline__ __half from_f<__half>(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

template <typename T>
__global__ void __launch_bounds__(128) paged_rows_kernel(const PagedArgs a) {
    grid_dep_launch_dependents();
    __shared__ float q_row[4][128];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const long long item = static_cast<long long>(blockIdx.x) * 4 + warp;
    const int token = static_cast<int>(item / a.heads), h = static_cast<int>(item - static_cast<long long>(token) * a.heads);
    grid_dep_wait();
    if (token >= a.seq.tokens) return;
    int b = -1;
    SeqSpan s = {0, 0, 0};
    for (int i = 0; i < a.seq.batch; ++i) {
        s = seq_span(a.seq, i);
        if (token >= s.first && token < s.end) { b = i; break; }
    }
    if (b < 0) return;
    const long long pos = static_cast<long long>(s.keys) - s.end + token;
    const int kh = h / a.group;
    for (int c = lane; c < a.head_dim; c += 32) q_row[warp][c] = to_f(static_cast<const T*>(a.q)[token * a.qs[0] + h * a.qs[1] + c]);
    __syncwarp();
    const float slope = a.alibi_slopes ? a.alibi_slopes[h] : 0.0f;
    float m = -INFINITY, l = 0.0f, acc[4] = {0.f, 0.f, 0.f, 0.f};
    bool bad = false;
    for (long long k0 = 0; k0 < s.keys; k0 += 32) {
        const long long key = k0 + lane;
        bool see = key < s.keys && (!a.is_causal || key <= pos) && (a.window_left < 0 || pos - key <= a.window_left) &&
                   (a.window_right < 0 || key - pos <= a.window_right);
        int page = -1;
        float score = -INFINITY;
        if (see) {
            const long long nth = key >> a.page_shift;
            if (nth < a.table_width) page = a.page_table[b * a.table_stride + nth];
            if (page < 0 || page >= a.num_pages) { bad = true; see = false; }
        }
        const long long slot = key & ((1 << a.page_shift) - 1);
        if (see) {
            const T* kr = static_cast<const T*>(a.k) + page * a.ks[0] + kh * a.ks[1] + slot * a.ks[2];
            float dot = 0.0f;
            for (int c = 0; c < a.head_dim; ++c) dot = fmaf(q_row[warp][c], to_f(kr[c]), dot);
            score = dot * a.scale - slope * fabsf(static_cast<float>(key - pos));
        }
        float m_new = score;
        for (int o = 16; o; o >>= 1) m_new = fmaxf(m_new, __shfl_xor_sync(0xffffffffu, m_new, o));
        m_new = fmaxf(m, m_new);
        const float base = m_new == -INFINITY ? 0.0f : m_new;
        const float f = expf(m - base), p = expf(score - base);
        m = m_new;
        float sum = p;
        for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        l = l * f + sum;
        for (int i = 0; i < 4; ++i) acc[i] *= f;
        for (int j = 0; j < 32; ++j) {
            if (!__shfl_sync(0xffffffffu, see ? 1 : 0, j)) continue;
            const float pj = __shfl_sync(0xffffffffu, p, j);
            const long long at = __shfl_sync(0xffffffffu, page, j) * a.vs[0] + kh * a.vs[1] + __shfl_sync(0xffffffffu, slot, j) * a.vs[2];
            for (int i = 0; i < 4; ++i)
                if (i * 32 + lane < a.head_dim) acc[i] = fmaf(pj, to_f(static_cast<const T*>(a.v)[at + i * 32 + lane]), acc[i]);
        }
    }
    bad = __any_sync(0xffffffffu, bad);
    if (bad && lane == 0 && a.status) atomicExch(a.status, FA_STATUS_PAGE);
    for (int i = 0; i < 4; ++i) {
        const int c = i * 32 + lane;
        if (c >= a.head_dim) continue;
        const float x = bad ? __int_as_float(0x7fc00000) : l > 0.0f ? acc[i] / l : l == 0.0f ? 0.0f : l;
        const long long at = token * a.os[0] + h * a.os[1] + c;
        if (a.o_is_fp32) static_cast<float*>(a.o)[at] = x;
        else static_cast<T*>(a.o)[at] = from_f<T>(x);
    }
    if (lane == 0 && a.lse) a.lse[static_cast<long long>(token) * a.heads + h] = bad ? __int_as_float(0x7fc00000) : l == 0.0f ? -INFINITY : m + logf(l);
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

}  // namespace

}  // namespace fa

using namespace fa;

extern "C" {

size_t fa_paged_fwd_workspace_bytes(const fa_paged_fwd_params* p) { return check_fwd(p) == FA_OK ? 0 : 0; }

int fa_paged_fwd(const fa_paged_fwd_params* p) {
    int rc = check_fwd(p);
    if (rc != FA_OK) return rc;
    int sms = 0, major = 0;
    if ((rc = current_device(&sms, &major)) != FA_OK) return rc;
    if (major != 10) return FA_ERR_NOT_SM100;
    const fa_paged_kv& c = p->cache;
    PagedArgs a = {};
    a.seq = {c.seqlens_k, c.cu_seqlens_q, c.batch, static_cast<int>(p->tokens)};
    a.q = p->q;
    a.k = c.k;
    a.v = c.v;
    a.o = p->o;
    a.lse = p->lse;
    a.page_table = c.page_table;
    a.table_stride = c.table_stride;
    a.table_width = c.table_width;
    a.num_pages = c.num_pages;
    while ((1 << a.page_shift) < c.page_size) ++a.page_shift;
    a.heads = p->heads;
    a.group = p->heads / c.heads;
    a.head_dim = c.head_dim;
    std::copy(p->q_stride, p->q_stride + 2, a.qs);
    std::copy(p->o_stride, p->o_stride + 2, a.os);
    std::copy(c.k_stride, c.k_stride + 3, a.ks);
    std::copy(c.v_stride, c.v_stride + 3, a.vs);
    a.scale = p->softmax_scale;
    a.is_causal = p->is_causal;
    a.window_left = p->window_left;
    a.window_right = p->window_right;
    a.alibi_slopes = p->alibi_slopes;
    a.o_is_fp32 = p->o_dtype == FA_DTYPE_FP32;
    a.status = p->status;
    const long long rows = p->tokens * p->heads;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>((rows + 3) / 4));
    cfg.blockDim = dim3(128);
    cfg.stream = static_cast<cudaStream_t>(p->stream);
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    const cudaError_t e = c.dtype == FA_DTYPE_BF16 ? cudaLaunchKernelEx(&cfg, paged_rows_kernel<__nv_bfloat16>, a)
                                                   : cudaLaunchKernelEx(&cfg, paged_rows_kernel<__half>, a);
    return e == cudaSuccess ? FA_OK : FA_ERR_CUDA;
}

}  // extern "C"
