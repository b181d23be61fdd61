// The end of a split item over a paged cache: the part that comes last puts the rows of all together.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include "paged_kernels.h"

namespace fa {
namespace {

// By the kThreads threads (named barrier 6) that wrote the part's rows: whether the part is the last of its item.
template <int kThreads>
__device__ __forceinline__ bool last_to_come(const PagedArgs& a, int slot, int parts, volatile int* flag) {
    asm volatile("bar.sync 6, %0;" ::"n"(kThreads) : "memory");
    if (threadIdx.x == 0) *flag = count_in(a.counts + slot, parts) ? 1 : 0;
    asm volatile("bar.sync 6, %0;" ::"n"(kThreads) : "memory");
    return *flag != 0;
}

// `slot`: where part 0 has left its rows (the others behind it), and the item's count.
// Rows [0, n_rows) of the block, whose first is row `row0` of the sequence, of K/V head `head_k`, by kWarps warps, kRows rows a warp at
// a time: sixteen 16-byte loads a lane are in flight, the weights' beside them.  What bounds it is one SM's way to L2, about a
// microsecond for 128 KB.
template <int D, bool kBf16, int kWarps, int kRows>
__device__ __forceinline__ void merge_parts(const PagedArgs& a, int slot, int parts, int head_k, int first, int row0, int n_rows, int warp) {
    constexpr int kUnroll = 16 / kRows;
    const int lane = threadIdx.x & 31;
    const bool mine = lane * 4 < D;
    for (int k0 = warp * kRows; k0 < n_rows; k0 += kWarps * kRows) {
        // lane i < kRows keeps row k0 + i's maximum and sum
        const bool row_lane = lane < kRows && k0 + lane < n_rows;
        float m = -INFINITY, l = 0.0f;
        float4 acc[kRows];
#pragma unroll
        for (int i = 0; i < kRows; ++i) acc[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        for (int j = 0; j < parts; j += kUnroll) {
            float4 v[kUnroll][kRows];
            float2 ml[kUnroll];
#pragma unroll
            for (int u = 0; u < kUnroll; ++u) {
                const long long at = (static_cast<long long>(slot) + j + u) * a.plan.rows + k0;
                const bool part = j + u < parts;
                ml[u] = row_lane && part ? __ldcg(a.ml_partial + at + lane) : make_float2(-INFINITY, 0.0f);
#pragma unroll
                for (int i = 0; i < kRows; ++i)
                    v[u][i] = mine && part && k0 + i < n_rows ? __ldcg(reinterpret_cast<const float4*>(a.o_partial + (at + i) * D) + lane)
                                                              : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            }
            float m_new = m;
#pragma unroll
            for (int u = 0; u < kUnroll; ++u) m_new = fmaxf(m_new, ml[u].x);
            const float base = m_new == -INFINITY ? 0.0f : m_new, keep = exp2f(m - base);
            l = j == 0 ? 0.0f : l * (m == -INFINITY ? 1.0f : keep);
            // (a part that saw no key has m = -inf, l = 0; one that saw only NaN has m = -inf, l = NaN)
            float wt[kUnroll];
#pragma unroll
            for (int u = 0; u < kUnroll; ++u) {
                wt[u] = exp2f(ml[u].x - base);
                l += ml[u].x == -INFINITY ? ml[u].y : wt[u] * ml[u].y;
            }
            m = m_new;
#pragma unroll
            for (int i = 0; i < kRows; ++i) {
                const float f = __shfl_sync(0xffffffffu, keep, i);
                if (j > 0) acc[i] = make_float4(acc[i].x * f, acc[i].y * f, acc[i].z * f, acc[i].w * f);
#pragma unroll
                for (int u = 0; u < kUnroll; ++u) {
                    const float x = __shfl_sync(0xffffffffu, wt[u], i);
                    if (x != 0.0f) {  // (a part without a key of the row has left 0, or what its masked values made of it)
                        acc[i].x = fmaf(x, v[u][i].x, acc[i].x);
                        acc[i].y = fmaf(x, v[u][i].y, acc[i].y);
                        acc[i].z = fmaf(x, v[u][i].z, acc[i].z);
                        acc[i].w = fmaf(x, v[u][i].w, acc[i].w);
                    }
                }
            }
        }
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;  // (NaN stays)
#pragma unroll
        for (int i = 0; i < kRows; ++i) {
            if (k0 + i >= n_rows) break;
            const float f = __shfl_sync(0xffffffffu, inv, i);
            const int tok = static_cast<int>(fast_div(a.div_group, static_cast<uint32_t>(row0 + k0 + i)));
            const int head = head_k * a.plan.group + row0 + k0 + i - tok * a.plan.group;
            const long long token = first + tok;
            if (lane * 4 < a.head_dim) {
                const long long at = token * a.o_stride[0] + head * a.o_stride[1] + lane * 4;
                const float4 o = make_float4(acc[i].x * f, acc[i].y * f, acc[i].z * f, acc[i].w * f);
                if (a.o_is_fp32) {
                    *reinterpret_cast<float4*>(static_cast<float*>(a.o) + at) = o;
                } else if (kBf16) {
                    const __nv_bfloat162 x = __floats2bfloat162_rn(o.x, o.y), y = __floats2bfloat162_rn(o.z, o.w);
                    *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.o) + at) =
                        make_uint2(*reinterpret_cast<const uint32_t*>(&x), *reinterpret_cast<const uint32_t*>(&y));
                } else {
                    const __half2 x = __floats2half2_rn(o.x, o.y), y = __floats2half2_rn(o.z, o.w);
                    *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.o) + at) =
                        make_uint2(*reinterpret_cast<const uint32_t*>(&x), *reinterpret_cast<const uint32_t*>(&y));
                }
            }
            if (lane == i && a.lse != nullptr) a.lse[token * a.heads + head] = l == 0.0f ? -INFINITY : fmaf(m, 0.6931471805599453f, logf(l));
        }
    }
}

}  // namespace
}  // namespace fa
