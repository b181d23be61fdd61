// Device helpers of the kernels that keep a query row a thread (S = Q K^T with M = N = 128, O += P V with P in tensor memory):
// packing, exponentials, the hand-over of P over named barriers, MMAs issued in blocks.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include "fa_internal.h"
#include "sm100_ptx.cuh"

namespace fa {
namespace {

template <bool kBf16>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    if constexpr (kBf16) {
        __nv_bfloat162 t = __floats2bfloat162_rn(lo, hi);
        return *reinterpret_cast<uint32_t*>(&t);
    } else {
        __half2 t = __floats2half2_rn(lo, hi);
        return *reinterpret_cast<uint32_t*>(&t);
    }
}

__device__ __forceinline__ float fast_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// exp2 on the FMA/ALU pipes for a pair of arguments x <= ~8: the MUFU unit (16 results per
// clock per SM) needs as long for the 128 x 128 exponentials of a tile pair as the tensor
// pipe needs for their MMAs, so part of them is computed here instead.  Round to the nearest
// integer n with the 1.5 * 2^23 trick, evaluate 2^f on f = x - n in [-0.5, 0.5] with a cubic
// (max relative error 7.5e-5, far below the 16-bit rounding of P), and add n to the exponent.
// Arguments below -126 give 2^-126 instead of 0.
__device__ __forceinline__ float2 poly_exp2_pair(float2 x) {
    x.x = fmaxf(x.x, -126.0f);
    x.y = fmaxf(x.y, -126.0f);
    const float2 magic = make_float2(12582912.0f, 12582912.0f);
    const float2 r = __fadd2_rn(x, magic);
    const float2 n = __fadd2_rn(r, make_float2(-12582912.0f, -12582912.0f));
    const float2 f = __ffma2_rn(n, make_float2(-1.0f, -1.0f), x);
    float2 p = __ffma2_rn(make_float2(0.0551716685f, 0.0551716685f), f, make_float2(0.2426111251f, 0.2426111251f));
    p = __ffma2_rn(p, f, make_float2(0.6932609677f, 0.6932609677f));
    p = __ffma2_rn(p, f, make_float2(0.9999280572f, 0.9999280572f));
    p.x = __int_as_float(__float_as_int(p.x) + (__float_as_int(r.x) << 23));
    p.y = __int_as_float(__float_as_int(p.y) + (__float_as_int(r.y) << 23));
    return p;
}

__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

// Whole-warp wait: the lanes poll together (one shared-memory access per poll).  A poll is
// slow while the tensor pipe streams operands from shared memory (several hundred cycles
// were measured), so the wait is a single phase with no second look.
__device__ __forceinline__ bool mbar_wait_warp(uint32_t bar, uint32_t parity, volatile int* abort_flag) {
    return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag) ? 1 : 0) != 0;
}

// Hardware named barriers carry the P hand-over: the 128 threads of a softmax warpgroup
// arrive (non-blocking), the MMA warp syncs.  Waking from a named barrier costs tens of
// cycles, while a poll of a shared-memory mbarrier took several hundred whenever the tensor
// pipe was streaming operands.  A named barrier cannot time out, so a softmax warp whose
// mbarrier wait gave up keeps walking its tile loop and posts every arrival it owes.
constexpr int kPBarrierThreads = 160;  // 128 softmax threads + the MMA warp (or + a keep-bit helper warp)
__device__ __forceinline__ void named_arrive(int id) {
    asm volatile("bar.arrive %0, %1;" ::"r"(id), "n"(kPBarrierThreads) : "memory");
}
__device__ __forceinline__ void named_sync(int id) {
    asm volatile("bar.sync %0, %1;" ::"r"(id), "n"(kPBarrierThreads) : "memory");
}

__device__ __forceinline__ bool elect_one() {
    uint32_t pred;
    asm volatile(
        "{\n\t.reg .pred P;\n\t"
        "elect.sync _|P, 0xffffffff;\n\t"
        "selp.u32 %0, 1, 0, P;\n\t}"
        : "=r"(pred));
    return pred != 0;
}

// Eight (D = 128) or four (D = 64) back-to-back MMAs of one S = Q K^T tile in a single
// asm block: the descriptors differ only in the low word (start address, 16-byte units),
// which is stepped inside the block, so the issuing thread does no other work between MMAs.
// Steps for a [128 x D] tile stored as 64-column boxes: 32 bytes per k-step inside a box
// (+2 units), next box after four steps (16 KB further: +1024 - 6 units).
#define FA_QK_STEP(inc)                                                                        \
    "add.u32 qa, qa, " #inc ";\n\tadd.u32 kb, kb, " #inc ";\n\t"                                 \
    "mov.b64 da, {qa, %3};\n\tmov.b64 db, {kb, %3};\n\t"                                        \
    "tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %4, p1;\n\t"
#define FA_QK_HEAD                                                                             \
    "{\n\t.reg .pred p0, p1;\n\t.reg .b32 qa, kb;\n\t.reg .b64 da, db;\n\t"                       \
    "setp.ne.b32 p0, 0, 0;\n\tsetp.eq.b32 p1, 0, 0;\n\t"                                        \
    "mov.b32 qa, %1;\n\tmov.b32 kb, %2;\n\t"                                                    \
    "mov.b64 da, {qa, %3};\n\tmov.b64 db, {kb, %3};\n\t"                                        \
    "tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %4, p0;\n\t"
template <int D>
__device__ __forceinline__ void issue_qk_block(uint32_t d_tmem, uint32_t qa_lo, uint32_t kb_lo, uint32_t desc_hi,
                                               uint32_t idesc) {
    if constexpr (D == 128) {
        asm volatile(FA_QK_HEAD FA_QK_STEP(2) FA_QK_STEP(2) FA_QK_STEP(2) FA_QK_STEP(1018) FA_QK_STEP(2)
                         FA_QK_STEP(2) FA_QK_STEP(2) "}"
                     ::"r"(d_tmem), "r"(qa_lo), "r"(kb_lo), "r"(desc_hi), "r"(idesc)
                     : "memory");
    } else {
        asm volatile(FA_QK_HEAD FA_QK_STEP(2) FA_QK_STEP(2) FA_QK_STEP(2) "}"
                     ::"r"(d_tmem), "r"(qa_lo), "r"(kb_lo), "r"(desc_hi), "r"(idesc)
                     : "memory");
    }
}

// Eight back-to-back MMAs of O += P V over the 128 keys of a tile: P advances 8 TMEM
// columns (16 packed elements) and V 16 rows (2048 bytes = 128 descriptor units) per step.
#define FA_PV_STEP                                                                             \
    "add.u32 pa, pa, 8;\n\tadd.u32 vb, vb, 128;\n\tmov.b64 db, {vb, %3};\n\t"                    \
    "tcgen05.mma.cta_group::1.kind::f16 [%0], [pa], db, %4, p1;\n\t"
#define FA_PV_HEAD                                                                             \
    "{\n\t.reg .pred p0, p1;\n\t.reg .b32 pa, vb;\n\t.reg .b64 db;\n\t"                          \
    "setp.ne.b32 p0, %5, 0;\n\tsetp.eq.b32 p1, 0, 0;\n\t"                                        \
    "mov.b32 pa, %1;\n\tmov.b32 vb, %2;\n\tmov.b64 db, {vb, %3};\n\t"                            \
    "tcgen05.mma.cta_group::1.kind::f16 [%0], [pa], db, %4, p0;\n\t"
// k-steps [0, kSplitSteps) of a tile: issued as soon as the first kSplitSteps*16 columns of P
// are in tensor memory; the rest follow when P is complete.
constexpr int kSplitSteps = 4;
__device__ __forceinline__ void issue_pv_first(uint32_t d_tmem, uint32_t a_tmem, uint32_t vb_lo, uint32_t desc_hi,
                                               uint32_t idesc, uint32_t accumulate) {
    asm volatile(FA_PV_HEAD FA_PV_STEP FA_PV_STEP FA_PV_STEP "}"
                 ::"r"(d_tmem), "r"(a_tmem), "r"(vb_lo), "r"(desc_hi), "r"(idesc), "r"(accumulate)
                 : "memory");
}
__device__ __forceinline__ void issue_pv_rest(uint32_t d_tmem, uint32_t a_tmem, uint32_t vb_lo, uint32_t desc_hi,
                                              uint32_t idesc) {
    asm volatile(FA_PV_HEAD FA_PV_STEP FA_PV_STEP FA_PV_STEP "}"
                 ::"r"(d_tmem), "r"(a_tmem + kSplitSteps * 8), "r"(vb_lo + kSplitSteps * 128), "r"(desc_hi), "r"(idesc), "r"(1u)
                 : "memory");
}

}  // namespace
}  // namespace fa
