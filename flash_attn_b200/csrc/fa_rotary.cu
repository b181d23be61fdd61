// Rotary positions, and the append of new tokens to a paged K/V cache with the rotation of K and Q fused in.
//
// Both are streams: each element is read once and written once, so HBM bounds them, and below some hundred kilobytes the launch.
// What a kernel adds to the bytes is the sine and cosine of a (position, pair), about fifty instructions, which all heads of a row
// share: a thread takes one row and one group of pairs -- the columns of two 16-byte vectors -- works its sines and cosines out once
// and goes through heads with them in registers.
//
// The angle of a far position is large (a million radians at 2^20), so position * inv_freq in 32 bits would be wrong by a tenth of
// a radian.  A turn is taken as 2^64 instead: inv_freq / 2 pi, less its whole turns, is rounded to a 64-bit fraction f, and
// position * f in wrapping integer arithmetic IS the angle modulo a turn, off by position * 2^-53 turns (what the double holds).
// Its upper 32 bits, as a signed number of half turns, are what sincospi is given: as a float of 24 bits, off by 2^-25 of a half turn at
// most (9.4e-8 of |a| + |b|: thousands of times less than the rounding of a 16-bit result; fp32 results are off by 4.5e-8 on the whole, where
// sines of 64-bit angles leave 3.4e-8).
#include <algorithm>
#include <cmath>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <type_traits>
#include "fa_internal.h"
#include "fa_paged.h"
#include "sm100_ptx.cuh"

namespace fa {

namespace {

constexpr int kRThreads = 256;
// Blocks an SM: 96 KB of loads in flight.  (bf16 [4, 32, 4096, 128]: with two blocks 44.0 us, three 42.2, four and two heads in flight
// 43.1; 6.4 TB/s.)
constexpr int kRBlocks = 3;
constexpr int kRUnroll = 4;       // heads whose vectors a thread has in flight
constexpr int kSeqStage = 1024;   // row numbers of sequences that a block keeps in shared memory

// kVec consecutive elements, loaded and stored as one and kept as they lie in memory: unpacked, 16-bit elements take a register each.
template <typename T, int kVec>
struct Vec {
    static constexpr int kBytes = static_cast<int>(sizeof(T)) * kVec, kWords = (kBytes + 3) / 4;
    uint32_t w[kWords];
    __device__ __forceinline__ void load(const T* p) {
        if constexpr (kBytes == 16) {
            const uint4 v = *reinterpret_cast<const uint4*>(p);
            w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
        } else if constexpr (kBytes == 8) {
            const uint2 v = *reinterpret_cast<const uint2*>(p);
            w[0] = v.x; w[1] = v.y;
        } else if constexpr (kBytes == 4) {
            w[0] = *reinterpret_cast<const uint32_t*>(p);
        } else {
            w[0] = *reinterpret_cast<const uint16_t*>(p);
        }
    }
    __device__ __forceinline__ void store(T* p) const {
        if constexpr (kBytes == 16) *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
        else if constexpr (kBytes == 8) *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
        else if constexpr (kBytes == 4) *reinterpret_cast<uint32_t*>(p) = w[0];
        else *reinterpret_cast<uint16_t*>(p) = static_cast<uint16_t>(w[0]);
    }
    __device__ __forceinline__ float get(int i) const {
        if constexpr (std::is_same_v<T, float>) return __uint_as_float(w[i]);
        else if constexpr (std::is_same_v<T, __nv_bfloat16>) return __uint_as_float((i & 1) ? w[i >> 1] & 0xffff0000u : w[i >> 1] << 16);
        else return __half2float(__ushort_as_half(static_cast<unsigned short>((i & 1) ? w[i >> 1] >> 16 : w[i >> 1])));
    }
    // elements i and i + 1 (i even; of a single element: x)
    __device__ __forceinline__ void set2(int i, float x, float y) {
        if constexpr (std::is_same_v<T, float>) {
            w[i] = __float_as_uint(x);
            if constexpr (kVec > 1) w[i + 1] = __float_as_uint(y);
        } else if constexpr (kVec == 1) {
            if constexpr (std::is_same_v<T, __nv_bfloat16>) w[0] = __bfloat16_as_ushort(__float2bfloat16_rn(x));
            else w[0] = __half_as_ushort(__float2half_rn(x));
        } else if constexpr (std::is_same_v<T, __nv_bfloat16>) {
            const __nv_bfloat162 v = __floats2bfloat162_rn(x, y);
            w[i >> 1] = *reinterpret_cast<const uint32_t*>(&v);
        } else {
            const __half2 v = __floats2half2_rn(x, y);
            w[i >> 1] = *reinterpret_cast<const uint32_t*>(&v);
        }
    }
};

struct Rotation {
    const double* inv_freq;
    int half;           // rotary_dim / 2; 0 = nothing turns
    int dim;            // head_dim
    float amplitude;
    float sine;         // +1 or -1 (inverse)
    int turn_groups;    // groups of kVec pairs
    int groups;         // and of two vectors that are copied, one behind the other
    int rows_per_block;
    FastDiv div_groups;
};

// The columns of a thread's two vectors.
template <int kVec, bool kInterleaved>
struct Columns {
    int a, b;
    bool turns, has_b;
    __device__ __forceinline__ Columns(const Rotation& r, int group) {
        turns = group < r.turn_groups;
        if (turns) {
            a = kInterleaved ? group * 2 * kVec : group * kVec;
            b = kInterleaved ? a + kVec : a + r.half;
            has_b = true;
        } else {
            a = 2 * r.half + (group - r.turn_groups) * 2 * kVec;
            b = a + kVec;
            has_b = b < r.dim;
        }
    }
};

template <int kVec>
__device__ __forceinline__ void angles(const Rotation& r, int group, long long position, float (&cs)[kVec], float (&sn)[kVec]) {
    if (group >= r.turn_groups) return;
#pragma unroll
    for (int i = 0; i < kVec; ++i) {
        double turns = __ldg(r.inv_freq + group * kVec + i) * 0.15915494309189533577;  // 1 / (2 pi)
        turns -= floor(turns);
        const unsigned long long f = __double2ull_rn(turns * 18446744073709549568.0) * static_cast<unsigned long long>(position);
        float s, c;
        sincospif(static_cast<float>(static_cast<int>(f >> 32)) * 4.656612873077393e-10f, &s, &c);  // 2^-31
        cs[i] = c * r.amplitude;
        sn[i] = s * r.amplitude * r.sine;
    }
}

template <typename T, int kVec, bool kInterleaved>
__device__ __forceinline__ void turn(Vec<T, kVec>& va, Vec<T, kVec>& vb, const float (&cs)[kVec], const float (&sn)[kVec]) {
    if constexpr (kInterleaved && kVec > 1) {  // pairs 0 .. kVec/2-1 lie in the first vector, the others in the second
#pragma unroll
        for (int i = 0; i < kVec; ++i) {
            Vec<T, kVec>& v = i < kVec / 2 ? va : vb;
            const int at = i < kVec / 2 ? 2 * i : 2 * i - kVec;
            const float x = v.get(at), y = v.get(at + 1);
            v.set2(at, fmaf(x, cs[i], -(y * sn[i])), fmaf(y, cs[i], x * sn[i]));
        }
    } else {
        constexpr int kStep = kVec > 1 ? 2 : 1;
#pragma unroll
        for (int i = 0; i < kVec; i += kStep) {
            float x[2] = {0.0f, 0.0f}, y[2] = {0.0f, 0.0f};
#pragma unroll
            for (int k = 0; k < kStep; ++k) {
                const float p = va.get(i + k), q = vb.get(i + k);
                x[k] = fmaf(p, cs[i + k], -(q * sn[i + k]));
                y[k] = fmaf(q, cs[i + k], p * sn[i + k]);
            }
            va.set2(i, x[0], x[1]);
            vb.set2(i, y[0], y[1]);
        }
    }
}

struct RotaryArgs {
    Rotation rot;
    const void* x;
    void* y;
    const void* positions;
    long long position_stride;
    int positions_64;
    int batch, heads, rows;
    int heads_per_block;
    long long xs[3], ys[3];
};

template <typename T, int kVec, bool kInterleaved>
__global__ void __launch_bounds__(kRThreads, kRBlocks) rotary_kernel(const RotaryArgs a) {
    grid_dep_launch_dependents();
    const int local = static_cast<int>(fast_div(a.rot.div_groups, threadIdx.x));
    const int group = static_cast<int>(threadIdx.x) - local * a.rot.groups;
    const long long row = static_cast<long long>(blockIdx.x) * a.rot.rows_per_block + local;
    if (local >= a.rot.rows_per_block || row >= a.rows) return;
    const Columns<kVec, kInterleaved> col(a.rot, group);
    const int h_lo = blockIdx.y * a.heads_per_block, h_hi = min(h_lo + a.heads_per_block, a.heads);
    using V = Vec<T, kVec>;
    grid_dep_wait();
    for (int b = blockIdx.z; b < a.batch; b += gridDim.z) {
        const long long at = b * a.position_stride + row;
        const long long position = a.positions_64 ? static_cast<const long long*>(a.positions)[at] : static_cast<const int*>(a.positions)[at];
        const T* x = static_cast<const T*>(a.x) + b * a.xs[0] + row * a.xs[2];
        T* y = static_cast<T*>(a.y) + b * a.ys[0] + row * a.ys[2];
        float cs[kVec], sn[kVec];
        bool have = false;
        for (int h0 = h_lo; h0 < h_hi; h0 += kRUnroll) {
            V va[kRUnroll], vb[kRUnroll];
#pragma unroll
            for (int u = 0; u < kRUnroll; ++u) {
                if (h0 + u >= h_hi) break;
                const T* p = x + (h0 + u) * a.xs[1];
                va[u].load(p + col.a);
                if (col.has_b) vb[u].load(p + col.b);
            }
            if (!have) {  // (under the first loads)
                angles<kVec>(a.rot, group, position, cs, sn);
                have = true;
            }
#pragma unroll
            for (int u = 0; u < kRUnroll; ++u) {
                if (h0 + u >= h_hi) break;
                if (col.turns) turn<T, kVec, kInterleaved>(va[u], vb[u], cs, sn);
                T* p = y + (h0 + u) * a.ys[1];
                va[u].store(p + col.a);
                if (col.has_b) vb[u].store(p + col.b);
            }
        }
    }
}

struct AppendArgs {
    Rotation rot;
    SeqTable seq;
    const int* page_table;
    long long table_stride;
    int table_width, num_pages, page_shift;
    int heads, heads_k;       // heads = 0: no Q
    int rows_per_thread;      // of the heads + 2 heads_k rows of a token
    const void *k, *v, *q;
    void *k_pages, *v_pages, *q_out;
    long long ks[2], vs[2], qs[2], qos[2], kps[3], vps[3];
    int* status;
};

// The sequence of a row: the last whose first row is at or before it.  In shared memory where the table fits.
__device__ __forceinline__ int sequence_of(const int* cu, int batch, int token) {
    int lo = 0, hi = batch;  // cu[lo] <= token < cu[hi], if the table ascends
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (cu[mid] <= token) lo = mid; else hi = mid;
    }
    return lo;
}

template <typename T, int kVec, bool kInterleaved>
__global__ void __launch_bounds__(kRThreads, kRBlocks) append_kernel(const AppendArgs a) {
    __shared__ int cu[kSeqStage];
    grid_dep_launch_dependents();
    const int local = static_cast<int>(fast_div(a.rot.div_groups, threadIdx.x));
    const int group = static_cast<int>(threadIdx.x) - local * a.rot.groups;
    const long long row = static_cast<long long>(blockIdx.x) * a.rot.rows_per_block + local;
    const Columns<kVec, kInterleaved> col(a.rot, group);
    using V = Vec<T, kVec>;
    grid_dep_wait();
    const bool staged = a.seq.cu_seqlens_q != nullptr && a.seq.batch < kSeqStage;
    if (staged) {
        for (int i = threadIdx.x; i <= a.seq.batch; i += kRThreads) cu[i] = a.seq.cu_seqlens_q[i];
        __syncthreads();
    }
    if (local >= a.rot.rows_per_block || row >= a.seq.tokens) return;
    const int token = static_cast<int>(row);
    const int b = a.seq.cu_seqlens_q == nullptr ? token : sequence_of(staged ? cu : a.seq.cu_seqlens_q, a.seq.batch, token);
    if (b >= a.seq.batch) return;  // (rows behind the last sequence)
    const SeqSpan span = seq_span(a.seq, b);
    if (token < span.first || token >= span.end) return;
    const int position = span.keys - span.end + token;
    // the token's page; one that is not in the pool takes nothing
    int page = -1;
    const int nth = position >> a.page_shift;
    if (position >= 0 && nth < a.table_width) page = a.page_table[b * a.table_stride + nth];
    const bool to_page = page >= 0 && page < a.num_pages;
    if (!to_page && group == 0 && blockIdx.y == 0 && a.status != nullptr) atomicExch(a.status, FA_STATUS_PAGE);
    const long long slot = position & ((1 << a.page_shift) - 1);

    const T* k = static_cast<const T*>(a.k) + token * a.ks[0];
    const T* v = static_cast<const T*>(a.v) + token * a.vs[0];
    const T* q = static_cast<const T*>(a.q) + token * a.qs[0];
    T* q_out = static_cast<T*>(a.q_out) + token * a.qos[0];
    T* k_to = static_cast<T*>(a.k_pages) + page * a.kps[0] + slot * a.kps[2];
    T* v_to = static_cast<T*>(a.v_pages) + page * a.vps[0] + slot * a.vps[2];
    // rows of a token: its query heads, its K heads, its V heads
    const int all = a.heads + 2 * a.heads_k;
    const int r_lo = blockIdx.y * a.rows_per_thread, r_hi = min(r_lo + a.rows_per_thread, all);
    float cs[kVec], sn[kVec];
    bool have = false;
    for (int r0 = r_lo; r0 < r_hi; r0 += kRUnroll) {
        V va[kRUnroll], vb[kRUnroll];
#pragma unroll
        for (int u = 0; u < kRUnroll; ++u) {
            const int r = r0 + u;
            if (r >= r_hi) break;
            const T* p = r < a.heads ? q + r * a.qs[1]
                         : r < a.heads + a.heads_k ? k + (r - a.heads) * a.ks[1] : v + (r - a.heads - a.heads_k) * a.vs[1];
            va[u].load(p + col.a);
            if (col.has_b) vb[u].load(p + col.b);
        }
        if (!have && r_lo < a.heads + a.heads_k) {
            angles<kVec>(a.rot, group, position, cs, sn);
            have = true;
        }
#pragma unroll
        for (int u = 0; u < kRUnroll; ++u) {
            const int r = r0 + u;
            if (r >= r_hi) break;
            if (col.turns && r < a.heads + a.heads_k) turn<T, kVec, kInterleaved>(va[u], vb[u], cs, sn);
            T* p = r < a.heads ? q_out + r * a.qos[1]
                   : r < a.heads + a.heads_k ? k_to + (r - a.heads) * a.kps[1] : v_to + (r - a.heads - a.heads_k) * a.vps[1];
            if (r < a.heads || to_page) {
                va[u].store(p + col.a);
                if (col.has_b) vb[u].store(p + col.b);
            }
        }
    }
}

// Elements of a vector that every row's columns can be read and written in: 16 bytes, 8, or one element.
struct VecRule {
    int elem;
    bool fits16 = true, fits8 = true;
    void columns(int n) { at(static_cast<uint64_t>(n) * elem); }
    void pointer(const void* p) { at(reinterpret_cast<uintptr_t>(p)); }
    void stride(int64_t s, int64_t steps) { if (steps > 1) at(static_cast<uint64_t>(s) * elem); }
    void at(uint64_t bytes) {
        if (bytes % 16 != 0) fits16 = false;
        if (bytes % 8 != 0) fits8 = false;
    }
    int bytes() const { return fits16 ? 16 : fits8 ? 8 : elem; }
};

void fill_rotation(Rotation* r, const double* inv_freq, int rotary_dim, int head_dim, float amplitude, bool inverse, int vec, bool copies) {
    r->inv_freq = inv_freq;
    r->half = rotary_dim / 2;
    r->dim = head_dim;
    r->amplitude = amplitude;
    r->sine = inverse ? -1.0f : 1.0f;
    r->turn_groups = r->half / vec;
    r->groups = r->turn_groups + (copies ? ((head_dim - rotary_dim) / vec + 1) / 2 : 0);
    r->rows_per_block = kRThreads / r->groups;
    r->div_groups = make_fastdiv(static_cast<uint32_t>(r->groups));
}

// Rows of a token that one thread goes through: eight of them share its sines and cosines (with two the instructions bound it, at
// eight HBM does), fewer where the launch would leave SMs idle.
int rows_a_thread(long long tokens, int groups, int rows, int sms) {
    int n = 8;
    while (n > 1 && tokens * groups * ((rows + n - 1) / n) < static_cast<long long>(sms) * 1024) n /= 2;
    while ((rows + n - 1) / n > 65535) n *= 2;
    return n;
}

template <typename F>
cudaError_t launch_rows(F kernel, dim3 grid, cudaStream_t stream, const void* args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(kRThreads);
    cfg.stream = stream;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    void* list[1] = {const_cast<void*>(args)};
    return cudaLaunchKernelExC(&cfg, reinterpret_cast<const void*>(kernel), list);
}

template <typename T>
auto rotary_of(int vec_bytes, bool inter) {
    constexpr int v16 = 16 / sizeof(T), v8 = 8 / sizeof(T);
    if (vec_bytes == 16) return inter ? rotary_kernel<T, v16, true> : rotary_kernel<T, v16, false>;
    if (vec_bytes == 8) return inter ? rotary_kernel<T, v8, true> : rotary_kernel<T, v8, false>;
    return inter ? rotary_kernel<T, 1, true> : rotary_kernel<T, 1, false>;
}
template <typename T>
auto append_of(int vec_bytes, bool inter) {
    if (vec_bytes == 16) return inter ? append_kernel<T, 8, true> : append_kernel<T, 8, false>;
    if (vec_bytes == 8) return inter ? append_kernel<T, 4, true> : append_kernel<T, 4, false>;
    return inter ? append_kernel<T, 1, true> : append_kernel<T, 1, false>;
}

int check_rotation(const double* inv_freq, int rotary_dim, int head_dim, float amplitude) {
    if (!inv_freq || (reinterpret_cast<uintptr_t>(inv_freq) & 7u)) return FA_ERR_INVALID_ARG;
    if (rotary_dim < 2 || rotary_dim % 2 != 0 || rotary_dim > head_dim) return FA_ERR_INVALID_ARG;
    return std::isfinite(amplitude) ? FA_OK : FA_ERR_INVALID_ARG;
}

}  // namespace

bool rows_apart(const int64_t* counts, const int64_t* strides, int n, int64_t columns) {
    int order[3], m = 0;
    for (int i = 0; i < n; ++i)
        if (counts[i] > 1) order[m++] = i;
    std::sort(order, order + m, [&](int x, int y) { return strides[x] < strides[y]; });
    int64_t reach = columns;  // elements from the first to behind the last of the dimensions so far
    for (int i = 0; i < m; ++i) {
        if (strides[order[i]] < reach || strides[order[i]] >= (1LL << 60) / counts[order[i]]) return false;
        reach += strides[order[i]] * (counts[order[i]] - 1);
    }
    return true;
}

int check_cache(const fa_paged_kv& c, int64_t tokens) {
    if (!c.k || !c.v || !c.page_table || !c.seqlens_k) return FA_ERR_INVALID_ARG;
    if (c.dtype != FA_DTYPE_FP16 && c.dtype != FA_DTYPE_BF16) return FA_ERR_UNSUPPORTED;
    if (c.num_pages < 1 || c.heads < 1 || c.head_dim < 1 || c.batch < 1 || c.table_width < 1 || tokens < 1) return FA_ERR_INVALID_ARG;
    if (c.page_size < 1) return FA_ERR_INVALID_ARG;
    if (c.head_dim > 128 || c.head_dim % 8 != 0 || c.page_size < 8 || (c.page_size & (c.page_size - 1)) != 0) return FA_ERR_UNSUPPORTED;
    if (c.table_stride < c.table_width && c.batch > 1) return FA_ERR_INVALID_ARG;
    if ((reinterpret_cast<uintptr_t>(c.k) | reinterpret_cast<uintptr_t>(c.v)) & 15u) return FA_ERR_INVALID_ARG;
    if ((reinterpret_cast<uintptr_t>(c.page_table) | reinterpret_cast<uintptr_t>(c.seqlens_k) | reinterpret_cast<uintptr_t>(c.cu_seqlens_q)) & 3u)
        return FA_ERR_INVALID_ARG;
    const int64_t counts[3] = {c.num_pages, c.heads, c.page_size};
    for (const int64_t* s : {c.k_stride, c.v_stride}) {
        for (int i = 0; i < 3; ++i) {
            if (counts[i] == 1) continue;
            if (s[i] % 8 != 0) return FA_ERR_INVALID_ARG;
            if (s[i] >= (1LL << 39)) return FA_ERR_TOO_LARGE;  // (a tensor map's strides are 40 bits of bytes)
        }
        if (!rows_apart(counts, s, 3, c.head_dim)) return FA_ERR_INVALID_ARG;
    }
    if (static_cast<long long>(c.table_width) * c.page_size >= kMostKeys) return FA_ERR_TOO_LARGE;
    if (tokens > 0x3fffffffLL || c.batch > 0x3fffffff) return FA_ERR_TOO_LARGE;
    if (!c.cu_seqlens_q && tokens < c.batch) return FA_ERR_INVALID_ARG;
    return FA_OK;
}

}  // namespace fa

using namespace fa;

extern "C" {

int fa_rotary_frequencies(int rotary_dim, double base, int kind, double factor, double original_length, double low_turns,
                          double high_turns, double* inv_freq, double* amplitude) {
    if (!inv_freq || rotary_dim < 2 || rotary_dim % 2 != 0 || !(base > 0.0) || !std::isfinite(base)) return FA_ERR_INVALID_ARG;
    if (kind < FA_ROTARY_PLAIN || kind > FA_ROTARY_RAMP) return FA_ERR_INVALID_ARG;
    if (kind != FA_ROTARY_PLAIN && (!(factor > 0.0) || !std::isfinite(factor))) return FA_ERR_INVALID_ARG;
    if (kind == FA_ROTARY_NTK) {
        if (rotary_dim < 4) return FA_ERR_INVALID_ARG;  // (the exponent is rotary_dim / (rotary_dim - 2))
        base *= std::pow(factor, static_cast<double>(rotary_dim) / (rotary_dim - 2));
    }
    if (kind == FA_ROTARY_RAMP && (!(original_length > 0.0) || !std::isfinite(original_length) || !(high_turns > low_turns) || !std::isfinite(high_turns - low_turns)))
        return FA_ERR_INVALID_ARG;
    for (int i = 0; i < rotary_dim / 2; ++i) {
        double w = std::pow(base, -2.0 * i / rotary_dim);
        if (kind == FA_ROTARY_LINEAR) w /= factor;
        if (kind == FA_ROTARY_RAMP) {
            const double turns = original_length * w / 6.283185307179586477;
            const double keep = std::min(1.0, std::max(0.0, (turns - low_turns) / (high_turns - low_turns)));
            w = w * keep + w / factor * (1.0 - keep);
        }
        inv_freq[i] = w;
    }
    if (amplitude) *amplitude = kind == FA_ROTARY_RAMP ? 0.1 * std::log(factor) + 1.0 : 1.0;
    return FA_OK;
}

int fa_rotary(const fa_rotary_params* p) {
    if (!p || !p->x || !p->y || !p->positions) return FA_ERR_INVALID_ARG;
    if (p->dtype != FA_DTYPE_FP16 && p->dtype != FA_DTYPE_BF16 && p->dtype != FA_DTYPE_FP32) return FA_ERR_UNSUPPORTED;
    if (p->batch < 1 || p->heads < 1 || p->rows < 1 || p->head_dim < 1) return FA_ERR_INVALID_ARG;
    if (p->head_dim > 256) return FA_ERR_UNSUPPORTED;  // (a row's groups of one pair are the threads of a block)
    int rc = check_rotation(p->inv_freq, p->rotary_dim, p->head_dim, p->amplitude);
    if (rc != FA_OK) return rc;
    const int elem = p->dtype == FA_DTYPE_FP32 ? 4 : 2;
    if ((reinterpret_cast<uintptr_t>(p->x) | reinterpret_cast<uintptr_t>(p->y)) % elem != 0) return FA_ERR_INVALID_ARG;
    if (reinterpret_cast<uintptr_t>(p->positions) % (p->positions_64 ? 8 : 4) != 0) return FA_ERR_INVALID_ARG;
    const int64_t counts[3] = {p->batch, p->heads, p->rows};
    const bool same = p->x == p->y;
    VecRule rule{elem};
    rule.pointer(p->x);
    rule.pointer(p->y);
    rule.columns(p->rotary_dim / 2);
    rule.columns(p->head_dim - p->rotary_dim);
    for (int i = 0; i < 3; ++i) {
        rule.stride(p->x_stride[i], counts[i]);
        rule.stride(p->y_stride[i], counts[i]);
        if (counts[i] > 1 && p->x_stride[i] < 0) return FA_ERR_INVALID_ARG;
        if (counts[i] > 1 && p->x_stride[i] != p->y_stride[i] && same) return FA_ERR_INVALID_ARG;
    }
    if (!rows_apart(counts, p->y_stride, 3, p->head_dim)) return FA_ERR_INVALID_ARG;
    int sms = 0, major = 0;
    if ((rc = current_device(&sms, &major)) != FA_OK) return rc;
    if (major != 10) return FA_ERR_NOT_SM100;
    RotaryArgs a = {};
    const int vec_bytes = rule.bytes(), vec = vec_bytes / elem;
    fill_rotation(&a.rot, p->inv_freq, p->rotary_dim, p->head_dim, p->amplitude, p->inverse != 0, vec, !same);
    a.x = p->x;
    a.y = p->y;
    a.positions = p->positions;
    a.positions_64 = p->positions_64;
    a.position_stride = p->position_stride;
    a.batch = p->batch;
    a.heads = p->heads;
    a.rows = p->rows;
    std::copy(p->x_stride, p->x_stride + 3, a.xs);
    std::copy(p->y_stride, p->y_stride + 3, a.ys);
    a.heads_per_block = rows_a_thread(static_cast<long long>(p->batch) * p->rows, a.rot.groups, p->heads, sms);
    const dim3 grid(static_cast<unsigned>((p->rows + a.rot.rows_per_block - 1) / a.rot.rows_per_block),
                    static_cast<unsigned>((p->heads + a.heads_per_block - 1) / a.heads_per_block),
                    static_cast<unsigned>(std::min(p->batch, 65535)));
    const bool inter = p->interleaved != 0;
    const auto kernel = p->dtype == FA_DTYPE_FP32 ? rotary_of<float>(vec_bytes, inter)
                        : p->dtype == FA_DTYPE_BF16 ? rotary_of<__nv_bfloat16>(vec_bytes, inter) : rotary_of<__half>(vec_bytes, inter);
    return launch_rows(kernel, grid, static_cast<cudaStream_t>(p->stream), &a) == cudaSuccess ? FA_OK : FA_ERR_CUDA;
}

int fa_paged_append(const fa_paged_append_params* p) {
    if (!p || !p->k || !p->v) return FA_ERR_INVALID_ARG;
    const fa_paged_kv& c = p->cache;
    int rc = check_cache(c, p->tokens);
    if (rc != FA_OK) return rc;
    if (p->q && (!p->q_out || p->heads < 1 || !p->inv_freq)) return FA_ERR_INVALID_ARG;
    if (!p->inv_freq && p->rotary_dim != 0) return FA_ERR_INVALID_ARG;
    if (p->inv_freq && (rc = check_rotation(p->inv_freq, p->rotary_dim, c.head_dim, p->amplitude)) != FA_OK) return rc;
    const int heads = p->q ? p->heads : 0;
    VecRule rule{2};
    auto rows = [&](const void* base, const int64_t* s, int n, bool writes) {
        if (reinterpret_cast<uintptr_t>(base) & 1u) rc = FA_ERR_INVALID_ARG;
        rule.pointer(base);
        const int64_t counts[2] = {p->tokens, n};
        for (int i = 0; i < 2; ++i) {
            rule.stride(s[i], counts[i]);
            if (counts[i] > 1 && s[i] < 0) rc = FA_ERR_INVALID_ARG;
        }
        if (writes && !rows_apart(counts, s, 2, c.head_dim)) rc = FA_ERR_INVALID_ARG;
    };
    rows(p->k, p->k_new_stride, c.heads, false);
    rows(p->v, p->v_new_stride, c.heads, false);
    if (p->q) {
        rows(p->q, p->q_stride, heads, false);
        rows(p->q_out, p->q_out_stride, heads, true);
        if (p->q == p->q_out && ((p->tokens > 1 && p->q_stride[0] != p->q_out_stride[0]) || (heads > 1 && p->q_stride[1] != p->q_out_stride[1])))
            return FA_ERR_INVALID_ARG;
    }
    if (rc != FA_OK) return rc;
    rule.columns(p->rotary_dim / 2);
    rule.columns(c.head_dim - p->rotary_dim);
    if (heads > 0x3fffffff - 2 * static_cast<long long>(c.heads)) return FA_ERR_TOO_LARGE;
    int sms = 0, major = 0;
    if ((rc = current_device(&sms, &major)) != FA_OK) return rc;
    if (major != 10) return FA_ERR_NOT_SM100;
    AppendArgs a = {};
    const int vec_bytes = rule.bytes();
    fill_rotation(&a.rot, p->inv_freq, p->rotary_dim, c.head_dim, p->amplitude, false, vec_bytes / 2, true);
    a.seq = {c.seqlens_k, c.cu_seqlens_q, c.batch, static_cast<int>(p->tokens)};
    a.page_table = c.page_table;
    a.table_stride = c.table_stride;
    a.table_width = c.table_width;
    a.num_pages = c.num_pages;
    while ((1 << a.page_shift) < c.page_size) ++a.page_shift;
    a.heads = heads;
    a.heads_k = c.heads;
    a.k = p->k;
    a.v = p->v;
    a.q = p->q;
    a.k_pages = c.k;
    a.v_pages = c.v;
    a.q_out = p->q_out;
    std::copy(p->k_new_stride, p->k_new_stride + 2, a.ks);
    std::copy(p->v_new_stride, p->v_new_stride + 2, a.vs);
    std::copy(p->q_stride, p->q_stride + 2, a.qs);
    std::copy(p->q_out_stride, p->q_out_stride + 2, a.qos);
    std::copy(c.k_stride, c.k_stride + 3, a.kps);
    std::copy(c.v_stride, c.v_stride + 3, a.vps);
    a.status = p->status;
    const int all = heads + 2 * c.heads;
    a.rows_per_thread = rows_a_thread(p->tokens, a.rot.groups, all, sms);
    const dim3 grid(static_cast<unsigned>((p->tokens + a.rot.rows_per_block - 1) / a.rot.rows_per_block),
                    static_cast<unsigned>((all + a.rows_per_thread - 1) / a.rows_per_thread));
    const bool inter = p->interleaved != 0;
    const auto kernel = c.dtype == FA_DTYPE_BF16 ? append_of<__nv_bfloat16>(vec_bytes, inter) : append_of<__half>(vec_bytes, inter);
    return launch_rows(kernel, grid, static_cast<cudaStream_t>(p->stream), &a) == cudaSuccess ? FA_OK : FA_ERR_CUDA;
}

}  // extern "C"
