// The call path of flash_attn_forward, and of the calls around a paged cache, on torch tensors: checks, output allocation, parameter block, stream and launch in
// one native function.  Successor of the host side of the reference's main() (src/main.cu:109-205) for callers whose memory
// torch owns.  A short call is bound by the host: [1,4,256,256,64] took 15.0 us a call through ctypes (two allocations through
// Python 5, argument handling 5, the library 4) and takes 6.1, of which the kernel is 4.8; a decode step over 1000 keys 16.4 and 6.6, of
// which the kernel is 5.1.  (On buffers seen before: a new one costs a tensor map each.)
#include <Python.h>
#include <ATen/ATen.h>
#include <ATen/core/grad_mode.h>
#include <c10/core/AutogradState.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <cuda_runtime_api.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <algorithm>
#include <cmath>
#include <cstring>
#include <optional>
#include "../../include/fa_b200.h"

namespace {

typedef int (*fwd_fn)(const fa_fwd_params*);
typedef size_t (*workspace_fn)(const fa_fwd_params*);
typedef int (*rotary_fn)(const fa_rotary_params*);
typedef int (*append_fn)(const fa_paged_append_params*);
typedef int (*paged_fn)(const fa_paged_fwd_params*);
typedef size_t (*paged_workspace_fn)(const fa_paged_fwd_params*);

// A Python error is set.
struct python_error_set {};

[[noreturn]] void value_error(const char* what) {
    PyErr_SetString(PyExc_ValueError, what);
    throw python_error_set();
}

// int(x), as the low bits that a C field of that width takes
unsigned long long bits_of(PyObject* x) {
    PyObject* n = PyLong_Check(x) ? Py_NewRef(x) : PyNumber_Long(x);
    if (!n) throw python_error_set();
    const unsigned long long v = PyLong_AsUnsignedLongLongMask(n);
    Py_DECREF(n);
    if (v == static_cast<unsigned long long>(-1) && PyErr_Occurred()) throw python_error_set();
    return v;
}
int int_of(PyObject* x) { return static_cast<int>(bits_of(x)); }
bool truth_of(PyObject* x) {
    const int t = PyObject_IsTrue(x);
    if (t < 0) throw python_error_set();
    return t != 0;
}
double float_of(PyObject* x) {
    if (PyFloat_CheckExact(x)) return PyFloat_AS_DOUBLE(x);
    PyObject* f = PyNumber_Float(x);
    if (!f) throw python_error_set();
    const double v = PyFloat_AS_DOUBLE(f);
    Py_DECREF(f);
    return v;
}
const at::Tensor& tensor_of(PyObject* x, const char* name) {
    if (!THPVariable_Check(x)) {
        PyErr_Format(PyExc_TypeError, "%s must be a tensor", name);
        throw python_error_set();
    }
    return THPVariable_Unpack(x);
}
// FA_DTYPE_* of a tensor that may be an output
int dtype_of(const at::Tensor& t) {
    switch (t.scalar_type()) {
        case at::kHalf: return FA_DTYPE_FP16;
        case at::kBFloat16: return FA_DTYPE_BF16;
        case at::kFloat: return FA_DTYPE_FP32;
        default:
            PyErr_Format(PyExc_KeyError, "no attention output of dtype %s", c10::toString(t.scalar_type()));
            throw python_error_set();
    }
}
bool same(at::IntArrayRef a, at::IntArrayRef b) { return a == b; }

// Kernels follow a pointer as it is, so memory that `device` does not reach is refused here.  A tensor on the device itself costs a
// comparison; pinned and managed host memory and an enabled peer's memory are reached too, which the runtime is asked about.
bool reaches(const c10::Device& device, const void* memory) {
    const c10::cuda::OptionalCUDAGuard guard(device);
    cudaPointerAttributes at;
    const bool known = cudaPointerGetAttributes(&at, memory) == cudaSuccess;
    if (!known) (void)cudaGetLastError();
    return known && at.devicePointer != nullptr;
}
void need_reach(const c10::Device& device, const at::Tensor& t, const char* name) {
    if (t.device() == device || t.numel() == 0 || reaches(device, t.data_ptr())) return;
    PyErr_Format(PyExc_ValueError, "%s must be on q's device, or in memory that this device reaches", name);
    throw python_error_set();
}

// (left, right) of whatever has two items
void window_of(PyObject* window, int* left, int* right) {
    for (int i = 0; i < 2; ++i) {
        PyObject* x;
        if (PyTuple_CheckExact(window) && PyTuple_GET_SIZE(window) > i) {
            x = Py_NewRef(PyTuple_GET_ITEM(window, i));
        } else {  // window[i] of whatever has items (a tensor is no sequence)
            PyObject* at = PyLong_FromLong(i);
            x = at ? PyObject_GetItem(window, at) : nullptr;
            Py_XDECREF(at);
        }
        if (!x) throw python_error_set();
        int w;
        try {
            w = int_of(x);
        } catch (...) {
            Py_DECREF(x);
            throw;
        }
        Py_DECREF(x);
        *(i == 0 ? left : right) = w;
    }
}

enum Arg {
    kFwd, kWorkspaceFn, kQ, kK, kV, kScale, kCausal, kWindow, kSlopes, kDropout, kSeed, kOffset, kSplits, kOut, kOutDtype,
    kReturnLse, kQPos0, kKPos0, kUnit0, kWorkspace, kStatus, kAccum, kAccumFirst, kAccumFinal, kLaunchIndex, kArgs
};

PyObject* forward_impl(PyObject* const* args) {
    const fwd_fn fwd = reinterpret_cast<fwd_fn>(bits_of(args[kFwd]));
    const workspace_fn workspace_bytes = reinterpret_cast<workspace_fn>(bits_of(args[kWorkspaceFn]));
    const at::Tensor &q = tensor_of(args[kQ], "q"), &k = tensor_of(args[kK], "k"), &v = tensor_of(args[kV], "v");
    if (!q.is_cuda()) value_error("flash_attn_forward needs CUDA tensors (use flash_attn_forward_host for host buffers)");
    if (q.dim() != 4) value_error("q must be [batch, heads, seqlen, head_dim]");
    const int64_t B = q.size(0), H = q.size(1), Nq = q.size(2), d = q.size(3);
    const c10::Device device = q.device();
    const bool accum = args[kAccum] != Py_None, accum_final = truth_of(args[kAccumFinal]);
    const bool writes_output = !accum || accum_final;
    at::Tensor out, lse;
    if (writes_output) {
        if (args[kOut] != Py_None) {
            out = tensor_of(args[kOut], "out");
        } else {
            at::ScalarType type = q.scalar_type();
            if (args[kOutDtype] != Py_None) {
                if (!THPDtype_Check(args[kOutDtype])) {
                    PyErr_SetString(PyExc_TypeError, "out_dtype must be a torch.dtype");
                    throw python_error_set();
                }
                type = reinterpret_cast<THPDtype*>(args[kOutDtype])->scalar_type;
            }
            out = at::empty({B, H, Nq, d}, q.options().dtype(type).layout(at::kStrided).requires_grad(false));
        }
        if (truth_of(args[kReturnLse])) lse = at::empty({B, H, Nq}, q.options().dtype(at::kFloat).layout(at::kStrided).requires_grad(false));
    }
    at::Tensor slopes;
    if (args[kSlopes] != Py_None) {
        slopes = tensor_of(args[kSlopes], "alibi_slopes").to(device, at::kFloat).contiguous();
        if (slopes.numel() < H) value_error("alibi_slopes must hold a slope for each head");
    }
    const at::Tensor& o = out.defined() ? out : q;
    if (k.dim() < 3) value_error("k and v must be [batch, heads_k, seqlen_k, head_dim] with heads a multiple of heads_k");
    const int64_t Hk = k.size(1), Nk = k.size(2);
    const int64_t kv[4] = {B, Hk, Nk, d};
    if (!same(k.sizes(), kv) || !same(v.sizes(), kv) || Hk < 1 || H % Hk != 0)
        value_error("k and v must be [batch, heads_k, seqlen_k, head_dim] with heads a multiple of heads_k");
    if (!(q.is_contiguous() && k.is_contiguous() && v.is_contiguous() && o.is_contiguous()))
        value_error("q, k, v, o must be contiguous [batch, heads, seqlen, head_dim]");
    const at::ScalarType type = q.scalar_type();
    if ((type != at::kHalf && type != at::kBFloat16) || k.scalar_type() != type || v.scalar_type() != type)
        value_error("q, k, v must share dtype float16 or bfloat16");
    // (an output of another shape is filled as [batch, heads, seqlen, head_dim] rows one behind the other: it has to hold them)
    if (o.numel() < q.numel()) value_error("out must hold [batch, heads, seqlen, head_dim]");
    need_reach(device, k, "k");
    need_reach(device, v, "v");
    need_reach(device, o, "out");

    fa_fwd_params p;
    std::memset(&p, 0, sizeof p);
    at::Tensor o_acc, lse_acc;
    if (accum) {
        PyObject* pair = PySequence_Fast(args[kAccum], "accum = (fp32 [B,H,Nq,d], fp32 [B,H,Nq]), contiguous");
        if (!pair) throw python_error_set();
        if (PySequence_Fast_GET_SIZE(pair) != 2) {
            Py_DECREF(pair);
            value_error("accum = (fp32 [B,H,Nq,d], fp32 [B,H,Nq]), contiguous");
        }
        PyObject *a = PySequence_Fast_GET_ITEM(pair, 0), *b = PySequence_Fast_GET_ITEM(pair, 1);
        const bool tensors = THPVariable_Check(a) && THPVariable_Check(b);
        if (tensors) {
            o_acc = THPVariable_Unpack(a);
            lse_acc = THPVariable_Unpack(b);
        }
        Py_DECREF(pair);
        const int64_t rows[4] = {B, H, Nq, d};
        if (!tensors || o_acc.scalar_type() != at::kFloat || lse_acc.scalar_type() != at::kFloat || !o_acc.is_contiguous() ||
            !lse_acc.is_contiguous() || !same(o_acc.sizes(), rows) || !same(lse_acc.sizes(), at::IntArrayRef(rows, 3)))
            value_error("accum = (fp32 [B,H,Nq,d], fp32 [B,H,Nq]), contiguous");
        need_reach(device, o_acc, "accum");
        need_reach(device, lse_acc, "accum");
        p.accum_o = static_cast<float*>(o_acc.data_ptr());
        p.accum_lse = static_cast<float*>(lse_acc.data_ptr());
        p.accum_flags = (truth_of(args[kAccumFirst]) ? FA_ACCUM_FIRST : 0) | (accum_final ? FA_ACCUM_FINAL : 0);
    }
    p.q = q.data_ptr();
    p.k = k.data_ptr();
    p.v = v.data_ptr();
    p.o = out.defined() ? out.data_ptr() : nullptr;
    p.lse = lse.defined() ? static_cast<float*>(lse.data_ptr()) : nullptr;
    p.dtype = dtype_of(q);
    p.o_dtype = dtype_of(o);
    p.batch = static_cast<int>(B);
    p.heads = static_cast<int>(H);
    p.heads_k = static_cast<int>(Hk);
    p.seqlen_q = static_cast<int>(Nq);
    p.seqlen_k = static_cast<int>(Nk);
    p.head_dim = static_cast<int>(d);
    if (args[kScale] != Py_None) {
        p.softmax_scale = static_cast<float>(float_of(args[kScale]));
    } else {
        if (d == 0) {
            PyErr_SetString(PyExc_ZeroDivisionError, "float division by zero");
            throw python_error_set();
        }
        p.softmax_scale = static_cast<float>(1.0 / std::sqrt(static_cast<double>(d)));
    }
    p.is_causal = truth_of(args[kCausal]) ? 1 : 0;
    window_of(args[kWindow], &p.window_left, &p.window_right);
    p.alibi_slopes = slopes.defined() ? static_cast<const float*>(slopes.data_ptr()) : nullptr;
    p.p_dropout = static_cast<float>(float_of(args[kDropout]));
    p.seed = bits_of(args[kSeed]);
    p.offset = bits_of(args[kOffset]);
    p.unit0 = bits_of(args[kUnit0]);
    p.launch_index = bits_of(args[kLaunchIndex]);
    p.num_splits = int_of(args[kSplits]);
    p.q_pos0 = static_cast<int64_t>(bits_of(args[kQPos0]));
    p.k_pos0 = static_cast<int64_t>(bits_of(args[kKPos0]));
    if (args[kStatus] != Py_None) {
        const at::Tensor& status = tensor_of(args[kStatus], "status");
        if (status.nbytes() < sizeof(int) || reinterpret_cast<uintptr_t>(status.data_ptr()) % sizeof(int) != 0)
            value_error("status must hold an aligned 32-bit word");
        need_reach(device, status, "status");
        p.status = static_cast<int*>(status.data_ptr());
    }

    const c10::cuda::OptionalCUDAGuard guard(device);  // (nothing where the device is the current one)
    at::Tensor workspace;
    if (p.num_splits != 1 || d % 8 != 0) {
        const size_t need = workspace_bytes(&p);
        if (need != 0) {
            if (args[kWorkspace] != Py_None) workspace = tensor_of(args[kWorkspace], "workspace");
            // (of a tensor that is not contiguous the byte count says nothing about the memory behind its first element)
            if (!workspace.defined() || workspace.nbytes() < need || !workspace.is_contiguous())
                workspace = at::empty({static_cast<int64_t>(need)}, at::TensorOptions().device(device).dtype(at::kByte));
            else
                need_reach(device, workspace, "workspace");
            p.workspace = workspace.data_ptr();
            p.workspace_bytes = workspace.nbytes();
        }
    }
    p.stream = c10::cuda::getCurrentCUDAStream(device.index()).stream();
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = fwd(&p);
    Py_END_ALLOW_THREADS
    if (rc != FA_OK) return PyLong_FromLong(rc);
    PyObject* first = !out.defined() ? Py_NewRef(Py_None) : args[kOut] != Py_None ? Py_NewRef(args[kOut]) : THPVariable_Wrap(std::move(out));
    PyObject* second = !lse.defined() ? Py_NewRef(Py_None) : THPVariable_Wrap(std::move(lse));
    PyObject* both = first && second ? PyTuple_Pack(2, first, second) : nullptr;
    Py_XDECREF(first);
    Py_XDECREF(second);
    return both;
}

// forward(address of fa_fwd, address of fa_fwd_workspace_bytes, the arguments of flash_attn_forward in order): (out, lse), or
// the library's error code.
PyObject* forward(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != kArgs) {
        PyErr_Format(PyExc_TypeError, "forward takes %d arguments, got %zd", static_cast<int>(kArgs), n);
        return nullptr;
    }
    try {
        return forward_impl(args);
    } catch (const python_error_set&) {
        return nullptr;
    }
    END_HANDLE_TH_ERRORS
}

// ---------------------------------------------------------------- rotary positions and the paged cache

[[noreturn]] void value_error_of(const char* name, const char* what) {
    PyErr_Format(PyExc_ValueError, "%s %s", name, what);
    throw python_error_set();
}
// The kernels are not recorded by autograd: a gradient or a tangent that would be lost in silence is refused.
void need_no_grad(const at::Tensor& t, const char* name) {
    if (c10::AutogradState::get_tls_state().get_fw_grad_mode() && t._fw_grad(0).defined()) value_error_of(name, "has a forward-mode tangent: unpack it first");
    if (t.requires_grad() && at::GradMode::is_enabled()) value_error_of(name, "requires grad: call this under torch.no_grad() or inside an autograd Function");
}
// A caller's tensor was written to: autograd's check of what it has saved is told, as torch's own calls do (under no_grad too).
void written(const at::Tensor& t) {
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}
// float(x) of a number or a tensor of one
double number_of(PyObject* x, const char* name) {
    if (THPVariable_Check(x)) need_no_grad(THPVariable_Unpack(x), name);
    return float_of(x);
}
bool sixteen_bit(const at::Tensor& t) { return t.scalar_type() == at::kHalf || t.scalar_type() == at::kBFloat16; }
void need_rows(const at::Tensor& t, const char* name) {
    if (t.size(-1) > 1 && t.stride(-1) != 1) value_error_of(name, "must be contiguous in its last dimension");
}
// What the device is told of an int32 tensor that it reads: one piece, on the device.
const int* ints(const at::Tensor& t, int64_t n, const c10::Device& device, const char* name, const char* what) {
    if (t.scalar_type() != at::kInt || t.dim() != 1 || t.size(0) != n || !t.is_contiguous()) value_error_of(name, what);
    need_reach(device, t, name);
    return static_cast<const int*>(t.data_ptr());
}
int* status_of(PyObject* x, const c10::Device& device) {
    if (x == Py_None) return nullptr;
    const at::Tensor& status = tensor_of(x, "status");
    if (status.nbytes() < sizeof(int) || reinterpret_cast<uintptr_t>(status.data_ptr()) % sizeof(int) != 0)
        value_error("status must hold an aligned 32-bit word");
    need_reach(device, status, "status");
    return static_cast<int*>(status.data_ptr());
}
int narrow_int(int64_t x) {
    if (x > 0x7fffffff) value_error("a size is beyond 31 bits");
    return static_cast<int>(x);
}

// rotary(address of fa_rotary, x, positions, inv_freq, amplitude, interleaved, inverse, out): out, or the library's error code.
PyObject* rotary_impl(PyObject* const* args) {
    const rotary_fn rotary = reinterpret_cast<rotary_fn>(bits_of(args[0]));
    const at::Tensor &x = tensor_of(args[1], "x"), &positions = tensor_of(args[2], "positions"), &inv_freq = tensor_of(args[3], "inv_freq");
    if (!x.is_cuda()) value_error("rotary_embedding needs CUDA tensors");
    if (x.dim() != 3 && x.dim() != 4) value_error("x must be [batch, heads, seqlen, head_dim] or [tokens, heads, head_dim]");
    if (!sixteen_bit(x) && x.scalar_type() != at::kFloat) value_error("x must be float16, bfloat16 or float32");
    need_no_grad(x, "x");
    need_rows(x, "x");
    const c10::Device device = x.device();
    const c10::cuda::OptionalCUDAGuard guard(device);
    const bool packed = x.dim() == 3;
    const int64_t B = packed ? 1 : x.size(0), H = x.size(1), N = packed ? x.size(0) : x.size(2), d = x.size(-1);
    if (positions.scalar_type() != at::kInt && positions.scalar_type() != at::kLong) value_error("positions must be int32 or int64");
    const bool one = positions.dim() == 1 && positions.size(0) == N;
    const bool each = !packed && positions.dim() == 2 && positions.size(0) == B && positions.size(1) == N;
    if ((!one && !each) || (N > 1 && positions.stride(-1) != 1)) value_error("positions must be [seqlen] or [batch, seqlen] ([tokens]), one behind the other");
    if (inv_freq.scalar_type() != at::kDouble || inv_freq.dim() != 1 || !inv_freq.is_contiguous() || inv_freq.numel() < 1 || 2 * inv_freq.numel() > d)
        value_error("inv_freq must be float64 [rotary_dim / 2], rotary_dim at most head_dim");
    need_no_grad(inv_freq, "inv_freq");
    need_reach(device, positions, "positions");
    need_reach(device, inv_freq, "inv_freq");
    at::Tensor out;
    if (args[7] != Py_None) {
        out = tensor_of(args[7], "out");
        if (!same(out.sizes(), x.sizes()) || out.scalar_type() != x.scalar_type()) value_error("out must have x's shape and dtype");
        need_rows(out, "out");
        need_no_grad(out, "out");
        need_reach(device, out, "out");
    } else {
        out = at::empty(x.sizes(), x.options().layout(at::kStrided).requires_grad(false));
    }
    fa_rotary_params p;
    std::memset(&p, 0, sizeof p);
    p.x = x.data_ptr();
    p.y = out.data_ptr();
    p.dtype = dtype_of(x);
    p.batch = narrow_int(B);
    p.heads = narrow_int(H);
    p.rows = narrow_int(N);
    p.head_dim = narrow_int(d);
    p.rotary_dim = static_cast<int>(2 * inv_freq.numel());
    const at::Tensor* both[2] = {&x, &out};
    int64_t* strides[2] = {p.x_stride, p.y_stride};
    for (int i = 0; i < 2; ++i) {
        strides[i][0] = packed ? 0 : both[i]->stride(0);
        strides[i][1] = both[i]->stride(1);
        strides[i][2] = both[i]->stride(packed ? 0 : 2);
    }
    p.positions = positions.data_ptr();
    p.positions_64 = positions.scalar_type() == at::kLong;
    p.position_stride = each ? positions.stride(0) : 0;
    p.inv_freq = static_cast<const double*>(inv_freq.data_ptr());
    p.amplitude = static_cast<float>(number_of(args[4], "amplitude"));
    p.interleaved = truth_of(args[5]) ? 1 : 0;
    p.inverse = truth_of(args[6]) ? 1 : 0;
    p.stream = c10::cuda::getCurrentCUDAStream(device.index()).stream();
    if (x.numel() != 0) {
        int rc;
        Py_BEGIN_ALLOW_THREADS
        rc = rotary(&p);
        Py_END_ALLOW_THREADS
        if (rc != FA_OK) return PyLong_FromLong(rc);
        written(out);
    }
    return args[7] != Py_None ? Py_NewRef(args[7]) : THPVariable_Wrap(std::move(out));
}

// The cache of a call: args k_pages, v_pages, page_table, seqlens_k, cu_seqlens_q.
fa_paged_kv cache_of(PyObject* const* args, const at::Tensor& rows, const c10::Device& device) {
    const at::Tensor &k = tensor_of(args[0], "k_pages"), &v = tensor_of(args[1], "v_pages"), &table = tensor_of(args[2], "page_table"),
                     &lens = tensor_of(args[3], "seqlens_k");
    if (k.dim() != 4 || !same(k.sizes(), v.sizes())) value_error("k_pages and v_pages must be [num_pages, heads_k, page_size, head_dim]");
    if (!sixteen_bit(k) || k.scalar_type() != v.scalar_type() || rows.scalar_type() != k.scalar_type())
        value_error("the new tokens and the pages must share dtype float16 or bfloat16");
    if (rows.size(2) != k.size(3)) value_error("the new tokens and the pages must have one head_dim");
    need_no_grad(k, "k_pages");
    need_no_grad(v, "v_pages");
    need_rows(k, "k_pages");
    need_rows(v, "v_pages");
    if (table.scalar_type() != at::kInt || table.dim() != 2 || (table.size(1) > 1 && table.stride(1) != 1))
        value_error("page_table must be int32 [batch, pages], a row in one piece");
    need_reach(device, k, "k_pages");
    need_reach(device, v, "v_pages");
    need_reach(device, table, "page_table");
    fa_paged_kv c;
    std::memset(&c, 0, sizeof c);
    c.k = k.data_ptr();
    c.v = v.data_ptr();
    c.dtype = dtype_of(k);
    c.num_pages = narrow_int(k.size(0));
    c.heads = narrow_int(k.size(1));
    c.page_size = narrow_int(k.size(2));
    c.head_dim = narrow_int(k.size(3));
    for (int i = 0; i < 3; ++i) {
        c.k_stride[i] = k.stride(i);
        c.v_stride[i] = v.stride(i);
    }
    c.page_table = static_cast<const int*>(table.data_ptr());
    c.table_stride = table.stride(0);
    c.table_width = narrow_int(table.size(1));
    c.batch = narrow_int(table.size(0));
    c.seqlens_k = ints(lens, c.batch, device, "seqlens_k", "must be int32 [batch], contiguous");
    if (args[4] != Py_None) c.cu_seqlens_q = ints(tensor_of(args[4], "cu_seqlens_q"), static_cast<int64_t>(c.batch) + 1, device, "cu_seqlens_q", "must be int32 [batch + 1], contiguous");
    else if (rows.size(0) != c.batch) value_error("without cu_seqlens_q there is one new token a sequence");
    return c;
}

enum AppendArg { kAppendFn, kNewK, kNewV, kAppendCache, kNewQ = kAppendCache + 5, kInvFreq, kAmplitude, kInterleaved, kQOut, kAppendStatus, kAppendArgs };

// append(address of fa_paged_append, the arguments of paged_kv_append in order): Q turned, None, or the library's error code.
PyObject* append_impl(PyObject* const* args) {
    const append_fn append = reinterpret_cast<append_fn>(bits_of(args[kAppendFn]));
    const at::Tensor &k = tensor_of(args[kNewK], "k"), &v = tensor_of(args[kNewV], "v");
    if (!k.is_cuda()) value_error("paged_kv_append needs CUDA tensors");
    if (k.dim() != 3 || !same(k.sizes(), v.sizes()) || k.scalar_type() != v.scalar_type()) value_error("k and v must be [tokens, heads_k, head_dim] of one dtype");
    need_no_grad(k, "k");
    need_no_grad(v, "v");
    need_rows(k, "k");
    need_rows(v, "v");
    const c10::Device device = k.device();
    const c10::cuda::OptionalCUDAGuard guard(device);
    need_reach(device, v, "v");
    fa_paged_append_params p;
    std::memset(&p, 0, sizeof p);
    p.cache = cache_of(args + kAppendCache, k, device);
    if (k.size(1) != p.cache.heads) value_error("k and v must have the heads of the pages");
    p.k = k.data_ptr();
    p.v = v.data_ptr();
    p.tokens = k.size(0);
    for (int i = 0; i < 2; ++i) {
        p.k_new_stride[i] = k.stride(i);
        p.v_new_stride[i] = v.stride(i);
    }
    if (args[kInvFreq] != Py_None) {
        const at::Tensor& f = tensor_of(args[kInvFreq], "inv_freq");
        if (f.scalar_type() != at::kDouble || f.dim() != 1 || !f.is_contiguous() || f.numel() < 1 || 2 * f.numel() > k.size(2))
            value_error("inv_freq must be float64 [rotary_dim / 2], rotary_dim at most head_dim");
        need_no_grad(f, "inv_freq");
        need_reach(device, f, "inv_freq");
        p.inv_freq = static_cast<const double*>(f.data_ptr());
        p.rotary_dim = static_cast<int>(2 * f.numel());
    }
    at::Tensor out;
    if (args[kNewQ] != Py_None) {
        const at::Tensor& q = tensor_of(args[kNewQ], "q");
        if (!p.inv_freq) value_error("q is only turned: it needs inv_freq");
        if (q.dim() != 3 || q.size(0) != k.size(0) || q.size(2) != k.size(2) || q.scalar_type() != k.scalar_type())
            value_error("q must be [tokens, heads, head_dim] of k's dtype");
        need_no_grad(q, "q");
        need_rows(q, "q");
        need_reach(device, q, "q");
        if (args[kQOut] != Py_None) {
            out = tensor_of(args[kQOut], "out");
            if (!same(out.sizes(), q.sizes()) || out.scalar_type() != q.scalar_type()) value_error("out must have q's shape and dtype");
            need_no_grad(out, "out");
            need_rows(out, "out");
            need_reach(device, out, "out");
        } else {
            out = at::empty(q.sizes(), q.options().layout(at::kStrided).requires_grad(false));
        }
        p.q = q.data_ptr();
        p.q_out = out.data_ptr();
        p.heads = narrow_int(q.size(1));
        for (int i = 0; i < 2; ++i) {
            p.q_stride[i] = q.stride(i);
            p.q_out_stride[i] = out.stride(i);
        }
    } else if (args[kQOut] != Py_None) {
        value_error("out is for q");
    }
    p.amplitude = static_cast<float>(number_of(args[kAmplitude], "amplitude"));
    p.interleaved = truth_of(args[kInterleaved]) ? 1 : 0;
    p.status = status_of(args[kAppendStatus], device);
    p.stream = c10::cuda::getCurrentCUDAStream(device.index()).stream();
    if (k.numel() != 0 || (out.defined() && out.numel() != 0)) {  // (pages without heads are refused where there is a Q to turn)
        int rc;
        Py_BEGIN_ALLOW_THREADS
        rc = append(&p);
        Py_END_ALLOW_THREADS
        if (rc != FA_OK) return PyLong_FromLong(rc);
        for (int i = 0; i < 2; ++i) written(THPVariable_Unpack(args[kAppendCache + i]));
        if (out.defined()) written(out);
    }
    return !out.defined() ? Py_NewRef(Py_None) : args[kQOut] != Py_None ? Py_NewRef(args[kQOut]) : THPVariable_Wrap(std::move(out));
}

enum PagedArg {
    kPagedFn, kPagedWorkspaceFn, kPagedQ, kPagedCache, kMaxSeqlenQ = kPagedCache + 5, kPagedScale, kPagedCausal, kPagedWindow, kPagedSlopes,
    kPagedOut, kPagedOutDtype, kPagedReturnLse, kPagedWorkspace, kPagedStatus, kPagedArgs
};

// paged(address of fa_paged_fwd, address of fa_paged_fwd_workspace_bytes, the arguments of paged_attn_forward in order): (out, lse),
// or the library's error code.
PyObject* paged_impl(PyObject* const* args) {
    const paged_fn fwd = reinterpret_cast<paged_fn>(bits_of(args[kPagedFn]));
    const paged_workspace_fn workspace_bytes = reinterpret_cast<paged_workspace_fn>(bits_of(args[kPagedWorkspaceFn]));
    at::Tensor q = tensor_of(args[kPagedQ], "q");
    if (!q.is_cuda()) value_error("paged_attn_forward needs CUDA tensors");
    if (q.dim() != 3) value_error("q must be [tokens, heads, head_dim]");
    need_no_grad(q, "q");
    need_rows(q, "q");
    const c10::Device device = q.device();
    const c10::cuda::OptionalCUDAGuard guard(device);
    const int64_t T = q.size(0), H = q.size(1), d = q.size(2);
    if ((T > 1 && q.stride(0) == 0) || (H > 1 && q.stride(1) == 0)) q = q.contiguous();  // (broadcast rows: the chunk kernel takes none)
    fa_paged_fwd_params p;
    std::memset(&p, 0, sizeof p);
    p.cache = cache_of(args + kPagedCache, q, device);
    if (p.cache.heads < 1 || H < 1 || H % p.cache.heads != 0) value_error("q's heads must be a multiple of the pages'");
    at::Tensor out, lse, slopes;
    if (args[kPagedOut] != Py_None) {
        out = tensor_of(args[kPagedOut], "out");
        if (!same(out.sizes(), q.sizes())) value_error("out must have q's shape");
        need_no_grad(out, "out");
        need_rows(out, "out");
        need_reach(device, out, "out");
    } else {
        at::ScalarType type = q.scalar_type();
        if (args[kPagedOutDtype] != Py_None) {
            if (!THPDtype_Check(args[kPagedOutDtype])) {
                PyErr_SetString(PyExc_TypeError, "out_dtype must be a torch.dtype");
                throw python_error_set();
            }
            type = reinterpret_cast<THPDtype*>(args[kPagedOutDtype])->scalar_type;
        }
        out = at::empty({T, H, d}, q.options().dtype(type).layout(at::kStrided).requires_grad(false));
    }
    if (truth_of(args[kPagedReturnLse])) lse = at::empty({T, H}, q.options().dtype(at::kFloat).layout(at::kStrided).requires_grad(false));
    if (args[kPagedSlopes] != Py_None) {
        need_no_grad(tensor_of(args[kPagedSlopes], "alibi_slopes"), "alibi_slopes");
        slopes = tensor_of(args[kPagedSlopes], "alibi_slopes").to(device, at::kFloat).contiguous();
        if (slopes.numel() < H) value_error("alibi_slopes must hold a slope for each head");
    }
    p.q = q.data_ptr();
    p.o = out.data_ptr();
    p.lse = lse.defined() ? static_cast<float*>(lse.data_ptr()) : nullptr;
    p.o_dtype = dtype_of(out);
    p.heads = narrow_int(H);
    p.tokens = T;
    for (int i = 0; i < 2; ++i) {
        p.q_stride[i] = q.stride(i);
        p.o_stride[i] = out.stride(i);
    }
    // (unsaid: as many as there are rows, or one)
    p.max_seqlen_q = args[kMaxSeqlenQ] != Py_None ? int_of(args[kMaxSeqlenQ]) : p.cache.cu_seqlens_q ? narrow_int(std::max<int64_t>(T, 1)) : 1;
    p.softmax_scale = static_cast<float>(args[kPagedScale] != Py_None ? number_of(args[kPagedScale], "softmax_scale") : 1.0 / std::sqrt(static_cast<double>(std::max<int64_t>(d, 1))));
    p.is_causal = truth_of(args[kPagedCausal]) ? 1 : 0;
    window_of(args[kPagedWindow], &p.window_left, &p.window_right);
    p.alibi_slopes = slopes.defined() ? static_cast<const float*>(slopes.data_ptr()) : nullptr;
    p.status = status_of(args[kPagedStatus], device);
    p.stream = c10::cuda::getCurrentCUDAStream(device.index()).stream();
    if (q.numel() != 0) {
        at::Tensor workspace;
        const size_t need = workspace_bytes(&p);
        if (need != 0) {
            if (args[kPagedWorkspace] != Py_None) workspace = tensor_of(args[kPagedWorkspace], "workspace");
            if (!workspace.defined() || workspace.nbytes() < need || !workspace.is_contiguous())
                workspace = at::empty({static_cast<int64_t>(need)}, at::TensorOptions().device(device).dtype(at::kByte));
            else
                need_reach(device, workspace, "workspace");
            p.workspace = workspace.data_ptr();
            p.workspace_bytes = workspace.nbytes();
        }
        int rc;
        Py_BEGIN_ALLOW_THREADS
        rc = fwd(&p);
        Py_END_ALLOW_THREADS
        if (rc != FA_OK) return PyLong_FromLong(rc);
        written(out);
    }
    PyObject* first = args[kPagedOut] != Py_None ? Py_NewRef(args[kPagedOut]) : THPVariable_Wrap(std::move(out));
    PyObject* second = !lse.defined() ? Py_NewRef(Py_None) : THPVariable_Wrap(std::move(lse));
    PyObject* both = first && second ? PyTuple_Pack(2, first, second) : nullptr;
    Py_XDECREF(first);
    Py_XDECREF(second);
    return both;
}

// A function of kCount positional arguments, with C++ and Python errors as Python has them.
template <PyObject* (*kImpl)(PyObject* const*), int kCount>
PyObject* entry(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != kCount) {
        PyErr_Format(PyExc_TypeError, "%d arguments are wanted, got %zd", kCount, n);
        return nullptr;
    }
    try {
        return kImpl(args);
    } catch (const python_error_set&) {
        return nullptr;
    }
    END_HANDLE_TH_ERRORS
}

PyMethodDef methods[] = {
    {"forward", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(forward)), METH_FASTCALL, nullptr},
    {"rotary", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(entry<rotary_impl, 8>)), METH_FASTCALL, nullptr},
    {"append", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(entry<append_impl, kAppendArgs>)), METH_FASTCALL, nullptr},
    {"paged", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(entry<paged_impl, kPagedArgs>)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_call", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__call() {
    PyObject* m = PyModule_Create(&module);
    if (m && PyModule_AddStringConstant(m, "built_for", FA_BUILT_FOR) != 0) {  // (torch's version: other versions have other classes)
        Py_DECREF(m);
        return nullptr;
    }
    return m;
}
