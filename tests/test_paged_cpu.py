"""The calls around a paged cache, as far as they go without a GPU: the ABI's structs, frequencies, refusals of the C entries."""
import ctypes
import math
import os
import subprocess
import tempfile

import pytest

from flash_attn_b200 import _lib, rotary_frequencies

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def lib():
    from flash_attn_b200 import build
    build.build()
    return _lib.load()


@pytest.mark.parametrize("name, mirror", [("fa_paged_kv", _lib.PagedKv), ("fa_rotary_params", _lib.RotaryParams),
                                          ("fa_paged_append_params", _lib.PagedAppendParams), ("fa_paged_fwd_params", _lib.PagedFwdParams)])
def test_struct_layouts_match_the_header(name, mirror):
    fields = [f[0] for f in mirror._fields_]
    src = f'#include <stdio.h>\n#include <stddef.h>\n#include "fa_b200.h"\nint main(void){{printf("%zu", sizeof({name}));\n'
    src += "".join(f'printf(" %zu", offsetof({name}, {f}));\n' for f in fields) + "return 0;}\n"
    with tempfile.TemporaryDirectory() as tmp:
        c, exe = os.path.join(tmp, "layout.c"), os.path.join(tmp, "layout")
        open(c, "w").write(src)
        subprocess.check_call(["gcc", "-std=c99", "-I", os.path.join(ROOT, "include"), c, "-o", exe])
        out = [int(x) for x in subprocess.check_output([exe]).split()]
    assert out == [ctypes.sizeof(mirror)] + [getattr(mirror, f).offset for f in fields]


# ------------------------------------------------------------------ frequencies
def test_frequencies_are_the_formulas(lib):
    n, base, f, length = 64, 10000.0, 8.0, 4096
    plain = [base ** (-2 * i / n) for i in range(n // 2)]
    near = lambda got, want: all(abs(a - b) <= 1e-14 * abs(b) for a, b in zip(got.tolist(), want)) and len(got) == len(want)  # noqa: E731
    got, t = rotary_frequencies(n, device="cpu")
    assert near(got, plain) and t == 1.0 and str(got.dtype) == "torch.float64"
    got, t = rotary_frequencies(n, scaling="linear", factor=f, device="cpu")
    assert near(got, [w / f for w in plain]) and t == 1.0
    got, t = rotary_frequencies(n, scaling="ntk", factor=f, device="cpu")
    assert near(got, [(base * f ** (n / (n - 2))) ** (-2 * i / n) for i in range(n // 2)]) and t == 1.0
    # the slowest pair turns exactly `factor` slower, the fastest as before
    assert abs(got[-1].item() * f / plain[-1] - 1) < 1e-12 and got[0].item() == 1.0
    got, t = rotary_frequencies(n, scaling="ramp", factor=f, original_length=length, low_turns=1, high_turns=4, device="cpu")
    want = []
    for w in plain:
        turns = length * w / (2 * math.pi)
        keep = 0.0 if turns <= 1 else 1.0 if turns >= 4 else (turns - 1) / 3
        want.append(w * keep + w / f * (1 - keep))
    assert near(got, want) and abs(t - (0.1 * math.log(f) + 1)) < 1e-15


@pytest.mark.parametrize("kw", [dict(rotary_dim=0), dict(rotary_dim=7), dict(rotary_dim=8, scaling="other"), dict(rotary_dim=8, scaling="ramp")])
def test_frequencies_refuse(lib, kw):
    with pytest.raises(ValueError):
        rotary_frequencies(device="cpu", **kw)


@pytest.mark.parametrize("kw", [dict(rotary_dim=8, base=0.0), dict(rotary_dim=8, base=math.inf), dict(rotary_dim=8, scaling="linear", factor=0.0),
                                dict(rotary_dim=8, scaling="linear", factor=math.nan), dict(rotary_dim=2, scaling="ntk", factor=2.0),
                                dict(rotary_dim=8, scaling="ramp", original_length=0), dict(rotary_dim=8, scaling="ramp", original_length=64, low_turns=4, high_turns=4)])
def test_frequencies_refuse_numbers(lib, kw):
    with pytest.raises(_lib.FaError):
        rotary_frequencies(device="cpu", **kw)


# ------------------------------------------------------------------ refusals: no pointer below is ever followed
def cache(c=None):
    c = c if c is not None else _lib.PagedKv()
    c.k, c.v, c.page_table, c.seqlens_k, c.cu_seqlens_q = 4096, 8192, 1024, 1024, 1024
    c.dtype, c.num_pages, c.page_size, c.heads, c.head_dim, c.batch, c.table_width, c.table_stride = 1, 10, 16, 8, 128, 4, 5, 5
    for s in (c.k_stride, c.v_stride):
        s[0], s[1], s[2] = 8 * 16 * 128, 16 * 128, 128
    return c


def fwd_params():
    p = _lib.PagedFwdParams()
    cache(p.cache)
    p.q, p.o, p.o_dtype, p.heads, p.tokens, p.max_seqlen_q, p.softmax_scale = 4096, 4096, 1, 32, 4, 1, 1.0
    p.window_left = p.window_right = -1
    for s in (p.q_stride, p.o_stride):
        s[0], s[1] = 32 * 128, 128
    return p


def append_params():
    p = _lib.PagedAppendParams()
    cache(p.cache)
    p.k, p.v, p.q, p.q_out, p.tokens, p.heads, p.rotary_dim, p.inv_freq, p.amplitude = 4096, 4096, 4096, 8192, 4, 32, 128, 4096, 1.0
    for s in (p.k_new_stride, p.v_new_stride):
        s[0], s[1] = 8 * 128, 128
    for s in (p.q_stride, p.q_out_stride):
        s[0], s[1] = 32 * 128, 128
    return p


def rotary_params():
    p = _lib.RotaryParams()
    p.x, p.y, p.dtype, p.batch, p.heads, p.rows, p.head_dim, p.rotary_dim = 4096, 8192, 1, 2, 4, 6, 128, 64
    for s in (p.x_stride, p.y_stride):
        s[0], s[1], s[2] = 4 * 6 * 128, 6 * 128, 128
    p.positions, p.inv_freq, p.amplitude = 4096, 4096, 1.0
    return p


BAD_CACHE = [("k", None, -1), ("v", None, -1), ("page_table", None, -1), ("seqlens_k", None, -1), ("k", 4100, -1), ("page_table", 1026, -1),
             ("dtype", 2, -2), ("dtype", 7, -2), ("num_pages", 0, -1), ("page_size", 0, -1), ("page_size", 4, -2), ("page_size", 48, -2),
             ("heads", 0, -1), ("head_dim", 136, -2), ("head_dim", 100, -2), ("batch", 0, -1), ("table_width", 0, -1), ("table_stride", 4, -1)]


@pytest.mark.parametrize("entry, make", [("fa_paged_fwd", fwd_params), ("fa_paged_append", append_params)])
@pytest.mark.parametrize("field, value, code", BAD_CACHE)
def test_a_cache_that_cannot_be_followed_is_refused(lib, entry, make, field, value, code):
    p = make()
    setattr(p.cache, field, value)
    assert getattr(lib, entry)(ctypes.byref(p)) == code


@pytest.mark.parametrize("entry, make", [("fa_paged_fwd", fwd_params), ("fa_paged_append", append_params)])
def test_pages_that_overlap_or_stand_askew_are_refused(lib, entry, make):
    call = lambda p: getattr(lib, entry)(ctypes.byref(p))  # noqa: E731
    for i, value in ((0, 8 * 16 * 128 - 8), (1, 16 * 128 - 8), (2, 120), (2, 132), (0, 0), (1, -128)):
        for name in ("k_stride", "v_stride"):
            p = make()
            getattr(p.cache, name)[i] = value
            assert call(p) == -1, (name, i, value)
    p = make()
    p.cache.v_stride[0] = 1 << 40
    assert call(p) == -7
    p = make()
    p.cache.cu_seqlens_q = None
    p.tokens = 3  # a row for each of four sequences is wanted
    assert call(p) == -1
    p = make()
    p.tokens = 1 << 31
    assert call(p) == -7
    assert getattr(lib, entry)(None) == -1


@pytest.mark.parametrize("field, value, code", [
    ("q", None, -1), ("o", None, -1), ("q", 4104, -1), ("o", 4104, -1), ("o_dtype", 0, -2), ("heads", 0, -1), ("heads", 12, -1),
    ("softmax_scale", 0.0, -1), ("softmax_scale", math.nan, -1), ("softmax_scale", math.inf, -1), ("window_left", -2, -1), ("window_right", -3, -1),
    ("max_seqlen_q", 0, -1), ("lse", 4097, -1), ("alibi_slopes", 4098, -1), ("status", 4098, -1)])
def test_attention_refuses(lib, field, value, code):
    p = fwd_params()
    setattr(p, field, value)
    assert lib.fa_paged_fwd(ctypes.byref(p)) == code
    assert lib.fa_paged_fwd_workspace_bytes(ctypes.byref(p)) == 0


def test_attention_refuses_rows_and_groups(lib):
    p = fwd_params()
    p.q_stride[1] = 132
    assert lib.fa_paged_fwd(ctypes.byref(p)) == -1
    p = fwd_params()
    p.o_stride[0] = 31 * 128  # rows of the output that overlap
    assert lib.fa_paged_fwd(ctypes.byref(p)) == -1
    p = fwd_params()
    p.heads = 8 * 129
    p.q_stride[0] = p.o_stride[0] = 8 * 129 * 128
    assert lib.fa_paged_fwd(ctypes.byref(p)) == -2


@pytest.mark.parametrize("field, value, code", [
    ("k", None, -1), ("v", None, -1), ("k", 4097, -1), ("q_out", None, -1), ("q_out", 8193, -1), ("heads", 0, -1), ("inv_freq", None, -1),
    ("inv_freq", 4100, -1), ("rotary_dim", 0, -1), ("rotary_dim", 7, -1), ("rotary_dim", 130, -1), ("amplitude", math.nan, -1)])
def test_append_refuses(lib, field, value, code):
    p = append_params()
    setattr(p, field, value)
    assert lib.fa_paged_append(ctypes.byref(p)) == code


def test_append_refuses_aliased_rows(lib):
    p = append_params()
    p.q_out_stride[0] = 31 * 128
    assert lib.fa_paged_append(ctypes.byref(p)) == -1
    p = append_params()
    p.q_out, p.q_out_stride[0] = p.q, 33 * 128  # in place, but at other places
    assert lib.fa_paged_append(ctypes.byref(p)) == -1


@pytest.mark.parametrize("field, value, code", [
    ("x", None, -1), ("y", None, -1), ("positions", None, -1), ("x", 4097, -1), ("positions", 4098, -1), ("inv_freq", None, -1), ("inv_freq", 4100, -1),
    ("dtype", 3, -2), ("batch", 0, -1), ("heads", 0, -1), ("rows", 0, -1), ("head_dim", 264, -2), ("rotary_dim", 0, -1), ("rotary_dim", 63, -1),
    ("rotary_dim", 130, -1), ("amplitude", math.inf, -1)])
def test_rotary_refuses(lib, field, value, code):
    p = rotary_params()
    setattr(p, field, value)
    assert lib.fa_rotary(ctypes.byref(p)) == code


def test_rotary_refuses_rows_that_overlap(lib):
    p = rotary_params()
    p.y_stride[2] = 0
    assert lib.fa_rotary(ctypes.byref(p)) == -1
    p = rotary_params()
    p.y, p.x_stride[1] = p.x, 7 * 128
    assert lib.fa_rotary(ctypes.byref(p)) == -1
    p = rotary_params()
    p.x_stride[0] = -1
    assert lib.fa_rotary(ctypes.byref(p)) == -1
