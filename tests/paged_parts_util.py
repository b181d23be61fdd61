"""The test build's view of how a launch over the paged cache is shared out (fa_test_paged_parts)."""
import ctypes
import os

import torch

FIELDS = ["b", "head", "first", "n", "keys", "row0", "n_rows", "part", "parts", "slot", "lo", "n_tiles", "vis_lo", "vis_hi"]


def test_library():
    from flash_attn_b200 import _lib, build
    path = build.TEST_LIB
    if not os.path.exists(path):
        path = build.build_test_variant()
    L = ctypes.CDLL(path)
    L.fa_test_paged_parts.argtypes = [ctypes.POINTER(_lib.PagedFwdParams), ctypes.c_void_p, ctypes.c_int, ctypes.c_void_p, ctypes.POINTER(ctypes.c_int64)]
    L.fa_test_paged_parts.restype = ctypes.c_int
    return L


def params(tokens, H, Hk, d, lens, cu, most, width, page=16, causal=True, window=(-1, -1)):
    """A call of these sizes; lens and cu (or None) on the device.  No page is ever followed, so one table entry serves all."""
    from flash_attn_b200 import _lib
    p = _lib.PagedFwdParams()
    c = p.cache
    c.k = c.v = p.q = p.o = 4096
    c.page_table = 4096
    c.dtype, c.num_pages, c.page_size, c.heads, c.head_dim = _lib.FA_DTYPE_BF16, 1 << 20, page, Hk, d
    for s in (c.k_stride, c.v_stride):
        s[0], s[1], s[2] = Hk * page * d, page * d, d
    c.table_stride = c.table_width = width
    c.batch = lens.numel()
    c.seqlens_k, c.cu_seqlens_q = lens.data_ptr(), cu.data_ptr() if cu is not None else None
    p.o_dtype, p.heads, p.tokens, p.max_seqlen_q, p.softmax_scale = _lib.FA_DTYPE_BF16, H, tokens, most, 1.0
    for s in (p.q_stride, p.o_stride):
        s[0], s[1] = H * d, d
    p.is_causal, p.window_left, p.window_right = int(causal), *window
    p.stream = torch.cuda.current_stream().cuda_stream
    return p


def parts(L, p, order=None):
    """(parts asked for as dicts or None, grid, room for partial rows, slots); order None: all numbers there may be and some more."""
    sizes = (ctypes.c_int64 * 3)()
    assert L.fa_test_paged_parts(ctypes.byref(p), None, 0, None, sizes) == 0
    if order is None:
        order = list(range(sizes[0] + 70))
    asked = torch.tensor(order, dtype=torch.int32).cuda()
    out = torch.zeros(len(order), 16, dtype=torch.int32, device="cuda")
    assert L.fa_test_paged_parts(ctypes.byref(p), asked.data_ptr(), len(order), out.data_ptr(), sizes) == 0
    found = [dict(zip(FIELDS, row)) if row[FIELDS.index("n_rows")] > 0 else None for row in out.cpu().tolist()]
    return found, *sizes
