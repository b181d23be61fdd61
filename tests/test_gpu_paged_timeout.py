"""Bounded waits of the attention over pages, exercised without faulting or hanging anything: a test build (waits give up after
about 2 ms) whose first CTA leaves out the loads of a tile and of all behind it.  The rows of that CTA's parts are NaN, everyone
else's as ever, the status word says so, and the workspace serves the next call."""
import ctypes
import os

import pytest
import torch

import paged_util as pu

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def test_lib():
    from flash_attn_b200 import _lib, build
    path = build.TEST_LIB
    if not os.path.exists(path):
        path = build.build_test_variant()
    L = ctypes.CDLL(path)
    for name, result in (("fa_paged_fwd", ctypes.c_int), ("fa_paged_fwd_workspace_bytes", ctypes.c_size_t)):
        getattr(L, name).argtypes = [ctypes.POINTER(_lib.PagedFwdParams)]
        getattr(L, name).restype = result
    L.fa_test_leave_out_paged_tiles.argtypes = [ctypes.c_int]
    return L


# single tokens whose items are cut, whole items one behind the other, chunks of one and two query tiles, cut and whole
@pytest.mark.parametrize("lens_q, lens_k, H, Hk, d", [
    ([1] * 4, [30000, 20000, 900, 100], 8, 2, 128), ([1] * 300, [700] * 300, 4, 4, 64), ([3] * 200, [400] * 200, 4, 2, 128),
    ([20] * 3, [9000, 300, 20], 4, 1, 128), ([200] * 4, [9000, 3000, 300, 200], 8, 2, 128), ([300] * 30, [300] * 30, 8, 2, 64)])
@pytest.mark.parametrize("first", [0, 1, 5])
def test_a_part_whose_wait_gave_up_is_nan_and_the_others_are_right(test_lib, lens_q, lens_k, H, Hk, d, first):
    from flash_attn_b200 import _lib
    t, L = torch.bfloat16, test_lib
    k, v, table = pu.make_cache(lens_k, 64, Hk, d, t, seed=1)
    T = sum(lens_q)
    q = torch.randn(T, H, d, device="cuda").to(t)
    lens, cu = torch.tensor(lens_k, dtype=torch.int32).cuda(), pu.cumulated(lens_q)
    p = _lib.PagedFwdParams()
    c = p.cache
    c.k, c.v, c.dtype, c.num_pages, c.page_size, c.heads, c.head_dim = k.data_ptr(), v.data_ptr(), _lib.FA_DTYPE_BF16, k.shape[0], 64, Hk, d
    c.k_stride[:], c.v_stride[:] = k.stride()[:3], v.stride()[:3]
    c.page_table, c.table_stride, c.table_width, c.batch = table.data_ptr(), table.stride(0), table.shape[1], len(lens_k)
    c.seqlens_k, c.cu_seqlens_q = lens.data_ptr(), cu.data_ptr()
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    p.q = p.o = q.data_ptr()  # (the output: for the size of the workspace only)
    p.o_dtype, p.heads, p.tokens, p.max_seqlen_q = _lib.FA_DTYPE_BF16, H, T, max(lens_q)
    p.q_stride[:] = p.o_stride[:] = q.stride()[:2]
    p.softmax_scale, p.is_causal, p.window_left, p.window_right = d ** -0.5, 1, -1, -1
    room = torch.empty(max(L.fa_paged_fwd_workspace_bytes(ctypes.byref(p)), 16), dtype=torch.uint8, device="cuda")
    p.workspace, p.workspace_bytes, p.status = room.data_ptr(), room.numel(), status.data_ptr()
    p.stream = torch.cuda.current_stream().cuda_stream

    def call(leave_out):
        o, lse = torch.full_like(q, 5.0), torch.full((T, H), 5.0, device="cuda")
        p.o, p.lse = o.data_ptr(), lse.data_ptr()
        status.zero_()
        L.fa_test_leave_out_paged_tiles(leave_out)
        try:
            assert L.fa_paged_fwd(ctypes.byref(p)) == 0
        finally:
            L.fa_test_leave_out_paged_tiles(-1)
        torch.cuda.synchronize()
        return o, lse, int(status)
    want = call(-1)
    assert want[2] == 0 and not want[0].isnan().any()
    for _ in range(2):
        o, lse, code = call(first)
        lost = lse.isnan()
        if code == 0:  # (the first CTA has fewer tiles than are loaded)
            assert not lost.any()
        else:
            assert 300 < code < 330 and lost.any() and not lost.all()
        assert torch.equal(o.isnan().all(-1), lost) and torch.equal(o.isnan().any(-1), lost)
        assert torch.equal(o[~lost], want[0][~lost]) and torch.equal(lse[~lost], want[1][~lost])
        again = call(-1)
        assert again[2] == 0 and torch.equal(again[0], want[0]) and torch.equal(again[1], want[1])
