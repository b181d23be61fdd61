"""Calls around a paged cache that the kernels do not take: each is refused by name, or done another way."""
import pytest
import torch

import paged_util as pu

pytestmark = pytest.mark.gpu


def fa():
    import flash_attn_b200
    return flash_attn_b200


def test_queries_beside_pages_without_heads():
    """There is nothing to append, but q was to be turned: refused, not handed back as it was allocated."""
    from flash_attn_b200._lib import FaError
    t = torch.bfloat16
    lens, table = torch.tensor([5, 9], dtype=torch.int32).cuda(), torch.zeros(2, 1, dtype=torch.int32, device="cuda")
    none, pages = torch.empty(2, 0, 64, dtype=t, device="cuda"), torch.empty(4, 0, 16, 64, dtype=t, device="cuda")
    q = torch.randn(2, 4, 64, device="cuda").to(t)
    f, _ = fa().rotary_frequencies(64)
    with pytest.raises(FaError):
        fa().paged_kv_append(none, none, pages, pages.clone(), table, lens, q=q, inv_freq=f)
    assert fa().paged_kv_append(none, none, pages, pages.clone(), table, lens) is None
    assert fa().paged_kv_append(none, none, pages, pages.clone(), table, lens, q=q[:, :0], inv_freq=f).shape == (2, 0, 64)


@pytest.mark.parametrize("lens_q", [[1, 1, 1], [40, 3, 20]])
def test_broadcast_queries(lens_q):
    """One row for all heads, or for all tokens: as if each had its own.  From C, chunks of such rows are refused."""
    import ctypes

    import paged_parts_util as pp
    from flash_attn_b200 import _lib
    t, lens_k, H, d, T = torch.bfloat16, [300, 40, 20], 4, 64, sum(lens_q)
    k, v, table = pu.make_cache(lens_k, 16, 2, d, t, seed=1)
    lens, cu = torch.tensor(lens_k, dtype=torch.int32).cuda(), pu.cumulated(lens_q)
    call = lambda q: fa().paged_attn_forward(q, k, v, table, lens, cu, max(lens_q), causal=True)  # noqa: E731
    for q in (torch.randn(T, 1, d, device="cuda").to(t).expand(T, H, d), torch.randn(1, H, d, device="cuda").to(t).expand(T, H, d),
              torch.randn(1, 1, d, device="cuda").to(t).expand(T, H, d)):
        got, want = call(q), call(q.contiguous())
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    if max(lens_q) * H // 2 > 16:
        for i in range(2):
            p = pp.params(T, H, 2, d, lens, cu, max(lens_q), table.shape[1])
            room = torch.empty(_lib.load().fa_paged_fwd_workspace_bytes(ctypes.byref(p)) + 16, dtype=torch.uint8, device="cuda")
            p.workspace, p.workspace_bytes = room.data_ptr(), room.numel()
            p.q_stride[i] = 0
            assert _lib.load().fa_paged_fwd(ctypes.byref(p)) == -1
