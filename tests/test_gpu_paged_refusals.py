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
