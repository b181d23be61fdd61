"""How far a value of V that is not finite reaches: the rows that see it, and at most the others of their block (256 rows of a chunk,
16 of few rows: a row is a token and a query head of one K/V head)."""
import pytest
import torch

import paged_util as pu

pytestmark = pytest.mark.gpu


def fa():
    import flash_attn_b200
    return flash_attn_b200


@pytest.mark.parametrize("before", [0, 37, 128])  # keys of the cache, so that the tiles of keys and of rows lie askew
@pytest.mark.parametrize("n, H, Hk, most, d", [(600, 1, 1, 600, 64), (300, 4, 2, 300, 128), (100, 1, 1, 100, 128), (40, 4, 1, 4, 64), (50, 1, 1, 8, 128)])
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_a_value_that_is_not_finite_stays_in_its_block(before, n, H, Hk, most, d, value):
    t, n_k, group = torch.bfloat16, before + n, H // Hk
    k, v, table = pu.make_cache([n_k], 16, Hk, d, t, seed=1)
    q = torch.randn(n, H, d, device="cuda").to(t)
    lens, cu = torch.tensor([n_k], dtype=torch.int32).cuda(), pu.cumulated([n])
    call = lambda v: fa().paged_attn_forward(q, k, v, table, lens, cu, most, causal=True)  # noqa: E731
    want = call(v)
    rows = min(most, n) * group
    block = 256 if rows > 128 else 128 if rows > 16 else 16  # (rows; a group that divides 128 here)
    for at in (0, n // 3, 130, n - 1):  # the new token whose V it is
        if at >= n:
            continue
        bad = v.clone()
        key = before + at
        bad[table[0, key // 16].long(), :, key % 16] = value
        o, lse = call(bad)
        first = max(0, at * group - block + 1) // group  # no row of a token before this one shares a block with one that sees the key
        assert torch.equal(o[:first], want[0][:first])
        assert not bool(o[at:].isfinite().all(-1).any())
        assert torch.equal(lse, want[1])  # (V has no part in it)
