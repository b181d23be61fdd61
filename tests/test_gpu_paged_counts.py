"""The counts by which the parts of an item know who comes last, in workspaces that something else was written to in between."""
import pytest
import torch

import paged_util as pu

pytestmark = pytest.mark.gpu


def fa():
    import flash_attn_b200
    return flash_attn_b200


@pytest.mark.parametrize("lens_q, lens_k, H, Hk, d", [([1, 1], [9000, 20000], 8, 1, 128), ([60, 60], [8000, 9000], 4, 1, 64), ([200], [7000], 8, 1, 128)])
@pytest.mark.parametrize("piece", range(4))
def test_a_count_that_was_written_to_in_part_is_none(lens_q, lens_k, H, Hk, d, piece):
    """A 16-bit piece of every word, as a tensor of 16-bit values leaves it where memory is handed on."""
    t = torch.bfloat16
    k, v, table = pu.make_cache(lens_k, 16, Hk, d, t, seed=1)
    q = torch.randn(sum(lens_q), H, d, device="cuda").to(t)
    lens, cu = torch.tensor(lens_k, dtype=torch.int32).cuda(), pu.cumulated(lens_q)
    room = torch.zeros(64 << 20, dtype=torch.uint8, device="cuda")
    call = lambda: fa().paged_attn_forward(q, k, v, table, lens, cu, max(lens_q), causal=True, workspace=room)  # noqa: E731
    want = call()
    pu.check_attention(*want, pu.attention(q, k, v, table, lens_k, lens_q, causal=True), t, max(lens_k))
    counts = room[: 16384].view(torch.int16).view(-1, 4)  # (they lie in front)
    for value in (0, 1, 2, 3, 7, 100, -1):
        counts[:, piece] = value
        got = call()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]), value
    for value in (1, 2, 3):  # off by as many as would come
        counts[:, piece] += value
        got = call()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]), value
