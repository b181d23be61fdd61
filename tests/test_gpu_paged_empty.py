"""Batches over the paged cache of which most sequences hold nothing (a padded batch of a captured step): a CTA that has done a part
with keys takes many without any.  Against the 64-bit form of tests/paged_util.py."""
import pytest
import torch

import paged_util as pu

pytestmark = pytest.mark.gpu


def fa():
    import flash_attn_b200
    return flash_attn_b200


def ints(x):
    return torch.tensor(x, dtype=torch.int32).cuda()


def check(got, status, q, cache, lens_q, lens_k, t, **kw):
    torch.cuda.synchronize()
    assert int(status) == 0
    want = pu.attention(q, *cache, [max(n, 0) for n in lens_k], lens_q, **kw)
    pu.check_attention(got[0], got[1], want, t, max(lens_k))
    nothing = torch.isneginf(want[1])
    assert bool((got[0].cpu()[nothing] == 0).all())


def spread(live, empty, B):
    """The sequences that hold something first, last, or among the others."""
    return {"first": live + empty * (B - len(live)), "last": empty * (B - len(live)) + live,
            "between": sum(([x] + empty * (B // len(live) - 1) for x in live), [])}


# one, four, eight and sixteen rows a block
@pytest.mark.parametrize("H, Hk, d", [(8, 8, 128), (16, 4, 64), (32, 8, 128), (64, 8, 64), (64, 4, 128)])
@pytest.mark.parametrize("place", ["first", "last", "between"])
def test_single_tokens_beside_many_empty_sequences(H, Hk, d, place):
    t, B = torch.bfloat16, 1024
    lens_k = spread([300 + 13 * i for i in range(64)], [0], B)[place]
    cache = pu.make_cache(lens_k, 16, Hk, d, t, seed=1, poison=float("nan"))
    q = torch.randn(B, H, d, device="cuda").to(t)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    for _ in range(3):
        got = fa().paged_attn_forward(q, *cache, ints(lens_k), causal=True, status=status)
        check(got, status, q, cache, [1] * B, lens_k, t, causal=True)


def test_lengths_below_zero_and_rows_before_the_first_key():
    t, B = torch.float16, 700
    lens_k = spread([900, 40, 513, 1], [-3], B)["first"]
    cache = pu.make_cache([max(n, 0) for n in lens_k], 32, 2, 64, t, seed=2)
    q = torch.randn(B, 8, 64, device="cuda").to(t)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    got = fa().paged_attn_forward(q, *cache, ints(lens_k), causal=True, status=status)
    check(got, status, q, cache, [1] * B, lens_k, t, causal=True)
    lens_q, lens_k = [3] * B, [1300, 700, 2] + [0] * (B - 3)  # three rows each, of which most have no key at all
    q = torch.randn(3 * B, 8, 64, device="cuda").to(t)
    cache = pu.make_cache(lens_k, 32, 2, 64, t, seed=2)
    got = fa().paged_attn_forward(q, *cache, ints(lens_k), pu.cumulated(lens_q), 3, causal=True, status=status)
    check(got, status, q, cache, lens_q, lens_k, t, causal=True)


@pytest.mark.parametrize("said", [1, 16])
def test_a_long_prompt_whose_length_was_not_said(said):
    """The few-rows kernel on a causal prompt: its first blocks own no tile of some of their parts."""
    t, n = torch.bfloat16, 4000
    cache = pu.make_cache([n], 64, 1, 64, t, seed=3)
    q = torch.randn(n, 1, 64, device="cuda").to(t)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    got = fa().paged_attn_forward(q, *cache, ints([n]), pu.cumulated([n]), said, causal=True, status=status)
    check(got, status, q, cache, [n], [n], t, causal=True)


def test_a_captured_step_whose_batch_runs_empty():
    t, B, Hk = torch.bfloat16, 512, 8
    most = [500 + i for i in range(B)]
    cache = pu.make_cache(most, 64, Hk, 64, t, seed=4)
    q = torch.randn(B, Hk, 64, device="cuda").to(t)
    lens, status = ints([1] * B), torch.zeros(1, dtype=torch.int32, device="cuda")
    step = lambda: fa().paged_attn_forward(q, *cache, lens, causal=True, status=status)  # noqa: E731
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for live in (B, 40, 1, 0, 300):
        lens_k = most[:live] + [0] * (B - live)
        lens.copy_(ints(lens_k))
        graph.replay()
        check(got, status, q, cache, [1] * B, lens_k, t, causal=True)
