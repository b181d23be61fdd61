"""The calls around a paged cache and autograd: nothing is recorded, so nothing that a gradient hangs on is taken or passed by."""
import pytest
import torch

import paged_util as pu

pytestmark = pytest.mark.gpu


def fa():
    import flash_attn_b200
    return flash_attn_b200


def made():
    """Each call with its arguments, by name."""
    t = torch.float16
    lens = torch.tensor([20, 30], dtype=torch.int32).cuda()
    k_pages, v_pages, table = pu.make_cache([20, 30], 16, 2, 64, t, seed=1)
    f, _ = fa().rotary_frequencies(64)
    rand = lambda *s: torch.randn(*s, device="cuda").to(t)  # noqa: E731
    cache = dict(k_pages=k_pages, v_pages=v_pages, page_table=table, seqlens_k=lens)
    one = lambda: torch.ones((), dtype=torch.float64, device="cuda")  # noqa: E731
    return {
        "rotary": (fa().rotary_embedding, dict(x=rand(2, 4, 64), positions=torch.arange(2, device="cuda"), inv_freq=f, amplitude=one(), out=rand(2, 4, 64))),
        "append": (fa().paged_kv_append, dict(k=rand(2, 2, 64), v=rand(2, 2, 64), **cache, q=rand(2, 4, 64), inv_freq=f, amplitude=one(), out=rand(2, 4, 64))),
        "attention": (fa().paged_attn_forward, dict(q=rand(2, 4, 64), **cache, softmax_scale=one() / 8, alibi_slopes=torch.ones(4, device="cuda"), out=rand(2, 4, 64)))}


FLOATS = [("rotary", n) for n in ("x", "inv_freq", "amplitude", "out")] + [("append", n) for n in ("k", "v", "k_pages", "v_pages", "q", "inv_freq", "amplitude", "out")] + [
    ("attention", n) for n in ("q", "k_pages", "v_pages", "softmax_scale", "alibi_slopes", "out")]


@pytest.mark.parametrize("name, argument", FLOATS)
def test_a_tensor_that_requires_grad_is_refused(name, argument):
    call, args = made()[name]
    call(**args)
    args[argument] = args[argument].clone().requires_grad_()
    with pytest.raises(ValueError, match=f"{argument} requires grad"):
        call(**args)
    with torch.no_grad():
        call(**args)
    args[argument] = args[argument].detach()
    call(**args)


@pytest.mark.parametrize("name, argument", FLOATS)
def test_a_tensor_with_a_tangent_is_refused(name, argument):
    from torch.autograd import forward_ad
    call, args = made()[name]
    with forward_ad.dual_level():
        plain = args[argument]
        args[argument] = forward_ad.make_dual(plain, torch.ones_like(plain))
        with pytest.raises(ValueError, match=f"{argument} has a forward-mode tangent"):
            call(**args)
        with torch.no_grad(), pytest.raises(ValueError, match="tangent"):  # (no_grad leaves forward mode on)
            call(**args)
        args[argument] = forward_ad.unpack_dual(args[argument]).primal
        call(**args)
    args[argument] = plain
    call(**args)


@pytest.mark.parametrize("name, outputs", [("rotary", ["out"]), ("append", ["k_pages", "v_pages", "out"]), ("attention", ["out"])])
def test_autograd_learns_what_was_written_to(name, outputs):
    """A tensor that a graph has saved and a call has overwritten since is named by backward, not used."""
    call, args = made()[name]
    before = {n: x._version for n, x in args.items()}
    with torch.no_grad():
        call(**args)
    assert {n for n, x in args.items() if x._version != before[n]} == set(outputs)
    for n in outputs:
        w = torch.ones((), dtype=args[n].dtype, device="cuda", requires_grad=True)
        loss = (w * args[n]).float().sum()
        call(**args)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()
    with torch.inference_mode():  # (tensors of inference mode count nothing)
        args = {n: x.clone() for n, x in args.items()}
        call(**args)


def test_a_rotation_in_place_is_seen():
    x = torch.randn(1, 2, 8, 64, device="cuda")
    f, _ = fa().rotary_frequencies(64)
    w = torch.ones((), device="cuda", requires_grad=True)
    loss = (w * x).sum()
    fa().rotary_embedding(x, torch.arange(8, device="cuda"), f, out=x)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
