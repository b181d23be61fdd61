"""Rotary positions against the 64-bit form: layouts, part of the head, odd sizes and strides, far positions, the gradient."""
import pytest
import torch

import paged_util as pu

pytestmark = pytest.mark.gpu


def call(*a, **kw):
    import flash_attn_b200 as fa
    return fa.rotary_embedding(*a, **kw)


def freqs(r, **kw):
    import flash_attn_b200 as fa
    return fa.rotary_frequencies(r, **kw)


def check(x, positions, f, got, **kw):
    flat = {k: v for k, v in kw.items() if k != "inverse"}
    want = pu.turned(x.cpu(), positions.cpu(), f.cpu(), **kw)
    bound = pu.turn_bound(x.cpu(), want, x.dtype, f.cpu(), positions.cpu(), **flat)
    off = (got.cpu().double() - want).abs()
    assert not torch.isnan(off).any() and bool((off <= bound).all()), float((off / bound).max())


CASES = [  # B, H, N, d, rotary_dim, interleaved, inverse, dtype
    (1, 1, 1, 64, 64, False, False, "bfloat16"), (2, 3, 5, 128, 128, False, False, "float16"), (2, 3, 5, 128, 128, True, True, "bfloat16"),
    (1, 32, 1, 128, 128, False, False, "bfloat16"), (3, 5, 257, 96, 48, False, True, "float32"), (3, 5, 257, 96, 48, True, False, "float32"),
    (1, 40, 300, 128, 64, True, False, "float16"), (2, 9, 33, 80, 40, False, False, "bfloat16"), (2, 9, 33, 80, 40, True, True, "bfloat16"),
    (1, 7, 19, 31, 30, False, False, "float16"), (1, 7, 19, 31, 14, True, False, "float32"), (1, 2, 70, 256, 256, False, True, "float32"),
    (1, 2, 70, 256, 2, True, False, "bfloat16"), (1, 1, 100000, 64, 64, False, False, "bfloat16"), (70000, 1, 1, 8, 8, True, False, "float16"),
    (2, 24, 1501, 96, 64, True, True, "float32"), (1, 64, 200, 128, 128, False, False, "float32"), (1, 3, 9, 12, 4, False, False, "float32"),
]


@pytest.mark.parametrize("B, H, N, d, r, interleaved, inverse, dtype", CASES)
def test_rows_are_turned(B, H, N, d, r, interleaved, inverse, dtype):
    torch.manual_seed(B * 7 + N)
    f, _ = freqs(r)
    x = torch.randn(B, H, N, d, device="cuda").to(pu.DT[dtype])
    each = torch.randint(0, 200000, (B, N), device="cuda")
    kw = dict(amplitude=1.25, interleaved=interleaved, inverse=inverse)
    check(x, each[:, None], f, call(x, each, f, **kw), **kw)
    one = torch.arange(N, device="cuda", dtype=torch.int32) + 11
    check(x, one, f, call(x, one, f, **kw), **kw)


@pytest.mark.parametrize("dtype", ["float16", "bfloat16", "float32"])
@pytest.mark.parametrize("T, H, d, r, interleaved", [(1, 8, 128, 128, False), (333, 5, 64, 32, True), (50, 28, 128, 96, False)])
def test_tokens_one_behind_the_other(T, H, d, r, interleaved, dtype):
    torch.manual_seed(T)
    f, _ = freqs(r)
    x = torch.randn(T, H, d, device="cuda").to(pu.DT[dtype])
    at = torch.randint(0, 1 << 20, (T,), device="cuda")
    check(x, at[:, None], f, call(x, at, f, interleaved=interleaved), interleaved=interleaved)


@pytest.mark.parametrize("interleaved", [False, True])
def test_far_positions_keep_their_angles(interleaved):
    f, _ = freqs(128)
    at = torch.tensor([0, 1, 2 ** 20 - 1, 2 ** 24 + 1, 2 ** 31 - 1, 2 ** 31 + 12345, 2 ** 40 + 7, -1, -77], device="cuda")
    x = torch.randn(len(at), 2, 128, device="cuda")
    check(x, at[:, None], f, call(x, at, f, interleaved=interleaved), interleaved=interleaved)


@pytest.mark.parametrize("kind", [dict(scaling="linear", factor=4.0), dict(scaling="ntk", factor=8.0), dict(scaling="ramp", factor=16.0, original_length=4096)])
def test_scaled_for_long_contexts(kind):
    f, t = freqs(64, **kind)
    x = torch.randn(1, 4, 129, 64, device="cuda").bfloat16()
    at = torch.arange(129, device="cuda") * 511
    check(x, at, f, call(x, at, f, t), amplitude=t)


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_strides_offsets_and_in_place(dtype):
    torch.manual_seed(5)
    f, _ = freqs(128)
    f40, _ = freqs(40)
    t = pu.DT[dtype]
    at = torch.arange(37, device="cuda") * 3
    # heads inside tokens, Q out of a fused projection
    fused = torch.randn(37, 3, 8, 128, device="cuda").to(t)
    q = fused[:, 1]
    check(q, at[:, None], f, call(q, at, f))
    x4 = torch.randn(2, 37, 4, 128, device="cuda").to(t).transpose(1, 2)
    check(x4, at, f, call(x4, at, f))
    # rows that start at odd elements: no vector fits
    raw = torch.randn(37 * 5 * 131 + 1, device="cuda").to(t)
    odd = raw[1:].view(37, 5, 131)[..., :128]
    check(odd, at[:, None], f, call(odd, at, f))
    # an expanded input
    wide = torch.randn(1, 1, 37, 128, device="cuda").to(t).expand(2, 3, 37, 128)
    check(wide, at, f, call(wide, at, f))
    # in place, the rest of the buffer as it was
    before = fused.clone()
    out = call(q, at, f, out=q)
    assert out is q
    check(before[:, 1], at[:, None], f, fused[:, 1])
    assert torch.equal(fused[:, 0], before[:, 0]) and torch.equal(fused[:, 2], before[:, 2])
    # in place with columns that are not turned
    part = torch.randn(37, 5, 96, device="cuda").to(t)
    before = part.clone()
    call(part, at, f40, out=part)
    check(before, at[:, None], f40, part)
    assert torch.equal(part[..., 40:], before[..., 40:])
    # into a view
    room = torch.full((37, 8, 160), 7.0, device="cuda").to(t)
    call(q, at, f, out=room[..., 16:144])
    assert bool((room[..., :16] == 7).all()) and bool((room[..., 144:] == 7).all())


def test_non_finite_values_stay_in_their_pairs():
    f, _ = freqs(64)
    at = torch.arange(4, device="cuda") + 1
    x = torch.randn(4, 2, 128, device="cuda")
    y = x.clone()
    y[1, 1, 3] = float("nan")
    y[2, 0, 100] = float("inf")  # not turned: copied
    a, b = call(x, at, f), call(y, at, f)
    hit = a != b
    assert hit.sum() == 3 and bool(hit[1, 1, 3]) and bool(hit[1, 1, 35]) and bool(hit[2, 0, 100])


def test_nothing_to_turn():
    f, _ = freqs(64)
    for shape in ((0, 4, 64), (5, 0, 64)):
        x = torch.empty(shape, device="cuda")
        assert call(x, torch.arange(shape[0], device="cuda"), f).shape == x.shape


@pytest.mark.parametrize("interleaved", [False, True])
def test_the_gradient_is_the_formulas_and_the_differences(interleaved):
    torch.manual_seed(9)
    f, _ = freqs(24)
    at = torch.tensor([3, 1000, 7, 65537], device="cuda")
    x, g = (torch.randn(4, 3, 32, device="cuda") for _ in range(2))
    kw = dict(amplitude=1.5, interleaved=interleaved)
    got = call(g, at, f, inverse=True, **kw).cpu().double()
    # the formula's, by autograd through the 64-bit form
    leaf = x.cpu().double().requires_grad_()
    y = pu.turned(leaf, at.cpu()[:, None], f.cpu(), **kw)
    (want,) = torch.autograd.grad((y * g.cpu().double()).sum(), leaf)
    bound = pu.turn_bound(g.cpu(), want, torch.float32, f.cpu(), at.cpu()[:, None], **kw)
    assert bool(((got - want).abs() <= bound).all())
    # differences of the kernel itself: the map is linear, so a step of 1 gives the derivative, up to the two results' own errors
    for row, head, col in ((0, 0, 0), (1, 2, 13), (2, 1, 23), (3, 0, 31)):
        step = torch.zeros_like(x)
        step[row, head, col] = 1.0
        up, down = call(x + step, at, f, **kw), call(x - step, at, f, **kw)
        moved = float(((up.double() - down.double()) / 2 * g.double()).sum())
        size = float((x.abs().max() + 1) * g.double().abs().sum(-1).max())
        assert abs(moved - float(got[row, head, col])) <= 8 * 4e-7 * 1.5 * size


def test_turning_back_and_the_calls_refusals():
    f, _ = freqs(64)
    at = torch.arange(9, device="cuda")
    x = torch.randn(9, 2, 64, device="cuda")
    back = call(call(x, at, f), at, f, inverse=True)
    assert float((back - x).abs().max()) <= 4 * 4e-7 * float(2 * x.abs().max()) + 2 * 2.0 ** -23 * float(x.abs().max())
    bad = [((x.cpu(), at, f), {}), ((x[0], at, f), {}), ((x.double(), at, f), {}), ((x, at.float(), f), {}), ((x, at[:8], f), {}), ((x, at, f.float()), {}),
           ((x, at, freqs(66)[0]), {}), ((x, at, f), dict(out=x.half())), ((x, at, f), dict(out=x[:8])), ((x.transpose(1, 2).contiguous().transpose(1, 2), at, f), {}),
           ((x.clone().requires_grad_(), at, f), {}), ((x, at.cpu(), f), {}), ((x, at, f.cpu()), {})]
    for args, kw in bad:
        with pytest.raises(ValueError):
            call(*args, **kw)
    from flash_attn_b200._lib import FaError
    with pytest.raises(FaError):
        call(x, at, f, out=x[:1].expand(9, 2, 64))  # rows of the result in one place
    with pytest.raises(TypeError):
        call(x, [1, 2], f)
    with torch.no_grad():
        call(x.clone().requires_grad_(), at, f)


def test_captured_and_replayed_on_a_stream_of_its_own():
    f, _ = freqs(128)
    x = torch.randn(4, 8, 65, 128, device="cuda").half()
    at = torch.arange(65, device="cuda")
    out = torch.empty_like(x)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        call(x, at, f, out=out)
        side.synchronize()
        with torch.cuda.graph(g, stream=side):
            call(x, at, f, out=out)
    for shift in (5, 100000):
        x.copy_(torch.randn(x.shape, device="cuda"))
        at.copy_(torch.arange(65, device="cuda") + shift)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, call(x, at, f))
