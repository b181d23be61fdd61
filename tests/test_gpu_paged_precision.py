"""What the attention over pages leaves of 32 bits: scores whose exponentials are powers of two, so that neither their products nor the
16 bits of P lose anything, and the kernels' own arithmetic shows.  An exponential that is off by a few 1e-5 fails."""
import math

import pytest
import torch

import paged_util as pu

pytestmark = pytest.mark.gpu


def fa():
    import flash_attn_b200
    return flash_attn_b200


# one to sixteen rows a block, one and two query tiles; in one part and in several
@pytest.mark.parametrize("n_q, H, Hk", [(1, 1, 1), (1, 4, 1), (2, 4, 1), (4, 8, 2), (30, 4, 1), (150, 8, 2)])
@pytest.mark.parametrize("n_k", [256, 4096])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("dtype, alibi", [("bfloat16", False), ("float16", False), ("bfloat16", True)])
def test_exponentials_and_sums_are_in_32_bits(n_q, H, Hk, n_k, d, dtype, alibi):
    """Scores are whole numbers s of -4 .. 4 times ln 2 (and with ALiBi less whole distances times ln 2, of which those below 2^-20 count
    for nothing here).  In units of 2^-24, relative:
      the exponent x = s scale log2 e: scale, log2 e and their product are rounded, 3 |x|, and the sum with the maximum, |x - m|: with
        |x| <= 4 and |x - m| <= 8 for what counts (ALiBi: |x - m| <= 20, and the bias rounded twice more, 2 * 20): 20 (72), times ln 2;
      ex2.approx: 4;
      the sum: 16 terms of a chain, 8 chains, n_k / 128 tiles, and up to 40 parts put together with two factors each: 16 + 8 + n_k / 128 + 80;
      LSE: logarithm, ln 2 and one sum, 2 each of at most |lse| + 8.
    O: the exponential twice over, the sum, and the tensor core's sums of n_k terms, 16 a step, each step taken as cut off at 2 of
    2^-24 of the largest sum: 4 (n_k / 16 + 16), all of sum p |v|; and its own rounding."""
    t, step = pu.DT[dtype], 2.0 ** -24
    g = torch.Generator().manual_seed(n_q * n_k + d)
    whole = lambda *s: torch.randint(-2, 3, s, generator=g).to(t)  # noqa: E731
    k, v, table = pu.make_cache([n_k], 16, Hk, d, t, seed=1)
    flat = torch.randn(k.shape, generator=g).to(t)
    flat[..., 0], flat[..., d - 1] = whole(*k.shape[:3]), whole(*k.shape[:3])
    k.copy_(flat)
    q = torch.zeros(n_q, H, d, dtype=t)
    q[..., 0] = q[..., d - 1] = 1.0  # (all other columns of K meet zeros)
    q = q.cuda()
    slopes = torch.full((H,), math.log(2.0), device="cuda") if alibi else None
    o, lse = fa().paged_attn_forward(q, k, v, table, torch.tensor([n_k], dtype=torch.int32).cuda(), pu.cumulated([n_q]), n_q, softmax_scale=math.log(2.0),
                                     causal=True, alibi_slopes=slopes, out_dtype=torch.float32)
    want, want_lse, size, _ = pu.attention(q, k, v, table, [n_k], [n_q], scale=math.log(2.0), causal=True, slopes=slopes)
    power = (72 if alibi else 20) * math.log(2.0) + 4
    total = 16 + 8 + n_k / 128 + 80
    off = (lse.cpu().double() - want_lse).abs()
    bound = step * (power + total + 6 * (want_lse.abs() + 8))
    assert bool((off <= bound).all()), float((off / bound).max())
    off = (o.cpu().double() - want).abs()
    bound = step * ((2 * power + total + 4 * (n_k / 16 + 16)) * size + want.abs())
    if alibi:
        bound = bound + 2.0 ** -20 * n_k * 6 * step  # (P of what counts for nothing: subnormal in no type here)
    assert bool((off <= bound).all()), float((off / bound).max())
