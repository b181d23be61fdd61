"""Plain 64-bit forms of the operators around a paged cache, on the CPU, and caches to run them on."""
import math

import torch

DT = {"float16": torch.float16, "bfloat16": torch.bfloat16, "float32": torch.float32}


def half_step(dtype):
    """Largest relative error of one rounding."""
    return torch.finfo(dtype).eps / 2


# ------------------------------------------------------------------ rotation
def turned(x, positions, inv_freq, amplitude=1.0, interleaved=False, inverse=False):
    """x [..., d] in 64 bits, positions broadcast against its leading dimensions."""
    x, r = x.double(), 2 * inv_freq.numel()
    angle = positions.double()[..., None] * inv_freq.double()
    c, s = amplitude * torch.cos(angle), (-amplitude if inverse else amplitude) * torch.sin(angle)
    y = x.clone()
    a, b = (slice(0, r, 2), slice(1, r, 2)) if interleaved else (slice(0, r // 2), slice(r // 2, r))
    y[..., a] = x[..., a] * c - x[..., b] * s
    y[..., b] = x[..., b] * c + x[..., a] * s
    return y


def turn_bound(x, want, dtype, inv_freq, positions, amplitude=1.0, interleaved=False):
    """One rounding of the result; before it, in 32 bits: the half turns rounded to 2^-25 (times pi: 9.4e-8), sincospi to two units of
    2^-24, cos * amplitude and the products to half a step each -- 9.4e-8 + 5 * 2^-24 < 4e-7 of |a| + |b|; and the angle of both sides
    to its 64-bit product, 2^-52 of the angle."""
    r = 2 * inv_freq.numel()
    x = x.double().abs()
    pair = x.clone()
    if interleaved:
        pair[..., 0:r:2] = pair[..., 1:r:2] = x[..., 0:r:2] + x[..., 1:r:2]
    else:
        pair[..., : r // 2] = pair[..., r // 2: r] = x[..., : r // 2] + x[..., r // 2: r]
    pair[..., r:] = 0.0
    far = 2.0 ** -51 * float(positions.double().abs().max()) * float(inv_freq.abs().max())
    tiny = torch.finfo(dtype).tiny * torch.finfo(dtype).eps  # (a step of the subnormals)
    return half_step(dtype) * want.abs() * 1.001 + (4e-7 + far) * amplitude * pair + tiny


# ------------------------------------------------------------------ caches
def make_cache(lens_k, page, heads, d, dtype, seed, slots_first=False, spare=3, poison=None):
    """(k_pages, v_pages, page_table) on the GPU: every token random, what no token holds `poison` (or random too)."""
    g = torch.Generator().manual_seed(seed)
    pages = [-(-n // page) for n in lens_k]
    total, width = sum(pages), max(max(pages), 1)
    shape = (total + spare, page, heads, d) if slots_first else (total + spare, heads, page, d)
    pools = [torch.randn(*shape, generator=g).to(dtype) for _ in range(2)]
    pools = [p.transpose(1, 2) if slots_first else p for p in pools]
    order = torch.randperm(total + spare, generator=g)[:total].to(torch.int32)
    table = torch.full((len(lens_k), width), -1, dtype=torch.int32)
    at = 0
    held = torch.zeros(total + spare, page, dtype=torch.bool)
    for b, n in enumerate(pages):
        table[b, :n] = order[at: at + n]
        for i in range(n):
            held[order[at + i], : min(page, lens_k[b] - i * page)] = True
        at += n
    if poison is not None:
        for p in pools:
            p.transpose(1, 2)[~held] = poison
    on_gpu = []
    for p in pools:
        q = p.transpose(1, 2).contiguous().cuda().transpose(1, 2) if slots_first else p.contiguous().cuda()
        on_gpu.append(q)
    return on_gpu[0], on_gpu[1], table.cuda()


def cumulated(lens_q):
    return torch.tensor([0] + list(torch.tensor(lens_q).cumsum(0)), dtype=torch.int32).cuda()


def tokens_of(pages, table, b, n):
    """[n, heads, d] in 64 bits: the first n tokens of sequence b."""
    page = pages.shape[2]
    rows = pages[table[b, : -(-n // page)].long()].transpose(1, 2).reshape(-1, pages.shape[1], pages.shape[3])
    return rows[:n].double()


def attention(q, k_pages, v_pages, table, lens_k, lens_q, scale=None, causal=False, window=(-1, -1), slopes=None):
    """(o, lse, sum of p |v|, bound of the scores' error) in 64 bits; rows of all sequences one behind the other."""
    q, k_pages, v_pages, table = q.cpu().double(), k_pages.cpu(), v_pages.cpu(), table.cpu()
    T, H, d = q.shape
    Hk = k_pages.shape[1]
    scale = scale if scale is not None else d ** -0.5
    o, lse = torch.zeros(T, H, d, dtype=torch.float64), torch.full((T, H), -math.inf, dtype=torch.float64)
    size, slack = torch.zeros(T, H, d, dtype=torch.float64), torch.zeros(T, H, dtype=torch.float64)
    first = 0
    for b, (n, nk) in enumerate(zip(lens_q, lens_k)):
        rows = slice(first, first + n)
        first += n
        if n == 0 or nk == 0:
            continue
        at, key = torch.arange(nk - n, nk), torch.arange(nk)
        ahead = key[None] - at[:, None]
        see = torch.ones(n, nk, dtype=torch.bool)
        if causal:
            see &= ahead <= 0
        if window[0] >= 0:
            see &= -ahead <= window[0]
        if window[1] >= 0:
            see &= ahead <= window[1]
        k, v = tokens_of(k_pages, table, b, nk), tokens_of(v_pages, table, b, nk)
        k = torch.nan_to_num(k.repeat_interleave(H // Hk, 1), 0.0, 0.0, 0.0)
        v = torch.nan_to_num(v.repeat_interleave(H // Hk, 1), 0.0, 0.0, 0.0)
        s = torch.einsum("nhd,khd->hnk", q[rows], k) * scale
        reach = torch.einsum("nhd,khd->hnk", q[rows].abs(), k.abs()) * scale
        if slopes is not None:
            bias = slopes.cpu().double()[:, None, None] * ahead.abs().double()
            s, reach = s - bias, reach + bias
        s = torch.where(see, s, -math.inf)
        reach = torch.where(see, reach, 0.0)
        lse[rows] = torch.logsumexp(s, -1).transpose(0, 1)
        p = torch.nan_to_num(torch.softmax(s, -1), 0.0)
        o[rows] = torch.einsum("hnk,khd->nhd", p, v)
        size[rows] = torch.einsum("hnk,khd->nhd", p, v.abs())
        slack[rows] = reach.amax(-1).transpose(0, 1)
    return o, lse, size, slack


def check_attention(got_o, got_lse, want, dtype, keys, out_dtype=None):
    """The tolerances, in terms of A = sum p |v| of the exact softmax:
      one rounding of the output: half a step of |o|;
      P rounded to 16 bits before P V: half a step of A, and in fp16 half a subnormal step (2^-25) a key: of at most `keys` |v|, where
        the largest P is at least 1/2 and max |v| < 6 (values of 100 000 normal deviates stay below 5);
      a score's error e is P's relative error: products of 16-bit values are exact, d <= 128 of them summed in 32 bits and the scale,
        bias and maximum each rounded: e <= (128 + 4) 2^-24 < 8e-6 of scale |q| |k| + bias, in numerator and denominator: 1.6e-5 of it;
      exponentials: ex2.approx 2^-22, the cubic 7.5e-5, twice over in the quotient: 1.5e-4;
      sums of up to 2^17 terms in 32 bits: 128 threads' partial sums of 2^10 terms, 2^10 2^-24 = 6.1e-5.
    LSE: the scores' error once, and the logarithm of a sum that is off by 7.5e-5 + 6.1e-5 at most."""
    o, lse, size, slack = want
    out_dtype = out_dtype or dtype
    u = half_step(dtype)
    rel = u + 1.6e-5 * slack[..., None] + 1.5e-4 + 1.3e-4
    bound = half_step(out_dtype) * o.abs() + rel * size * 1.01 + 1e-30
    if dtype == torch.float16:
        bound = bound + keys * 6.0 * 2.0 ** -25
    off = (got_o.cpu().double() - o).abs()
    worst = float((off / bound).max()) if off.numel() else 0.0
    assert not torch.isnan(off).any(), "NaN in the output"
    assert worst <= 1.0, f"output off by {worst:.2f} of its bound"
    if got_lse is not None:
        got_lse = got_lse.cpu().double()
        none = torch.isinf(lse)
        assert torch.equal(torch.isneginf(got_lse), none), "rows without keys"
        off = (got_lse - lse)[~none].abs()
        assert off.numel() == 0 or bool((off <= 8e-6 * slack[~none] + 1.4e-4 + 2.0 ** -23 * lse[~none].abs()).all()), float(off.max())
