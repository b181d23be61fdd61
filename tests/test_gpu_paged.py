"""The append of new tokens to a paged K/V cache and their attention over it, against 64-bit forms."""
import itertools

import pytest
import torch

import paged_util as pu

pytestmark = pytest.mark.gpu


def fa():
    import flash_attn_b200
    return flash_attn_b200


def ints(x):
    return torch.tensor(x, dtype=torch.int32).cuda()


def attend(q, cache, lens_k, lens_q, dtype, out_dtype=None, cu=True, most=None, **kw):
    """One call checked against the 64-bit form; returns its outputs."""
    k, v, table = cache
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    o, lse = fa().paged_attn_forward(q, k, v, table, ints(lens_k), pu.cumulated(lens_q) if cu else None,
                                     (max(lens_q) if most is None else most) if cu else None, out_dtype=out_dtype, status=status, **kw)
    torch.cuda.synchronize()
    assert int(status) == 0
    window = kw.get("window", (-1, -1))
    want = pu.attention(q, k, v, table, lens_k, lens_q, kw.get("softmax_scale"), kw.get("causal", False), window, kw.get("alibi_slopes"))
    n = sum(lens_q)
    pu.check_attention(o[:n], lse[:n], tuple(x[:n] for x in want), dtype, max(max(lens_k), 1), out_dtype)
    return o, lse


def slopes(h):
    return torch.pow(2.0, -8.0 * torch.arange(1, h + 1) / h).cuda()


# heads, heads_k, d, page: groups that do and do not divide 128, one K/V head, 64-wide and narrower heads, every size of page
SHAPES = [(8, 2, 128, 16), (4, 4, 64, 8), (7, 1, 128, 32), (12, 4, 80, 16), (16, 2, 64, 64), (5, 5, 128, 128), (6, 2, 96, 256), (64, 1, 64, 16),
          (3, 1, 40, 512), (32, 2, 128, 16), (2, 2, 8, 16)]


@pytest.mark.parametrize("H, Hk, d, page", SHAPES)
@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
def test_single_tokens(H, Hk, d, page, dtype):
    lens_k = [1, 2, page - 1, page, page + 1, 127, 128, 129, 500, 1023, 2050]
    t = pu.DT[dtype]
    cache = pu.make_cache(lens_k, page, Hk, d, t, seed=H + d, slots_first=page % 3 == 1, poison=float("nan"))
    q = torch.randn(len(lens_k), H, d, device="cuda").to(t)
    attend(q, cache, lens_k, [1] * len(lens_k), t, cu=False, causal=True)
    attend(q, cache, lens_k, [1] * len(lens_k), t, cu=True, window=(100, -1), causal=True, alibi_slopes=slopes(H))


@pytest.mark.parametrize("H, Hk, d, page", SHAPES)
@pytest.mark.parametrize("causal", [False, True])
def test_chunks_of_unequal_lengths(H, Hk, d, page, causal):
    lens_q = [1, 7, 0, 64, 130, 3, 257]
    lens_k = [300, 7, 40, 64, 1000, 0, 290]
    t = torch.bfloat16 if causal else torch.float16
    cache = pu.make_cache(lens_k, page, Hk, d, t, seed=H + d, slots_first=page % 3 == 1, poison=float("nan"))
    q = torch.randn(sum(lens_q), H, d, device="cuda").to(t)
    attend(q, cache, lens_k, lens_q, t, causal=causal)


MASKS = [dict(), dict(causal=True), dict(window=(0, 0)), dict(window=(17, 5)), dict(causal=True, window=(129, -1)), dict(window=(-1, 0)),
         dict(window=(3, -1)), dict(causal=True, alibi_slopes=True), dict(window=(40, 90), alibi_slopes=True)]


@pytest.mark.parametrize("mask", MASKS)
@pytest.mark.parametrize("lens_q, lens_k", [([1, 1, 1], [5, 700, 129]), ([5, 2, 8], [900, 2, 77]), ([300, 20, 150], [300, 1000, 151])])
def test_masks(mask, lens_q, lens_k):
    mask = dict(mask)
    H, Hk, d = 8, 2, 64
    if mask.get("alibi_slopes"):
        mask["alibi_slopes"] = slopes(H)
    for t in (torch.bfloat16, torch.float16):
        cache = pu.make_cache(lens_k, 16, Hk, d, t, seed=4, poison=float("inf"))
        q = torch.randn(sum(lens_q), H, d, device="cuda").to(t)
        attend(q, cache, lens_k, lens_q, t, **mask)


@pytest.mark.parametrize("lens_q, lens_k", [([4, 3], [2, 0]), ([1, 1], [0, 1]), ([200], [50]), ([9], [1])])
def test_rows_that_see_nothing(lens_q, lens_k):
    """More new tokens than the cache holds: the first stand before its first key; empty caches."""
    t = torch.bfloat16
    cache = pu.make_cache(lens_k, 16, 2, 128, t, seed=4, poison=float("nan"))
    q = torch.randn(sum(lens_q), 4, 128, device="cuda").to(t)
    o, lse = attend(q, cache, lens_k, lens_q, t, causal=True)
    none = torch.isneginf(lse)
    assert bool(none.any()) and bool((o[none] == 0).all())
    attend(q, cache, lens_k, lens_q, t, causal=False)
    # ... or behind everything that the window leaves
    attend(q, cache, lens_k, lens_q, t, causal=False, window=(-1, 0))


def test_output_types_scales_and_strides():
    t = torch.float16
    lens_q, lens_k = [1, 30, 140], [900, 30, 400]
    k, v, table = pu.make_cache(lens_k, 16, 2, 96, t, seed=1)
    n = sum(lens_q)
    fused = torch.randn(n, 8 + 2 + 2, 96, device="cuda").to(t)
    q = fused[:, :8]  # tokens 12 heads apart
    attend(q, (k, v, table), lens_k, lens_q, t, causal=True, softmax_scale=0.3)
    attend(q, (k, v, table), lens_k, lens_q, t, out_dtype=torch.float32, causal=True)
    heads_first = torch.randn(8, n, 96, device="cuda").to(t).transpose(0, 1)
    attend(heads_first, (k, v, table), lens_k, lens_q, t, causal=True)
    room = torch.full((n, 10, 112), 3.0, device="cuda", dtype=t)
    wide = torch.full((table.shape[0], table.shape[1] + 5), -1, dtype=torch.int32, device="cuda")
    wide[:, : table.shape[1]] = table
    out = room[:, 1:9, :96]
    o, lse = fa().paged_attn_forward(q, k, v, wide[:, : table.shape[1]], ints(lens_k), pu.cumulated(lens_q), 140, causal=True, out=out)
    assert o is out
    again, lse2 = fa().paged_attn_forward(q, k, v, table, ints(lens_k), pu.cumulated(lens_q), 140, causal=True)
    assert torch.equal(o, again) and torch.equal(lse, lse2)
    assert bool((room[:, 0] == 3).all()) and bool((room[:, 9] == 3).all()) and bool((room[..., 96:] == 3).all())
    none, no_lse = fa().paged_attn_forward(q, k, v, table, ints(lens_k), pu.cumulated(lens_q), 140, causal=True, return_lse=False)
    assert no_lse is None and torch.equal(none, again)


@pytest.mark.parametrize("lens_q", [[1, 1, 1, 1], [2, 9, 1, 33], [140, 1, 260, 20]])
@pytest.mark.parametrize("H, Hk", [(4, 4), (8, 2), (10, 2)])
def test_rows_behind_the_last_sequence_are_left(lens_q, H, Hk):
    t = torch.bfloat16
    lens_k = [n + 50 * i for i, n in enumerate(lens_q)]
    k, v, table = pu.make_cache(lens_k, 16, Hk, 64, t, seed=2)
    n = sum(lens_q)
    q = torch.randn(n + 37, H, 64, device="cuda").to(t)
    out = torch.full_like(q, 5.0)
    o, _ = fa().paged_attn_forward(q, k, v, table, ints(lens_k), pu.cumulated(lens_q), max(lens_q), causal=True, out=out)
    assert bool((o[n:] == 5).all())
    want, _ = fa().paged_attn_forward(q[:n], k, v, table, ints(lens_k), pu.cumulated(lens_q), max(lens_q), causal=True)
    assert torch.equal(o[:n], want)
    # and rows before the first
    cu = pu.cumulated(lens_q) + 11
    out.fill_(5.0)
    o, _ = fa().paged_attn_forward(torch.cat((q[n: n + 11], q[:n])), k, v, table, ints(lens_k), cu, max(lens_q), causal=True, out=out[: n + 11])
    assert bool((o[:11] == 5).all()) and torch.equal(o[11:], want)


@pytest.mark.parametrize("lens_q", [[1, 1], [5, 3], [200, 150]])
def test_the_hint_of_the_most_new_tokens_changes_no_result_beyond_rounding(lens_q):
    t = torch.float16
    lens_k = [1000, 333]
    cache = pu.make_cache(lens_k, 32, 2, 128, t, seed=8)
    q = torch.randn(sum(lens_q), 8, 128, device="cuda").to(t)
    for most in (1, 2, 7, 64, 4096):
        attend(q, cache, lens_k, lens_q, t, causal=True, most=most)


def test_long_caches_and_many_sequences():
    t = torch.bfloat16
    lens_k = [70001, 1, 333]
    cache = pu.make_cache(lens_k, 64, 1, 128, t, seed=3)
    attend(torch.randn(3, 4, 128, device="cuda").to(t), cache, lens_k, [1, 1, 1], t, cu=False, causal=True)
    lens_q = [40, 1, 300]
    attend(torch.randn(sum(lens_q), 4, 128, device="cuda").to(t), cache, lens_k, lens_q, t, causal=True)
    lens_k = [1 + (i * 37) % 90 for i in range(1500)]
    cache = pu.make_cache(lens_k, 16, 1, 64, t, seed=3)
    attend(torch.randn(1500, 2, 64, device="cuda").to(t), cache, lens_k, [1] * 1500, t, cu=False, causal=True)
    lens_q = [(i * 7) % 5 for i in range(1500)]
    attend(torch.randn(sum(lens_q), 2, 64, device="cuda").to(t), cache, lens_k, lens_q, t, causal=True)


def test_pages_beyond_four_gigabytes():
    """Element offsets past 2^32: a pool of 4.5 GB whose last pages are the ones in use."""
    t, page, Hk, d = torch.float16, 256, 8, 128
    n_pages = 8704
    k = torch.zeros(n_pages, Hk, page, d, dtype=t, device="cuda")
    v = torch.zeros_like(k)
    assert k.numel() > 2 ** 31 and k.nbytes > 2 ** 32
    lens_k = [600, 90]
    table = torch.full((2, 3), -1, dtype=torch.int32, device="cuda")
    table[0] = ints([n_pages - 1, n_pages - 3, n_pages - 2])
    table[1, 0] = n_pages - 4
    small_k, small_v, small = pu.make_cache(lens_k, page, Hk, d, t, seed=3, spare=0)
    for b in range(2):
        for i in range(-(-lens_k[b] // page)):
            k[table[b, i]], v[table[b, i]] = small_k[small[b, i]], small_v[small[b, i]]
    for lens_q in ([1, 1], [70, 80]):
        q = torch.randn(sum(lens_q), 16, d, device="cuda").to(t)
        o, lse = fa().paged_attn_forward(q, k, v, table, ints(lens_k), pu.cumulated(lens_q), max(lens_q), causal=True)
        want, want_lse = fa().paged_attn_forward(q, small_k, small_v, small, ints(lens_k), pu.cumulated(lens_q), max(lens_q), causal=True)
        assert torch.equal(o, want) and torch.equal(lse, want_lse)
    # the append's slots there too
    new = torch.randn(2, Hk, d, device="cuda").to(t)
    fa().paged_kv_append(new, new, k, v, table, ints([601, 91]))
    assert torch.equal(k[n_pages - 2, :, 600 % page], new[0]) and torch.equal(v[n_pages - 4, :, 90], new[1])


def test_masked_places_may_hold_anything():
    """What no row of a call sees -- slots past the length, pages outside of the window -- is not looked at."""
    t = torch.float16
    lens_k, page = [1000, 650], 16
    for lens_q, (H, Hk) in itertools.product(([1, 1], [3, 2], [40, 100]), ((4, 4), (8, 2))):
        q = torch.randn(sum(lens_q), H, 64, device="cuda").to(t)
        clean = pu.make_cache(lens_k, page, Hk, 64, t, seed=6)
        want = fa().paged_attn_forward(q, *clean, ints(lens_k), pu.cumulated(lens_q), max(lens_q), causal=True, window=(200, -1))
        for value in (float("nan"), float("inf"), -65504.0):
            k, v, table = (x.clone() for x in clean)
            free = table.clone()
            for b, (n, nk) in enumerate(zip(lens_q, lens_k)):
                first = nk - n - 200  # the first key that any row sees
                for p in range(table.shape[1]):
                    for at in range(p * page, (p + 1) * page):
                        if table[b, p] >= 0 and (at < first or at >= nk):
                            k[table[b, p], :, at % page] = value
                            v[table[b, p], :, at % page] = value
                    if (p + 1) * page <= first:
                        free[b, p] = -1 if p % 2 else 10 ** 9  # given back to the pool: not a page any more
            status = torch.zeros(1, dtype=torch.int32, device="cuda")
            got = fa().paged_attn_forward(q, k, v, free, ints(lens_k), pu.cumulated(lens_q), max(lens_q), causal=True, window=(200, -1), status=status)
            assert int(status) == 0
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]), (lens_q, H, value)


@pytest.mark.parametrize("lens_q", [[1, 1, 1], [4, 4, 4], [150, 10, 150]])
def test_a_page_that_is_not_in_the_pool_is_named_and_not_followed(lens_q):
    t = torch.bfloat16
    lens_k = [400, 300, 200]
    k, v, table = pu.make_cache(lens_k, 16, 2, 128, t, seed=6)
    q = torch.randn(sum(lens_q), 4, 128, device="cuda").to(t)
    cu = pu.cumulated(lens_q)
    want, _ = fa().paged_attn_forward(q, k, v, table, ints(lens_k), cu, max(lens_q), causal=True)
    for bad in (-1, k.shape[0], 2 ** 31 - 1, -2 ** 31):
        broken = table.clone()
        broken[1, 3] = bad
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        o, lse = fa().paged_attn_forward(q, k, v, broken, ints(lens_k), cu, max(lens_q), causal=True, status=status)
        torch.cuda.synchronize()
        assert int(status) == 400
        a, b = lens_q[0], lens_q[0] + lens_q[1]
        assert bool(torch.isnan(o[a:b]).all()) and bool(torch.isnan(lse[a:b]).all())
        assert torch.equal(o[:a], want[:a]) and torch.equal(o[b:], want[b:])
    # a length that the table has no pages for
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    o, _ = fa().paged_attn_forward(q, k, v, table, ints([table.shape[1] * 16 + 1, 300, 200]), cu, max(lens_q), causal=True, status=status)
    assert int(status) == 400 and bool(torch.isnan(o[lens_q[0] - 1]).all())
    # lengths and row numbers that make no sense stay inside the tensors
    for lens, rows in (([-5, 300, 200], cu), (lens_k, ints([0, -7, 10 ** 9, 5])), (lens_k, ints([-2 ** 31, 2 ** 31 - 1, 3, 2]))):
        fa().paged_attn_forward(q, k, v, table, ints(lens), rows, max(lens_q), causal=True)
        fa().paged_kv_append(k.new_zeros(sum(lens_q), 2, 128), k.new_zeros(sum(lens_q), 2, 128), k.clone(), v.clone(), table, ints(lens), rows)
    torch.cuda.synchronize()


# ------------------------------------------------------------------ append
@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("H, Hk, d, page, r, interleaved, lens_q", [
    (8, 2, 128, 16, 128, False, [1, 1, 1]), (4, 4, 64, 8, 32, True, [5, 0, 40]), (28, 4, 128, 32, 96, False, [200, 1, 33]),
    (12, 4, 80, 128, 40, False, [3, 17, 2]), (2, 1, 8, 16, 8, True, [9, 9, 9]), (64, 8, 128, 256, 128, True, [1, 700, 1])])
def test_new_tokens_go_to_their_slots(H, Hk, d, page, r, interleaved, lens_q, dtype):
    t = pu.DT[dtype]
    lens_k = [n + x for n, x in zip(lens_q, (0, 100, 333))]
    f, amp = fa().rotary_frequencies(r, scaling="ramp", factor=4.0, original_length=64)
    kp, vp, table = pu.make_cache(lens_k, page, Hk, d, t, seed=d, slots_first=page in (16, 128))
    before_k, before_v = kp.clone(), vp.clone()
    n = sum(lens_q)
    fused = torch.randn(n + 3, H + 2 * Hk, d, device="cuda").to(t)  # (three rows of padding)
    q, k, v = fused[:, :H], fused[:, H: H + Hk], fused[:, H + Hk:]
    out = torch.full((n + 3, H, d), 9.0, device="cuda", dtype=t)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    got = fa().paged_kv_append(k, v, kp, vp, table, ints(lens_k), pu.cumulated(lens_q), q=q, inv_freq=f, amplitude=amp, interleaved=interleaved,
                               out=out, status=status)
    assert got is out and int(status) == 0 and bool((out[n:] == 9).all())
    first = 0
    for b, (m, nk) in enumerate(zip(lens_q, lens_k)):
        at = torch.arange(nk - m, nk)
        rows = slice(first, first + m)
        first += m
        if not m:
            continue
        pages, slots = table[b].cpu().long()[at // page], at % page
        for x, y in ((q[rows], out[rows]), (k[rows], kp[pages.cuda(), :, slots.cuda()])):
            x = x.cpu()
            want = pu.turned(x, at[:, None], f.cpu(), amp, interleaved)
            bound = pu.turn_bound(x, want, t, f.cpu(), at, amp, interleaved)
            assert bool(((y.cpu().double() - want).abs() <= bound).all())
        assert torch.equal(vp[pages.cuda(), :, slots.cuda()], v[rows])
        before_k[pages.cuda(), :, slots.cuda()] = kp[pages.cuda(), :, slots.cuda()]
        before_v[pages.cuda(), :, slots.cuda()] = v[rows]
    assert torch.equal(kp, before_k) and torch.equal(vp, before_v)  # nothing else was touched
    # without a rotation; and q turned in place gives the same
    fa().paged_kv_append(k, v, kp, vp, table, ints(lens_k), pu.cumulated(lens_q))
    at = lens_k[0] - 1
    assert torch.equal(kp[table[0, at // page].long(), :, at % page], k[lens_q[0] - 1])
    want = out[:n].clone()
    fa().paged_kv_append(k, v, kp, vp, table, ints(lens_k), pu.cumulated(lens_q), q=q, inv_freq=f, amplitude=amp, interleaved=interleaved, out=q)
    assert torch.equal(q[:n], want)


def test_rows_at_odd_places_are_appended_element_by_element():
    t, lens = torch.float16, [5, 9]
    f, _ = fa().rotary_frequencies(30)
    raw = torch.randn(14 * 3 * 67 + 1, device="cuda").to(t)
    k = raw[1:].view(14, 3, 67)[..., :64]
    kp, vp, table = pu.make_cache(lens, 8, 3, 64, t, seed=1)
    fa().paged_kv_append(k, k, kp, vp, table, ints(lens), pu.cumulated(lens), inv_freq=f)
    even, even_v, _ = pu.make_cache(lens, 8, 3, 64, t, seed=1)
    fa().paged_kv_append(k.contiguous(), k.contiguous(), even, even_v, table, ints(lens), pu.cumulated(lens), inv_freq=f)
    assert torch.equal(kp, even) and torch.equal(vp, even_v)


def test_a_token_without_a_page_is_dropped_and_named():
    t = torch.bfloat16
    lens = [20, 40]
    kp, vp, table = pu.make_cache(lens, 16, 2, 64, t, seed=1)
    k = torch.randn(2, 2, 64, device="cuda").to(t)
    for bad in (-1, kp.shape[0], 2 ** 31 - 1):
        broken = table.clone()
        broken[1, 2] = bad
        a, b = kp.clone(), vp.clone()
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        fa().paged_kv_append(k, k, a, b, broken, ints(lens), status=status)
        assert int(status) == 400
        changed = (a != kp).any(-1).any(1).nonzero().tolist()
        assert changed == [[int(table[0, 1]), 3]]
    for lens_bad in ([20, 49], [20, 0], [20, -3]):  # beyond the table; before the first position
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        a, b = kp.clone(), vp.clone()
        fa().paged_kv_append(k, k, a, b, table, ints(lens_bad), status=status)
        assert int(status) == 400 and (a != kp).any(-1).any(1).sum() == 1


# ------------------------------------------------------------------ as they are used
def generate(steps, captured):
    """A prompt of each sequence, then steps of one token each, all through the cache; returns the outputs of every step."""
    t, H, Hk, d, page = torch.bfloat16, 8, 2, 64, 16
    g = torch.Generator(device="cuda").manual_seed(77)
    rand = lambda *s: torch.randn(*s, device="cuda", generator=g).to(t)  # noqa: E731
    prompts = [37, 5, 150]
    kp, vp = (torch.full((40, Hk, page, d), float("nan"), device="cuda", dtype=t) for _ in range(2))
    table = torch.arange(39, dtype=torch.int32, device="cuda").view(3, 13).flip(1).contiguous()
    f, _ = fa().rotary_frequencies(d)
    n = sum(prompts)
    q, k, v = rand(n, H, d), rand(n, Hk, d), rand(n, Hk, d)
    kept = [(q, k, v, list(prompts))]
    lens = ints(prompts)
    q = fa().paged_kv_append(k, v, kp, vp, table, lens, pu.cumulated(prompts), q=q, inv_freq=f)
    outs = [fa().paged_attn_forward(q, kp, vp, table, lens, pu.cumulated(prompts), max(prompts), causal=True)]
    q, k, v = rand(3, H, d), rand(3, Hk, d), rand(3, Hk, d)

    def step():
        return fa().paged_attn_forward(fa().paged_kv_append(k, v, kp, vp, table, lens, q=q, inv_freq=f), kp, vp, table, lens, causal=True)
    graph = None
    for _ in range(steps):
        for x in (q, k, v):
            x.copy_(rand(*x.shape))
        kept.append((q.clone(), k.clone(), v.clone(), [1, 1, 1]))
        lens += 1
        if captured:
            if graph is None:
                torch.cuda.synchronize()
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph):
                    out = step()
            graph.replay()
            outs.append(tuple(x.clone() for x in out))
        else:
            outs.append(step())
    torch.cuda.synchronize()
    return kept, outs, f


@pytest.mark.parametrize("captured", [False, True])
def test_a_prompt_and_its_answer_through_the_cache(captured):
    """Every step's output is that of attention over the whole sequence so far, laid out in one piece."""
    kept, outs, f = generate(20, captured)
    t = torch.bfloat16
    whole = [[], [], []]
    for (q, k, v, new), (o, lse) in zip(kept, outs):
        first = 0
        for b, n in enumerate(new):
            rows = slice(first, first + n)
            first += n
            at0 = sum(x[0].shape[0] for x in whole[b])
            at = torch.arange(at0, at0 + n)[:, None]
            turn = lambda x: pu.turned(x[rows].cpu(), at, f.cpu()).to(t)  # noqa: E731, B023
            whole[b].append((turn(k), v[rows].cpu()))
            ks, vs = (torch.cat([x[i] for x in whole[b]]) for i in range(2))
            pool = lambda x: x.transpose(0, 1)[None].contiguous()  # noqa: E731  (one page that holds it all)
            table = torch.zeros(1, 1, dtype=torch.int32)
            want = pu.attention(turn(q), pool(ks), pool(vs), table, [ks.shape[0]], [n], causal=True)
            # K and Q went through 64 bits and one rounding here, through 32 and one there: a tie in a thousand falls the other way,
            # by a step of 2^-8: allowed on every score at once, 2^-8 of scale |q| |k|, it is
            o64, lse64, size, slack = want
            slack = slack * (1 + 2 * 2.0 ** -8 / 1.6e-5 / 64)  # (of 64 products of which one in 64 differs)
            pu.check_attention(o[rows], lse[rows], (o64, lse64, size, slack), t, ks.shape[0])


def test_two_streams_two_workspaces_and_another_device():
    t = torch.bfloat16
    lens_k = [5000, 3000]
    k, v, table = pu.make_cache(lens_k, 16, 1, 128, t, seed=1)
    q = torch.randn(2, 4, 128, device="cuda").to(t)
    want = fa().paged_attn_forward(q, k, v, table, ints(lens_k))
    streams = [torch.cuda.Stream() for _ in range(2)]
    lens = ints(lens_k)
    torch.cuda.synchronize()
    got = []
    for _ in range(20):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(fa().paged_attn_forward(q, k, v, table, lens))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want[0]) and torch.equal(lse, want[1]) for o, lse in got)
    room = torch.empty(64 << 20, dtype=torch.uint8, device="cuda")
    for _ in range(3):
        o, lse = fa().paged_attn_forward(q, k, v, table, lens, workspace=room)
        assert torch.equal(o, want[0]) and torch.equal(lse, want[1])
    small = fa().paged_attn_forward(q, k, v, table, lens, workspace=room[:8])
    assert torch.equal(small[0], want[0])


def test_the_calls_refusals():
    t = torch.float16
    lens = ints([20, 30])
    k, v, table = pu.make_cache([20, 30], 16, 2, 64, t, seed=1)
    q = torch.randn(2, 4, 64, device="cuda").to(t)
    call = fa().paged_attn_forward
    bad = [((q.cpu(), k, v, table, lens), {}), ((q[0], k, v, table, lens), {}), ((q.bfloat16(), k, v, table, lens), {}), ((q, k, v.bfloat16(), table, lens), {}),
           ((q, k[0], v[0], table, lens), {}), ((q, k, v[:1], table, lens), {}), ((q[..., :32], k, v, table, lens), {}), ((q[:, :3], k, v, table, lens), {}),
           ((q, k, v, table.long(), lens), {}), ((q, k, v, table[0], lens), {}), ((q, k, v, table, lens.long()), {}), ((q, k, v, table, lens[:1]), {}),
           ((q, k, v, table, lens, lens), {}), ((q[:1], k, v, table, lens), {}), ((q, k, v, table, lens), dict(out=q[:1])), ((q, k, v, table, lens), dict(alibi_slopes=torch.ones(3))),
           ((q, k.cpu(), v, table, lens), {}), ((q, k, v, table.cpu(), lens), {}), ((q, k, v, table, lens.cpu()), {}),
           ((q.clone().requires_grad_(), k, v, table, lens), {}), ((q, k, v, table, lens), dict(status=torch.zeros(1, dtype=torch.int32))),
           ((q.transpose(1, 2).contiguous().transpose(1, 2), k, v, table, lens), {}), ((q, k, v, table.t().contiguous().t(), lens), {})]
    for i, (args, kw) in enumerate(bad):
        with pytest.raises(ValueError):
            call(*args, **kw)
            raise AssertionError(f"call {i} was taken")
    with pytest.raises(KeyError):
        call(q, k, v, table, lens, out_dtype=torch.float64)
    with pytest.raises(TypeError):
        call(q, k, v, table, lens, window=5)
    from flash_attn_b200._lib import FaError
    for args, kw in [((q, k, v, table, lens), dict(softmax_scale=-1.0)), ((q, k, v, table, lens), dict(out_dtype=torch.bfloat16)),
                     ((q, k[:, :, :12], v[:, :, :12], table, lens), {}), ((q, k, v, table, lens), dict(window=(-2, 0))),
                     ((q, k, v, table, lens, pu.cumulated([1, 1]), 0), {})]:
        with pytest.raises(FaError):
            call(*args, **kw)
    app = fa().paged_kv_append
    f, _ = fa().rotary_frequencies(64)
    kn = torch.randn(2, 2, 64, device="cuda").to(t)
    for args, kw in [((kn.cpu(), kn, k, v, table, lens), {}), ((kn, kn[:1], k, v, table, lens), {}), ((kn.bfloat16(), kn.bfloat16(), k, v, table, lens), {}),
                     ((kn[:, :1], kn[:, :1], k, v, table, lens), {}), ((kn, kn, k, v, table, lens), dict(q=q)), ((kn, kn, k, v, table, lens), dict(out=q)),
                     ((kn, kn, k, v, table, lens), dict(q=q[:1], inv_freq=f)), ((kn, kn, k, v, table, lens), dict(q=q, inv_freq=f.float())),
                     ((kn, kn, k, v, table, lens), dict(inv_freq=fa().rotary_frequencies(66)[0])), ((kn, kn, k, v, table, lens), dict(q=q, inv_freq=f, out=q.bfloat16())),
                     ((kn.clone().requires_grad_(), kn, k, v, table, lens), {})]:
        with pytest.raises(ValueError):
            app(*args, **kw)
    empty = call(q[:0], k, v, table, lens, ints([0, 0, 0]), 1)
    assert empty[0].shape == (0, 4, 64) and empty[1].shape == (0, 4)
    assert app(kn[:0], kn[:0], k, v, table, lens, ints([0, 0, 0])) is None
