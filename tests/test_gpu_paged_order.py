"""The parts of a launch over the paged cache: each is found by its number whatever was asked for before (CTAs are taken in no
promised order), and together they are every item's keys, once."""
import random

import pytest
import torch

import paged_parts_util as pp
import paged_util as pu

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def L():
    return pp.test_library()


def batches():
    r = random.Random(5)
    yield "long single tokens", [1] * 3, [9000, 40, 30000], 8, 2, 128
    yield "single tokens, a warp's sequences", [1] * 32, [r.randint(1, 9000) for _ in range(32)], 16, 4, 64
    yield "single tokens, more of them", [1] * 100, [r.randint(0, 9000) for _ in range(100)], 8, 8, 128
    yield "single tokens, a block's sequences", [1] * 700, [r.choice([0, 3, 200, r.randint(1, 5000)]) for _ in range(700)], 8, 2, 64
    yield "guessed tokens", [5] * 40, [r.randint(5, 6000) for _ in range(40)], 4, 4, 128
    yield "chunks", [r.randint(0, 300) for _ in range(20)], [r.randint(300, 9000) for _ in range(20)], 8, 1, 128
    yield "chunks beside single tokens", [700] + [1] * 50, [9000] + [r.randint(1, 4000) for _ in range(50)], 7, 1, 64


@pytest.mark.parametrize("lens_q, lens_k, H, Hk, d", [x[1:] for x in batches()], ids=[x[0] for x in batches()])
@pytest.mark.parametrize("window", [(-1, -1), (1000, -1)])
def test_parts_are_found_in_any_order(L, lens_q, lens_k, H, Hk, d, window):
    lens, cu = torch.tensor(lens_k, dtype=torch.int32).cuda(), pu.cumulated(lens_q)
    p = pp.params(sum(lens_q), H, Hk, d, lens, cu, max(lens_q), -(-max(lens_k) // 16), window=window)
    found, grid, room, slots = pp.parts(L, p)
    count = sum(x is not None for x in found)
    assert 0 < count <= grid and all(x is not None for x in found[:count])
    # every item's rows and tiles, once
    items = {}
    for x in found[:count]:
        items.setdefault((x["b"], x["head"], x["row0"]), []).append(x)
    rows, taken = {}, set()
    for (b, head, _), of in items.items():
        assert [x["part"] for x in sorted(of, key=lambda x: x["part"])] == list(range(of[0]["parts"]))
        of.sort(key=lambda x: x["part"])
        at = of[0]["lo"]
        for x in of:
            assert (x["slot"], x["parts"], x["n_rows"], x["vis_lo"], x["vis_hi"]) == tuple(of[0][k] for k in ("slot", "parts", "n_rows", "vis_lo", "vis_hi"))
            assert x["lo"] == at
            at += x["n_tiles"]
        lo, hi = of[0]["vis_lo"], of[0]["vis_hi"]
        assert sum(x["n_tiles"] for x in of) == (-(-hi // 128) - lo // 128 if hi > lo else 0)
        rows[b, head] = rows.get((b, head), 0) + of[0]["n_rows"]
        if of[0]["parts"] > 1:
            places = set(range(of[0]["slot"], of[0]["slot"] + of[0]["parts"]))
            assert not places & taken and max(places) < room
            taken |= places
    assert rows == {(b, h): n * (H // Hk) for b, n in enumerate(lens_q) if n for h in range(Hk)}
    # the same whatever comes before
    r = random.Random(1)
    orders = [list(reversed(range(len(found)))), r.sample(range(len(found)), len(found)), [r.randrange(len(found)) for _ in range(500)],
              [len(found) - 1, 0, len(found) - 1, count - 1, count, 0, count // 2]]
    for order in orders:
        again, *_ = pp.parts(L, p, order)
        assert again == [found[i] for i in order]


# cu_seqlens_q that go back and forth: every other sequence claims the same rows, which is more than a launch is sized for
@pytest.mark.parametrize("T, H, Hk, batch, keys, most", [(1, 1, 1, 32, 8192, 1), (1, 1, 1, 200, 8192, 1), (1, 4, 1, 700, 4096, 1), (5, 4, 4, 31, 9000, 5),
                                                         (300, 8, 2, 30, 9000, 300), (300, 8, 2, 600, 3000, 300), (2000, 4, 1, 400, 2500, 2000)])
def test_rows_that_many_sequences_claim_stay_inside_the_workspace(L, T, H, Hk, batch, keys, most):
    lens = torch.full((batch,), keys, dtype=torch.int32, device="cuda")
    cu = torch.tensor([T * (i % 2) for i in range(batch + 1)], dtype=torch.int32).cuda()
    p = pp.params(T, H, Hk, 64, lens, cu, most, -(-keys // 16))
    found, grid, room, _ = pp.parts(L, p)
    seen = {}
    for x in found:
        if x is not None:
            assert x["parts"] == 1 or 0 <= x["slot"] <= room - x["parts"]
            seen.setdefault((x["b"], x["head"], x["row0"]), []).append(x["part"])
            seen[x["b"], x["head"], x["row0"], "of"] = x["parts"]
    assert any(x is not None for x in found) and all(x is None for x in found[grid:])
    for item, of in seen.items():
        if len(item) == 3:  # an item is done with all of its parts, or not at all
            assert sorted(of) == list(range(seen[(*item, "of")]))


@pytest.mark.parametrize("T, H, Hk, batch, keys, most", [(1, 1, 1, 32, 8192, 1), (1, 4, 1, 700, 4096, 1), (300, 8, 2, 30, 9000, 300), (5, 4, 4, 31, 9000, 5)])
def test_a_workspace_outlives_rows_that_many_sequences_claim(T, H, Hk, batch, keys, most):
    import ctypes

    import flash_attn_b200 as fa
    from flash_attn_b200 import _lib
    t, d = torch.bfloat16, 64
    k, v, one = pu.make_cache([keys], 16, Hk, d, t, seed=1)
    table, lens = one.expand(batch, -1).contiguous(), torch.full((batch,), keys, dtype=torch.int32, device="cuda")
    q = torch.randn(T, H, d, device="cuda").to(t)
    good = torch.tensor([0] + [T] * batch, dtype=torch.int32).cuda()
    bad = torch.tensor([T * (i % 2) for i in range(batch + 1)], dtype=torch.int32).cuda()
    need = _lib.load().fa_paged_fwd_workspace_bytes(ctypes.byref(pp.params(T, H, Hk, d, lens, bad, most, table.shape[1])))
    assert need > 0
    room = torch.full((need + (1 << 20),), 0x5a, dtype=torch.uint8, device="cuda")
    call = lambda cu: fa.paged_attn_forward(q, k, v, table, lens, cu, most, causal=True, workspace=room[:need])  # noqa: E731
    want = call(good)
    pu.check_attention(*want, pu.attention(q, k, v, table, [keys], [T], causal=True), t, keys)
    for _ in range(3):
        call(bad)
        got = call(good)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert bool((room[need:] == 0x5a).all())


@pytest.mark.parametrize("lens_q, H, Hk, d", [([1, 1, 1], 4, 1, 64), ([3, 1, 2], 4, 2, 128), ([200, 1, 40], 4, 1, 128), ([300, 1, 40], 4, 1, 64)])
@pytest.mark.parametrize("window", [(-1, -1), (100, -1), (-1, 100)])
@pytest.mark.parametrize("causal", [False, True])
def test_a_length_beyond_the_table_costs_no_more_than_the_table(L, lens_q, H, Hk, d, window, causal):
    """No more tiles than the table has and the first that it lacks; the rows that meet it are NaN, the others as ever."""
    import flash_attn_b200 as fa
    t, room = torch.bfloat16, 512
    cu = pu.cumulated(lens_q)
    k, v, table = pu.make_cache([room, 300, room], 16, Hk, d, t, seed=2)
    q = torch.randn(sum(lens_q), H, d, device="cuda").to(t)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    for far in (room + 1, room + 150, 10 ** 6, 2 ** 30, 2 ** 31 - 1):
        lens = torch.tensor([far, 300, room], dtype=torch.int32).cuda()
        p = pp.params(sum(lens_q), H, Hk, d, lens, cu, max(lens_q), room // 16, causal=causal, window=window)
        walked = {}
        for x in pp.parts(L, p)[0]:
            if x is not None:
                walked[x["b"], x["head"], x["row0"]] = walked.get((x["b"], x["head"], x["row0"]), 0) + x["n_tiles"]
        assert max(walked.values()) <= room // 128 + 1
        status.zero_()
        o, lse = fa.paged_attn_forward(q, k, v, table, lens, cu, max(lens_q), causal=causal, window=window, status=status)
        assert int(status) == 400
        # the last row sees its own place, which the table has no page for (a causal row before the table's end sees none such)
        assert bool(o[lens_q[0] - 1].isnan().all()) and bool(lse[lens_q[0] - 1].isnan().all())
        if far >= 10 ** 6:
            assert bool(o[: lens_q[0]].isnan().all()) and bool(lse[: lens_q[0]].isnan().all())
        n = lens_q[0]
        want = pu.attention(q[n:], k, v, table[1:], [300, room], lens_q[1:], causal=causal, window=window)
        pu.check_attention(o[n:], lse[n:], want, t, room)
