"""How a launch over the paged cache is shared out: many sequences, long ones cut into parts, parts of many items a CTA, pools in any
layout, workspaces that hold anything.  Against the 64-bit form of tests/paged_util.py, and bit by bit against other layouts."""
import random

import pytest
import torch

import paged_util as pu

pytestmark = pytest.mark.gpu


def fa():
    import flash_attn_b200
    return flash_attn_b200


def ints(x):
    return torch.tensor(x, dtype=torch.int32).cuda()


def made(lens_q, lens_k, H, Hk, d, page, t, seed=0, **kw):
    k, v, table = pu.make_cache(lens_k, page, Hk, d, t, seed, **kw)
    g = torch.Generator().manual_seed(seed + 1)
    q = torch.randn(sum(lens_q), H, d, generator=g).to(t).cuda()
    return q, k, v, table


def run(q, k, v, table, lens_q, lens_k, **kw):
    cu = None if all(n == 1 for n in lens_q) else pu.cumulated(lens_q)
    return fa().paged_attn_forward(q, k, v, table, ints(lens_k), cu, max(lens_q), **kw)


def check(got, q, k, v, table, lens_q, lens_k, t, out_dtype=None, **kw):
    want = pu.attention(q, k, v, table, lens_k, lens_q, **kw)
    pu.check_attention(got[0], got[1], want, t, max(lens_k), out_dtype)


# 32 sequences are a lane's each, up to 256 one warp's, more the block's
@pytest.mark.parametrize("B", [31, 32, 33, 65, 256, 257, 700])
def test_single_tokens_of_many_sequences(B):
    r, t = random.Random(B), torch.bfloat16
    lens_k = [r.choice([1, 2, 127, 128, 129, r.randint(1, 700)]) for _ in range(B)]
    q, k, v, table = made([1] * B, lens_k, 4, 2, 64, 16, t)
    check(run(q, k, v, table, [1] * B, lens_k, causal=True), q, k, v, table, [1] * B, lens_k, t, causal=True)


@pytest.mark.parametrize("B, most", [(33, 5), (40, 40), (257, 3), (300, 70)])
def test_chunks_of_many_sequences_some_empty(B, most):
    r, t = random.Random(B), torch.float16
    lens_q = [r.choice([0, 1, r.randint(0, most)]) for _ in range(B)]
    lens_q[B // 2] = most
    lens_k = [n + r.choice([0, 0, r.randint(0, 300)]) for n in lens_q]
    q, k, v, table = made(lens_q, lens_k, 4, 1, 64, 16, t)
    check(run(q, k, v, table, lens_q, lens_k, causal=True), q, k, v, table, lens_q, lens_k, t, causal=True)


@pytest.mark.parametrize("lens_q, lens_k", [([1] * 3, [9000, 40, 30000]), ([3] * 2, [20000, 6001]), ([40, 1, 40], [12000, 9000, 41])])
@pytest.mark.parametrize("H, Hk, d", [(8, 2, 128), (7, 1, 80), (16, 1, 64), (2, 2, 96)])
def test_long_sequences_are_cut_and_put_together_the_same_way_each_time(H, Hk, d, lens_q, lens_k):
    t = torch.bfloat16
    q, k, v, table = made(lens_q, lens_k, H, Hk, d, 32, t)
    got = run(q, k, v, table, lens_q, lens_k, causal=True)
    check(got, q, k, v, table, lens_q, lens_k, t, causal=True)
    for _ in range(10):
        again = run(q, k, v, table, lens_q, lens_k, causal=True)
        assert torch.equal(again[0], got[0]) and torch.equal(again[1], got[1])


@pytest.mark.parametrize("lens_q", [[1, 1, 1], [150, 1, 70]])
@pytest.mark.parametrize("d, page", [(128, 16), (128, 256), (64, 8), (96, 32)])
def test_a_pools_layout_changes_nothing(d, page, lens_q):
    """Whole-row boxes, half-row boxes and their coordinates: the same keys and values wherever they lie."""
    t, Hk, lens_k = torch.bfloat16, 3, [500, 131, 1000]
    q, k, v, table = made(lens_q, lens_k, 6, Hk, d, page, t)
    n = k.shape[0]
    want = run(q, k, v, table, lens_q, lens_k, causal=True)
    check(want, q, k, v, table, lens_q, lens_k, t, causal=True)

    def laid(x, shape, cut):
        room = torch.full(shape, float("nan"), dtype=t, device="cuda")
        view = cut(room)
        view.copy_(x)
        return view
    layouts = {
        "slots first": lambda x: laid(x, (n, page, Hk, d), lambda r: r.transpose(1, 2)),
        "heads first": lambda x: laid(x, (Hk, n, page, d), lambda r: r.transpose(0, 1)),
        "beside others": lambda x: laid(x, (n, 2, Hk, page, d), lambda r: r[:, 1]),
        "wide slots": lambda x: laid(x, (n, Hk, page, d + 8), lambda r: r[..., :d]),
        "odd pages": lambda x: laid(x, (n, Hk * page * d + 8), lambda r: r[:, : Hk * page * d].view(n, Hk, page, d)),
        "odd heads": lambda x: laid(x, (n, Hk, page * d + 8), lambda r: r[..., : page * d].unflatten(-1, (page, d))),
    }
    for name, lay in layouts.items():
        for a, b in ((lay(k), lay(v)), (k, lay(v))):  # (both ways, and each pool its own)
            got = run(q, a, b, table, lens_q, lens_k, causal=True)
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]), name


@pytest.mark.parametrize("H, Hk, d", [(8, 2, 128), (4, 4, 128), (14, 2, 64), (32, 1, 128), (8, 2, 80)])
@pytest.mark.parametrize("wide, out_dtype", [(0, None), (4, None), (8, None), (0, torch.float32)])
def test_rows_of_chunks_are_written_where_they_belong(H, Hk, d, wide, out_dtype):
    """By TMA where 32 rows are whole tokens, by hand where they are not, in strides of 4 and 8 elements; nothing beside them."""
    t, lens_q, lens_k = torch.bfloat16, [129, 3, 70], [129, 900, 4000]
    q, k, v, table = made(lens_q, lens_k, H, Hk, d, 16, t)
    T = sum(lens_q)
    room = torch.full((T + 2, H, d + wide), 77.0, dtype=out_dtype or t, device="cuda")
    out = room[1: T + 1, :, :d]
    got = run(q, k, v, table, lens_q, lens_k, causal=True, out=out, out_dtype=out_dtype)
    check((out, got[1]), q, k, v, table, lens_q, lens_k, t, out_dtype, causal=True)
    assert bool((room[0] == 77).all()) and bool((room[T + 1] == 77).all()) and bool((room[..., d:] == 77).all())


def test_a_workspace_may_hold_anything_and_serve_one_call_behind_another():
    t = torch.bfloat16
    calls = []
    for lens_q, lens_k, H, Hk, d in [([1, 1], [9000, 20000], 8, 1, 128), ([60, 60], [8000, 9000], 4, 1, 64), ([200], [7000], 8, 1, 128), ([4], [30000], 4, 4, 64)]:
        args = made(lens_q, lens_k, H, Hk, d, 16, t)
        calls.append((args, lens_q, lens_k, run(*args, lens_q, lens_k, causal=True)))
    g = torch.Generator(device="cuda").manual_seed(3)
    for fill in (0x00, 0xff, 0x9d, None):
        room = torch.empty(64 << 20, dtype=torch.uint8, device="cuda")
        if fill is None:
            room.random_(0, 256, generator=g)
        else:
            room.fill_(fill)
        for _ in range(3):
            for args, lens_q, lens_k, want in calls:
                got = run(*args, lens_q, lens_k, causal=True, workspace=room)
                assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]), fill


def test_two_captured_calls_share_a_workspace_and_follow_the_lengths():
    """Replayed one behind the other on lengths that were not those of the capture: from one part to many and back."""
    t, H, Hk, d, page = torch.float16, 8, 2, 128, 16
    most = [20000, 3000, 700]
    q1, k, v, table = made([1] * 3, most, H, Hk, d, page, t)
    q2 = torch.randn(90, H, d, device="cuda").to(t)
    lens, cu, room = ints([1, 1, 1]), ints([0, 0, 0, 0]), torch.empty(64 << 20, dtype=torch.uint8, device="cuda")
    one = lambda: fa().paged_attn_forward(q1, k, v, table, lens, causal=True, workspace=room)  # noqa: E731
    many = lambda: fa().paged_attn_forward(q2, k, v, table, lens, cu, 90, causal=True, workspace=room)  # noqa: E731
    one(), many()
    torch.cuda.synchronize()
    graphs = []
    for f in (one, many):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = f()
        graphs.append((graph, out))
    for lens_k, lens_q in [(most, [30, 0, 60]), ([1, 1, 1], [1, 1, 1]), ([5000, 3000, 1], [90, 0, 0]), ([20000, 128, 129], [0, 45, 45]), (most, [1, 1, 88])]:
        lens.copy_(ints(lens_k))
        cu.copy_(pu.cumulated(lens_q))
        for graph, _ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        check(graphs[0][1], q1, k, v, table, [1] * 3, lens_k, t, causal=True)
        n = sum(lens_q)
        check(tuple(x[:n] for x in graphs[1][1]), q2[:n], k, v, table, lens_q, lens_k, t, causal=True)


@pytest.mark.parametrize("lens_q", [[1], [5], [64]])
def test_a_length_beyond_the_table_is_named_and_every_row_is_written(lens_q):
    t = torch.bfloat16
    q, k, v, table = made(lens_q, [256], 4, 1, 64, 16, t)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    for far in (257, 100_000, 2 ** 31 - 1):
        out = torch.zeros_like(q)
        status.zero_()
        o, lse = fa().paged_attn_forward(q, k, v, table, ints([far]), pu.cumulated(lens_q), max(lens_q), window=(300, -1), out=out, status=status)
        assert int(status) == 400 and bool(o.isnan().all()) and bool(lse.isnan().all()), far
    got = run(q, k, v, table, lens_q, [256], causal=True)
    check(got, q, k, v, table, lens_q, [256], t, causal=True)
