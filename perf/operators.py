"""What the operators around a paged K/V cache are measured on: rotary positions, the append of new tokens to the cache's
pages, and the attention of new tokens over them -- the three calls that a layer of a serving step makes, and the first of
them as training makes it, with its gradient.

A case is a plain dict:
  op     "rotary":  one rotary_embedding of a [B, H, N, d] tensor (packed: [N, H, d], positions in any order)
         "append":  one paged_kv_append of the new tokens of B sequences, Q rotated beside K
         "attend":  one paged_attn_forward of the new tokens of B sequences over their pages
  dtype, H, Hk, d;  rotary_dim, interleaved, scaling, factor (of the rotation)
  B, chunks, q_lo, q_hi, k_lo, k_hi, lens_seed: the first `chunks` sequences bring q_lo .. q_hi new tokens, the others one;
         a cache holds k_lo .. k_hi tokens with the new ones (never fewer than those)
  page   tokens of a page;  slots_first: pages are [page_size, heads_k, d] in memory, else [heads_k, page_size, d]
  causal, window_left, alibi
"""
import math
import random

import numpy as np
import torch

own = False

_DT = {"float16": torch.float16, "bfloat16": torch.bfloat16, "float32": torch.float32}
_ROTARY = dict(op="rotary", dtype="bfloat16", B=1, H=1, N=1, d=128, rotary_dim=128, interleaved=False, inverse=False, packed=False,
               scaling="none", factor=1.0, far=4096)
_CACHE = dict(dtype="bfloat16", B=1, H=32, Hk=8, d=128, chunks=0, q_lo=1, q_hi=1, k_lo=1, k_hi=1, lens_seed=0, page=16, slots_first=False)
_APPEND = dict(_CACHE, op="append", rotary_dim=128, interleaved=False, scaling="none", factor=1.0)
_ATTEND = dict(_CACHE, op="attend", causal=True, window_left=-1, alibi=False)


def listed():
    return [
        # Q of a training or prompt pass in the layout of flash_attn_forward, positions interpolated for a long context
        dict(_ROTARY, name="rotary_heads", B=4, H=32, N=4096, scaling="linear", factor=4.0),
        # the gradient of a rotation of part of the head, neighbouring columns paired, kept in 32 bits; odd length
        dict(_ROTARY, name="rotary_gradient", dtype="float32", B=2, H=24, N=1501, d=96, rotary_dim=64, interleaved=True, inverse=True),
        # a decode step of a full batch: one new token a sequence
        dict(_APPEND, name="append_step", B=64, k_lo=100, k_hi=8192, lens_seed=1),
        # prompts of several requests going into the cache at once, scaled rotation
        dict(_APPEND, name="append_prompts", B=6, chunks=6, q_lo=500, q_hi=4000, k_lo=1, k_hi=1, lens_seed=2, scaling="ramp", factor=8.0),
        # one request being answered: latency
        dict(_ATTEND, name="decode_one", k_lo=1000, k_hi=1000, lens_seed=3),
        # a decode step of a full batch of requests of unequal lengths
        dict(_ATTEND, name="decode_batch", B=64, k_lo=100, k_hi=8192, lens_seed=4),
        # few requests with long contexts
        dict(_ATTEND, name="decode_long", B=4, k_lo=98304, k_hi=131072, lens_seed=5, page=64),
        # the check of four guessed tokens, a head of K/V for each query head, 64-wide heads
        dict(_ATTEND, name="verify_d64", dtype="float16", B=24, H=16, Hk=16, d=64, chunks=24, q_lo=5, q_hi=5, k_lo=500, k_hi=4000,
             lens_seed=6, page=32, slots_first=True),
        # prompts of several requests at once, nothing cached before
        dict(_ATTEND, name="prompts", B=6, chunks=6, q_lo=200, q_hi=2048, k_lo=1, k_hi=1, lens_seed=7),
        # the next part of two long documents with a sliding window and ALiBi
        dict(_ATTEND, name="local_chunks", dtype="float16", B=2, H=16, Hk=4, d=64, chunks=2, q_lo=700, q_hi=1100, k_lo=9000, k_hi=16000,
             lens_seed=8, page=128, window_left=1024, alibi=True),
        # a step that carries a part of a prompt beside the decodes of other requests
        dict(_ATTEND, name="mixed", B=33, chunks=1, q_lo=512, q_hi=512, k_lo=512, k_hi=8192, lens_seed=9),
        # the last part of a long prompt
        dict(_ATTEND, name="long_chunk", chunks=1, q_lo=2048, q_hi=2048, k_lo=32768, k_hi=32768, lens_seed=10, page=64),
    ]


# ------------------------------------------------------------------ more of the same
def _log_int(r, lo, hi):
    return int(round(math.exp(r.uniform(math.log(lo), math.log(hi)))))


def _rotation(r, d):
    part = r.choice([d, d, d // 2 // 8 * 8])
    scaling = r.choice(["none", "none", "linear", "ntk", "ramp"])
    return dict(rotary_dim=part, interleaved=r.random() < 0.4, scaling=scaling, factor=1.0 if scaling == "none" else r.choice([2.0, 4.0, 8.0]))


def _draw_rotary(r):
    d = r.choice([64, 80, 96, 128, 128])
    n = _log_int(r, 1, 8192)
    return dict(_ROTARY, dtype=r.choice(["float16", "bfloat16", "bfloat16", "float32"]), B=max(1, min(8, _log_int(r, 1, 16384) // n)),
                H=r.choice([1, 8, 16, 24, 32]), N=n, d=d, inverse=r.random() < 0.4, packed=r.random() < 0.5, far=_log_int(r, 4096, 1048576),
                **_rotation(r, d))


def _cache(r):
    h, hk = r.choice([(32, 8), (32, 8), (16, 16), (28, 4), (64, 8), (16, 2), (8, 1)])
    return dict(dtype=r.choice(["float16", "bfloat16"]), H=h, Hk=hk, d=r.choice([64, 128, 128, 96, 80]), page=r.choice([8, 16, 16, 32, 64, 128, 256]),
                slots_first=r.random() < 0.4, lens_seed=r.randrange(1 << 30))


def _draw_append(r):
    c = _cache(r)
    b = _log_int(r, 1, 128)
    chunks = r.choice([0, 0, b, r.randint(0, b)])
    most = max(1, min(4000, 16384 // max(1, chunks)))
    return dict(_APPEND, **c, **_rotation(r, c["d"]), B=b, chunks=chunks, q_lo=1, q_hi=most, k_lo=1, k_hi=_log_int(r, 16, 65536 // b + 16))


def _draw_decode(r):
    c = _cache(r)
    k = _log_int(r, 64, 65536)
    b = max(1, min(128, _log_int(r, 512, 262144) // k))
    n = r.choice([1, 1, 1, r.randint(2, 8)])
    return dict(_ATTEND, **c, B=b, chunks=b if n > 1 else 0, q_lo=n, q_hi=n, k_lo=max(1, int(k * r.choice([0.02, 0.2, 1.0]))), k_hi=k,
                window_left=r.choice([-1, -1, -1, 1024]), alibi=r.random() < 0.2)


def _draw_chunks(r):
    c = _cache(r)
    q = _log_int(r, 16, 2048)
    k = _log_int(r, q, 15000)
    # (what the plain form holds at once: every head's scores of the longest of both, twice over)
    most = max(1, 500_000_000 // (c["H"] * q * max(q, k)))
    b = min(most, _log_int(r, 1, 24))
    return dict(_ATTEND, **c, B=b, chunks=r.choice([b, b, max(1, b // 4)]), q_lo=max(1, q // 8), q_hi=q, k_lo=1, k_hi=k,
                causal=r.random() < 0.85, window_left=r.choice([-1, -1, -1, 512]), alibi=r.random() < 0.2)


def draw(rng):
    return rng.choice([_draw_rotary, _draw_append, _draw_decode, _draw_decode, _draw_chunks, _draw_chunks])(rng)


# ------------------------------------------------------------------ inputs
def _lengths(c):
    """New tokens and cached tokens (the new ones among them) of each sequence: the case's own, whatever the seed."""
    r = random.Random(c["lens_seed"])
    n = [_log_int(r, c["q_lo"], c["q_hi"]) if b < c["chunks"] else 1 for b in range(c["B"])]
    return n, [max(x, _log_int(r, c["k_lo"], c["k_hi"])) for x in n]


def _frequencies(c, device):
    """Angle of each pair a position (64 bits) and the amplitude of the rotation."""
    r, f = c["rotary_dim"], c["factor"]
    i = torch.arange(r // 2, dtype=torch.float64)
    if c["scaling"] == "ntk":
        return torch.pow(10000.0 * f ** (r / (r - 2)), -2 * i / r).to(device), 1.0
    w = torch.pow(torch.tensor(10000.0, dtype=torch.float64), -2 * i / r)
    if c["scaling"] == "linear":
        return (w / f).to(device), 1.0
    if c["scaling"] == "ramp":
        turns = 4096 * w / (2 * math.pi)  # over the length that was trained on
        keep = ((turns - 1.0) / (32.0 - 1.0)).clamp(0.0, 1.0)
        return (w * keep + w / f * (1 - keep)).to(device), 0.1 * math.log(f) + 1.0
    return w.to(device), 1.0


def prepare(case, seed):
    c = case
    dev, dt = "cuda", _DT[c["dtype"]]
    g = torch.Generator(device=dev).manual_seed(seed)
    rand = lambda *shape: torch.randn(*shape, device=dev, dtype=dt, generator=g)  # noqa: E731
    s = {"case": c}
    if c["op"] == "rotary":
        s["inv_freq"], s["amplitude"] = _frequencies(c, dev)
        if c["packed"]:  # the tokens of many sequences one behind the other
            s["x"] = rand(c["B"] * c["N"], c["H"], c["d"])
            s["positions"] = torch.randint(0, c["far"], (c["B"] * c["N"],), device=dev, generator=g)
        else:
            s["x"] = rand(c["B"], c["H"], c["N"], c["d"])
            s["positions"] = torch.arange(c["N"], device=dev) + max(0, c["far"] - c["N"])
        return s
    n, k = _lengths(c)
    pages = [-(-x // c["page"]) for x in k]
    total, width = sum(pages), max(pages)
    shape = (total + 3, c["page"], c["Hk"], c["d"]) if c["slots_first"] else (total + 3, c["Hk"], c["page"], c["d"])
    pools = [rand(*shape) for _ in range(2)]
    s["k_pages"], s["v_pages"] = [p.transpose(1, 2) if c["slots_first"] else p for p in pools]
    order = torch.randperm(total + 3, device=dev, generator=g)[:total].to(torch.int32)
    held = torch.arange(width)[None] < torch.tensor(pages)[:, None]
    s["page_table"] = torch.full((c["B"], width), -1, dtype=torch.int32, device=dev)
    s["page_table"][held.to(dev)] = order
    s["seqlens_k"] = torch.tensor(k, dtype=torch.int32).to(dev)
    s["cu_seqlens_q"] = torch.tensor([0] + list(np.cumsum(n)), dtype=torch.int32).to(dev) if c["chunks"] else None
    s["max_seqlen_q"] = max(n)
    s["q"] = rand(sum(n), c["H"], c["d"])
    if c["op"] == "append":
        s["inv_freq"], s["amplitude"] = _frequencies(c, dev)
        s["k"], s["v"] = rand(sum(n), c["Hk"], c["d"]), rand(sum(n), c["Hk"], c["d"])
    elif c["alibi"]:
        s["slopes"] = torch.pow(2.0, -8.0 * torch.arange(1, c["H"] + 1, dtype=torch.float32) / c["H"]).to(dev)
    return s


# ------------------------------------------------------------------ plain forms
def _rotated(x, positions, inv_freq, amplitude, interleaved, inverse):
    """x [..., heads or rows, d] in 32 bits; positions broadcast against its leading dimensions."""
    r = 2 * inv_freq.numel()
    angle = positions[..., None].double() * inv_freq
    cos, sin = (angle.cos() * amplitude).float(), (angle.sin() * (-amplitude if inverse else amplitude)).float()
    part, rest = x[..., :r].float(), x[..., r:].float()
    if interleaved:
        a, b = part[..., 0::2], part[..., 1::2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = part[..., : r // 2], part[..., r // 2:]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((turned, rest), -1).to(x.dtype)


def _places(s, tokens):
    """Sequence, place among its new tokens and position of each new token."""
    k = s["seqlens_k"].long()
    if s["cu_seqlens_q"] is None:
        seq = torch.arange(tokens, device=k.device)
        return seq, torch.zeros_like(seq), k - 1
    cu = s["cu_seqlens_q"].long()
    at = torch.arange(tokens, device=k.device)
    seq = torch.bucketize(at, cu[1:], right=True)
    return seq, at - cu[seq], k[seq] - cu[seq + 1] + at


def _plain_append(s):
    seq, _, position = _places(s, s["k"].shape[0])
    turn = lambda x: _rotated(x, position[:, None], s["inv_freq"], s["amplitude"], s["case"]["interleaved"], False)  # noqa: E731
    page = s["page_table"][seq, position // s["case"]["page"]].long()
    slot = position % s["case"]["page"]
    s["k_pages"][page, :, slot] = turn(s["k"])
    s["v_pages"][page, :, slot] = s["v"]
    return turn(s["q"])


def _plain_attention(s):
    c, q = s["case"], s["q"]
    B, P = s["page_table"].shape
    H, Hk, d, n = c["H"], c["Hk"], c["d"], s["max_seqlen_q"]
    seq, place, position = _places(s, q.shape[0])
    rows = torch.zeros(B, n, H, d, device=q.device)
    rows[seq, place] = q.float()
    rows = rows.reshape(B, n, Hk, H // Hk, d).permute(0, 2, 3, 1, 4).reshape(B, Hk, H // Hk * n, d)
    table = s["page_table"].clamp(min=0).long()
    gather = lambda pages: pages[table].permute(0, 2, 1, 3, 4).reshape(B, Hk, P * c["page"], d).float()  # noqa: E731
    score = torch.matmul(rows, gather(s["k_pages"]).transpose(2, 3)).mul_(d ** -0.5).view(B, Hk, H // Hk, n, P * c["page"])
    key = torch.arange(P * c["page"], device=q.device)
    at = torch.zeros(B, n, dtype=torch.long, device=q.device)
    at[seq, place] = position
    ahead = key - at[..., None]  # [B, n, keys]
    hidden = (key >= s["seqlens_k"].long()[:, None])[:, None, :] | torch.zeros_like(ahead, dtype=torch.bool)
    if c["causal"]:
        hidden |= ahead > 0
    if c["window_left"] >= 0:
        hidden |= -ahead > c["window_left"]
    if c["alibi"]:
        score -= s["slopes"].view(Hk, H // Hk, 1, 1) * ahead.abs().float()[:, None, None]
    score.masked_fill_(hidden[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    p = score.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p.view(B, Hk, H // Hk * n, P * c["page"]), gather(s["v_pages"])).view(B, Hk, H // Hk, n, d)
    out = torch.where(total > 0, out / total, 0.0)
    lse = (top + total.log()).squeeze(-1)
    out = out.permute(0, 3, 1, 2, 4).reshape(B, n, H, d)[seq, place].to(q.dtype)
    return out, lse.permute(0, 3, 1, 2).reshape(B, n, H)[seq, place]


# ------------------------------------------------------------------ one pass
def run(state):
    s, c = state, state["case"]
    if own:
        import flash_attn_b200 as fa
        if c["op"] == "rotary":
            return fa.rotary_embedding(s["x"], s["positions"], s["inv_freq"], s["amplitude"], interleaved=c["interleaved"], inverse=c["inverse"])
        if c["op"] == "append":
            q = fa.paged_kv_append(s["k"], s["v"], s["k_pages"], s["v_pages"], s["page_table"], s["seqlens_k"], s["cu_seqlens_q"], q=s["q"],
                                   inv_freq=s["inv_freq"], amplitude=s["amplitude"], interleaved=c["interleaved"])
            return {"q": q, "k_pages": s["k_pages"], "v_pages": s["v_pages"]}
        return fa.paged_attn_forward(s["q"], s["k_pages"], s["v_pages"], s["page_table"], s["seqlens_k"], s["cu_seqlens_q"], s["max_seqlen_q"],
                                     causal=c["causal"], window=(c["window_left"], -1), alibi_slopes=s.get("slopes"))
    if c["op"] == "rotary":
        positions = s["positions"][:, None] if c["packed"] else s["positions"]
        return _rotated(s["x"], positions, s["inv_freq"], s["amplitude"], c["interleaved"], c["inverse"])
    if c["op"] == "append":
        return {"q": _plain_append(s), "k_pages": s["k_pages"], "v_pages": s["v_pages"]}
    return _plain_attention(s)


# ------------------------------------------------------------------ what a pass cannot do without
def _visible(c, n, k):
    """(query, key) pairs that the masks leave, and the keys that any query sees, of one sequence."""
    at = np.arange(k - n, k, dtype=np.int64)
    hi = np.minimum(at + 1, k) if c["causal"] else np.full(n, k)
    lo = np.maximum(at - c["window_left"], 0) if c["window_left"] >= 0 else np.zeros(n, dtype=np.int64)
    return int(np.maximum(hi - lo, 0).sum()), int(hi.max() - lo.min())


def work(case):
    c = case
    e = 4 if c["dtype"] == "float32" else 2
    if c["op"] == "rotary":
        x = c["B"] * c["H"] * c["N"]
        return {"bytes": 2 * x * c["d"] * e + 8 * c["N"] * (c["B"] if c["packed"] else 1), "flops": 3 * x * c["rotary_dim"]}
    n, k = _lengths(c)
    t = sum(n)
    if c["op"] == "append":
        return {"bytes": 2 * t * (c["H"] + 2 * c["Hk"]) * c["d"] * e, "flops": 3 * t * (c["H"] + c["Hk"]) * c["rotary_dim"]}
    seen = [_visible(c, *x) for x in zip(n, k)]
    return {"bytes": 2 * t * c["H"] * c["d"] * e + 4 * t * c["H"] + 2 * sum(x[1] for x in seen) * c["Hk"] * c["d"] * e,
            "flops": 4 * c["d"] * c["H"] * sum(x[0] for x in seen)}


# ------------------------------------------------------------------ the same in 64 bits
def _turn64(x, position, inv_freq, amplitude, interleaved, inverse):
    """Rows [n, heads, d] by complex multiplication, one position a row."""
    r = 2 * inv_freq.numel()
    x = x.double()
    pairs = x[..., :r].reshape(*x.shape[:-1], r // 2, 2) if interleaved else x[..., :r].reshape(*x.shape[:-1], 2, r // 2).transpose(-1, -2)
    phase = position.double()[:, None, None] * inv_freq
    z = torch.view_as_complex(pairs.contiguous()) * torch.polar(torch.full_like(phase, amplitude), -phase if inverse else phase)
    pairs = torch.view_as_real(z)
    return torch.cat(((pairs if interleaved else pairs.transpose(-1, -2)).reshape(*x.shape[:-1], r), x[..., r:]), -1)


def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["op"] == "rotary":
        turn = lambda x: _turn64(x, s["positions"], s["inv_freq"], s["amplitude"], c["interleaved"], c["inverse"])  # noqa: E731
        if c["packed"]:
            return turn(s["x"])
        return torch.stack([turn(x.transpose(0, 1)).transpose(0, 1) for x in s["x"]])
    n, k = _lengths(c)
    dev, first = s["q"].device, 0
    if c["op"] == "append":
        q, kp, vp = torch.empty_like(s["q"], dtype=torch.float64), s["k_pages"].double(), s["v_pages"].double()
        for b in range(c["B"]):
            rows = slice(first, first + n[b])
            at = torch.arange(k[b] - n[b], k[b], device=dev)
            turn = lambda x: _turn64(x[rows], at, s["inv_freq"], s["amplitude"], c["interleaved"], False)  # noqa: E731
            q[rows] = turn(s["q"])
            where = (s["page_table"][b].long()[at // c["page"]], slice(None), at % c["page"])
            kp[where], vp[where] = turn(s["k"]), s["v"][rows].double()
            first += n[b]
        return {"q": q, "k_pages": kp, "v_pages": vp}
    out = torch.empty_like(s["q"], dtype=torch.float64)
    lse = torch.empty(s["q"].shape[:2], dtype=torch.float64, device=dev)
    group = c["H"] // c["Hk"]
    for b in range(c["B"]):
        rows, at, key = slice(first, first + n[b]), torch.arange(k[b] - n[b], k[b], device=dev), torch.arange(k[b], device=dev)
        first += n[b]
        pages = s["page_table"][b, : -(-k[b] // c["page"])].long()
        seen = torch.ones(n[b], k[b], dtype=torch.bool, device=dev)
        if c["causal"]:
            seen &= key[None] <= at[:, None]
        if c["window_left"] >= 0:
            seen &= key[None] >= at[:, None] - c["window_left"]
        for h in range(c["H"]):
            keys, values = (s[x][pages, h // group].reshape(-1, c["d"])[: k[b]].double() for x in ("k_pages", "v_pages"))
            score = s["q"][rows, h].double() @ keys.T / math.sqrt(c["d"])
            if c["alibi"]:
                score = score - float(s["slopes"][h]) * (at[:, None] - key[None]).abs()
            score = torch.where(seen, score, -math.inf)
            lse[rows, h] = score.logsumexp(-1)
            out[rows, h] = score.softmax(-1) @ values
    return out, lse
