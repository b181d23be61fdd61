"""Serving from a paged K/V cache, on torch tensors: rotary positions, the append of new tokens to their pages, and the
attention of the new tokens over what the cache holds.

The cache is a pool `k_pages`, `v_pages` [num_pages, heads_k, page_size, head_dim] (fp16 or bf16; any strides of the first three
dimensions, so a pool that is [num_pages, page_size, heads_k, head_dim] in memory is given as `pool.transpose(1, 2)`).  Token t of
sequence b lies in page `page_table[b, t // page_size]` (int32 [batch, pages]), slot `t % page_size`; `seqlens_k` (int32 [batch])
counts the tokens of each sequence, the new ones of this step included.  The new tokens of all sequences are rows one behind the
other, `cu_seqlens_q[b] .. cu_seqlens_q[b + 1]` (int32 [batch + 1], ascending) those of sequence b; without it there is one row a sequence.
The j-th of n new tokens has position `seqlens_k[b] - n + j`.  Rows behind the last sequence are left as they were.

Lengths and tables live on the device and are read there, so a step can be captured into a CUDA graph and replayed on new ones.
A step of a layer is `q = paged_kv_append(k, v, ..., q=q, inv_freq=f)`, then `paged_attn_forward(q, ...)`.

Nothing here is recorded by autograd: a tensor that requires grad, whichever argument it is, is refused while grad mode is on, and so is
one with a forward-mode tangent.  The gradient of
rotary_embedding is rotary_embedding(grad, ..., inverse=True).
"""
import ctypes

import torch

from . import _lib

_KINDS = {None: _lib.FA_ROTARY_PLAIN, "linear": _lib.FA_ROTARY_LINEAR, "ntk": _lib.FA_ROTARY_NTK, "ramp": _lib.FA_ROTARY_RAMP}


def rotary_frequencies(rotary_dim, base=10000.0, scaling=None, factor=1.0, original_length=None, low_turns=1.0, high_turns=32.0,
                       device="cuda"):
    """(inv_freq, amplitude): float64 [rotary_dim / 2] on `device`, what each pair of columns turns by from one position to the
    next, and what the turned columns are multiplied by.

    `scaling` None: base^(-2 i / rotary_dim).  "linear": divided by `factor`.  "ntk": the base raised to
    base * factor^(rotary_dim / (rotary_dim - 2)).  "ramp": pairs that make `low_turns` or fewer over `original_length` positions
    are divided by `factor`, those that make `high_turns` or more are kept, linearly between; amplitude 0.1 ln(factor) + 1 (1 for
    the others; a model that was trained with another passes its own to the calls)."""
    if scaling not in _KINDS:
        raise ValueError(f"scaling must be one of {', '.join(map(repr, _KINDS))}")
    if scaling == "ramp" and original_length is None:
        raise ValueError("scaling 'ramp' needs original_length")
    n = int(rotary_dim)
    if n < 2 or n % 2:
        raise ValueError("rotary_dim must be even and positive")
    out = (ctypes.c_double * (n // 2))()
    amplitude = ctypes.c_double()
    _lib.check(_lib.load().fa_rotary_frequencies(n, float(base), _KINDS[scaling], float(factor), float(original_length or 0),
                                                 float(low_turns), float(high_turns), out, ctypes.byref(amplitude)),
               "fa_rotary_frequencies")
    return torch.tensor(list(out), dtype=torch.float64).to(device), amplitude.value


def rotary_embedding(x, positions, inv_freq, amplitude=1.0, interleaved=False, inverse=False, out=None):
    """The rows of x turned by their positions, on the current CUDA stream of x's device.

    x [batch, heads, seqlen, head_dim] or [tokens, heads, head_dim], fp16, bf16 or fp32, any strides with the last dimension in one
    piece; positions int32 or int64 [seqlen], [batch, seqlen] or [tokens]; inv_freq float64 [rotary_dim / 2] (rotary_frequencies).
    Pair i is columns (i, i + rotary_dim / 2), `interleaved`: (2 i, 2 i + 1); columns from rotary_dim on are copied.  `inverse`
    turns back, which is also the gradient's way: it multiplies by the transposed map.  `out` may be x (in place) or memory that
    does not overlap it.

    position * inv_freq is taken modulo a turn in 64-bit fixed point, so that far positions lose nothing; the angle that is left is
    rounded to 32 bits for sine and cosine (an error of 1e-7 of the pair's |a| + |b|), and the products are in 32 bits."""
    call = _lib.rotary or (_lib.load_call() and _lib.rotary)
    done = call(x, positions, inv_freq, amplitude, interleaved, inverse, out)
    if type(done) is int:
        _lib.check(done, "fa_rotary")
    return done


def paged_kv_append(k, v, k_pages, v_pages, page_table, seqlens_k, cu_seqlens_q=None, q=None, inv_freq=None, amplitude=1.0,
                    interleaved=False, out=None, status=None):
    """Puts the new tokens' k and v [tokens, heads_k, head_dim] into their slots of the pages, on the current CUDA stream, with k
    turned by the tokens' positions where `inv_freq` is given (as rotary_embedding does).  With `q` [tokens, heads, head_dim]
    returns q turned too (in `out`, which may be q), else None.  One launch.

    Of two tokens that have the same slot one or the other is kept, in pieces of 16 bytes.  A token whose page is not in the
    pool is dropped, and `status` (an int32 word on the device, zeroed by the caller) becomes 400."""
    call = _lib.append or (_lib.load_call() and _lib.append)
    done = call(k, v, k_pages, v_pages, page_table, seqlens_k, cu_seqlens_q, q, inv_freq, amplitude, interleaved, out, status)
    if type(done) is int:
        _lib.check(done, "fa_paged_append")
    return done


def paged_attn_forward(q, k_pages, v_pages, page_table, seqlens_k, cu_seqlens_q=None, max_seqlen_q=None, softmax_scale=None,
                       causal=False, window=(-1, -1), alibi_slopes=None, out=None, out_dtype=None, return_lse=True, workspace=None,
                       status=None):
    """(o, lse): attention of the new tokens q [tokens, heads, head_dim] over their sequences' pages, on the current CUDA stream
    of q's device.  heads is a multiple of heads_k; query head h reads K/V head h // (heads // heads_k).

    Masks and biases are flash_attn_forward's, on the positions of the cache: `causal` hides keys behind the query's position (so a
    chunk of new tokens sees the cache and itself), `window` = (left, right) with -1 = unbounded, `alibi_slopes` fp32 [heads].
    A row that sees no key gets o = 0, lse = -inf.  `max_seqlen_q`: the most new tokens that a sequence brings, known to the host
    (unsaid: it may be as many as there are); it says which kernel suits, the results are right whatever it is.
    lse is fp32 [tokens, heads].  Scores, sums and o are in 32 bits, but each probability is rounded to q's dtype for the product with
    V, as in flash_attn_forward and whatever `out_dtype` is.  Slots past a sequence's length may hold anything, and so may pages that
    its rows' masks hide whole; a value of V that is not finite may reach all of the up to 256 rows (a row is a token and a query head
    of one K/V head) of a block of which one sees it.

    `workspace`: room for partial results (allocated where it is missing or too small); two calls that may run at once need one
    each.  `status`: an int32 word on the device, zeroed by the caller: 400 where a visible page is not in the pool (the rows that
    met it are NaN), 300 + n where a bounded wait inside the kernel gave up (the results are undefined; zero a workspace of your own
    before its next use)."""
    call = _lib.paged or (_lib.load_call() and _lib.paged)
    done = call(q, k_pages, v_pages, page_table, seqlens_k, cu_seqlens_q, max_seqlen_q, softmax_scale, causal, window, alibi_slopes, out,
                out_dtype, return_lse, workspace, status)
    if type(done) is int:
        _lib.check(done, "fa_paged_fwd")
    return done
