"""Serving operators: a paged key-value cache with rotated keys, the attention of
one new token over it, and causal attention over whole packed prompts.

The reference's attention is unmasked over one fixed grid of tokens
(fa_rope_full .py:91-315); a model that generates token by token with the same
pair rotation and the same ``[N_pos, D/2]`` tables needs these three next to it:

    q, k = paged_rope_append(q, k, v, k_cache, v_cache, block_table, start_lens, COSP, SINP, ...)
    o = prompt_attention(q, k, v, cu_seqlens)                       # a prompt's tokens, or
    o = paged_decode_attention(q, k_cache, v_cache, block_table, seq_lens)   # one new token each

Tensors: packed tokens ``[T, heads, D]`` (``Hkv`` dividing ``Hq``; query head
``h`` reads kv head ``h // (Hq // Hkv)``), caches ``[pages, Hkv, page_size,
D]``, all bf16 or f16, ``D`` a multiple of 8 up to 128; index arrays int32 on
the same device. Strided tokens whose rows are 16-byte aligned are read in
place, others are copied; the caches are used in place and must be so
addressable. Everything runs on torch's current stream, without a host
synchronisation. Index values outside their range (a page, a position, a
length) are not followed; ``frsa_query_status`` of the C ABI reports them.
There is no derivative: inputs that ask for a gradient, or carry a forward-mode
tangent, are refused. What is not finite in a token's keys and values counts as
in the formula for those that see it, and not at all for others.
"""
from __future__ import annotations

from . import _lib
from .attention import _ext


def paged_rope_append(q, k, v, k_cache, v_cache, block_table, start_lens, cosp, sinp,
                      cu_seqlens=None, positions=None):
    """Rotate new tokens and append their keys and values to a paged cache.

    ``q [T, Hq, D]``, ``k``, ``v [T, Hkv, D]``: the new tokens of all sequences,
    sequence ``b`` holding ``[cu_seqlens[b], cu_seqlens[b+1])``; without
    ``cu_seqlens`` one token per sequence. ``start_lens [B]``: tokens cached
    before the call. Token ``j`` of sequence ``b`` gets index ``i =
    start_lens[b] + j`` and goes to slot ``i % page_size`` of page
    ``block_table[b, i // page_size]``. It is rotated with table row ``i``, or
    ``positions[t]`` (``[T]``; -1: not rotated, as a CLS token) where given.

    Returns the rotated ``(q, k)``, contiguous, rounded once; ``k_cache`` and
    ``v_cache`` are written in place (their version counters rise). Tokens outside ``[cu_seqlens[0],
    cu_seqlens[-1])`` belong to no sequence: neither rotated nor stored.
    """
    q_out, k_out, rc = _ext().paged_append(q, k, v, k_cache, v_cache, block_table, start_lens,
                                           cosp, sinp, cu_seqlens, positions)
    if rc:
        _lib.check(rc, "frsa_paged_append")
    return q_out, k_out


def paged_decode_attention(q, k_cache, v_cache, block_table, seq_lens, scale=None,
                           return_lse: bool = False):
    """Attention of one (rotated) query token per sequence over its cached tokens.

    ``q [B, Hq, D]``, ``seq_lens [B]``: cached tokens, the new one included
    (0: the output is 0 and the LSE -inf). ``scale`` (positive, finite) defaults
    to ``1/sqrt(D)``.
    Returns ``o [B, Hq, D]``, with ``return_lse`` also the natural-log row LSE
    (float32 ``[B, Hq]``). The split over the cache's length is joined in a
    fixed order: equal inputs give equal bits.
    """
    o, lse, rc = _ext().paged_decode(q, k_cache, v_cache, block_table, seq_lens, scale, return_lse)
    if rc:
        _lib.check(rc, "frsa_paged_decode")
    return (o, lse) if return_lse else o


def prompt_attention(q, k, v, cu_seqlens, scale=None, return_lse: bool = False):
    """Causal attention over whole packed prompts of different lengths.

    ``q [T, Hq, D]``, ``k``, ``v [T, Hkv, D]`` (q and k rotated), sequence ``b``
    holding the tokens ``[cu_seqlens[b], cu_seqlens[b+1])``; a token sees itself
    and the earlier tokens of its sequence. ``Hq // Hkv`` is at most 128.
    Returns ``o [T, Hq, D]``, with ``return_lse`` also the natural-log row LSE
    (float32 ``[Hq, T]``). Tokens outside ``[cu_seqlens[0], cu_seqlens[-1])``
    belong to no sequence: output 0, LSE -inf.
    """
    o, lse, rc = _ext().prompt(q, k, v, cu_seqlens, scale, return_lse)
    if rc:
        _lib.check(rc, "frsa_prompt_fwd")
    return (o, lse) if return_lse else o
