"""64-bit definitions of the serving operators for their tests, with the bounds
that a 16-bit result of 32-bit arithmetic has to keep.

Bounds. u is half an ulp of the output type relative to the value (bf16 2^-8,
f16 2^-11). With A = sum_j p_j |v_j| per output element:

* the output is rounded once: u |o|, and at least half the type's smallest
  step (f16: 2^-25);
* where the probabilities are rounded to the type before the second product
  (prompt): u A; where they enter as two 16-bit parts (decode): u^2 A, and for
  f16 the low part's smallest step, 2^-25 per key, sum_j |v_j| 2^-25;
* a score of D products summed in 32 bits is off by at most
  d = (D + 2) 2^-24 scale sum |q k|, which moves a probability by the factor
  exp(+-d), in numerator and denominator: 2 d A; the sums over n keys and the
  approximate exponential (2^-22): (n 2^-23 + 2^-20) A.
"""
from __future__ import annotations

import math

import torch

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def rope_tables(n, D, device="cuda", base=100.0):
    inv = base ** (-torch.arange(D // 2, dtype=torch.float64) / (D // 2))
    ang = torch.arange(n, dtype=torch.float64)[:, None] * inv
    return ang.cos().float().to(device), ang.sin().float().to(device)


def rotate64(x, pos, cosp, sinp):
    """x [T, H, D] rotated by table rows pos [T] (-1: as it is), in 64 bits."""
    x = x.double()
    c = torch.ones(x.shape[0], x.shape[2] // 2, dtype=torch.float64, device=x.device)
    s = torch.zeros_like(c)
    on = pos >= 0
    c[on], s[on] = cosp.double()[pos[on].long()], sinp.double()[pos[on].long()]
    c, s = c[:, None], s[:, None]
    e, o = x[..., 0::2], x[..., 1::2]
    return torch.stack((e * c - o * s, o * c + e * s), dim=-1).flatten(-2)


def attend64(q, k, v, scale, mask, dtype, split_p):
    """q [H, M, D], k, v [H, N, D], mask [M, N] (True: seen). Returns o, its
    bound, lse and its bound; rows that see nothing: o = 0, lse = -inf."""
    q, k, v = q.double(), k.double(), v.double()
    D, n = q.shape[-1], k.shape[-2]
    x = (q @ k.transpose(-1, -2)) * scale
    x = x.masked_fill(~mask, -math.inf)
    lse = torch.logsumexp(x, dim=-1) if n else torch.full(x.shape[:-1], -math.inf,
                                                          device=q.device, dtype=torch.float64)
    p = torch.exp(x - lse.clamp_min(-1e300)[..., None])
    o, A = p @ v, p @ v.abs()
    S = ((q.abs() @ k.abs().transpose(-1, -2)) * scale).masked_fill(~mask, 0.0)
    d = (D + 2) * 2.0 ** -24 * (S.amax(-1) if n else torch.zeros_like(lse))
    u = U[dtype]
    tiny = 2.0 ** -25 if dtype == torch.float16 else 2.0 ** -130
    tol = u * o.abs() + tiny + (2 * d[..., None] + n * 2.0 ** -23 + 2.0 ** -20) * A
    tol = tol + (u * u if split_p else u) * A
    if dtype == torch.float16:
        tol = tol + 2.0 ** -25 * (mask.double() @ v.abs())
    return o, tol, lse, d + n * 2.0 ** -23 + 2.0 ** -20 * (1 + lse.abs().clamp_max(1e300))


def check(got, want, tol, what=""):
    got = got.double()
    assert torch.isfinite(got).all() or not torch.isfinite(want).all(), f"{what}: not finite"
    over = (got - want).abs() - tol
    worst = float(over.max()) if over.numel() else -1.0
    assert worst <= 0, f"{what}: {worst:.3e} over its bound at {int(over.argmax())}"


def check_lse(got, want, tol, what=""):
    empty = torch.isinf(want)
    assert torch.equal(torch.isinf(got), empty), what
    check(got[~empty], want[~empty], tol[~empty], what)


def prompt64(q, k, v, lens, scale, dtype):
    """Packed causal prompts: o [T, Hq, D], bound, lse [Hq, T], bound."""
    T, hq, D = q.shape
    g = hq // k.shape[1]
    o = torch.zeros(T, hq, D, dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(o)
    lse = torch.full((hq, T), -math.inf, dtype=torch.float64, device=q.device)
    ltol = torch.zeros_like(lse)
    t = 0
    for n in lens:
        s = slice(t, t + n)
        if n:
            mask = torch.ones(n, n, dtype=torch.bool, device=q.device).tril()
            kk, vv = (x[s].transpose(0, 1).repeat_interleave(g, 0) for x in (k, v))
            r = attend64(q[s].transpose(0, 1), kk, vv, scale, mask, dtype, False)
            o[s], tol[s] = r[0].transpose(0, 1), r[1].transpose(0, 1)
            lse[:, s], ltol[:, s] = r[2], r[3]
        t += n
    return o, tol, lse, ltol


def gather(cache, table, n):
    """The first n cached tokens of one sequence: [Hkv, n, D]."""
    page = cache.shape[2]
    i = torch.arange(n, device=cache.device)
    return cache[table[i // page].long(), :, i % page].transpose(0, 1)


def decode64(q, kc, vc, table, lens, scale, dtype):
    """One token per sequence: o [B, Hq, D], bound, lse [B, Hq], bound."""
    B, hq, D = q.shape
    g = hq // kc.shape[1]
    o = torch.zeros(B, hq, D, dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(o)
    lse = torch.full((B, hq), -math.inf, dtype=torch.float64, device=q.device)
    ltol = torch.zeros_like(lse)
    for b, n in enumerate(lens):
        if n == 0:
            continue
        kk, vv = (gather(c, table[b], n).repeat_interleave(g, 0) for c in (kc, vc))
        mask = torch.ones(1, n, dtype=torch.bool, device=q.device)
        r = attend64(q[b][:, None], kk, vv, scale, mask, dtype, True)
        o[b], tol[b], lse[b], ltol[b] = (x[:, 0] for x in r)
    return o, tol, lse, ltol


def paged(lens, hkv, page, D, dtype, gen, spare=2, order="phsd", fill=None, width=0):
    """A pool of pages handed out in no order: k_cache, v_cache and the block
    table (unused entries 0). order: memory order of (page, head, slot)."""
    npages = [-(-n // page) for n in lens]
    pool = sum(npages) + spare
    shape = {"p": pool, "h": hkv, "s": page, "d": D}
    caches = []
    for _ in range(2):
        c = torch.randn([shape[a] for a in order], device="cuda", generator=gen).to(dtype)
        caches.append(c.permute([order.index(a) for a in "phsd"]))
    ids = torch.randperm(pool, device="cuda", generator=gen).to(torch.int32)
    table = torch.zeros(len(lens), max(width, max(npages), 1), device="cuda", dtype=torch.int32)
    at = 0
    for b, n in enumerate(npages):
        table[b, :n] = ids[at:at + n]
        at += n
    if fill is not None:   # slots that hold no token, and pages that nobody owns
        for c in caches:
            for page_id in ids[at:].tolist():
                c[page_id] = fill
            for b, n in enumerate(lens):
                if n % page:
                    c[int(table[b, n // page]), :, n % page:] = fill
    return caches[0], caches[1], table
