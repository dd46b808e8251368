"""The serving operators where the values are hard: infinities and NaN that a
token may see, probabilities far below the largest one, and what a call must
refuse or report. Against 64-bit definitions; bounds: tests/serving_ref.py and
at each test."""
from __future__ import annotations

import math

import pytest
import torch

from serving_ref import U, check, check_lse, decode64, paged

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16


def frsa():
    import triton_fused_rope_flash_attn_b200 as m
    return m


def status():
    from triton_fused_rope_flash_attn_b200 import _lib
    return _lib.load().frsa_query_status()


def gen(seed=0):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, *shape, dtype=BF, amp=1.0):
    return (torch.randn(*shape, device="cuda", generator=g) * amp).to(dtype)


def ints(v):
    return torch.tensor(v, device="cuda", dtype=torch.int32)


def bounds(lens):
    return ints([sum(lens[:i]) for i in range(len(lens) + 1)])


# ------------------------------------------------------------------ decode: visible infinities
@pytest.mark.parametrize("bad,want", [((math.inf,), math.inf), ((-math.inf,), -math.inf),
                                      ((math.inf, -math.inf), math.nan),
                                      ((math.inf, math.nan), math.nan)])
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("n,hq,hkv,D,page", [(1, 2, 2, 64, 16), (90, 8, 2, 128, 16),
                                             (500, 4, 2, 80, 24), (700, 17, 1, 72, 64),
                                             (30000, 8, 2, 128, 16)])
def test_decode_carries_visible_infinities(n, hq, hkv, D, page, dtype, bad, want):
    """A probability is positive, so an infinity in v makes its column infinite, two
    of opposite sign or a NaN make it NaN; the other columns, kv heads and
    sequences do not see it."""
    if len(bad) > n:
        pytest.skip("one token holds one value")
    g = gen(n + D)
    lens = [n, 333]
    kc, vc, table = paged(lens, hkv, page, D, dtype, g)
    q = randn(g, 2, hq, D, dtype=dtype)
    clean = decode64(q, kc, vc, table, lens, 1 / math.sqrt(D), dtype)
    for i, x in enumerate(bad):
        j = min(n - 1, n // 3 + 70 * i + i)
        vc[int(table[0, j // page]), hkv - 1, j % page, 5] = x
    o, lse = frsa().paged_decode_attention(q, kc, vc, table, ints(lens), return_lse=True)
    assert status() == 0
    hit = torch.zeros_like(o, dtype=torch.bool)
    hit[0, hq - hq // hkv:, 5] = True
    got = o[hit].double()
    assert torch.isnan(got).all() if math.isnan(want) else bool((got == want).all())
    check(o[~hit], clean[0][~hit], clean[1][~hit], "o")
    check_lse(lse, clean[2], clean[3], "lse")
    assert torch.equal(torch.nan_to_num(o), torch.nan_to_num(
        frsa().paged_decode_attention(q, kc, vc, table, ints(lens))))


def test_decode_infinity_of_small_weight():
    """An infinity 60 nats below the largest score: its probability is small, not zero."""
    for dtype in (BF, HF):
        n, D = 2000, 64
        kc, vc, table = paged([n], 1, 16, D, dtype, gen(1))
        kc.zero_()
        kc[int(table[0, 0]), 0, 3, 0] = 60.0
        vc[int(table[0, 100]), 0, 7, 9] = -math.inf
        q = torch.zeros(1, 2, D, device="cuda", dtype=dtype)
        q[..., 0] = 1.0
        o = frsa().paged_decode_attention(q, kc, vc, table, ints([n]), scale=1.0)
        assert (o[0, :, 9] == -math.inf).all()
        assert int(torch.isfinite(o).sum()) == 2 * (D - 1)


# ------------------------------------------------------------------ f16: small probabilities
def tail_rows(n, tail, D):
    """q, k, v of one head in f16: token 0 scores 0 and has v = 0, every other one
    scores -tail and has a v of about one."""
    q, k = (torch.zeros(n, 1, D, device="cuda", dtype=HF) for _ in range(2))
    q[..., 0] = 1.0
    k[1:, :, 0] = -tail
    v = 1.0 + 0.25 * torch.rand(n, 1, D, device="cuda", generator=gen(n), dtype=torch.float32)
    v[0] = 0.0
    return q, k, v.to(HF)


def tail_tol(o, A, V, n, D, floor, u):
    """Relative to the largest probability a held one is off by u of itself or by
    half a step at `floor`, and counts |v|; the rest as in serving_ref. (The score
    is one product, so exact but for the rounding of its base-2 form: 18 nats
    times 2^-23.)"""
    return U[HF] * o.abs() + 2.0 ** -25 + (u + 2 * 18 * 2.0 ** -23 + n * 2.0 ** -24 +
                                           2.0 ** -20) * A + floor * V


@pytest.mark.parametrize("n", [300, 4096, 131072])
@pytest.mark.parametrize("tail", [14.0, 16.0, 17.0, 17.40625, 18.0])
def test_f16_decode_keeps_small_probabilities(n, tail):
    """An attention sink over a long cache: what lies far below the largest
    probability is all of the output. Two parts of 2^-11 each carry 2^-22 of a
    probability; f16's smallest half step is 2^-25, at least 2^14 below which the
    largest probability has to lie: floor 2^-39."""
    D, page = 64, 16
    q, k, v = tail_rows(n, tail, D)
    kc, vc, table = paged([n], 1, page, D, HF, gen(2))
    at = torch.arange(n, device="cuda")
    kc[table[0, at // page].long(), :, at % page] = k
    vc[table[0, at // page].long(), :, at % page] = v
    o, lse = frsa().paged_decode_attention(q[:1], kc, vc, table, ints([n]), scale=1.0,
                                           return_lse=True)
    w = math.exp(-tail)
    V = v[:, 0].double().sum(0)
    want = V * w / (1 + (n - 1) * w)
    tol = tail_tol(want, want, V, n, D, 2.0 ** -39, 2.0 ** -22)
    check(o[0, 0], want, tol, "o")
    check(lse[0], torch.full((1,), math.log1p((n - 1) * w), dtype=torch.float64, device="cuda"),
          torch.full((1,), 2.0 ** -19 + n * 2.0 ** -24 * n * w, dtype=torch.float64, device="cuda"))


def big_scores(D, dtype):
    """Scores of 2^27 and more that rise by 2^17 from key to key: each row is its
    last key's v alone, and a probability's rounding of 2^4 (half a step of the
    score's base-2 form) must not take it out of f16's range."""
    n = 1000
    q, k = (torch.zeros(n, 1, D, device="cuda", dtype=dtype) for _ in range(2))
    q[..., 0] = 2.0 ** 13
    k[:, 0, 0] = 2.0 ** 14 + 16 * torch.arange(n, device="cuda")
    return q, k, randn(gen(D), n, 1, D, dtype=dtype)


@pytest.mark.parametrize("D", [64, 128])
def test_f16_decode_large_scores(D):
    q, k, v = big_scores(D, HF)
    kc, vc, table = paged([1000], 1, 8, D, HF, gen(2))
    at = torch.arange(1000, device="cuda")
    kc[table[0, at // 8].long(), :, at % 8] = k
    vc[table[0, at // 8].long(), :, at % 8] = v
    for n in (1, 100, 1000):
        o = frsa().paged_decode_attention(q[:1], kc, vc, table, ints([n]), scale=1.0)
        assert torch.equal(o[0, 0], v[n - 1, 0])


@pytest.mark.parametrize("n,D,at", [(300, 64, 0), (4096, 64, 0), (4096, 128, 0), (4096, 80, 1500)])
@pytest.mark.parametrize("tail", [14.0, 16.0, 17.0, 17.40625, 18.0])
def test_f16_prompt_keeps_small_probabilities(n, D, at, tail):
    """The same in a prompt, with the large score first or in the middle. One part
    of a probability carries 2^-11 of it; with the largest one at 2^11 or above
    f16's smallest half step is a floor of 2^-36."""
    q, k, v = tail_rows(n, tail, D)
    k[0], k[at] = k[at].clone(), k[0].clone()
    v[0], v[at] = v[at].clone(), v[0].clone()
    o, lse = frsa().prompt_attention(q, k, v, bounds([n]), scale=1.0, return_lse=True)
    assert status() == 0
    x = k[:, 0, 0].double()
    p = torch.exp(x)
    V = v[:, 0].double().cumsum(0)
    l = p.cumsum(0)[:, None]
    want = (p[:, None] * v[:, 0].double()).cumsum(0) / l
    # rows before the large score: probabilities relative to the largest of the row
    top = torch.cummax(x, 0).values.exp()[:, None]
    tol = tail_tol(want, want, V * top / l, n, D, 2.0 ** -36, 2.0 ** -11)
    check(o[:, 0], want, tol, "o")
    check(lse[0], l[:, 0].log(), torch.full((n,), 2.0 ** -18 + n * 2.0 ** -23, dtype=torch.float64,
                                            device="cuda"))


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("D", [64, 128])
def test_prompt_large_scores(D, dtype):
    q, k, v = big_scores(D, dtype)
    if dtype == BF:   # 2^14 + 16 j in steps of 2^7
        k, v = k[::16], v[::16]
        q = q[:k.shape[0]]
    k[:, 0, 0] = k[:, 0, 0].sort().values
    o = frsa().prompt_attention(q, k, v, bounds([k.shape[0]]), scale=1.0)
    assert k[:, 0, 0].double().diff().min() >= 16
    assert status() == 0 and torch.equal(o[:, 0], v[:, 0])
