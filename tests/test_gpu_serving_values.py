"""The serving operators where the values are hard: infinities and NaN that a
token may see, probabilities far below the largest one, and what a call must
refuse or report. Against 64-bit definitions; bounds: tests/serving_ref.py and
at each test."""
from __future__ import annotations

import math

import pytest
import torch

from serving_ref import U, check, check_lse, decode64, paged, prompt64, rope_tables

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


# ------------------------------------------------------------------ prompt: values that are not finite
def fastest_ms(fn, runs=7):
    fn()
    best = math.inf
    for _ in range(runs):
        a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        torch.cuda.synchronize()
        a.record()
        fn()
        b.record()
        b.synchronize()
        best = min(best, a.elapsed_time(b))
    return best


@pytest.mark.parametrize("D,dtype", [(64, BF), (64, HF), (128, BF), (128, HF)])
def test_prompt_nan_early_in_a_long_prompt(D, dtype):
    """One NaN in the first token of 8192: the result where it is not seen and where
    it is, no status, and about the time of a call without it (all rows behind it
    hold a NaN that is theirs)."""
    n, hq, hkv = 8192, 4, 2
    g = gen(D)
    q, k, v = (randn(g, n, h, D, dtype=dtype) for h in (hq, hkv, hkv))
    cu = bounds([n])
    want = prompt64(q, k, v, [n], 1 / math.sqrt(D), dtype)
    clean = fastest_ms(lambda: frsa().prompt_attention(q, k, v, cu))
    for what in ("element", "row", "key"):
        k2, v2 = k.clone(), v.clone()
        hit = torch.zeros(n, hq, D, dtype=torch.bool, device="cuda")
        if what == "element":
            v2[0, 1, 7] = math.nan
            hit[:, 2:, 7] = True
        elif what == "row":
            v2[0, 1] = math.nan
            hit[:, 2:] = True
        else:
            k2[0, 1] = math.nan
            hit[:, 2:] = True
        o, lse = frsa().prompt_attention(q, k2, v2, cu, return_lse=True)
        assert status() == 0
        assert torch.isnan(o[hit]).all()
        check(o[~hit], want[0][~hit], want[1][~hit], what)
        if what == "key":
            assert torch.isnan(lse[2:]).all()
            check_lse(lse[:2], want[2][:2], want[3][:2])
        else:
            check_lse(lse, want[2], want[3])
        ms = fastest_ms(lambda: frsa().prompt_attention(q, k2, v2, cu))
        assert ms < 3 * clean + 0.1, f"{what}: {ms:.3f} ms, without {clean:.3f}"


@pytest.mark.parametrize("hq,hkv,D,dtype", [(2, 2, 64, BF), (8, 2, 128, HF), (12, 4, 80, BF),
                                            (3, 1, 72, HF), (16, 1, 128, BF)])
def test_prompt_masked_values_beside_visible_ones(hq, hkv, D, dtype):
    """Early tokens with an infinity or NaN that later rows see, and later tokens
    with others that earlier rows of the same tiles must not see; the last token
    of one sequence and the first of the next."""
    g = gen(hq * D)
    lens = [300, 41, 200]
    cu = bounds(lens)
    q, k, v = (randn(g, 541, h, D, dtype=dtype) for h in (hq, hkv, hkv))
    want = prompt64(q, k, v, lens, 1 / math.sqrt(D), dtype)
    v2 = v.clone()
    col = torch.zeros(541, hkv, D, dtype=torch.float64, device="cuda")   # what rows get instead
    ends = [300, 341, 541]
    for t, x, c in ((10, math.inf, 3), (130, math.nan, 3), (131, math.nan, 5), (200, -math.inf, 9),
                    (299, math.nan, 0), (300, math.inf, 1), (340, -math.inf, D - 1),
                    (341, math.nan, 0), (540, math.inf, 2)):
        v2[t, 0, c] = x
        end = min(e for e in ends if e > t)
        col[t:end, 0, c] += x
    o = frsa().prompt_attention(q, k, v2, cu).double()
    assert status() == 0
    put = col.repeat_interleave(hq // hkv, 1)
    hit = put != 0
    assert torch.equal(torch.isnan(o[hit]), torch.isnan(put[hit]))
    same = hit & ~torch.isnan(put)
    assert torch.equal(o[same], put[same])
    check(o[~hit], want[0][~hit], want[1][~hit])


@pytest.mark.parametrize("D", [64, 128])
def test_prompt_infinity_of_small_weight(D):
    """An infinity 60 nats below the largest score is seen all the same, in f16 too,
    whose rounded probability there is 0."""
    for dtype in (BF, HF):
        n = 3000
        q, k = (torch.zeros(n, 1, D, device="cuda", dtype=dtype) for _ in range(2))
        q[..., 0] = 1.0
        k[0, 0, 0] = 60.0
        v = randn(gen(D), n, 1, D, dtype=dtype)
        v[100, 0, 9] = -math.inf
        o = frsa().prompt_attention(q, k, v, bounds([n]), scale=1.0)
        assert status() == 0
        assert (o[100:, 0, 9] == -math.inf).all()
        assert int(torch.isfinite(o).sum()) == n * D - (n - 100)


@pytest.mark.parametrize("D,dtype", [(64, BF), (128, BF), (64, HF), (80, HF)])
def test_prompt_scores_of_minus_infinity(D, dtype):
    """Keys whose score is -inf count nothing, also where they fill whole tiles
    before the first other one; rows that see nothing else have lse -inf."""
    n = 700
    g = gen(D)
    for holes in ([(0, 200)], [(0, 64), (100, 500)], [(0, 128)], [(0, 400), (401, 650)]):
        q, k, v = (randn(g, n, h, D, dtype=dtype) for h in (2, 1, 1))
        q[..., 0] = 1.0
        k[..., 0] = 0.0
        out = torch.zeros(n, dtype=torch.bool, device="cuda")
        for a, b in holes:
            k[a:b, 0, 0] = -math.inf
            out[a:b] = True
        o, lse = frsa().prompt_attention(q, k, v, bounds([n]), return_lse=True)
        assert status() == 0
        first = int((~out).nonzero()[0])
        k2 = k.clone()
        k2[out] = 0
        from serving_ref import attend64
        mask = torch.ones(n, n, dtype=torch.bool, device="cuda").tril() & ~out
        want = attend64(q.transpose(0, 1), k2.transpose(0, 1).repeat_interleave(2, 0),
                        v.transpose(0, 1).repeat_interleave(2, 0), 1 / math.sqrt(D), mask, dtype,
                        False)
        check(o.transpose(0, 1)[:, first:], want[0][:, first:], want[1][:, first:])
        check_lse(lse, want[2], want[3])


def test_prompt_large_values():
    """v near the end of bf16's range, a score that rises by 2^7.9 within the first
    tile: the sum over probabilities of at most 1 stays in f32's range."""
    for D in (64, 128):
        n = 128
        q, k = (torch.zeros(n, 1, D, device="cuda", dtype=BF) for _ in range(2))
        q[..., 0] = 1.0
        k[64:, 0, 0] = 7.875 * math.log(2.0)
        v = torch.full((n, 1, D), 2.0 ** 120, device="cuda", dtype=BF)
        o = frsa().prompt_attention(q, k, v, bounds([n]), scale=1.0)
        assert status() == 0
        assert ((o.double() / 2.0 ** 120 - 1).abs() <= 2.0 ** -8 + 2.0 ** -8).all()


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("power", [10, 24, 40, 59])
def test_prompt_scores_far_past_their_step(D, power):
    """bf16 scores of 2^(2 power): every row is the v of its largest score, the last
    key's, which is twice the one before it (and so on, eight times over)."""
    n = 200
    q, k = (torch.zeros(n, 1, D, device="cuda", dtype=BF) for _ in range(2))
    q[..., 0] = 2.0 ** power
    for lens in ([n], [1] * n, [8] * 25):
        first = [0]
        for m in lens:
            first.append(first[-1] + m)
        j = torch.cat([torch.arange(m) for m in lens]).cuda()
        k[:, 0, 0] = 2.0 ** (power - 8 + (j % 8).float()) * (1 + (j // 8).float() / 128)
        v = randn(gen(D), n, 1, D)
        o, lse = frsa().prompt_attention(q, k, v, bounds(lens), scale=1.0, return_lse=True)
        assert status() == 0
        s = (q[:, 0, 0].double() * k[:, 0, 0].double())
        for a, b in zip(first[:-1], first[1:]):
            top, at = torch.cummax(s[a:b], 0)
            assert torch.equal(o[a:b, 0], v[a:b, 0][at])
            assert ((lse[0, a:b].double() - top).abs() <= top.abs() * 2.0 ** -22).all()


@pytest.mark.parametrize("hq,hkv,D,dtype", [(4, 2, 64, HF), (2, 1, 128, BF)])
def test_prompt_many_values_that_are_not_finite(hq, hkv, D, dtype):
    """One element of v in a hundred is not finite: nearly every row has masked ones
    in its last tile, and each column is what its visible values make it."""
    n = 3000
    g = gen(D)
    q, k, v = (randn(g, n, h, D, dtype=dtype) for h in (hq, hkv, hkv))
    want = prompt64(q, k, v, [n], 1 / math.sqrt(D), dtype)
    u = torch.rand(n, hkv, D, device="cuda", generator=g)
    u[:1000, :, 3:] = 1.0     # (first only three columns, so that others stay finite)
    u[:, :, D // 2:] = 1.0
    v[u < 0.01] = math.inf
    v[(u >= 0.01) & (u < 0.015)] = -math.inf
    v[(u >= 0.015) & (u < 0.016)] = math.nan
    put = torch.where(torch.isfinite(v.double()), 0.0, v.double()).cumsum(0)
    put = put.repeat_interleave(hq // hkv, 1)
    o = frsa().prompt_attention(q, k, v, bounds([n])).double()
    assert status() == 0
    hit = put != 0
    assert torch.equal(torch.isnan(o[hit]), torch.isnan(put[hit]))
    same = hit & ~torch.isnan(put)
    assert torch.equal(o[same], put[same])
    check(o[~hit], want[0][~hit], want[1][~hit])


# ------------------------------------------------------------------ append: sequence boundaries
def test_append_reports_boundaries_outside_the_tokens():
    """Sequence boundaries below 0, past the tokens or out of order are reported,
    wherever they stand; a sequence that begins below 0 is not stored."""
    g = gen(31)
    kc, vc, table = paged([48] * 3, 2, 16, 64, BF, g)
    cosp, sinp = rope_tables(64, 64)
    q, k, v = (randn(g, 40, h, 64) for h in (4, 2, 2))
    before = kc.clone(), vc.clone()

    def call(cu):
        out = frsa().paged_rope_append(q, k, v, kc, vc, table, ints([0, 0, 0]), cosp, sinp,
                                       cu_seqlens=ints(cu))
        return out, status()

    (qr, kr), code = call([-3, 40, 40, 40])
    assert code == 11
    assert torch.equal(qr, q) and torch.equal(kr, k)
    assert torch.equal(kc, before[0]) and torch.equal(vc, before[1])
    for cu in ([0, 20, 30, 41], [0, 30, 20, 40], [0, -1, 20, 40], [0, 20, 1 << 30, 40]):
        assert call(cu)[1] == 11, cu
    for cu in ([0, 20, 30, 40], [5, 5, 30, 38], [40, 40, 40, 40], [0, 0, 0, 0]):
        assert call(cu)[1] == 0, cu
    many = [0] * 500 + [40] * 500
    many[700] = -7
    table = table[:1].expand(999, -1)
    out = frsa().paged_rope_append(q, k, v, kc, vc, table, ints([0] * 999), cosp, sinp,
                                   cu_seqlens=ints(many))
    assert status() == 11


@pytest.mark.parametrize("which", ["prompt", "decode"])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_infinity_of_no_weight_in_a_row_computed_again(which, dtype):
    """An infinity 200 nats below the largest score (zero in 32 bits) in a row that is
    computed again for another column: a key of -inf score whose v is infinite (0
    times an infinity: NaN) in the decode, a masked value in the prompt."""
    n, D = 300, 64
    g = gen(77)
    q, k = (torch.zeros(n, 1, D, device="cuda", dtype=dtype) for _ in range(2))
    q[..., 0] = 1.0
    k[0, 0, 0] = 200.0
    v = randn(g, n, 1, D, dtype=dtype)
    v[100, 0, 9] = math.inf
    if which == "prompt":
        v[250, 0, 20] = math.nan   # masked for rows 192..249 of its tile
        o = frsa().prompt_attention(q, k, v, bounds([n]), scale=1.0)[192:250, 0]
        bad = []
    else:
        k[150, 0, 0] = -math.inf
        v[150, 0, 20] = math.inf
        kc, vc, table = paged([n], 1, 16, D, dtype, g)
        at = torch.arange(n, device="cuda")
        kc[table[0, at // 16].long(), :, at % 16] = k
        vc[table[0, at // 16].long(), :, at % 16] = v
        o = frsa().paged_decode_attention(q[:1], kc, vc, table, ints([n]), scale=1.0)[0]
        bad = [20]
    assert status() == 0
    assert (o[:, 9] == math.inf).all()
    rest = [c for c in range(D) if c != 9 and c not in bad]
    assert torch.equal(o[:, rest], v[0, 0, rest].expand(o.shape[0], -1))
    assert torch.isnan(o[:, bad]).all()
