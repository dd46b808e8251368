"""The serving operators where the values are hard: infinities and NaN that a
token may see, probabilities far below the largest one, and what a call must
refuse or report. Against 64-bit definitions; bounds: tests/serving_ref.py and
at each test."""
from __future__ import annotations

import math

import pytest
import torch

from serving_ref import check, check_lse, decode64, paged

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
