"""The serving operators on the GPU against their 64-bit definitions: sizes and
masks where they can go wrong, strides and memory orders, values in masked
places, streams and graphs, index values outside their range. Bounds:
tests/serving_ref.py."""
from __future__ import annotations

import math

import pytest
import torch

from serving_ref import (U, check, check_lse, decode64, paged, prompt64, rope_tables, rotate64)

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


# ------------------------------------------------------------------ prompt
@pytest.mark.parametrize("lens,hq,hkv,D,dtype", [
    ([1], 1, 1, 64, BF), ([1], 4, 2, 128, HF), ([2, 1, 3], 3, 3, 8, BF),
    ([127, 128, 129], 2, 2, 64, BF), ([31, 32, 33, 63, 64, 65], 8, 2, 128, HF),
    ([197], 12, 12, 64, BF), ([0, 5, 0, 0, 300, 0], 4, 4, 80, BF),
    ([1370], 4, 1, 80, HF), ([700, 13], 6, 2, 72, BF), ([401], 10, 2, 128, BF),
    ([260, 259], 7, 1, 104, HF), ([150], 16, 1, 32, BF), ([77, 300], 17, 1, 48, BF),
    ([40], 128, 1, 64, HF), ([90], 100, 1, 128, BF), ([255, 256, 257, 511, 512, 513], 2, 1, 128, BF),
    ([3] * 40 + [500] + [0] * 5 + [130] * 3, 4, 4, 64, BF), ([2048], 8, 2, 128, BF),
    ([(37 * i) % 200 for i in range(70)], 8, 4, 128, HF), ([3000, 1, 1100], 32, 8, 64, HF)])
def test_prompt_against_definition(lens, hq, hkv, D, dtype):
    g = gen(sum(lens) + hq + D)
    T = sum(lens)
    q, k, v = (randn(g, T, h, D, dtype=dtype) for h in (hq, hkv, hkv))
    o, lse = frsa().prompt_attention(q, k, v, bounds(lens), return_lse=True)
    assert status() == 0
    assert o.shape == q.shape and o.dtype == dtype and lse.shape == (hq, T)
    want = prompt64(q, k, v, lens, 1 / math.sqrt(D), dtype)
    check(o, want[0], want[1], "o")
    check_lse(lse, want[2], want[3], "lse")
    assert torch.equal(o, frsa().prompt_attention(q, k, v, bounds(lens)))


@pytest.mark.parametrize("amp", [8.0, 0.01])
def test_prompt_sharp_and_flat_scores(amp):
    """Large scores raise the softmax base again and again; small ones never do."""
    g = gen(3)
    lens = [600, 333]
    q, k, v = randn(g, 933, 4, 128, amp=amp), randn(g, 933, 2, 128, amp=amp), randn(g, 933, 2, 128)
    k *= torch.linspace(0.1, 1.0, 933, device="cuda").to(BF)[:, None, None]   # later keys score higher
    o, lse = frsa().prompt_attention(q, k, v, bounds(lens), scale=0.3, return_lse=True)
    assert status() == 0
    want = prompt64(q, k, v, lens, 0.3, BF)
    check(o, want[0], want[1], "o")
    check_lse(lse, want[2], want[3], "lse")


def test_prompt_reads_strided_tokens_in_place():
    """q, k, v as views of one projection output, and an odd offset that is copied."""
    g = gen(4)
    lens = [190, 77]
    qkv = randn(g, 267, 8 + 2 + 2, 80)
    q, k, v = qkv[:, :8], qkv[:, 8:10], qkv[:, 10:]
    o = frsa().prompt_attention(q, k, v, bounds(lens))
    assert torch.equal(o, frsa().prompt_attention(q.contiguous(), k.contiguous(), v.contiguous(),
                                                  bounds(lens)))
    odd = randn(g, 267 * 8 * 80 + 1)[1:].view(267, 8, 80)   # 2 bytes past a 16-byte boundary
    wide = randn(g, 267, 2, 84)[..., 2:82]                  # rows that are not 16-byte aligned
    o = frsa().prompt_attention(odd, wide, v, bounds(lens))
    assert torch.equal(o, frsa().prompt_attention(odd.clone(), wide.contiguous(), v, bounds(lens)))
    heads_first = randn(g, 8, 267, 80).transpose(0, 1)      # [H, T, D] memory order
    want = prompt64(heads_first, k, v, lens, 1 / math.sqrt(80), BF)
    check(frsa().prompt_attention(heads_first, k, v, bounds(lens)), want[0], want[1])
    assert status() == 0


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("hq,hkv,D", [(2, 2, 64), (8, 2, 128)])
def test_prompt_masked_values_do_not_spread(bad, hq, hkv, D):
    """Values that are not finite in a token reach neither earlier tokens of its
    sequence nor other sequences; tokens after it are computed as defined."""
    g = gen(5)
    lens = [150, 170]
    cu = bounds(lens)
    q, k, v = (randn(g, 320, h, D) for h in (hq, hkv, hkv))
    clean = prompt64(q, k, v, lens, 1 / math.sqrt(D), BF)
    at = 150 + 97
    k2, v2 = k.clone(), v.clone()
    k2[at] = bad
    v2[at] = bad
    o, lse = frsa().prompt_attention(q, k2, v2, cu, return_lse=True)
    keep = torch.tensor([t < at for t in range(320)], device="cuda")
    check(o[keep], clean[0][keep], clean[1][keep])
    check_lse(lse[:, keep], clean[2][:, keep], clean[3][:, keep])
    # One element of v alone: later tokens carry it in that column only.
    v3 = v.clone()
    v3[at, 0, 3] = bad
    o = frsa().prompt_attention(q, k, v3, cu).double()
    hit = torch.zeros(320, hq, D, dtype=torch.bool, device="cuda")
    hit[at:, :hq // hkv, 3] = True
    assert torch.equal(torch.isfinite(o), ~hit)
    check(o[~hit], clean[0][~hit], clean[1][~hit])
    if math.isinf(bad):
        assert (o[hit] == bad).all()
    assert status() == 0


def test_prompt_tokens_of_no_sequence():
    g = gen(6)
    q, k, v = (randn(g, 50, h, 64) for h in (4, 2, 2))
    k[41:], v[41:] = math.nan, math.nan
    cu = ints([0, 30, 41])
    o, lse = frsa().prompt_attention(q, k, v, cu, return_lse=True)
    want = prompt64(q[:41], k[:41], v[:41], [30, 11], 0.125, BF)
    check(o[:41], want[0], want[1])
    assert (o[41:] == 0).all() and (lse[:, 41:] == -math.inf).all()
    cu = ints([9, 30, 41])
    o, lse = frsa().prompt_attention(q, k, v, cu, return_lse=True)
    want = prompt64(q[9:41], k[9:41], v[9:41], [21, 11], 0.125, BF)
    check(o[9:41], want[0], want[1])
    assert (o[:9] == 0).all() and (lse[:, :9] == -math.inf).all() and (o[41:] == 0).all()
    o, lse = frsa().prompt_attention(q, k, v, ints([0, 0, 0]), return_lse=True)
    assert (o == 0).all() and (lse == -math.inf).all()
    o, lse = frsa().prompt_attention(q, k, v, ints([0]), return_lse=True)
    assert (o == 0).all() and (lse == -math.inf).all()
    assert frsa().prompt_attention(q[:0], k[:0], v[:0], ints([0, 0])).shape == (0, 4, 64)
    assert status() == 0
    for cu in ([0, 60], [-3, 50], [0, 30, 20, 50]):   # boundaries outside the tokens
        assert torch.isfinite(frsa().prompt_attention(q[:41], k[:41], v[:41], ints(cu)).float()).all()
        assert status() == 11
    assert status() == 0


# ------------------------------------------------------------------ decode
@pytest.mark.parametrize("lens,hq,hkv,D,page,dtype", [
    ([1], 1, 1, 64, 16, BF), ([0], 4, 2, 64, 16, BF), ([63, 64, 65, 1, 0, 128], 4, 4, 64, 16, HF),
    ([197], 12, 12, 64, 16, BF), ([5000], 8, 1, 128, 16, BF), ([20011, 3], 4, 2, 128, 48, HF),
    ([300, 0, 17], 16, 1, 80, 1, BF), ([300, 200, 17], 6, 2, 72, 3, HF), ([777], 5, 1, 8, 7, BF),
    ([513, 1024, 15], 17, 1, 96, 256, BF), ([130], 40, 1, 128, 24, HF), ([90, 91], 3, 3, 104, 8, BF),
    ([400] * 150, 4, 2, 64, 32, BF), ([(61 * i) % 300 for i in range(400)], 8, 2, 32, 16, HF),
    ([64 * 37], 2, 2, 16, 64, BF), ([2500, 1, 9000, 70], 32, 8, 128, 64, BF)])
def test_decode_against_definition(lens, hq, hkv, D, page, dtype):
    g = gen(sum(lens) + D)
    kc, vc, table = paged(lens, hkv, page, D, dtype, g, fill=math.nan)
    q = randn(g, len(lens), hq, D, dtype=dtype)
    o, lse = frsa().paged_decode_attention(q, kc, vc, table, ints(lens), return_lse=True)
    assert status() == 0
    want = decode64(q, kc, vc, table, lens, 1 / math.sqrt(D), dtype)
    check(o, want[0], want[1], "o")
    check_lse(lse, want[2], want[3], "lse")
    for _ in range(3):   # the joined sum does not depend on timing
        assert torch.equal(o, frsa().paged_decode_attention(q, kc, vc, table, ints(lens)))


@pytest.mark.parametrize("order", ["phsd", "pshd", "hpsd", "sphd"])
def test_decode_memory_orders(order):
    g = gen(7)
    lens = [333, 40, 1200]
    kc, vc, table = paged(lens, 2, 24, 80, BF, g, order=order, width=60)
    qkv = randn(g, 3, 8 + 4, 80)
    q = qkv[:, :8]
    o = frsa().paged_decode_attention(q, kc, vc, table, ints(lens), scale=0.2)
    want = decode64(q, kc, vc, table, lens, 0.2, BF)
    check(o, want[0], want[1])
    part = torch.empty(3, 200, device="cuda", dtype=torch.int32)[:, :table.shape[1]]
    part.copy_(table)   # a wider table's rows
    assert torch.equal(o, frsa().paged_decode_attention(q, kc, vc, part, ints(lens), scale=0.2))
    assert status() == 0


def test_decode_sharp_scores():
    g = gen(8)
    lens = [4000]
    kc, vc, table = paged(lens, 2, 16, 128, BF, g)
    q = randn(g, 1, 8, 128, amp=12.0)
    o, lse = frsa().paged_decode_attention(q, kc, vc, table, ints(lens), return_lse=True)
    want = decode64(q, kc, vc, table, lens, 1 / math.sqrt(128), BF)
    check(o, want[0], want[1])
    check_lse(lse, want[2], want[3])


def test_decode_rows_do_not_share_what_is_not_finite():
    """An infinity or NaN in one sequence's cache stays with that sequence."""
    g = gen(9)
    lens = [500, 600]
    kc, vc, table = paged(lens, 2, 16, 64, BF, g)
    q = randn(g, 2, 4, 64)
    want = decode64(q, kc, vc, table, lens, 0.125, BF)
    vc[int(table[0, 3]), 1, 5] = math.nan
    kc[int(table[0, 7]), 0, 2] = math.inf
    o = frsa().paged_decode_attention(q, kc, vc, table, ints(lens))
    check(o[1], want[0][1], want[1][1])
    assert torch.isnan(o[0, 2:]).all()


def test_decode_index_values_outside():
    g = gen(10)
    lens = [100, 50]
    kc, vc, table = paged(lens, 2, 16, 64, BF, g)
    q = randn(g, 2, 4, 64)
    good = frsa().paged_decode_attention(q, kc, vc, table, ints(lens))
    assert status() == 0
    for page in (-1, kc.shape[0], 1 << 30):
        t = table.clone()
        t[0, 1] = page
        o = frsa().paged_decode_attention(q, kc, vc, t, ints(lens))
        assert status() == 11
        assert torch.equal(o[1], good[1])
    o, lse = frsa().paged_decode_attention(q, kc, vc, table, ints([-5, 50]), return_lse=True)
    assert status() == 11
    assert (o[0] == 0).all() and (lse[0] == -math.inf).all() and torch.equal(o[1], good[1])
    o = frsa().paged_decode_attention(q, kc, vc, table, ints([10 ** 9, 50]))   # past the table
    assert status() == 11
    assert torch.equal(o[1], good[1])
    assert frsa().paged_decode_attention(q[:0], kc, vc, table[:0], ints([])).shape == (0, 4, 64)
    assert status() == 0


# ------------------------------------------------------------------ append
def append64(q, k, v, kc, vc, table, start, cosp, sinp, new, positions, dtype):
    B = len(new)
    idx = torch.cat([torch.arange(n) + start[b] for b, n in enumerate(new)]).cuda()
    seq = torch.cat([torch.full((n,), b) for b, n in enumerate(new)]).cuda()
    pos = idx if positions is None else positions
    q64, k64 = rotate64(q, pos, cosp, sinp), rotate64(k, pos, cosp, sinp)
    page = kc.shape[2]
    where = table[seq, idx // page].long()
    kc64, vc64 = kc.double(), vc.double()
    kc64[where, :, idx % page] = k64
    vc64[where, :, idx % page] = v.double()
    assert B == table.shape[0]
    return q64, k64, kc64, vc64


@pytest.mark.parametrize("new,start,hq,hkv,D,page,dtype,cls", [
    ([1], [0], 1, 1, 64, 16, BF, False), ([1, 1, 1], [5, 0, 31], 8, 2, 128, 16, HF, False),
    ([7, 0, 1, 40], [0, 3, 15, 9], 4, 4, 80, 3, BF, True), ([197], [0], 12, 12, 64, 16, BF, True),
    ([300, 5], [100, 0], 16, 1, 8, 1, HF, False), ([50], [7], 48, 16, 128, 24, BF, False),
    ([(13 * i) % 29 for i in range(80)], [i % 7 for i in range(80)], 6, 3, 72, 256, BF, False),
    ([1] * 1500, [i % 100 for i in range(1500)], 4, 2, 32, 32, HF, True),
    ([1] * 700 + [0] * 500 + [3] * 100, [0] * 1300, 2, 1, 40, 8, BF, False)])
@pytest.mark.parametrize("order", ["phsd", "pshd"])
def test_append_against_definition(new, start, hq, hkv, D, page, dtype, cls, order):
    g = gen(sum(new) + D)
    T = sum(new)
    total = [n + s for n, s in zip(new, start)]
    kc, vc, table = paged(total, hkv, page, D, dtype, g, order=order, spare=3)
    cosp, sinp = rope_tables(max(total) + 1, D)
    q, k, v = (randn(g, T, h, D, dtype=dtype) for h in (hq, hkv, hkv))
    positions = None
    if cls:
        positions = torch.cat([torch.arange(n) + start[b] - 1 for b, n in enumerate(new)])
        positions = positions.to("cuda", torch.int32)
    want = append64(q, k, v, kc, vc, table, start, cosp, sinp, new, positions, dtype)
    one_each = all(n == 1 for n in new)
    cu = None if one_each else bounds(new)
    before = kc.clone(), vc.clone()
    got = frsa().paged_rope_append(q, k, v, kc, vc, table, ints(start), cosp, sinp, cu_seqlens=cu,
                                   positions=positions)
    assert status() == 0
    u = U[dtype]

    def close(a, b):   # |e c| + |o s| <= 2 max: two products and a sum in 32 bits, one rounding
        a, big = a.double(), 8.0
        assert ((a - b).abs() <= u * b.abs() + 2.0 ** -22 * big + 2.0 ** -25).all()

    close(got[0], want[0])
    close(got[1], want[1])
    close(kc, want[2])
    assert torch.equal(vc.double(), want[3])
    same = want[2] == before[0].double()
    assert torch.equal(kc[same], before[0][same])   # slots of no new token are as they were
    if one_each:
        kc2, vc2 = before
        again = frsa().paged_rope_append(q, k, v, kc2, vc2, table, ints(start), cosp, sinp,
                                         cu_seqlens=bounds(new), positions=positions)
        assert all(torch.equal(a, b) for a, b in zip((*got, kc, vc), (*again, kc2, vc2)))


def test_append_strided_tokens():
    g = gen(11)
    kc, vc, table = paged([64], 2, 16, 80, BF, g)
    cosp, sinp = rope_tables(64, 80)
    qkv = randn(g, 64, 12, 80)
    q, k, v = qkv[:, :8], qkv[:, 8:10], qkv[:, 10:]
    got = frsa().paged_rope_append(q, k, v, kc, vc, table, ints([0]), cosp, sinp,
                                   cu_seqlens=ints([0, 64]))
    kc2, vc2 = torch.zeros_like(kc), torch.zeros_like(vc)
    want = frsa().paged_rope_append(q.contiguous(), k.contiguous(), v.contiguous(), kc2, vc2, table,
                                    ints([0]), cosp, sinp, cu_seqlens=ints([0, 64]))
    own = table[0, :4].long()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert torch.equal(kc[own], kc2[own]) and torch.equal(vc[own], vc2[own])


def test_append_index_values_outside():
    g = gen(12)
    kc, vc, table = paged([32, 32], 2, 16, 64, BF, g, width=2)
    cosp, sinp = rope_tables(40, 64)
    q, k, v = (randn(g, 2, h, 64) for h in (4, 2, 2))
    before = kc.clone(), vc.clone()

    def call(start, tab=table, positions=None, cu=None):
        frsa().paged_rope_append(q, k, v, kc, vc, tab, ints(start), cosp, sinp, cu_seqlens=cu,
                                 positions=positions)
        return status()

    assert call([32, 32]) == 11          # past the block table
    assert call([-1, -7]) == 11
    bad = table.clone()
    bad[:] = kc.shape[0]
    assert call([0, 0], bad) == 11
    bad[:] = -1
    assert call([0, 0], bad) == 11
    assert call([0, 0], cu=ints([0, 0, 0])) == 0   # tokens of no sequence go nowhere
    assert call([0, 0], cu=ints([2, 2, 2])) == 0
    qr, kr = frsa().paged_rope_append(q, k, v, kc, vc, table, ints([7, 7]), cosp, sinp,
                                      cu_seqlens=ints([2, 2, 2]))
    assert torch.equal(qr, q) and torch.equal(kr, k) and status() == 0
    assert torch.equal(kc, before[0]) and torch.equal(vc, before[1])
    assert call([0, 0], positions=ints([40, 0])) == 11
    assert call([0, 0], positions=ints([-2, 0])) == 11
    assert call([0, 0], positions=ints([39, -1])) == 0


# ------------------------------------------------------------------ large offsets
def test_cache_offsets_past_32_bits():
    """Pages whose elements lie past 2^32: append and decode there give the bits
    of a small cache."""
    g = gen(20)
    hkv, page, D, n = 8, 64, 128, 150
    pages = 2 ** 32 // (hkv * page * D) + 8
    big = [torch.empty(pages, hkv, page, D, device="cuda", dtype=BF) for _ in range(2)]
    small = [torch.empty(8, hkv, page, D, device="cuda", dtype=BF) for _ in range(2)]
    cosp, sinp = rope_tables(n + 1, D)
    q, k, v = (randn(g, n, h, D) for h in (16, hkv, hkv))
    table = ints([[4, 1, 6]])
    outs = []
    for (kc, vc), t in ((small, table), (big, table + (pages - 8))):
        qr, _ = frsa().paged_rope_append(q, k, v, kc, vc, t, ints([0]), cosp, sinp,
                                         cu_seqlens=ints([0, n]))
        outs.append(frsa().paged_decode_attention(qr[-1:], kc, vc, t, ints([n])))
    assert status() == 0
    assert torch.equal(outs[0], outs[1])
    want = decode64(qr[-1:], *small, table, [n], 1 / math.sqrt(D), BF)
    check(outs[0], want[0], want[1])


def test_prompt_offsets_past_31_bits():
    """More than 2^31 elements of q in 1800 packed sequences: the last ones give
    the bits of a call of their own."""
    g = gen(21)
    n, B, hq, D = 300, 1800, 32, 128
    T = n * B
    assert T * hq * D > 2 ** 31
    q = torch.empty(T, hq, D, device="cuda", dtype=BF).normal_(generator=g)
    k, v = (torch.empty(T, 1, D, device="cuda", dtype=BF).normal_(generator=g) for _ in range(2))
    o = frsa().prompt_attention(q, k, v, bounds([n] * B))
    assert status() == 0
    for b in (0, 901, B - 1):
        s = slice(b * n, (b + 1) * n)
        assert torch.equal(o[s], frsa().prompt_attention(q[s], k[s], v[s], bounds([n])))


# ------------------------------------------------------------------ together
def test_other_streams_and_graphs():
    """The operators run on the current stream; a captured step can be replayed,
    and two streams do not share the decode's scratch."""
    g = gen(13)
    lens = [3000, 2900]
    kc, vc, table = paged([n + 64 for n in lens], 2, 16, 128, BF, g)
    cosp, sinp = rope_tables(4000, 128)
    q, k, v = (randn(g, 2, h, 128) for h in (8, 2, 2))
    n = ints(lens)
    torch.cuda.synchronize()

    def step(q, k, v, n):
        qr, _ = frsa().paged_rope_append(q, k, v, kc, vc, table, n, cosp, sinp)
        n += 1
        return frsa().paged_decode_attention(qr, kc, vc, table, n)

    want = [step(q, k, v, n) for _ in range(4)]
    torch.cuda.synchronize()
    n.copy_(ints(lens))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [step(q, k, v, n) for _ in range(4)]
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    n.copy_(ints(lens))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(q, k, v, n)
    n.copy_(ints(lens))
    for w in want:
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, w)
    # the two streams at once, on different data
    q2 = randn(g, 2, 8, 128)
    n.copy_(ints(lens))
    torch.cuda.synchronize()
    a = frsa().paged_decode_attention(q, kc, vc, table, n)
    b = frsa().paged_decode_attention(q2, kc, vc, table, n)
    torch.cuda.synchronize()
    outs = []
    for _ in range(50):
        x = frsa().paged_decode_attention(q, kc, vc, table, n)
        with torch.cuda.stream(side):
            y = frsa().paged_decode_attention(q2, kc, vc, table, n)
        outs.append((x, y))
    torch.cuda.synchronize()
    assert all(torch.equal(x, a) and torch.equal(y, b) for x, y in outs)
    assert status() == 0


def test_early_started_kernels_see_what_comes_before():
    """Calls that follow one another without a wait (each may start while the one
    before it ends) give the bits of calls with the device idle in between:
    the step's output is the next step's input, and buffers are reused."""
    g = gen(15)
    lens = [700, 1, 65]
    kc0, vc0, table = paged([n + 80 for n in lens], 2, 16, 64, BF, g)
    cosp, sinp = rope_tables(800, 64)
    x0 = randn(g, 3, 8, 64)
    cu = ints([0, 1, 2, 3])

    def chain(wait):
        kc, vc, n, x = kc0.clone(), vc0.clone(), ints(lens), x0
        for _ in range(60):
            q, k = frsa().paged_rope_append(x, x[:, :2], x[:, 2:4], kc, vc, table, n, cosp, sinp)
            wait()
            n += 1
            x = frsa().paged_decode_attention(q, kc, vc, table, n)
            wait()
            x = x + frsa().prompt_attention(q, k, x[:, 4:6], cu)
            wait()
        return x, kc, vc

    want = chain(torch.cuda.synchronize)
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(chain(lambda: None), want))
    assert status() == 0


def test_refusals_on_the_gpu():
    m = frsa()
    g = gen(14)
    kc, vc, table = paged([32], 2, 16, 64, BF, g)
    cosp, sinp = rope_tables(64, 64)
    q, k = randn(g, 1, 4, 64), randn(g, 1, 2, 64)
    n = ints([1])

    def raises(kind, *a, fn=m.paged_decode_attention, **kw):
        with pytest.raises(kind):
            fn(*a, **kw)

    raises(TypeError, q.float(), kc.float(), vc.float(), table, n)
    raises(TypeError, q, kc.half(), vc.half(), table, n)
    raises(TypeError, q, kc, vc, table.long(), n)
    raises(TypeError, q, kc, vc, table, n.long())
    raises(RuntimeError, q, kc, vc, table, ints([1, 1]))
    raises(RuntimeError, q, kc, vc[:, :1], table, n)
    raises(RuntimeError, q, kc, vc, table.cpu(), n)
    raises(RuntimeError, q.cpu(), kc, vc, table, n)
    raises(RuntimeError, randn(g, 1, 3, 64), kc, vc, table, n)          # heads do not divide
    raises(RuntimeError, randn(g, 1, 4, 60), *(randn(g, 4, 2, 16, 60) for _ in range(2)), table, n)
    raises(RuntimeError, randn(g, 1, 4, 136), *(randn(g, 4, 2, 16, 136) for _ in range(2)), table, n)
    raises(RuntimeError, q, *(randn(g, 4, 2, 16, 68)[..., :64] for _ in range(2)), table, n)
    for scale in (0.0, -1.0, math.nan):
        raises(ValueError, q, kc, vc, table, n, scale=scale)
        raises(ValueError, q, k, k, ints([0, 1]), scale=scale, fn=m.prompt_attention)
    raises(RuntimeError, q.clone().requires_grad_(), kc, vc, table, n)
    with torch.no_grad():
        m.paged_decode_attention(q.clone().requires_grad_(), kc, vc, table, n)
    raises(RuntimeError, q, k, k, kc, vc, table, ints([0, 0]), cosp, sinp, fn=m.paged_rope_append)
    raises(TypeError, q, k, k, kc, vc, table, ints([0]), cosp.double(), sinp.double(),
           fn=m.paged_rope_append)
    raises(RuntimeError, q, k, k, kc, vc, table, ints([0]), cosp[:, :8], sinp[:, :8],
           fn=m.paged_rope_append)
    raises(RuntimeError, q, k, randn(g, 1, 4, 64), kc, vc, table, ints([0]), cosp, sinp,
           fn=m.paged_rope_append)
    raises(RuntimeError, q, randn(g, 2, 2, 64), k, ints([0, 1]), fn=m.prompt_attention)
    raises(TypeError, q, k, k, ints([0, 1]).long(), fn=m.prompt_attention)
    raises(TypeError, q, k.half(), k, ints([0, 1]), fn=m.prompt_attention)
    raises(RuntimeError, randn(g, 1, 129, 64), randn(g, 1, 1, 64), randn(g, 1, 1, 64), ints([0, 1]),
           fn=m.prompt_attention)
    raises(RuntimeError, q.clone().requires_grad_(), k, k, ints([0, 1]), fn=m.prompt_attention)
    assert status() == 0
