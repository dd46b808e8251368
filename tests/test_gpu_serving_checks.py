"""What the serving operators must refuse, and what a caller of torch must see of
their writes."""
from __future__ import annotations

import math

import pytest
import torch
import torch.autograd.forward_ad as fwad

from serving_ref import paged, rope_tables

pytestmark = pytest.mark.gpu


def frsa():
    import triton_fused_rope_flash_attn_b200 as m
    return m


def ints(v):
    return torch.tensor(v, device="cuda", dtype=torch.int32)


def case(seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    kc, vc, table = paged([32], 2, 16, 64, torch.bfloat16, g)
    q, k, v = (torch.randn(1, h, 64, device="cuda", generator=g).bfloat16() for h in (4, 2, 2))
    return q, k, v, kc, vc, table, rope_tables(64, 64)


def test_forward_mode_tangents_are_refused():
    q, k, v, kc, vc, table, (cosp, sinp) = case()
    append = (q, k, v, kc, vc, table, ints([0]), cosp, sinp)
    decode = (q, kc, vc, table, ints([1]))
    prompt = (q, k, v, ints([0, 1]))
    for fn, args, which in ((frsa().paged_rope_append, append, (0, 1, 2, 3, 4, 7, 8)),
                            (frsa().paged_decode_attention, decode, (0, 1, 2)),
                            (frsa().prompt_attention, prompt, (0, 1, 2))):
        for i in which:
            with fwad.dual_level(), pytest.raises(RuntimeError, match="tangent"):
                dual = fwad.make_dual(args[i], torch.ones_like(args[i]))
                fn(*args[:i], dual, *args[i + 1:])
        fn(*args)


def test_tables_that_ask_for_a_gradient_are_refused():
    q, k, v, kc, vc, table, (cosp, sinp) = case()
    for c, s in ((cosp.clone().requires_grad_(), sinp), (cosp, sinp.clone().requires_grad_())):
        with pytest.raises(RuntimeError, match="no_grad"):
            frsa().paged_rope_append(q, k, v, kc, vc, table, ints([0]), c, s)
        with torch.no_grad():
            frsa().paged_rope_append(q, k, v, kc, vc, table, ints([0]), c, s)


def test_append_counts_as_a_write_of_the_caches():
    """As after an in-place operation of torch: a graph that saved a cache refuses its
    backward, caches made in inference mode work inside and outside of it."""
    q, k, v, kc, vc, table, (cosp, sinp) = case()
    w = torch.ones((), device="cuda", dtype=torch.bfloat16, requires_grad=True)
    for saved in (kc, vc):
        y = (saved * w).sum()
        before = kc._version, vc._version
        frsa().paged_rope_append(q, k, v, kc, vc, table, ints([0]), cosp, sinp)
        assert kc._version > before[0] and vc._version > before[1]
        with pytest.raises(RuntimeError, match="inplace"):
            y.backward()
    before = kc._version
    frsa().paged_decode_attention(q, kc, vc, table, ints([1]))
    assert kc._version == before
    with torch.inference_mode():
        kc2, vc2 = kc.clone(), vc.clone()
        frsa().paged_rope_append(q, k, v, kc2, vc2, table, ints([0]), cosp, sinp)
        frsa().paged_rope_append(q, k, v, kc, vc, table, ints([0]), cosp, sinp)
    frsa().paged_rope_append(q, k, v, kc2, vc2, table, ints([0]), cosp, sinp)
    assert torch.equal(kc, kc2) and torch.equal(vc, vc2)
    whole = torch.zeros(2, *kc.shape, device="cuda", dtype=torch.bfloat16)   # views share a counter
    frsa().paged_rope_append(q, k, v, whole[0], whole[1], table, ints([0]), cosp, sinp)
    assert whole._version > 0


@pytest.mark.parametrize("scale", [math.inf, 1e300, 3e38, 1e-60])
def test_scales_past_their_range_are_refused(scale):
    q, k, v, kc, vc, table, _ = case()
    with pytest.raises(ValueError, match="scale"):
        frsa().paged_decode_attention(q, kc, vc, table, ints([1]), scale=scale)
    with pytest.raises(ValueError, match="scale"):
        frsa().prompt_attention(q, k, v, ints([0, 1]), scale=scale)
    with pytest.raises(ValueError, match="scale"):   # no call that returns early lets it pass
        frsa().prompt_attention(q[:0], k[:0], v[:0], ints([0]), scale=scale)
