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
