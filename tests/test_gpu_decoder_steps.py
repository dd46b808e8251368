"""The causal layer over its paged cache on the GPU: its documented use, up to
the last position of its table."""
from __future__ import annotations

import textwrap

import pytest
import torch

pytestmark = pytest.mark.gpu


def status():
    from triton_fused_rope_flash_attn_b200 import _lib
    return _lib.load().frsa_query_status()


def test_documented_example_runs_as_printed():
    import triton_fused_rope_flash_attn_b200 as m
    from triton_fused_rope_flash_attn_b200 import decoder
    code = textwrap.dedent("\n".join(l for l in decoder.__doc__.splitlines()
                                     if l.startswith("    ")))
    g = torch.Generator(device="cuda").manual_seed(0)
    names = dict(torch=torch, CosSinTable=m.CosSinTable, PagedKVCache=m.PagedKVCache,
                 CausalRopeAttention=m.CausalRopeAttention,
                 x=torch.randn(257, 1024, device="cuda", generator=g).bfloat16(),
                 x_new=torch.randn(2, 1024, device="cuda", generator=g).bfloat16())
    exec(code, names)
    assert names["y"].shape == (2, 1024)
    with torch.no_grad():
        for _ in range(59):   # sequence 0 reaches the table's last position
            names["attn"].step(names["x_new"], names["cache"])
        assert status() == 0
        with pytest.raises(ValueError, match="256 positions"):
            names["attn"].step(names["x_new"], names["cache"])
    assert names["cache"].host_lens == [257, 120]
