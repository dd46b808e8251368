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


def test_sequences_come_and_go():
    """A finished sequence rests while the others go on, and a new prompt takes its
    place: every output is that of the whole sequence in 64 bits."""
    from test_gpu_decoder import layer64
    from triton_fused_rope_flash_attn_b200 import CausalRopeAttention, CosSinTable, PagedKVCache
    torch.manual_seed(1)
    dim, heads, kv = 256, 4, 2
    attn = CausalRopeAttention(dim, heads, kv, CosSinTable(100.0, 14, 64, device="cuda"),
                               device="cuda", dtype=torch.bfloat16)
    cache = PagedKVCache(3, 196, kv, 64, page_size=16, num_pages=18)
    fed, got = [[], [], []], [[], [], []]   # tokens and outputs of the sequence in each slot
    done = []

    def tokens(n):
        return torch.randn(n, dim, device="cuda").bfloat16()

    def prefill(lens):
        x = [tokens(n) for n in lens]
        for b, y in enumerate(attn.prefill(torch.cat(x), lens, cache).split(lens)):
            fed[b] += list(x[b])
            got[b] += list(y)

    def step(ids, **kw):
        x = tokens(len(ids))
        y = attn.step(x, cache, **kw)
        for i, b in enumerate(ids):
            fed[b].append(x[i])
            got[b].append(y[i])

    def end(b):
        done.append((torch.stack(fed[b]), torch.stack(got[b])))
        fed[b], got[b] = [], []
        cache.release(b)

    with torch.no_grad():
        prefill([100, 33, 60])
        for _ in range(5):
            step([0, 1, 2])
        end(1)
        free = len(cache._free)
        for _ in range(4):
            step([2, 0], active=[2, 0])
        assert cache.host_lens == [109, 0, 69] and cache.lens.tolist() == [109, 0, 69]
        assert len(cache._free) == free   # the resting sequence drew no page
        prefill([0, 77, 0])
        for _ in range(3):
            step([0, 1, 2])
        step([1], active=[1])
        end(0)
        step([1, 2], active=[1, 2])
        end(1)
        end(2)
        assert status() == 0 and len(cache._free) == 18
        for x, y in done:
            w, = layer64(attn, x, [x.shape[0]])
            d, size = (y.double() - w).abs(), float(w.abs().max())
            # four roundings to bf16 on the way: qkv, rotation, o, output
            assert float(d.max()) <= 4 * 2.0 ** -8 * size and float(d.mean()) <= 2.0 ** -8 * size
