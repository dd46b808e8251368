"""The serving operators used together: a causal attention layer that prefills
packed prompts into its paged cache and goes on one token a step, against the
same layer in 64 bits, and a captured step replayed."""
from __future__ import annotations

import math

import pytest
import torch

from serving_ref import rotate64

pytestmark = pytest.mark.gpu


def layer64(attn, x, lens):
    """The layer over whole sequences, 64 bits throughout."""
    hq, hkv, D = attn.num_heads, attn.num_kv_heads, attn.head_dim
    cosp, sinp = attn.rope.tables()
    outs, t = [], 0
    for n in lens:
        y = x[t:t + n].double() @ attn.qkv.weight.double().T + attn.qkv.bias.double()
        q, k, v = y.view(n, -1, D).split((hq, hkv, hkv), dim=1)
        pos = torch.arange(n, device=x.device) - int(attn.has_cls)
        q, k = rotate64(q, pos, cosp, sinp), rotate64(k, pos, cosp, sinp)
        k, v = (z.repeat_interleave(hq // hkv, 1) for z in (k, v))
        s = torch.einsum("qhd,khd->hqk", q, k) / math.sqrt(D)
        s = s.masked_fill(~torch.ones(n, n, dtype=torch.bool, device=x.device).tril(), -math.inf)
        o = torch.einsum("hqk,khd->qhd", s.softmax(-1), v).flatten(1)
        outs.append(o @ attn.proj.weight.double().T + attn.proj.bias.double())
        t += n
    return outs


@pytest.mark.parametrize("dim,heads,kv_heads,page,has_cls", [(256, 4, 2, 16, True),
                                                              (768, 12, 12, 64, True),
                                                              (640, 8, 2, 24, False)])
def test_prefill_and_steps_against_the_layer_in_64_bits(dim, heads, kv_heads, page, has_cls):
    from triton_fused_rope_flash_attn_b200 import (CausalRopeAttention, CosSinTable, PagedKVCache,
                                                   _lib)
    torch.manual_seed(0)
    D = dim // heads
    attn = CausalRopeAttention(dim, heads, kv_heads, CosSinTable(100.0, 14, D, device="cuda"),
                               has_cls, device="cuda", dtype=torch.bfloat16)
    prompts, steps = [180, 1, 57], 12
    total = [n + steps for n in prompts]
    x = [torch.randn(n, dim, device="cuda").bfloat16() for n in total]
    cache = PagedKVCache(3, 196, kv_heads, D, page)
    with torch.no_grad():
        want = layer64(attn, torch.cat(x), total)
        y = attn.prefill(torch.cat([a[:n] for a, n in zip(x, prompts)]), prompts, cache)
        got = [list(p.unbind(0)) for p in y.split(prompts)]
        for i in range(steps):
            y = attn.step(torch.stack([a[n + i] for a, n in zip(x, prompts)]), cache)
            for b in range(3):
                got[b].append(y[b])
    assert _lib.load().frsa_query_status() == 0
    # Four roundings to bf16 (2^-8 each) lie on the way: qkv, rotation, o, output.
    for g, w in zip(got, want):
        d = (torch.stack(g).double() - w).abs()
        size = float(w.abs().max())
        assert float(d.max()) <= 4 * 2.0 ** -8 * size and float(d.mean()) <= 2.0 ** -8 * size
    cache.release(1)
    assert cache.host_lens[1] == 0


def test_needs_no_grad():
    from triton_fused_rope_flash_attn_b200 import CausalRopeAttention, CosSinTable, PagedKVCache
    attn = CausalRopeAttention(256, 4, 2, CosSinTable(100.0, 14, 64, device="cuda"), device="cuda",
                               dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="no_grad"):
        attn.prefill(torch.zeros(5, 256, device="cuda", dtype=torch.bfloat16), [5],
                     PagedKVCache(1, 64, 2, 64))


def test_registered_ops_trace_and_agree():
    """The registered forms give the same bits, pass opcheck, and a compiled step
    holds them in one graph."""
    from triton_fused_rope_flash_attn_b200 import (CosSinTable, paged_decode_attention,
                                                   paged_rope_append, prompt_attention)
    cs = CosSinTable(100.0, 14, 64, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(3)

    def rand(*s):
        return torch.randn(*s, device="cuda", generator=g).bfloat16()

    q, k, v = rand(40, 4, 64), rand(40, 2, 64), rand(40, 2, 64)
    kc, vc = rand(8, 2, 16, 64), rand(8, 2, 16, 64)
    table = torch.tensor([[1, 5], [2, 7]], device="cuda", dtype=torch.int32)
    zero = torch.zeros(2, device="cuda", dtype=torch.int32)
    cu = torch.tensor([0, 25, 40], device="cuda", dtype=torch.int32)
    lens = torch.tensor([25, 15], device="cuda", dtype=torch.int32)

    def chain(q, k, v, kc, vc):
        q, k = torch.ops.frsa.paged_append(q, k, v, kc, vc, table, zero, cs.COSP, cs.SINP, cu)
        o = torch.ops.frsa.prompt_attn(q, k, v, cu)
        return o, torch.ops.frsa.paged_decode(q[:2], kc, vc, table, lens)

    kc1, vc1 = kc.clone(), vc.clone()
    qr, kr = paged_rope_append(q, k, v, kc1, vc1, table, zero, cs.COSP, cs.SINP, cu_seqlens=cu)
    want = (prompt_attention(qr, kr, v, cu), paged_decode_attention(qr[:2], kc1, vc1, table, lens))
    kc2, vc2 = kc.clone(), vc.clone()
    got = torch.compile(chain, fullgraph=True)(q, k, v, kc2, vc2)
    assert all(torch.equal(a, b) for a, b in zip((*got, kc2, vc2), (*want, kc1, vc1)))
    torch.library.opcheck(torch.ops.frsa.paged_append.default,
                          (q, k, v, kc2, vc2, table, zero, cs.COSP, cs.SINP, cu))
    torch.library.opcheck(torch.ops.frsa.prompt_attn.default, (q, k, v, cu))
    torch.library.opcheck(torch.ops.frsa.paged_decode.default, (q[:2], kc, vc, table, lens))
