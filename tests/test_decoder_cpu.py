"""Host side of the causal layer and its paged cache without a GPU: what the
layer refuses before it reserves a page, and the lists it makes of sequences."""
from __future__ import annotations

import pytest
import torch

from triton_fused_rope_flash_attn_b200 import CausalRopeAttention, CosSinTable, PagedKVCache


def layer(side=4, has_cls=True):
    return CausalRopeAttention(256, 4, 2, CosSinTable(100.0, side, 64, device="cpu"), has_cls)


@pytest.mark.parametrize("has_cls,most", [(True, 17), (False, 16)])
def test_positions_past_the_table_are_refused(has_cls, most):
    """A table of 16 rows: 16 rotated tokens, and a CLS token in front."""
    attn = layer(4, has_cls)
    cache = PagedKVCache(2, 64, 2, 64, page_size=4, device="cpu")
    free = len(cache._free)
    with pytest.raises(ValueError, match="16 positions"):
        attn.prefill(torch.zeros(most + 4, 256), [3, most + 1], cache)
    assert len(cache._free) == free and cache.host_lens == [0, 0]
    cache.reserve([3, most])
    cache.advance([3, most])
    free = len(cache._free)
    with pytest.raises(ValueError, match="16 positions"):
        attn.step(torch.zeros(2, 256), cache)
    assert len(cache._free) == free and cache.host_lens == [3, most]


def test_prefill_and_step_name_their_sequences():
    attn = layer()
    cache = PagedKVCache(3, 17, 2, 64, page_size=4, device="cpu")
    cache.reserve([5, 0, 4])
    cache.advance([5, 0, 4])
    free = len(cache._free)
    with pytest.raises(ValueError, match="sequence 2 holds 4 tokens"):
        attn.prefill(torch.zeros(4, 256), [0, 3, 1], cache)
    for active in ([0, 0], [3], [-1]):
        with pytest.raises(ValueError, match="once each"):
            attn.step(torch.zeros(len(active), 256), cache, active)
    with pytest.raises(ValueError, match="2 tokens for 1 sequences"):
        attn.step(torch.zeros(2, 256), cache, [0])
    with pytest.raises(ValueError, match="2 counts for 3"):
        attn.step(torch.zeros(2, 256), cache)
    assert len(cache._free) == free and cache.host_lens == [5, 0, 4]
    # Past these checks the operators refuse the CPU.
    with pytest.raises(RuntimeError, match="CUDA"), torch.no_grad():
        attn.step(torch.zeros(1, 256), cache, [2])
    with pytest.raises(RuntimeError, match="CUDA"), torch.no_grad():
        attn.prefill(torch.zeros(3, 256), [0, 3, 0], cache)
