"""Host side of the serving operators without a GPU: the C ABI's argument checks
(only calls that return before a device is touched), the wrappers' refusals,
and the paged cache's page accounting."""
from __future__ import annotations

import ctypes

import pytest
import torch

from triton_fused_rope_flash_attn_b200 import (CausalRopeAttention, CosSinTable, PagedKVCache, _lib,
                                               paged_decode_attention, paged_rope_append,
                                               prompt_attention)
from triton_fused_rope_flash_attn_b200.build import build_library

P = 0x1000   # a 16-byte aligned stand-in; nothing is read before the device check


@pytest.fixture(scope="module")
def lib():
    build_library()
    return _lib.load()


def fill(struct, pointers, values, changes):
    a = struct()
    for name in pointers:
        setattr(a, name, P)
    for name, v in {**values, **changes}.items():
        if isinstance(v, list):
            getattr(a, name)[:] = v
        else:
            setattr(a, name, v)
    return a


SHAPE = dict(B=2, Hq=8, Hkv=2, D=64, num_pages=10, page_size=16, max_pages=4, block_table_stride=4)


def append_args(**kw):
    return fill(_lib.FrsaPagedAppendArgs,
                ("q", "k", "v", "q_out", "k_out", "k_cache", "v_cache", "block_table", "start_lens",
                 "cu_seqlens", "positions", "cosp", "sinp"), dict(SHAPE, T=7, n_pos=64), kw)


def decode_args(lib, **kw):
    return fill(_lib.FrsaPagedDecodeArgs,
                ("q", "k_cache", "v_cache", "o", "lse", "block_table", "seq_lens", "workspace"),
                dict(SHAPE, scale=0.125, workspace_bytes=lib.frsa_paged_decode_workspace_bytes()), kw)


def prompt_args(**kw):
    return fill(_lib.FrsaPromptArgs, ("q", "k", "v", "o", "lse", "cu_seqlens"),
                dict(T=50, B=2, Hq=8, Hkv=2, D=64, scale=0.125), kw)


COMMON = [(dict(D=60), 3), (dict(D=136), 3), (dict(Hq=9), 2), (dict(Hkv=0), 2), (dict(B=0), 2),
          (dict(dtype=_lib.FRSA_DTYPE_F32), 4), (dict(q=P + 8), 5), (dict(q=None), 1),
          (dict(q_strides=[512, 60]), 5), (dict(q_strides=[0, 64]), 5),
          (dict(q_strides=[-512, 64]), 5), (dict(q_strides=[1 << 40, 64]), 5), ({}, 8)]
CACHE = [(dict(num_pages=0), 2), (dict(page_size=0), 2), (dict(max_pages=0), 2),
         (dict(block_table_stride=-1), 2), (dict(page_size=1 << 29, max_pages=1 << 10), 2),
         (dict(cache_strides=[2048, 1024, 60]), 5), (dict(block_table=None), 1),
         (dict(block_table=P + 2), 5), (dict(v_cache=P + 4), 5), (dict(k_cache=None), 1)]


@pytest.mark.parametrize("kw,code", COMMON + CACHE + [
    (dict(T=0), 2), (dict(cu_seqlens=None), 2), (dict(cu_seqlens=None, T=2), 8),
    (dict(positions=None, k_out=None), 8), (dict(start_lens=None), 1), (dict(cosp=None), 1),
    (dict(sinp=P + 4), 5), (dict(n_pos=-1), 2), (dict(positions=P + 1), 5),
    (dict(v_strides=[132, 64]), 5), (dict(cache_strides=[128, 1 << 20, 128]), 8)])
def test_append_argument_checks(lib, kw, code):
    assert lib.frsa_paged_append(ctypes.byref(append_args(**kw)), None) == code


@pytest.mark.parametrize("kw,code", COMMON + CACHE + [
    (dict(lse=None), 8), (dict(seq_lens=None), 1), (dict(workspace=None), 9),
    (dict(workspace_bytes=64), 9), (dict(workspace=P + 4), 5), (dict(scale=0.0), 2),
    (dict(scale=float("nan")), 2), (dict(cache_strides=[1 << 36, 1024, 64]), 2),
    (dict(B=1 << 20, max_pages=1 << 20), 2), (dict(Hq=512, Hkv=2), 8)])
def test_decode_argument_checks(lib, kw, code):
    assert lib.frsa_paged_decode(ctypes.byref(decode_args(lib, **kw)), None) == code


@pytest.mark.parametrize("kw,code", COMMON + [
    (dict(lse=None), 8), (dict(T=0), 2), (dict(cu_seqlens=None), 1), (dict(cu_seqlens=P + 2), 5),
    (dict(Hq=258, Hkv=2), 2), (dict(Hq=256, Hkv=2), 8), (dict(scale=-1.0), 2),
    (dict(k_strides=[128, 68]), 5), (dict(o=None), 1), (dict(T=1 << 31), 2)])
def test_prompt_argument_checks(lib, kw, code):
    assert lib.frsa_prompt_fwd(ctypes.byref(prompt_args(**kw)), None) == code


def test_null_args_and_messages(lib):
    assert lib.frsa_paged_append(None, None) == 1
    assert lib.frsa_paged_decode(None, None) == 1
    assert lib.frsa_prompt_fwd(None, None) == 1
    assert b"index" in lib.frsa_strerror(11)
    assert lib.frsa_paged_decode_workspace_bytes() > 0


def test_cpu_tensors_are_refused():
    q, kv = torch.zeros(2, 4, 64).bfloat16(), torch.zeros(2, 2, 64).bfloat16()
    cache = torch.zeros(4, 2, 16, 64).bfloat16()
    table, one = torch.zeros(2, 2, dtype=torch.int32), torch.ones(2, dtype=torch.int32)
    tab = torch.zeros(32, 32)
    with pytest.raises(RuntimeError, match="CUDA"):
        paged_rope_append(q, kv, kv, cache, cache, table, one, tab, tab)
    with pytest.raises(RuntimeError, match="CUDA"):
        paged_decode_attention(q, cache, cache, table, one)
    with pytest.raises(RuntimeError, match="CUDA"):
        prompt_attention(q, kv, kv, one)


def test_cache_hands_out_and_takes_back_pages():
    c = PagedKVCache(batch=3, max_len=40, num_kv_heads=2, head_dim=64, page_size=16, num_pages=6,
                     device="cpu")
    c.reserve([17, 0, 40])
    c.advance([17, 0, 40])
    used = c.block_table[0, :2].tolist() + c.block_table[2, :3].tolist()
    assert len(set(used)) == 5 and c.lens.tolist() == [17, 0, 40]
    c.reserve([15, 16, 0])          # 32 tokens of sequence 0 fill its two pages
    c.advance([15, 16, 0])
    assert set(used + [int(c.block_table[1, 0])]) == set(range(6))
    with pytest.raises(RuntimeError, match="out of pages"):
        c.reserve([1, 0, 0])
    with pytest.raises(ValueError, match="41 tokens"):
        c.reserve([0, 0, 1])
    with pytest.raises(ValueError):
        c.reserve([1, 1])
    c.release(2)
    assert c.host_lens == [32, 16, 0] and c.lens.tolist() == [32, 16, 0]
    c.reserve([8, 1, 0])
    with pytest.raises(ValueError):
        PagedKVCache(batch=0, max_len=4, num_kv_heads=1, head_dim=8, device="cpu")


def test_layer_checks_its_arguments():
    rope = CosSinTable(100.0, 4, 64, device="cpu")
    with pytest.raises(AssertionError):
        CausalRopeAttention(256, 4, 3, rope)
    attn = CausalRopeAttention(256, 4, 2, rope)
    cache = PagedKVCache(1, 17, 2, 64, device="cpu")
    with pytest.raises(ValueError, match="tokens for prompts"):
        attn.prefill(torch.zeros(3, 256), [4], cache)
    cache.host_lens = [3]
    with pytest.raises(ValueError, match="empty cache"):
        attn.prefill(torch.zeros(4, 256), [4], cache)
