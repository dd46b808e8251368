"""A caller of the serving operators: a causal self-attention layer that keeps
its keys and values in a paged cache.

``CausalRopeAttention`` is the generating counterpart of ``block.RopeAttention``
(the ViT block of reference README:156-159): the same projections, pair
rotation and tables, but causal, with fewer kv heads than query heads if
wanted, prompts of different lengths packed without padding, and one new token
per sequence and step:

    rope = CosSinTable(100.0, 16, 64)   # 256 positions: a CLS token and 256 patches
    cache = PagedKVCache(batch=2, max_len=257, num_kv_heads=4, head_dim=64)
    attn = CausalRopeAttention(1024, 16, 4, rope, device="cuda", dtype=torch.bfloat16)
    with torch.no_grad():
        y = attn.prefill(x, [197, 60], cache)     # x [257, 1024]: the prompts' tokens
        y = attn.step(x_new, cache)               # x_new [2, 1024]: a token each

A sequence that is done gives its pages back (``cache.release(b)``); the others go
on (``step`` with ``active``), and a new prompt can take its place (``prefill``
with no tokens for those that run).
"""
from __future__ import annotations

import torch
from torch import nn

from .serving import paged_decode_attention, paged_rope_append, prompt_attention


class PagedKVCache:
    """Keys and values of ``batch`` sequences in pages of ``page_size`` tokens.

    ``k``, ``v``: ``[num_pages, num_kv_heads, page_size, head_dim]``;
    ``block_table`` (int32 ``[batch, pages per sequence]``) and ``lens`` (int32
    ``[batch]``) live on the device as the operators read them. Pages are handed
    out on the host by ``reserve`` and given back by ``release``.
    """

    def __init__(self, batch: int, max_len: int, num_kv_heads: int, head_dim: int,
                 page_size: int = 64, num_pages: int | None = None, device="cuda",
                 dtype=torch.bfloat16):
        per_seq = -(-max_len // page_size)
        if batch < 1 or per_seq < 1:
            raise ValueError("a cache holds at least one sequence of one token")
        pages = batch * per_seq if num_pages is None else num_pages
        shape = (pages, num_kv_heads, page_size, head_dim)
        self.k = torch.empty(shape, device=device, dtype=dtype)
        self.v = torch.empty(shape, device=device, dtype=dtype)
        self.page_size = page_size
        self.max_len = max_len
        self.block_table = torch.zeros(batch, per_seq, device=device, dtype=torch.int32)
        self.lens = torch.zeros(batch, device=device, dtype=torch.int32)
        self.host_lens = [0] * batch
        self._pages = [[] for _ in range(batch)]
        self._free = list(range(pages - 1, -1, -1))

    def reserve(self, new) -> None:
        """Make room for ``new[b]`` more tokens of each sequence ``b``."""
        if len(new) != len(self.host_lens):
            raise ValueError(f"{len(new)} counts for {len(self.host_lens)} sequences")
        want = []
        for b, n in enumerate(new):
            total = self.host_lens[b] + n
            if n < 0 or total > self.max_len:
                raise ValueError(f"sequence {b}: {total} tokens, the cache holds {self.max_len}")
            want.append(-(-total // self.page_size) - len(self._pages[b]))
        if sum(max(w, 0) for w in want) > len(self._free):
            raise RuntimeError("the cache is out of pages")
        for b, w in enumerate(want):
            if w > 0:
                first = len(self._pages[b])
                self._pages[b] += [self._free.pop() for _ in range(w)]
                self.block_table[b, first:first + w] = torch.tensor(
                    self._pages[b][first:], dtype=torch.int32)

    def advance(self, new) -> None:
        """Count ``new[b]`` appended tokens of each sequence."""
        self.host_lens = [n + m for n, m in zip(self.host_lens, new)]
        if len(set(new)) == 1:   # a step: no copy from the host
            self.lens += new[0]
        else:
            self.lens.copy_(torch.tensor(self.host_lens, dtype=torch.int32))

    def release(self, b: int) -> None:
        """Sequence ``b`` is done: its pages are free again."""
        self._free += reversed(self._pages[b])
        self._pages[b] = []
        self.host_lens[b] = 0
        self.lens[b] = 0


class CausalRopeAttention(nn.Module):
    """Causal multi-head self-attention with grouped kv heads over a paged cache.

    ``rope`` is any module with ``tables()`` (``CosSinTable`` for patches in
    raster order); token ``i`` of a sequence is rotated with table row ``i -
    has_cls``, the CLS token not at all. A token whose row the table does not
    have is refused. Inference only: call it under ``torch.no_grad()``.
    """

    def __init__(self, dim: int, num_heads: int, num_kv_heads: int, rope, has_cls: bool = True,
                 qkv_bias: bool = True, device=None, dtype=None):
        super().__init__()
        assert dim % num_heads == 0, "dim must be divisible by num_heads"
        assert num_heads % num_kv_heads == 0, "num_heads must be divisible by num_kv_heads"
        self.num_heads, self.num_kv_heads = num_heads, num_kv_heads
        self.head_dim = dim // num_heads
        self.has_cls = has_cls
        self.rope = rope
        self.qkv = nn.Linear(dim, (num_heads + 2 * num_kv_heads) * self.head_dim, bias=qkv_bias,
                             device=device, dtype=dtype)
        self.proj = nn.Linear(dim, dim, device=device, dtype=dtype)

    def _project(self, x):
        qkv = self.qkv(x).view(x.shape[0], -1, self.head_dim)
        return qkv.split((self.num_heads, self.num_kv_heads, self.num_kv_heads), dim=1)

    def _tables(self, new, cache: PagedKVCache):
        """The rotation tables, which have to reach ``new[b]`` more tokens of each sequence."""
        cosp, sinp = self.rope.tables()
        for b, (have, n) in enumerate(zip(cache.host_lens, new)):
            if n and have + n - int(self.has_cls) > cosp.shape[0]:
                raise ValueError(f"sequence {b}: {have + n} tokens, the rotation table has "
                                 f"{cosp.shape[0]} positions")
        return cosp, sinp

    def prefill(self, x: torch.Tensor, lens, cache: PagedKVCache) -> torch.Tensor:
        """Whole prompts, ``x [sum(lens), dim]``: ``lens[b]`` tokens for sequence ``b``,
        which has to be empty; those with no tokens here stay as they are."""
        for b, (have, n) in enumerate(zip(cache.host_lens, lens)):
            if have and n:
                raise ValueError(f"sequence {b} holds {have} tokens: prefill starts from an empty "
                                 "cache")
        if x.shape[0] != sum(lens):
            raise ValueError(f"{x.shape[0]} tokens for prompts of {sum(lens)}")
        tables = self._tables(lens, cache)
        cache.reserve(lens)
        q, k, v = self._project(x)
        bounds, index = [0], []
        for n in lens:
            bounds.append(bounds[-1] + n)
            index.append(torch.arange(n, dtype=torch.int32) - int(self.has_cls))
        cu = torch.tensor(bounds, dtype=torch.int32).to(x.device)
        q, k = paged_rope_append(q, k, v, cache.k, cache.v, cache.block_table, cache.lens,
                                 *tables, cu_seqlens=cu,
                                 positions=torch.cat(index).to(x.device))
        cache.advance(lens)
        o = prompt_attention(q, k, v, cu)
        return self.proj(o.flatten(1))

    def step(self, x: torch.Tensor, cache: PagedKVCache, active=None) -> torch.Tensor:
        """One new token of every sequence in ``active`` (a list, in any order; by default
        all of them), ``x [len(active), dim]``."""
        batch = len(cache.host_lens)
        if active is None:
            new = [1] * x.shape[0]
        else:
            active = list(active)
            if len(set(active)) != len(active) or not all(0 <= b < batch for b in active):
                raise ValueError(f"active must name sequences of {batch} once each, got {active}")
            if x.shape[0] != len(active):
                raise ValueError(f"{x.shape[0]} tokens for {len(active)} sequences")
            new = [int(b in active) for b in range(batch)]
        tables = self._tables(new, cache)
        cache.reserve(new)
        q, k, v = self._project(x)
        table, lens = cache.block_table, cache.lens
        if active is not None:
            at = torch.tensor(active, dtype=torch.int64).to(x.device)
            table, lens = table[at], lens[at]
        q, _ = paged_rope_append(q, k, v, cache.k, cache.v, table, lens, *tables,
                                 positions=lens - 1 if self.has_cls else None)
        cache.advance(new)
        o = paged_decode_attention(q, cache.k, cache.v, table,
                                   cache.lens if active is None else lens + 1)
        return self.proj(o.flatten(1))
