"""The serving operators as a user calls them, and their plain forms, over the
sizes that decoders with rotary positions meet: appending rotated keys to a
paged key-value cache, the attention of one new token over that cache, and the
causal attention over whole packed prompts.

``own`` false: ``run`` computes the operators with elementary torch operations
in 32 bits, rounded once at the end. ``own`` true: ``run`` calls this
repository's operators. A case is a dict of plain values; the sequence lengths
follow from its ``lo``, ``hi`` and ``mix`` alone, the data from the seed.

Layouts: packed tokens ``[T, heads, D]``; caches ``[pages, kv heads,
page_size, D]``; ``block_table[b, i]`` is the page that holds tokens
``[i * page_size, (i + 1) * page_size)`` of sequence ``b``; rotation tables
``[positions, D/2]`` with adjacent-pair rotation.
"""
from __future__ import annotations

import math
import random

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}


def listed():
    def case(name, op, B, lo, hi, hq, hkv, D, page, dtype, mix=0, new=0, cls=0):
        return dict(name=name, op=op, B=B, lo=lo, hi=hi, hq=hq, hkv=hkv, D=D, page=page,
                    dtype=dtype, mix=mix, new=new, cls=cls)

    return [
        # One new token of one sequence: the append of a single-user chat step.
        case("append_token_b1", "append", 1, 300, 300, 16, 4, 64, 16, "bf16", new=1),
        # One new token of each of 64 running sequences: a serving step.
        case("append_token_b64", "append", 64, 1, 4000, 32, 8, 128, 16, "f16", mix=1, new=1),
        # Image prompts of different sizes (37 x 37 patches and a CLS token at
        # most), positions from the patch grid, the CLS token not rotated.
        case("append_images", "append", 11, 50, 1370, 16, 16, 80, 32, "bf16", mix=2, cls=1),
        # A long document into an empty cache.
        case("append_prompt_8192", "append", 1, 8192, 8192, 32, 8, 128, 64, "bf16"),
        # A short caption step: one sequence of one image's tokens.
        case("decode_b1_197", "decode", 1, 197, 197, 12, 12, 64, 16, "bf16"),
        # Eight sequences over images of different sizes, odd page size.
        case("decode_b8_images", "decode", 8, 1, 1370, 16, 4, 80, 24, "f16", mix=3),
        # A full serving batch with mixed lengths.
        case("decode_b64_mixed", "decode", 64, 33, 8000, 32, 8, 128, 64, "bf16", mix=4),
        # One sequence with a very long cache: the length has to be split.
        case("decode_b1_131072", "decode", 1, 131072, 131072, 32, 8, 128, 16, "bf16"),
        # One image as a prompt (ViT-B heads).
        case("prompt_b1_197", "prompt", 1, 197, 197, 12, 12, 64, 16, "bf16"),
        # Packed prompts from one token to a 37 x 37 image and a CLS token.
        case("prompt_b9_images", "prompt", 9, 1, 1370, 16, 4, 80, 16, "f16", mix=5),
        # Packed documents of mixed lengths.
        case("prompt_b6_mixed", "prompt", 6, 500, 3000, 32, 8, 128, 16, "bf16", mix=6),
        # A long document.
        case("prompt_b1_8192", "prompt", 1, 8192, 8192, 32, 8, 128, 16, "bf16"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    op = rng.choice(("append", "decode", "prompt"))
    hkv = rng.choice((1, 2, 3, 4, 8, 12, 16))
    group = rng.choice((1, 2, 3, 4, 5, 7, 8, 16))
    while hkv * group > 48:
        group = rng.choice((1, 2, 3))
    D = rng.choice((32, 48, 64, 64, 72, 80, 96, 104, 128, 128))
    page = rng.choice((8, 16, 16, 24, 32, 48, 64, 128, 256))
    dtype = rng.choice(("bf16", "f16"))
    mix = rng.randrange(1, 1 << 20)
    c = dict(op=op, hq=hkv * group, hkv=hkv, D=D, page=page, dtype=dtype, mix=mix, new=0, cls=0)
    if op == "append":
        c["new"] = rng.choice((0, 1))
        c["cls"] = rng.choice((0, 1))
        c["B"] = _log_int(rng, 1, 128 if c["new"] else 24)
        c["hi"] = _log_int(rng, 1, 8192)
        rows = c["hq"] + 4 * hkv
        while c["hi"] > 1 and c["B"] * c["hi"] * (4 * hkv if c["new"] else rows) * D > 8192 * 64 * 128:
            c["hi"] = max(1, c["hi"] // 2)
    elif op == "decode":
        c["B"] = _log_int(rng, 1, 128)
        c["hi"] = _log_int(rng, 1, 131072)
        while c["hi"] > 1 and (c["B"] * c["hi"] * hkv * D > 131072 * 8 * 128
                               or c["B"] * c["hi"] * c["hq"] > 131072 * 32):
            c["hi"] = max(1, c["hi"] // 2)
    else:
        c["B"] = _log_int(rng, 1, 48)
        c["hi"] = _log_int(rng, 1, 8192)
        while c["hi"] > 1 and c["B"] * c["hi"] ** 2 * c["hq"] > 8192 * 8192 * 32:
            c["hi"] = max(1, c["hi"] // 2)
    c["lo"] = max(1, min(c["hi"], rng.choice((1, c["hi"] // 2, c["hi"]))))
    return c


def _lens(case):
    """Tokens per sequence: spread over [lo, hi], the longest exactly hi."""
    r = random.Random(1000003 * case["mix"] + case["B"])
    n = [r.randint(case["lo"], case["hi"]) for _ in range(case["B"])]
    n[r.randrange(case["B"])] = case["hi"]
    return n


def _rope_tables(n, D, device):
    inv = 10000.0 ** (-torch.arange(0, D // 2, device=device, dtype=torch.float64) / (D // 2))
    ang = torch.arange(n, device=device, dtype=torch.float64)[:, None] * inv
    return ang.cos().float().contiguous(), ang.sin().float().contiguous()


def prepare(case, seed):
    dev = torch.device("cuda")
    dt = _DTYPES[case["dtype"]]
    g = torch.Generator(device=dev).manual_seed(seed)
    D, hq, hkv, page = case["D"], case["hq"], case["hkv"], case["page"]
    lens = _lens(case)
    B, longest = len(lens), max(lens)

    def rand(*shape):
        return torch.randn(*shape, device=dev, generator=g, dtype=torch.float32).to(dt)

    def ints(v):
        return torch.tensor(v, device=dev, dtype=torch.int32)

    s = dict(op=case["op"], scale=1.0 / math.sqrt(D), longest=longest)
    if case["op"] == "prompt":
        T = sum(lens)
        s.update(q=rand(T, hq, D), k=rand(T, hkv, D), v=rand(T, hkv, D),
                 cu_seqlens=ints([sum(lens[:i]) for i in range(B + 1)]))
        return s
    # A pool of pages handed out in no order, as a server's allocator does.
    npages = [-(-n // page) for n in lens]
    pool = sum(npages) + 3
    ids = torch.randperm(pool, device=dev, generator=g).to(torch.int32)
    width = max(npages)
    first = ints([sum(npages[:i]) for i in range(B)])[:, None]
    col = torch.arange(width, device=dev, dtype=torch.int32)[None, :]
    used = col < ints(npages)[:, None]
    s["block_table"] = torch.where(used, ids[torch.where(used, first + col, 0).long()],
                                   torch.zeros((), device=dev, dtype=torch.int32)).contiguous()
    s["k_cache"], s["v_cache"] = rand(pool, hkv, page, D), rand(pool, hkv, page, D)
    if case["op"] == "decode":
        s.update(q=rand(B, hq, D), seq_lens=ints(lens))
        return s
    new = [1] * B if case["new"] else lens
    T = sum(new)
    s.update(q=rand(T, hq, D), k=rand(T, hkv, D), v=rand(T, hkv, D),
             start_lens=ints([n - 1 if case["new"] else 0 for n in lens]),
             cu_seqlens=None if case["new"] else ints([sum(new[:i]) for i in range(B + 1)]))
    s["cosp"], s["sinp"] = _rope_tables(longest, D, dev)
    s["positions"] = None
    if case["cls"]:   # the first token of each sequence carries no position
        cu = ints([sum(new[:i]) for i in range(B + 1)])
        b = torch.searchsorted(cu[1:].contiguous(), torch.arange(T, device=dev, dtype=torch.int32),
                               right=True)
        t = torch.arange(T, device=dev, dtype=torch.int32)
        s["positions"] = (s["start_lens"][b] + t - cu[b] - 1).to(torch.int32)
    return s


def _rotate(x, positions, cosp, sinp):
    x = x.float()
    row = positions.clamp_min(0).long()
    turn = (positions >= 0)[:, None]
    c = torch.where(turn, cosp[row], torch.ones_like(cosp[row]))[:, None]
    s = torch.where(turn, sinp[row], torch.zeros_like(sinp[row]))[:, None]
    e, o = x[..., 0::2], x[..., 1::2]
    return torch.stack((e * c - o * s, o * c + e * s), dim=-1).flatten(-2)


def _plain_append(s):
    T = s["q"].shape[0]
    t = torch.arange(T, device=s["q"].device)
    if s["cu_seqlens"] is None:
        b, at = t, s["start_lens"].long()
    else:
        b = torch.searchsorted(s["cu_seqlens"][1:].long().contiguous(), t, right=True)
        at = s["start_lens"].long()[b] + t - s["cu_seqlens"].long()[b]
    pos = at if s["positions"] is None else s["positions"]
    page = s["k_cache"].shape[2]
    where = s["block_table"].long()[b, at // page]
    q = _rotate(s["q"], pos, s["cosp"], s["sinp"]).to(s["q"].dtype)
    k = _rotate(s["k"], pos, s["cosp"], s["sinp"]).to(s["k"].dtype)
    s["k_cache"][where, :, at % page] = k
    s["v_cache"][where, :, at % page] = s["v"]
    return dict(q=q, k=k, k_cache=s["k_cache"], v_cache=s["v_cache"])


def _plain_decode(s):
    B, hq, D = s["q"].shape
    hkv, page = s["k_cache"].shape[1], s["k_cache"].shape[2]
    n = s["block_table"].shape[1] * page

    def pages(c):
        return c[s["block_table"].long()].transpose(1, 2).reshape(B, hkv, n, D).float()

    q = s["q"].view(B, hkv, hq // hkv, D).float()
    x = (q @ pages(s["k_cache"]).transpose(-1, -2)) * s["scale"]
    seen = torch.arange(n, device=q.device)[None] < s["seq_lens"][:, None]
    x = x.masked_fill(~seen[:, None, None], float("-inf"))
    p = torch.exp(x - x.amax(-1, keepdim=True))
    o = (p @ pages(s["v_cache"])) / p.sum(-1, keepdim=True)
    return o.reshape(B, hq, D).to(s["q"].dtype)


def _plain_prompt(s):
    T, hq, D = s["q"].shape
    hkv, n = s["k"].shape[1], s["longest"]
    cu = s["cu_seqlens"].long()
    B = cu.numel() - 1
    i = torch.arange(n, device=cu.device)
    held = i < (cu[1:] - cu[:-1])[:, None]
    tok = torch.where(held, cu[:-1, None] + i, 0)

    def padded(x, heads):   # [B, kv heads, rows, D]
        return x[tok].view(B, n, hkv, heads // hkv, D).permute(0, 2, 3, 1, 4).reshape(
            B, hkv, heads // hkv * n, D).float()

    x = (padded(s["q"], hq) @ padded(s["k"], hkv).transpose(-1, -2)) * s["scale"]
    x = x.view(B, hkv, hq // hkv, n, n)
    x = x.masked_fill(i[None, :] > i[:, None], float("-inf"))
    p = torch.exp(x - x.amax(-1, keepdim=True))
    o = p.view(B, hkv, hq // hkv * n, n) @ padded(s["v"], hkv)
    o = o.view(B, hkv, hq // hkv, n, D) / p.sum(-1, keepdim=True)
    t = torch.arange(T, device=cu.device)
    b = torch.searchsorted(cu[1:].contiguous(), t, right=True)
    return o.permute(0, 3, 1, 2, 4).reshape(B, n, hq, D)[b, t - cu[b]].to(s["q"].dtype)


def run(s):
    if not own:
        if s["op"] == "append":
            return _plain_append(s)
        return _plain_decode(s) if s["op"] == "decode" else _plain_prompt(s)
    import triton_fused_rope_flash_attn_b200 as frsa
    if s["op"] == "append":
        q, k = frsa.paged_rope_append(s["q"], s["k"], s["v"], s["k_cache"], s["v_cache"],
                                      s["block_table"], s["start_lens"], s["cosp"], s["sinp"],
                                      cu_seqlens=s["cu_seqlens"], positions=s["positions"])
        return dict(q=q, k=k, k_cache=s["k_cache"], v_cache=s["v_cache"])
    if s["op"] == "decode":
        return frsa.paged_decode_attention(s["q"], s["k_cache"], s["v_cache"], s["block_table"],
                                           s["seq_lens"])
    return frsa.prompt_attention(s["q"], s["k"], s["v"], s["cu_seqlens"])


def work(case):
    lens = _lens(case)
    D, hq, hkv = case["D"], case["hq"], case["hkv"]
    if case["op"] == "append":
        T = len(lens) if case["new"] else sum(lens)
        # q, k, v in; q and k rotated out; k and v into the cache; one row of
        # both tables for each position that a token has.
        rows = min(T, max(lens))
        return {"bytes": 2 * T * D * (2 * hq + 5 * hkv) + 4 * rows * D,
                "flops": 3 * T * D * (hq + hkv)}
    if case["op"] == "decode":
        return {"bytes": 2 * D * (2 * hkv * sum(lens) + 2 * hq * len(lens)),
                "flops": 4 * D * hq * sum(lens)}
    return {"bytes": 2 * D * sum(lens) * (2 * hq + 2 * hkv),
            "flops": 4 * D * hq * sum(n * (n + 1) // 2 for n in lens)}


def exact(case, seed):
    """The definitions in 64 bits, one sequence and one kv head after another."""
    s = prepare(case, seed)
    if case["op"] == "append":
        D, page = case["D"], case["page"]
        kc, vc = s["k_cache"].double(), s["v_cache"].double()
        new = [1] * case["B"] if case["new"] else _lens(case)
        outs, t = {"q": [], "k": []}, 0
        for b, n in enumerate(new):
            at = int(s["start_lens"][b]) + torch.arange(n, device="cuda")
            pos = at - 1 if case["cls"] else at
            c, d = (x.double()[pos.clamp_min(0)] for x in (s["cosp"], s["sinp"]))
            c[pos < 0], d[pos < 0] = 1.0, 0.0
            z = torch.complex(c, d)[:, None]
            for name in ("q", "k"):
                x = torch.view_as_complex(s[name][t:t + n].double().reshape(n, -1, D // 2, 2))
                outs[name].append(torch.view_as_real(x * z).reshape(n, -1, D))
            pages = s["block_table"][b].long()[at // page]
            kc[pages, :, at % page] = outs["k"][-1]
            vc[pages, :, at % page] = s["v"][t:t + n].double()
            t += n
        return dict(q=torch.cat(outs["q"]), k=torch.cat(outs["k"]), k_cache=kc, v_cache=vc)
    group = case["hq"] // case["hkv"]
    out = torch.empty(s["q"].shape, device="cuda", dtype=torch.float64)
    first = 0
    for b, n in enumerate(_lens(case)):
        for h in range(case["hkv"]):
            heads = slice(h * group, (h + 1) * group)
            if case["op"] == "decode":
                at = s["block_table"][b].long()
                k, v = (s[c][at, h].reshape(-1, case["D"])[:n].double()
                        for c in ("k_cache", "v_cache"))
                w = torch.softmax(s["q"][b, heads].double() @ k.T / math.sqrt(case["D"]), dim=-1)
                out[b, heads] = w @ v
            else:
                own_rows = slice(first, first + n)
                k, v = s["k"][own_rows, h].double(), s["v"][own_rows, h].double()
                past = torch.ones(n, n, device="cuda", dtype=torch.bool).tril()
                for j in range(h * group, (h + 1) * group):
                    x = s["q"][own_rows, j].double() @ k.T / math.sqrt(case["D"])
                    out[own_rows, j] = torch.softmax(x.masked_fill(~past, -math.inf), dim=-1) @ v
        first += n
    return out
