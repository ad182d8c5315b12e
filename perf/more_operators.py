"""Workloads of the operators of the 8-bit paged KV cache: the rotary step that quantises K and V as
it writes them, decode attention over the quantised cache, and the read-back of whole requests in
bf16.

A cache holds e4m3 codes [blocks, block_size, KV heads, head_dim] and one power-of-two scale for
each row of head_dim codes, [blocks, block_size, KV heads] in e8m0: a row x is held with the least
whole e for which its largest magnitude is at most 448 * 2^e, e in [-60, 60], as x * 2^-e rounded
to e4m3.

`run` computes one pass: in elementary torch operations where `own` is false, through svllm_ops
where it is true. Both take what `prepare` made. Request lengths follow from the case alone
(`lengths`), values from the seed.
"""

from __future__ import annotations

import math
import os
import sys

import numpy as np
import torch

own = False

DEV = "cuda"
E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu
E_MIN, E_MAX = -60, 60
EPS = 1e-6
LLAMA_SCALING = (8.0, 1.0, 4.0, 8192)  # factor, low and high frequency factor, original length
_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _ops():
    path = os.path.join(_ROOT, "small-vllm_b200", "python")
    if path not in sys.path:
        sys.path.insert(0, path)
    import svllm_ops

    return svllm_ops


# ------------------------------------------------------------------------------------- cases

def _write(name, tokens, heads, kv_heads, dim, norm, max_pos, block=16, pad=0):
    return {"name": name, "op": "write", "tokens": tokens, "heads": heads, "kv_heads": kv_heads,
            "dim": dim, "norm": norm, "max_pos": max_pos, "block": block, "pad": pad}


def _attn(name, requests, lo, hi, heads, kv_heads, dim, block=16):
    return {"name": name, "op": "attention", "requests": requests, "lo": lo, "hi": hi,
            "heads": heads, "kv_heads": kv_heads, "dim": dim, "block": block}


def _read(name, requests, lo, hi, kv_heads, dim, block=16):
    return {"name": name, "op": "read", "requests": requests, "lo": lo, "hi": hi,
            "kv_heads": kv_heads, "dim": dim, "block": block}


def listed():
    return [
        # one user's decode step: latency is everything
        _write("write 1 token", 1, 16, 8, 128, True, 700),
        # a full decode batch, far positions, some rows padding
        _write("write 256 decode", 256, 16, 8, 128, True, 131071, pad=7),
        # an odd chunk of a prompt without norms, three query heads per KV head, 12-token pages
        _write("write 5003 llama", 5003, 24, 8, 64, False, 131071, block=12, pad=1),
        # a packed prefill of long prompts: the largest
        _write("write 64k prefill", 65536, 16, 8, 128, True, 32768),
        # one user right after a short prompt
        _attn("attn 1 over 200", 1, 200, 200, 16, 8, 128),
        # one user with a long document: the cache has to be split over the GPU
        _attn("attn 1 over 32k", 1, 32760, 32760, 16, 8, 128),
        # odd everything: 3 query heads per KV head, 12-token pages, lengths from 1 on
        _attn("attn odd 13 over 1-2500", 13, 1, 2500, 24, 8, 64, block=12),
        # many query heads per KV head
        _attn("attn 48 over 1-4k", 48, 1, 4096, 32, 4, 128),
        # a full serving batch over ordinary contexts: the largest
        _attn("attn 64 over 2k-4k", 64, 2048, 4096, 16, 8, 128),
        # one short request handed to a prefill step
        _read("read 1 of 100", 1, 100, 100, 8, 128),
        # requests of all lengths, behind which most of the rectangle is empty
        _read("read odd 9 of 0-3001", 9, 0, 3001, 4, 64, block=12),
        # a batch of long prompts read for the next chunk: the largest
        _read("read 32 of 4k-8k", 32, 4096, 8192, 8, 128),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["write", "write", "attention", "attention", "attention", "read"])
    heads, kv, dim = rng.choice([(16, 8, 128), (32, 8, 64), (8, 8, 128), (24, 8, 64), (28, 4, 128),
                                 (20, 4, 128), (32, 4, 128), (8, 1, 64), (6, 2, 64), (32, 2, 128)])
    block = rng.choice([1, 8, 12, 16, 16, 32, 64, 256])
    if op == "write":
        most = 65536 * 32 * 128 // ((heads + 2 * kv) * dim)
        return {"op": op, "tokens": _log_int(rng, 1, most), "heads": heads, "kv_heads": kv,
                "dim": dim, "norm": rng.choice([True, False]),
                "max_pos": rng.choice([4095, 32768, 131071]), "block": block,
                "pad": rng.choice([0, 0, 3])}
    if op == "attention":
        hi = _log_int(rng, 1, 32768)
        most = 64 * 3000 * 8 * 128 // (hi * kv * dim)
        return {"op": op, "requests": _log_int(rng, 1, max(1, min(64, most))),
                "lo": rng.randint(0, hi), "hi": hi, "heads": heads, "kv_heads": kv, "dim": dim,
                "block": block}
    hi = _log_int(rng, 1, 8192)
    most = 32 * 8192 * 8 * 128 // (hi * kv * dim)
    return {"op": op, "requests": _log_int(rng, 1, max(1, min(64, most))),
            "lo": rng.randint(0, hi), "hi": hi, "kv_heads": kv, "dim": dim, "block": block}


def lengths(case):
    """Cached tokens of every request: spread over the case's range, the first request at its top."""
    part = np.arange(case["requests"]) * 0.6180339887 % 1
    return case["hi"] - np.floor(part * (case["hi"] - case["lo"] + 1)).astype(np.int64)


# ------------------------------------------------------------------------------------- inputs

def _quantise(x):
    """Codes and scales of rows [..., head_dim]."""
    amax = x.abs().amax(-1)
    m, e = torch.frexp(amax)  # amax = m * 2^e, m in [0.5, 1); 448 = 0.875 * 2^9
    e = torch.where(m <= 0.875, e - 9, e - 8).clamp(E_MIN, E_MAX)
    e = torch.where(amax > 0, e, E_MIN)
    codes = (x * torch.exp2(-e.to(x.dtype))[..., None]).clamp(-448, 448).to(E4M3)
    return codes, (e + 127).to(torch.uint8).view(E8M0)


def _rows(gen, *shape):
    """bf16 rows of K or V: normal values, rows of different magnitudes."""
    x = torch.randn(*shape, device=DEV, generator=gen)
    size = torch.exp(torch.randn(*shape[:-1], 1, device=DEV, generator=gen))
    return (x * size).bfloat16()


def _inv_freq(case):
    """Hugging Face's fp32 table, an input of the rotation: 1 / theta^(2i / dim), and for the
    kind without norms its llama3 rule on top."""
    dim = case["dim"]
    theta = 1e6 if case["norm"] else 5e5
    exponent = torch.arange(0, dim, 2).float() / float(dim)
    table = torch.reciprocal(torch.pow(theta, exponent))
    if case["norm"]:
        return table
    factor, low, high, length = LLAMA_SCALING
    wave = torch.reciprocal(table) * (2 * math.pi)
    scaled = torch.where(wave > length / low, table / factor, table)
    smooth = (torch.reciprocal(wave) * length - low) / (high - low)
    smoothed = (1 - smooth) * scaled / factor + smooth * scaled
    medium = ~(wave < length / high) & ~(wave > length / low)
    return torch.where(medium, smoothed, scaled)


def _dev(a, dtype=None):
    t = torch.from_numpy(np.ascontiguousarray(a))
    return t.to(DEV, dtype=dtype) if dtype else t.to(DEV)


def prepare(case, seed):
    rng = np.random.default_rng(seed)
    gen = torch.Generator(device=DEV).manual_seed(seed)
    kv, dim, block = case["kv_heads"], case["dim"], case["block"]
    if case["op"] == "write":
        tokens, heads = case["tokens"], case["heads"]
        num_blocks = -(-tokens // block) + 2
        # tokens fill random pages in order; the last ones are padding
        pages = torch.randperm(num_blocks, generator=gen, device=DEV)
        t = torch.arange(tokens, device=DEV)
        slots = pages[t // block] * block + t % block
        slots[max(0, tokens - case["pad"]):] = -1
        qkv = torch.randn(tokens, (heads + 2 * kv) * dim, device=DEV, generator=gen).bfloat16()
        q, k, v = qkv.split([heads * dim, kv * dim, kv * dim], 1)
        old = _quantise(_rows(gen, 2, num_blocks, block, kv, dim).float())
        weight = 1 + 0.1 * torch.randn(2, dim, device=DEV, generator=gen)
        return {"case": case, "q": q.view(tokens, heads, dim), "k": k.view(tokens, kv, dim),
                "v": v.view(tokens, kv, dim), "q_weight": weight[0].bfloat16(),
                "k_weight": weight[1].bfloat16(), "slot_mapping": slots,
                "positions": torch.randint(0, case["max_pos"] + 1, (tokens,), device=DEV,
                                           generator=gen),
                "k_cache": old[0][0], "v_cache": old[0][1], "k_scale": old[1][0],
                "v_scale": old[1][1], "inv_freq": _inv_freq(case).to(DEV),
                "theta": 1e6 if case["norm"] else 5e5}
    n = lengths(case)
    need = -(-n // block)
    num_blocks = int(need.sum()) + 3
    order = rng.permutation(num_blocks)
    width = max(1, int(need.max(initial=1)))
    tables = np.zeros((len(n), width), np.int32)
    first = np.concatenate([[0], np.cumsum(need)])
    for s in range(len(n)):
        tables[s, : need[s]] = order[first[s]: first[s + 1]]
    state = {"case": case, "block_tables": _dev(tables), "seq_lens": _dev(n, torch.int32)}
    for name in "kv":
        state[name + "_cache"], state[name + "_scale"] = _quantise(
            _rows(gen, num_blocks, block, kv, dim).float())
    if case["op"] == "attention":
        heads = case["heads"]
        qkv = torch.randn(len(n), (heads + 2 * kv) * dim, device=DEV, generator=gen).bfloat16()
        state["q"] = qkv[:, : heads * dim].view(len(n), heads, dim)
        state["scale"] = dim ** -0.5
    return state


# ------------------------------------------------------------------------------- plain forms

def _rotate(x, weight, cos, sin):
    """Norm (where there is a weight) and rotation of heads [T, H, D] in fp32."""
    x = x.float()
    if weight is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * weight.float()
    a, b = x.chunk(2, -1)
    cos, sin = cos[:, None], sin[:, None]
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)


def _plain_write(s):
    # angles of far positions lose what matters in 32 bits
    angle = s["positions"].double()[:, None] * s["inv_freq"].double()
    cos, sin = torch.cos(angle).float(), torch.sin(angle).float()
    norm = s["case"]["norm"]
    q = _rotate(s["q"], s["q_weight"] if norm else None, cos, sin)
    k = _rotate(s["k"], s["k_weight"] if norm else None, cos, sin)
    live = s["slot_mapping"] >= 0
    at = s["slot_mapping"][live]
    for name, x in (("k", k), ("v", s["v"].float())):
        codes, scale = _quantise(x[live])
        s[name + "_cache"].view(torch.uint8).flatten(0, 1)[at] = codes.view(torch.uint8)
        s[name + "_scale"].view(torch.uint8).flatten(0, 1)[at] = scale.view(torch.uint8)
    s["q"].copy_(q)
    return {x: s[x] for x in ("q", "k_cache", "v_cache", "k_scale", "v_scale")}


def _gathered(s, name):
    """A cache's rows of every request, [S, rows, KV heads, D] in fp32."""
    at = s["block_tables"].long()
    codes = s[name + "_cache"].view(torch.uint8)[at].view(E4M3)
    scale = s[name + "_scale"].view(torch.uint8)[at].view(E8M0)
    return codes.flatten(1, 2).float() * scale.flatten(1, 2).float()[..., None]


def _plain_read(s):
    out = []
    for name in "kv":
        x = _gathered(s, name)
        live = torch.arange(x.shape[1], device=x.device) < s["seq_lens"][:, None]
        out.append(torch.where(live[:, :, None, None], x, 0).bfloat16())
    return out


def _plain_attention(s):
    k, v = _gathered(s, "k"), _gathered(s, "v")
    seqs, rows, kv, dim = k.shape
    q = s["q"].float().view(seqs, kv, -1, dim)
    x = torch.einsum("shgd,slhd->shgl", q, k) * s["scale"]
    live = torch.arange(rows, device=x.device) < s["seq_lens"][:, None]
    x = x.masked_fill(~live[:, None, None], -math.inf)
    top = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(top == -math.inf, 0, top))
    total = p.sum(-1, keepdim=True)
    p = torch.where(total > 0, p / total, 0)
    o = torch.einsum("shgl,slhd->shgd", p, v)
    return o.reshape(seqs, -1, dim).to(s["q"].dtype)


def run(s):
    op = s["case"]["op"]
    if not own:
        return {"write": _plain_write, "attention": _plain_attention, "read": _plain_read}[op](s)
    ops = _ops()
    caches = (s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"])
    if op == "attention":
        return ops.decode_attention_fp8(s["q"], *caches, s["block_tables"], s["seq_lens"],
                                        s["scale"])
    if op == "read":
        return ops.cache_read_fp8(*caches, s["block_tables"], s["seq_lens"])
    if s["case"]["norm"]:
        ops.qk_norm_rope_cache_fp8(s["q"], s["k"], s["v"], s["q_weight"], s["k_weight"],
                                   s["positions"], s["slot_mapping"], *caches, EPS, s["theta"])
    else:
        ops.rope_cache_fp8(s["q"], s["k"], s["v"], s["positions"], s["slot_mapping"], *caches,
                           s["theta"], ops.Llama3RopeScaling(*LLAMA_SCALING))
    return {x: s[x] for x in ("q", "k_cache", "v_cache", "k_scale", "v_scale")}


# ------------------------------------------------------------------------------ work, 64 bits

def work(case):
    kv, dim = case["kv_heads"], case["dim"]
    row = 2 * kv * (dim + 1)  # a token's codes and scales, K and V
    if case["op"] == "write":
        tokens, heads = case["tokens"], case["heads"]
        # q in and out, k and v in, position and slot; padding writes no cache
        return {"bytes": tokens * (4 * heads * dim + 4 * kv * dim + 16) +
                max(0, tokens - case["pad"]) * row,
                "flops": tokens * (heads + kv) * dim * (8 if case["norm"] else 3)}
    n = lengths(case)
    pages = -(-n // case["block"])
    cached = int(n.sum()) * row + 4 * int(pages.sum()) + 4 * len(n)
    if case["op"] == "read":
        rows = len(n) * max(1, int(pages.max(initial=1))) * case["block"]
        return {"bytes": cached + rows * 4 * kv * dim, "flops": 0}
    return {"bytes": cached + 4 * len(n) * case["heads"] * dim,
            "flops": 4 * case["heads"] * dim * int(n.sum())}


def exact(case, seed):
    """The definitions in 64 bits: request by request, and for the caches the values before they
    are rounded to codes."""
    s = prepare(case, seed)
    kv, dim = case["kv_heads"], case["dim"]
    if case["op"] == "write":
        angle = s["positions"].double().unsqueeze(1) * s["inv_freq"].double()
        turn = torch.polar(torch.ones_like(angle), angle).unsqueeze(1)  # one complex factor a pair
        new = {"v": s["v"].double()}
        for name in "qk":
            x = s[name].double()
            if case["norm"]:
                x = x / (x.square().sum(-1, keepdim=True) / dim + EPS).sqrt()
                x = x * s[name + "_weight"].double()
            y = torch.complex(x[..., : dim // 2], x[..., dim // 2:]) * turn
            new[name] = torch.cat([y.real, y.imag], -1)
        out = {"q": new["q"]}
        put = torch.nonzero(s["slot_mapping"] >= 0).flatten()
        for name in "kv":
            x = new[name][put]
            e = torch.ceil(torch.log2(x.abs().amax(-1) / 448)).clamp(E_MIN, E_MAX)
            codes, scale = s[name + "_cache"].double(), s[name + "_scale"].double()
            codes.view(-1, kv, dim)[s["slot_mapping"][put]] = x / torch.exp2(e).unsqueeze(-1)
            scale.view(-1, kv)[s["slot_mapping"][put]] = torch.exp2(e)
            out[name + "_cache"], out[name + "_scale"] = codes, scale
        return out
    tables, n = s["block_tables"].cpu().numpy().astype(np.int64), lengths(case)
    block = case["block"]
    rows = tables.shape[1] * block
    if case["op"] == "read":
        out = [torch.zeros(len(n), rows, kv, dim, dtype=torch.float64, device=DEV) for _ in "kv"]
    else:
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    for b in range(len(n)):
        j = np.arange(n[b])
        slot = _dev(tables[b][j // block] * block + j % block)
        k, v = (s[x + "_cache"].view(-1, kv, dim).view(torch.uint8)[slot].view(E4M3).double() *
                s[x + "_scale"].view(-1, kv).view(torch.uint8)[slot].view(E8M0).double()
                .unsqueeze(-1) for x in "kv")
        if case["op"] == "read":
            out[0][b, : n[b]], out[1][b, : n[b]] = k, v
        elif n[b]:
            for h in range(case["heads"]):
                g = h * kv // case["heads"]
                p = torch.softmax(k[:, g] @ s["q"][b, h].double() * s["scale"], 0)
                out[b, h] = p @ v[:, g]
    return out
