"""The 8-bit KV cache's operators in 64 bits, for the tests, and how far an implementation with fp32
arithmetic may be from them."""

from __future__ import annotations

import math

import torch

E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu
E_MIN, E_MAX = -60, 60


def quantise(x):
    """Codes, scales (e8m0) and exponents of rows [..., D] of doubles."""
    finite = torch.isfinite(x)
    amax = torch.where(finite, x.abs(), 0).amax(-1)
    e = torch.full(amax.shape, E_MIN)
    for n in range(E_MAX, E_MIN - 1, -1):  # the least one that holds the row
        e = torch.where(amax <= 448 * 2.0 ** n, n, e)
    e = torch.where(amax > 448 * 2.0 ** E_MAX, E_MAX, e)
    # a multiple of a power of two: the scaled values are exact in fp32 wherever x is a bf16 number
    scaled = (x * torch.exp2(-e.double())[..., None]).clamp(-448, 448)
    codes = torch.where(finite, scaled, math.nan).float().to(E4M3)
    return codes, (e + 127).to(torch.uint8).view(E8M0), e


def values(codes, scale):
    return codes.double() * scale.double()[..., None]


def rotate(x, weight, positions, inv_freq, eps):
    """Norm (where there is a weight) and rotation of heads [T, H, D], and a bound on what fp32
    arithmetic may be off: the sum of squares of up to 128 terms 2^-18 of the norm's factor, its
    other steps, the two products, cos and sin together less than 2^-18 of the two terms."""
    x = x.double()
    if weight is not None:
        x = x / ((x * x).mean(-1, keepdim=True) + eps).sqrt() * weight.double()
    angle = positions.double()[:, None, None] * inv_freq.double()
    c, s = torch.cos(angle), torch.sin(angle)
    a, b = x.chunk(2, -1)
    size = 2.0 ** -17 * (a.abs() + b.abs())
    return torch.cat([a * c - b * s, b * c + a * s], -1), torch.cat([size, size], -1)


def make_cache(seed, num_blocks, block, kv_heads, dim, spread=1.0):
    """Random K and V caches of rows whose magnitudes spread: codes, scales."""
    g = torch.Generator().manual_seed(seed)
    out = []
    for _ in range(2):
        x = torch.randn(num_blocks, block, kv_heads, dim, generator=g)
        x = x * torch.exp(spread * torch.randn(num_blocks, block, kv_heads, 1, generator=g))
        out.append(quantise(x.bfloat16().double())[:2])
    return out[0][0], out[1][0], out[0][1], out[1][1]


def make_tables(seed, lens, block, spare=2, width=None):
    """Pages in random order: block tables [S, width] int32 and the number of blocks."""
    need = [-(-n // block) for n in lens]
    total = sum(need) + spare
    order = torch.randperm(total, generator=torch.Generator().manual_seed(seed)).tolist()
    width = max(need + [1]) if width is None else width
    tables, at = [], 0
    for n in need:
        tables.append(order[at: at + n] + [0] * (width - n))
        at += n
    return torch.tensor(tables, dtype=torch.int32).view(len(lens), width), total


def rows_of(cache, scale, table, n):
    """The first n cached rows of a request, [n, Hk, D] doubles."""
    block = cache.shape[1]
    j = torch.arange(n)
    slot = table.long()[j // block] * block + j % block
    v = values(cache, scale)
    return v.flatten(0, 1)[slot]


def attention(q, k_cache, v_cache, k_scale, v_scale, tables, lens, scale):
    """Output in 64 bits and the bound of an element: half a bf16 step of the result, and of the sum
    of weighted magnitudes 2^-11 for weights rounded to f16, 2^-17 (1 + size of the scores) twice
    for the scores' fp32 sums and the exponential, numerator and denominator, and 2^-23 a row for
    the fp32 sums over the rows."""
    seqs, heads, dim = q.shape
    kv_heads = k_cache.shape[2]
    out = torch.zeros(seqs, heads, dim, dtype=torch.float64)
    bound = torch.zeros_like(out)
    for s, n in enumerate(lens):
        if n == 0:
            continue
        k, v = rows_of(k_cache, k_scale, tables[s], n), rows_of(v_cache, v_scale, tables[s], n)
        for h in range(heads):
            kh = h // (heads // kv_heads)
            x = q[s, h].double()
            p = torch.softmax(k[:, kh] @ x * scale, 0)
            out[s, h] = p @ v[:, kh]
            size = (k[:, kh].abs() @ x.abs()).max().item() * scale
            part = 2.0 ** -11 + 2.0 ** -16 * (1 + size) + n * 2.0 ** -23
            bound[s, h] = 2.0 ** -8 * out[s, h].abs() + part * (p @ v[:, kh].abs())
    return out, bound
