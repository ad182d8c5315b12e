"""decode_attention_fp8 over rows whose V scales lie at both ends of their range, 2^-60 to 2^60: what a
row adds to the denominator does not depend on its V's scale, whatever the weights of the numerators
are held as."""

from __future__ import annotations

import math

import pytest
import torch

import fp8_reference as ref
import svllm_ops
from test_cache_fp8 import check_attention

LN2 = math.log(2.0)  # as the scale: scores in base 2 are q . k


def one_request(n, kv_heads, dim, scores, exponents, seed, nil=False):
    """A request of n rows over pages in order: K rows that give the scores, V rows of magnitudes 224 to
    448 times 2^exponent (or, where nil, zeros in place of the smallest): caches, K and V in doubles."""
    g = torch.Generator().manual_seed(seed)
    k = torch.zeros(n, kv_heads, dim, dtype=torch.float64)
    k[:, :, 0] = scores[:, None]
    size = (224 + 224 * torch.rand(n, kv_heads, dim, generator=g)).bfloat16().double()
    sign = torch.randint(0, 2, (n, kv_heads, dim), generator=g) * 2 - 1
    v = (size * sign).clamp(-448, 448) * torch.exp2(exponents.double())[:, None, None]
    if nil:
        v[exponents == ref.E_MIN] = 0
    block = 16
    pages = -(-n // block)
    caches = []
    for x in (k, v):
        codes, scale, _ = ref.quantise(x)
        held = torch.zeros(pages * block, kv_heads, dim, dtype=torch.uint8)
        held[:n] = codes.view(torch.uint8)
        rows = torch.full((pages * block, kv_heads), 127, dtype=torch.uint8)
        rows[:n] = scale.view(torch.uint8)
        caches.append((held.view(pages, block, kv_heads, dim).view(ref.E4M3),
                       rows.view(pages, block, kv_heads).view(ref.E8M0), ref.values(codes, scale)))
    (kc, ks, k), (vc, vs, v) = caches
    assert torch.equal(k[:, :, 0], scores[:, None].expand(n, kv_heads))  # the scores are exact
    assert torch.equal(vs.view(torch.uint8).flatten(0, 1)[:n, 0].long() - 127, exponents)
    return (kc, vc, ks, vs), v


def check(device, n, requests, heads, kv_heads, dim, width, scores, exponents, nil=False):
    caches, v = one_request(n, kv_heads, dim, scores, exponents, n + requests, nil)
    pages = -(-n // 16)
    tables = torch.zeros(requests, width or pages, dtype=torch.int32)
    tables[:, :pages] = torch.arange(pages)  # every request reads the same pages
    q = torch.zeros(requests, heads, dim, dtype=torch.bfloat16)
    q[:, :, 0] = 1
    out = svllm_ops.decode_attention_fp8(
        q.to(device), *(c.to(device) for c in caches), tables.to(device),
        torch.full((requests,), n, dtype=torch.int32, device=device), LN2).cpu().double()
    p = torch.exp2(scores - scores.max())
    p = p / p.sum()
    want = torch.einsum("n,nhd->hd", p, v).repeat_interleave(heads // kv_heads, 0)
    parts = torch.einsum("n,nhd->hd", p, v.abs()).repeat_interleave(heads // kv_heads, 0)
    # half a bf16 step; as fp8_reference.attention, of the parts' magnitudes: weights rounded to f16,
    # scores and exponentials, fp32 sums; weights below 2^-31 of the largest lost, each times codes
    # that are at most twice those of the largest
    size = scores.abs().max().item() * LN2
    off = 2.0 ** -8 * want.abs() + parts * (2.0 ** -11 + 2.0 ** -16 * (1 + size) +
                                            n * (2.0 ** -23 + 2.0 ** -30))
    wrong = (out - want).abs() / off
    assert (wrong <= 1).all(), f"off by up to {wrong.max():.3g} bounds, " \
        f"{(out / want).abs().max():.3g} of the value"


def mixture(n, place, high, low, high_exponent=ref.E_MAX, low_exponent=ref.E_MIN):
    """One row of score `high` and a large V among rows of score `low` and small ones."""
    scores = torch.full((n,), float(low), dtype=torch.float64)
    exponents = torch.full((n,), low_exponent)
    at = {"first": 0, "middle": n // 2, "last": n - 1}[place]
    scores[at], exponents[at] = high, high_exponent
    return scores, exponents


@pytest.mark.parametrize("high, low, high_exponent", [
    (0, -13, 60),    # a low row's weight is 2^-127 after its V's scale
    (0, -7, 60),     # the maxima of parts without the high row lie 127 lower
    (13, 0, 60),
    (0, -22, 51),
    (0, 104, 60),    # the low rows have all of the sum, the high one most of the result
    (0, 0, 60),
    (0, -60, 60),
])
@pytest.mark.parametrize("place", ["first", "middle", "last"])
def test_one_large_row_among_many_small(device, high, low, high_exponent, place):
    """By items: a CTA, or a cluster, an item."""
    scores, exponents = mixture(250, place, high, low, high_exponent)
    check(device, 250, 2, 4, 2, 64, None, scores, exponents)
    check(device, 250, 1, 3, 1, 128, None, scores, exponents, nil=True)
    scores, exponents = mixture(1900, place, high, low, high_exponent)
    check(device, 1900, 1, 2, 1, 128, None, scores, exponents)
    check(device, 1900, 2, 4, 2, 64, None, scores, exponents, nil=True)


@pytest.mark.gpu
@pytest.mark.parametrize("n, requests, heads, kv_heads, dim, width", [
    (250, 2, 4, 2, 64, 4000),      # whole items in a table far wider
    (250, 2, 5, 1, 128, 4000),
    (32000, 1, 8, 4, 128, None),   # many parts an item
    (32000, 1, 8, 4, 64, None),
    (9000, 3, 9, 3, 64, None),
    (2000, 30, 16, 8, 128, None),  # few parts an item
    (2000, 64, 16, 8, 64, None),   # KV heads in pairs
    (2000, 40, 33, 3, 64, None),
])
@pytest.mark.parametrize("high, low, high_exponent",
                         [(0, -13, 60), (0, -7, 60), (0, -22, 51), (0, 104, 60)])
@pytest.mark.parametrize("place", ["first", "middle", "last"])
def test_by_lines(cuda, n, requests, heads, kv_heads, dim, width, high, low, high_exponent, place):
    scores, exponents = mixture(n, place, high, low, high_exponent)
    check(cuda, n, requests, heads, kv_heads, dim, width, scores, exponents)


@pytest.mark.parametrize("seed", range(4))
def test_scales_spread_over_the_whole_range(device, seed):
    g = torch.Generator().manual_seed(seed)
    n = 1500
    exponents = torch.randint(ref.E_MIN, ref.E_MAX + 1, (n,), generator=g)
    scores = torch.randint(-15, 16, (n,), generator=g).double() * 2.0 ** seed
    check(device, n, 2, 4, 2, 128, None, scores, exponents)


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("top", [2, 3])
def test_scores_whose_steps_pass_the_slack(cuda, dim, top):
    """Scores of 2^27, where fp32 holds only multiples of 16: a maximum one or two such steps above the
    running one still moves it, and the row of the largest score has all the weight."""
    n, base = 64, 2.0 ** 27
    g = torch.Generator().manual_seed(dim)
    k = torch.zeros(n, 1, dim, dtype=torch.float64)
    k[:, 0, 0], k[:, 0, 1] = 128, 1
    k[n - 1, 0, 1] = top  # in the second step of a warp
    v = (128 + 256 * torch.rand(n, 1, dim, generator=g)).bfloat16().double()  # scales of 1
    caches = []
    for x in (k, v):
        codes, scale, _ = ref.quantise(x)
        caches.append((codes.view(4, 16, 1, dim), scale.view(4, 16, 1)))
    tables = torch.zeros(1, 1000, dtype=torch.int32)
    tables[0, :4] = torch.arange(4)
    q = torch.zeros(1, 3, dim, dtype=torch.bfloat16)
    q[:, :, 0], q[:, :, 1] = base / 128, 16
    out = svllm_ops.decode_attention_fp8(
        q.to(cuda), *(t.to(cuda) for t in (caches[0][0], caches[1][0], caches[0][1], caches[1][1])),
        tables.to(cuda), torch.tensor([n], dtype=torch.int32, device=cuda), LN2).cpu().double()
    want = ref.values(*caches[1]).view(n, dim)[n - 1].expand(3, dim)
    # the others weigh 63 * 2^-16 together, their values at most four times this row's
    assert ((out[0] - want).abs() <= (2.0 ** -8 + 2.0 ** -11 + 4 * 63 * 2.0 ** -16) * want).all()


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("power", [-120, 100, 116, 120])
def test_query_magnitudes(device, power, dim):
    """Queries anywhere in bf16's range under a scale that brings the scores back."""
    check_attention(device, [1, 40, 200], 4, 2, dim, 16, spread=0.3, size=2.0 ** power,
                    scale=2.0 ** (-2 - power))


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("power", [90, 127])
def test_large_queries_across_large_keys(device, dim, power):
    """Scores of exactly 0 between the largest queries and the largest rows of K: the mean of V."""
    n, block = 70, 16
    g = torch.Generator().manual_seed(dim)
    k = (224 + 224 * torch.rand(n + 10, 2, dim, generator=g)).bfloat16().double() * 2.0 ** 60
    k[:, :, 0] = 0
    v = (1 + torch.rand(n + 10, 2, dim, generator=g)).bfloat16().double()
    caches = []
    for x in (k, v):
        codes, scale, _ = ref.quantise(x)
        caches.append((codes.view(5, block, 2, dim), scale.view(5, block, 2)))
    q = torch.zeros(1, 4, dim, dtype=torch.bfloat16)
    q[:, :, 0] = 2.0 ** power
    want = ref.values(*caches[1]).flatten(0, 1)[:n].mean(0).repeat_interleave(2, 0)
    for width in (5, 2000):
        tables = torch.zeros(1, width, dtype=torch.int32)
        tables[0, :5] = torch.arange(5)
        out = svllm_ops.decode_attention_fp8(
            q.to(device), *(t.to(device) for t in (caches[0][0], caches[1][0], caches[0][1],
                                                   caches[1][1])),
            tables.to(device), torch.tensor([n], dtype=torch.int32, device=device)).cpu().double()
        assert ((out[0] - want).abs() <= (2.0 ** -8 + 2.0 ** -11 + n * 2.0 ** -23) * want).all()
