"""The 8-bit paged KV cache on CPU and GPU: qk_norm_rope_cache_fp8 / rope_cache_fp8, cache_read_fp8
and decode_attention_fp8 against the definitions in 64 bits, and their refusals."""

from __future__ import annotations

import math

import pytest
import torch

import fp8_reference as ref
import svllm_capi as capi
import svllm_ops
from fp8_reference import E4M3, E8M0

EPS, THETA = 1e-6, 1e6
LLAMA = svllm_ops.Llama3RopeScaling(8.0, 1.0, 4.0, 8192)


def bits(t):
    return t.cpu().view(torch.uint8)


# ------------------------------------------------------------------- the quantising rotary step

def write_case(seed, tokens, heads, kv_heads, dim, *, block=16, max_pos=131071, spread=1.0, pad=0):
    g = torch.Generator().manual_seed(seed)
    num_blocks = -(-max(tokens, 1) // block) + 2
    slots = torch.randperm(num_blocks * block, generator=g)[:tokens]
    if pad:
        slots[-pad:] = -1
    x = torch.randn(tokens, (heads + 2 * kv_heads), dim, generator=g)
    x = x * torch.exp(spread * torch.randn(tokens, heads + 2 * kv_heads, 1, generator=g))
    k_cache, v_cache, k_scale, v_scale = ref.make_cache(seed, num_blocks, block, kv_heads, dim)
    return {"qkv": x.bfloat16().flatten(1), "slots": slots, "caches": (k_cache, v_cache, k_scale,
                                                                       v_scale),
            "positions": torch.randint(0, max_pos + 1, (tokens,), generator=g),
            "weights": (1 + 0.1 * torch.randn(2, dim, generator=g)).bfloat16()}


def split(qkv, heads, kv_heads, dim):
    q, k, v = qkv.split([heads * dim, kv_heads * dim, kv_heads * dim], 1)
    n = len(qkv)
    return q.view(n, heads, dim), k.view(n, kv_heads, dim), v.view(n, kv_heads, dim)


def call_write(c, device, heads, kv_heads, dim, norm, scaling=None, qkv=None, positions=None):
    """Runs the step on a copy of the case; returns q and the caches on the CPU and the inputs."""
    qkv = c["qkv"].to(device).clone() if qkv is None else qkv
    q, k, v = split(qkv, heads, kv_heads, dim)
    caches = [t.clone().to(device) for t in c["caches"]]
    w = c["weights"].to(device)
    pos = (c["positions"] if positions is None else positions).to(device)
    slots = c["slots"].to(device)
    if norm:
        svllm_ops.qk_norm_rope_cache_fp8(q, k, v, w[0], w[1], pos, slots, *caches, EPS, THETA,
                                         scaling)
    else:
        svllm_ops.rope_cache_fp8(q, k, v, pos, slots, *caches, THETA, scaling)
    return q.cpu(), [t.cpu() for t in caches], (k.cpu(), v.cpu())


def check_write(c, got, heads, kv_heads, dim, norm, scaling=None):
    q, (k_cache, v_cache, k_scale, v_scale), (k_after, v_after) = got
    q0, k0, v0 = split(c["qkv"], heads, kv_heads, dim)
    assert torch.equal(k_after, k0) and torch.equal(v_after, v0)  # read only
    inv = svllm_ops.rope_inv_freq(THETA, dim, scaling)
    w = c["weights"] if norm else (None, None)
    want, off = ref.rotate(q0, w[0], c["positions"], inv, EPS)
    assert ((q.double() - want).abs() <= 2.0 ** -8 * want.abs() + off).all()
    old_k, old_v, old_ks, old_vs = c["caches"]
    live = c["slots"] >= 0
    at = c["slots"][live]
    rows = [bits(t).flatten(0, 1)[at] for t in (k_cache, v_cache, k_scale, v_scale)]
    # v: whole bf16 numbers scaled by powers of two, so its codes and scales are known to the bit
    codes, scale, _ = ref.quantise(v0.double()[live])
    assert torch.equal(rows[1], bits(codes)) and torch.equal(rows[3], bits(scale))
    # k: the scale holds the row, and no smaller one would; each code is a rounding of the value
    want, off = ref.rotate(k0, w[1], c["positions"], inv, EPS)
    want, off = want[live], off[live]
    e = rows[2].double() - 127
    amax, slack = want.abs().amax(-1), off.amax(-1)
    assert (amax <= 448 * torch.exp2(e) + slack).all()
    assert ((amax > 224 * torch.exp2(e) - slack) | (e == ref.E_MIN)).all()
    held = rows[0].view(E4M3).double() * torch.exp2(e)[..., None]
    assert ((held - want).abs() <= 2.0 ** -4 * want.abs() + 2.0 ** -10 * torch.exp2(e)[..., None] +
            off).all()
    # every other row is as it was
    others = torch.ones(k_cache.shape[0] * k_cache.shape[1], dtype=torch.bool)
    others[at] = False
    for new, old in zip((k_cache, v_cache, k_scale, v_scale), (old_k, old_v, old_ks, old_vs)):
        assert torch.equal(bits(new).flatten(0, 1)[others], bits(old).flatten(0, 1)[others])


@pytest.mark.parametrize("norm", [True, False], ids=["norm", "plain"])
@pytest.mark.parametrize("tokens, heads, kv_heads, dim, block, pad", [
    (1, 16, 8, 128, 16, 0),
    (1, 1, 1, 64, 1, 0),
    (7, 6, 2, 64, 12, 2),     # passes that mix q, k and v heads
    (33, 5, 5, 128, 16, 0),
    (130, 24, 8, 64, 12, 1),
    (64, 20, 4, 128, 3, 64),  # padding alone
    (300, 32, 2, 128, 256, 5),
    (5, 0, 3, 128, 16, 0),    # no query heads
])
def test_write(device, norm, tokens, heads, kv_heads, dim, block, pad):
    c = write_case(tokens + heads, tokens, heads, kv_heads, dim, block=block, pad=pad)
    scaling = None if norm else LLAMA
    got = call_write(c, device, heads, kv_heads, dim, norm, scaling)
    check_write(c, got, heads, kv_heads, dim, norm, scaling)


@pytest.mark.gpu
@pytest.mark.parametrize("norm", [True, False], ids=["norm", "plain"])
@pytest.mark.parametrize("tokens, heads, kv_heads, dim", [
    (9000, 16, 8, 128), (5003, 24, 8, 64), (20000, 6, 2, 64), (2500, 40, 8, 128)])
def test_write_many_tokens(cuda, norm, tokens, heads, kv_heads, dim):
    c = write_case(3, tokens, heads, kv_heads, dim, pad=3)
    check_write(c, call_write(c, cuda, heads, kv_heads, dim, norm), heads, kv_heads, dim, norm)


@pytest.mark.gpu
@pytest.mark.parametrize("offset, gap", [(1, 0), (8, 0), (0, 5), (0, 8), (3, 3)])
def test_write_rows_off_alignment(cuda, offset, gap):
    """Rows off 16 bytes and at odd strides give the same bits."""
    heads, kv_heads, dim = 6, 2, 128
    c = write_case(4, 40, heads, kv_heads, dim)
    want = call_write(c, cuda, heads, kv_heads, dim, True)
    width = c["qkv"].shape[1]
    room = torch.zeros(40 * (width + gap) + offset, dtype=torch.bfloat16, device=cuda)
    qkv = room[offset:].view(40, width + gap)[:, :width]
    qkv.copy_(c["qkv"])
    got = call_write(c, cuda, heads, kv_heads, dim, True, qkv=qkv)
    assert torch.equal(got[0], want[0])
    for a, b in zip(got[1], want[1]):
        assert torch.equal(bits(a), bits(b))


def test_write_int32_positions_and_no_tokens(device):
    c = write_case(5, 9, 4, 2, 64)
    a = call_write(c, device, 4, 2, 64, True)
    b = call_write(c, device, 4, 2, 64, True, positions=c["positions"].int())
    assert torch.equal(a[0], b[0]) and torch.equal(bits(a[1][0]), bits(b[1][0]))
    empty = write_case(5, 0, 4, 2, 64)
    got = call_write(empty, device, 4, 2, 64, True)
    assert torch.equal(bits(got[1][0]), bits(empty["caches"][0]))


def test_write_far_positions(device):
    """Angles far past fp32's precision, the last position a whole number that fp64 still holds."""
    c = write_case(6, 4, 2, 1, 64)
    c["positions"] = torch.tensor([10 ** 6 + 1, 2 ** 31 - 1, 2 ** 33 + 5, 2 ** 25 + 1])
    q, _, _ = call_write(c, device, 2, 1, 64, False)
    inv = svllm_ops.rope_inv_freq(THETA, 64, None)
    q0 = split(c["qkv"], 2, 1, 64)[0]
    # 2^33 times an inverse frequency of at most 1, in fp64: the angle is off by 2^-20 at most
    want, off = ref.rotate(q0, None, c["positions"], inv, EPS)
    size = 2.0 ** 17 * off
    assert ((q.double() - want).abs() <= 2.0 ** -8 * want.abs() + off + 2.0 ** -19 * size).all()


def test_write_extreme_values(device):
    """Rows of zeros, of the smallest and the largest bf16 numbers, with infinities and NaN."""
    heads, kv_heads, dim = 2, 2, 64
    c = write_case(7, 10, heads, kv_heads, dim, spread=0.0)
    qkv = c["qkv"].view(10, 6, dim)
    big = torch.finfo(torch.bfloat16).max
    qkv[0, 4:] = 0
    qkv[1, 4:] *= 2.0 ** -58
    qkv[2, 4:] *= 2.0 ** -80   # below what the smallest scale holds: zeros
    qkv[3, 4:] *= 2.0 ** 55
    qkv[4, 4:] = big           # past the largest scale: saturated
    qkv[5, 4, 3] = math.inf
    qkv[5, 4, 9] = -math.nan
    qkv[6, 5] = math.nan
    qkv[7, 4] = 448 * 2.0 ** 3   # exactly a scale's largest
    qkv[8, 4] = 450 * 2.0 ** 3   # (a bf16 number) just above
    qkv[9, 4, ::2] = -0.0
    got = call_write(c, device, heads, kv_heads, dim, False)
    codes, scale, e = ref.quantise(qkv[:, 4:].double())
    at = c["slots"]
    assert torch.equal(bits(got[1][1]).flatten(0, 1)[at], bits(codes))
    assert torch.equal(bits(got[1][3]).flatten(0, 1)[at], bits(scale))
    assert e[7, 0] == 3 and e[8, 0] == 4 and e[0, 0] == -60 and e[4, 0] == 60
    held = ref.values(got[1][1], got[1][3]).flatten(0, 1)[at]
    assert held[4].unique().item() == 448 * 2.0 ** 60
    assert held[2].abs().max() == 0
    assert held[5, 0].isnan().sum() == 2 and held[5, 1].isfinite().all()


def test_write_k_that_is_not_finite_stays_in_its_row(device):
    c = write_case(8, 3, 4, 2, 128, spread=0.0)
    clean = call_write(c, device, 4, 2, 128, True)
    c["qkv"].view(3, 8, 128)[1, 4, 7] = math.nan  # k head 0 of token 1
    q, caches, _ = call_write(c, device, 4, 2, 128, True)
    assert torch.equal(q, clean[0])
    held = ref.values(caches[0], caches[2]).flatten(0, 1)[c["slots"]]
    want = ref.values(clean[1][0], clean[1][2]).flatten(0, 1)[c["slots"]]
    assert held[1, 0].isnan().all()  # the norm spreads it over the head
    held[1, 0] = want[1, 0] = 0
    assert torch.equal(held, want)


# --------------------------------------------------------------------------------- the read-back

@pytest.mark.parametrize("lens, kv_heads, dim, block, width", [
    ([100], 8, 128, 16, None),
    ([0, 1, 33, 12, 11, 13], 3, 64, 12, None),
    ([5, 300, 0], 1, 64, 1, None),
    ([17], 2, 128, 256, 3),
    ([0, 0], 2, 64, 16, 2),
    ([1, 16, 15], 20, 64, 16, 5),
])
def test_read(device, lens, kv_heads, dim, block, width):
    tables, total = ref.make_tables(1, lens, block, width=width)
    caches = ref.make_cache(2, total, block, kv_heads, dim, spread=6.0)
    k, v = svllm_ops.cache_read_fp8(*(t.to(device) for t in caches), tables.to(device),
                                    torch.tensor(lens, dtype=torch.int32, device=device))
    shape = (len(lens), tables.shape[1] * block, kv_heads, dim)
    for got, cache, scale in ((k, caches[0], caches[2]), (v, caches[1], caches[3])):
        assert got.shape == shape and got.dtype == torch.bfloat16
        for s, n in enumerate(lens):
            assert torch.equal(got[s, :n].cpu().double(), ref.rows_of(cache, scale, tables[s], n))
            assert (got[s, n:] == 0).all()


def test_read_every_code_and_scale(device):
    codes = torch.arange(256, dtype=torch.uint8).view(2, 128)[None, :, None].expand(121, 2, 1, 128)
    codes = codes.contiguous().view(E4M3)
    scale = (torch.arange(121, dtype=torch.uint8) + 67)[:, None, None].expand(121, 2, 1)
    scale = scale.contiguous().view(E8M0)
    tables = torch.arange(121, dtype=torch.int32)[None]
    k, v = svllm_ops.cache_read_fp8(*(t.to(device) for t in (codes, codes, scale, scale)),
                                    tables.to(device),
                                    torch.tensor([242], dtype=torch.int32, device=device))
    want = ref.values(codes, scale).flatten(0, 1)[None]
    assert torch.equal(k.cpu().double().nan_to_num(7.0), want.nan_to_num(7.0))
    assert torch.equal(v.cpu().isnan(), want.isnan())


# -------------------------------------------------------------------------------- the attention

def run_attention(device, q, caches, tables, lens, scale=None):
    out = svllm_ops.decode_attention_fp8(q.to(device), *(t.to(device) for t in caches),
                                         tables.to(device),
                                         torch.tensor(lens, dtype=torch.int32, device=device),
                                         scale)
    assert out.dtype == torch.bfloat16 and out.shape == q.shape and out.is_contiguous()
    return out.cpu()


def check_attention(device, lens, heads, kv_heads, dim, block, *, width=None, spread=1.0, size=1.0,
                    scale=None, seed=0):
    tables, total = ref.make_tables(seed, lens, block, width=width)
    caches = ref.make_cache(seed + 1, total, block, kv_heads, dim, spread)
    g = torch.Generator().manual_seed(seed + 2)
    q = (torch.randn(len(lens), heads, dim, generator=g) * size).bfloat16()
    out = run_attention(device, q, caches, tables, lens, scale)
    want, bound = ref.attention(q, *caches, tables, lens, scale or dim ** -0.5)
    off = (out.double() - want).abs()
    assert (off <= bound).all(), f"off by up to {(off / bound.clamp(min=1e-300)).max():.3g} bounds"
    return out


@pytest.mark.parametrize("heads, kv_heads, dim", [
    (16, 8, 128), (8, 8, 64), (6, 2, 64), (5, 1, 128), (16, 2, 64), (9, 1, 64), (20, 1, 128)])
@pytest.mark.parametrize("block", [1, 12, 16, 256])
def test_attention(device, heads, kv_heads, dim, block):
    check_attention(device, [0, 1, 2, 15, 16, 17, 31, 32, 33, 64, 65, 100], heads, kv_heads, dim,
                    block)


@pytest.mark.gpu
@pytest.mark.parametrize("lens, heads, kv_heads, dim, block, width", [
    ([5000], 4, 2, 128, 16, None),
    ([4097, 3, 1024], 6, 2, 64, 12, None),
    ([9001], 1, 1, 64, 1, None),
    ([700] * 40, 8, 4, 128, 16, None),
    ([129, 127, 128], 3, 3, 128, 7, 400),     # a table far wider than the requests
    ([2500, 1, 0, 777], 24, 8, 64, 12, None),
    (list(range(0, 520, 4)), 2, 2, 64, 16, None),
    ([30000], 2, 1, 128, 64, None),
    # by items, as clusters of 8, 4 and 2 CTAs, some of which find no rows
    ([1000], 16, 8, 128, 16, None),
    ([1, 2000, 0, 33], 3, 1, 128, 16, None),
    ([900] * 4, 16, 8, 64, 12, None),
    ([2000, 1500, 3], 27, 3, 64, 16, None),
    ([700] * 8, 8, 8, 128, 16, None),
    ([500, 1] * 10, 16, 16, 64, 16, None),
    # by lines, KV heads of 64 in pairs, the last one alone
    ([9000, 70, 0, 4000], 9, 3, 64, 16, None),
    ([9000, 33], 27, 3, 64, 12, None),
    ([600, 1, 77] * 50, 10, 5, 64, 16, None),
    ([3000, 5, 2000, 100] * 16, 8, 4, 64, 1, None),
    ([3000, 5, 2000, 100] * 12, 33, 3, 128, 16, None),
    ([700, 33, 0, 2000] * 4, 27, 3, 64, 16, 2000),
    ([700, 33, 1, 2000] * 4, 3, 1, 64, 12, 9000),
    ([90, 4100], 40, 5, 64, 256, 800),
    # items of few parts: KV heads in pairs with two groups of query heads each, several items a CTA
    ([600, 1, 77] * 50, 27, 3, 64, 16, None),
    ([600, 0, 77] * 50, 9, 3, 64, 16, None),
    ([900, 30, 2000] * 30, 9, 3, 128, 16, None),
    ([900, 30, 2000] * 30, 16, 8, 128, 12, None),
    ([3, 1, 0, 65] * 80, 3, 1, 128, 16, 40),
])
def test_attention_long(cuda, lens, heads, kv_heads, dim, block, width):
    check_attention(cuda, lens, heads, kv_heads, dim, block, width=width)


@pytest.mark.parametrize("spread, size, scale", [
    (8.0, 1.0, None),        # rows 2^-30 to 2^30 apart
    (1.0, 2.0 ** -100, None), (0.3, 2.0 ** 60, 2.0 ** -62), (0.5, 30.0, None), (1.0, 1.0, 1e-6)])
def test_attention_magnitudes(device, spread, size, scale):
    check_attention(device, [1, 40, 200], 4, 2, 64, 16, spread=spread, size=size, scale=scale)


def test_attention_rows_that_are_not_seen_do_not_matter(device):
    """NaN codes and odd scale bytes behind a request's last row and in other blocks."""
    lens, block = [5, 40, 0], 16
    tables, total = ref.make_tables(3, lens, block)
    caches = ref.make_cache(4, total, block, 2, 64)
    g = torch.Generator().manual_seed(5)
    q = torch.randn(3, 4, 64, generator=g).bfloat16()
    want = run_attention(device, q, caches, tables, lens)
    seen = torch.zeros(total * block, dtype=torch.bool)
    for s, n in enumerate(lens):
        j = torch.arange(n)
        seen[tables[s].long()[j // block] * block + j % block] = True
    bad = [bits(t).clone() for t in caches]
    for t, value in zip(bad, (0x7f, 0xff, 255, 0)):
        t.flatten(0, 1)[~seen] = value
    bad = [t.view(d) for t, d in zip(bad, (E4M3, E4M3, E8M0, E8M0))]
    assert torch.equal(run_attention(device, q, bad, tables, lens), want)
    assert (want[2] == 0).all()


def test_attention_a_seen_nan_stays_in_its_head(device):
    lens, block = [40], 16
    tables, total = ref.make_tables(3, lens, block)
    caches = [t.clone() for t in ref.make_cache(4, total, block, 2, 64)]
    q = torch.randn(1, 4, 64, generator=torch.Generator().manual_seed(5)).bfloat16()
    want = run_attention(device, q, caches, tables, lens)
    caches[0].view(torch.uint8)[tables[0, 1].long(), 3, 1, 9] = 0x7f  # K of KV head 1
    out = run_attention(device, q, caches, tables, lens)
    assert torch.equal(out[:, :2], want[:, :2]) and out[:, 2:].isnan().all()
    caches = [t.clone() for t in ref.make_cache(4, total, block, 2, 64)]
    caches[1].view(torch.uint8)[tables[0, 1].long(), 3, 1, 9] = 0x7f  # V, element 9
    out = run_attention(device, q, caches, tables, lens)
    assert out[:, 2:, 9].isnan().all()
    out[:, 2:, 9] = want[:, 2:, 9] = 0
    assert torch.equal(out, want)


def test_attention_of_rows_that_are_zero_and_of_a_zero_query(device):
    lens, block = [40, 7], 16
    tables, total = ref.make_tables(3, lens, block)
    x = torch.randn(total, block, 2, 64, generator=torch.Generator().manual_seed(1)).double()
    codes, scale, _ = ref.quantise(x.bfloat16().double())
    nil, low, _ = ref.quantise(torch.zeros_like(x))
    q = torch.zeros(2, 4, 64).bfloat16()
    out = run_attention(device, q, (codes, codes, scale, scale), tables, lens)
    for s, n in enumerate(lens):  # equal weights: the mean of the rows, rounded
        mean = ref.rows_of(codes, scale, tables[s], n)
        size = mean.abs().mean(0).repeat_interleave(2, 0)
        mean = mean.mean(0).repeat_interleave(2, 0)
        assert ((out[s].double() - mean).abs() <= 2.0 ** -8 * mean.abs() + 2.0 ** -10 * size).all()
    assert (run_attention(device, q + 1, (codes, nil, scale, low), tables, lens) == 0).all()


@pytest.mark.gpu
def test_attention_strides_streams_and_repeats(cuda):
    """q as a view of a qkv projection, another stream, two calls at once: the same bits."""
    lens, block = [900, 33, 1500, 4], 16
    tables, total = ref.make_tables(3, lens, block)
    caches = [t.to(cuda) for t in ref.make_cache(4, total, block, 4, 128)]
    g = torch.Generator().manual_seed(5)
    qkv = torch.randn(4, (8 + 8) * 128, generator=g).bfloat16().to(cuda)
    q = qkv[:, : 8 * 128].view(4, 8, 128)
    t, n = tables.to(cuda), torch.tensor(lens, dtype=torch.int32, device=cuda)
    want = svllm_ops.decode_attention_fp8(q.contiguous(), *caches, t, n)
    assert torch.equal(svllm_ops.decode_attention_fp8(q, *caches, t, n), want)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    outs = []
    for _ in range(5):
        for s in streams:
            with torch.cuda.stream(s):
                outs.append(svllm_ops.decode_attention_fp8(q, *caches, t, n))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


@pytest.mark.gpu
@pytest.mark.parametrize("lens", [[300, 17, 64], [9000, 17, 64]], ids=["by items", "by lines"])
def test_step_captured_and_replayed(cuda, lens):
    """Write, attention and read-back of one step in a graph; replays follow the data, the lengths
    too."""
    heads, kv_heads, dim, block = 8, 4, 128, 16
    tables, total = ref.make_tables(3, lens, block)
    caches = [t.to(cuda) for t in ref.make_cache(4, total, block, kv_heads, dim)]
    start = [t.clone() for t in caches]
    g = torch.Generator().manual_seed(5)
    w = torch.ones(2, dim).bfloat16().to(cuda)
    t, n = tables.to(cuda), torch.tensor(lens, dtype=torch.int32, device=cuda)
    pos = (n - 1).long()
    slots = t.long()[torch.arange(3, device=cuda), pos // block] * block + pos % block
    qkv = torch.zeros(3, (heads + 2 * kv_heads) * dim, device=cuda).bfloat16()

    def step(x):
        q, k, v = split(x, heads, kv_heads, dim)
        svllm_ops.qk_norm_rope_cache_fp8(q, k, v, w[0], w[1], pos, slots, *caches, EPS, THETA)
        return (svllm_ops.decode_attention_fp8(q, *caches, t, n),
                *svllm_ops.cache_read_fp8(*caches, t, n))

    step(qkv)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step(qkv)
    for seed in range(4):
        if seed == 2:  # other lengths in the same tables, one of them none
            n.copy_(torch.tensor([lens[0] // 2, 0, 50], dtype=torch.int32))
        fresh = torch.randn(qkv.shape, generator=g).bfloat16().to(cuda)
        for c, s in zip(caches, start):
            c.copy_(s)
        want = [x.clone() for x in step(fresh.clone())]
        for c, s in zip(caches, start):
            c.copy_(s)
        qkv.copy_(fresh)
        graph.replay()
        for a, b in zip(held, want):
            assert torch.equal(a, b)


@pytest.mark.gpu
def test_two_graphs_replay_at_once(cuda):
    """Graphs of the joined form, captured apart, replayed on two streams: each its own workspace."""
    block, lens = 16, [6000, 9000]
    tables, total = ref.make_tables(3, lens, block)
    caches = [t.to(cuda) for t in ref.make_cache(4, total, block, 2, 64)]
    t, n = tables.to(cuda), torch.tensor(lens, dtype=torch.int32, device=cuda)
    g = torch.Generator().manual_seed(5)
    qs = [torch.randn(2, 4, 64, generator=g).bfloat16().to(cuda) for _ in range(2)]
    want = [svllm_ops.decode_attention_fp8(q, *caches, t, n) for q in qs]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for q in qs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append([svllm_ops.decode_attention_fp8(q, *caches, t, n) for _ in range(20)])
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(5):
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for held, w in zip(outs, want):
        assert all(torch.equal(o, w) for o in held)


@pytest.mark.gpu
def test_slots_past_32_bits(cuda):
    """Rows behind 4 GB of codes: written, attended to and read back."""
    kv_heads, dim, block = 1, 128, 16
    blocks = (1 << 32) // (block * kv_heads * dim) + 64
    caches = [torch.zeros(blocks, block, kv_heads, dim, dtype=torch.uint8, device=cuda).view(E4M3)
              for _ in range(2)]
    caches += [torch.full((blocks, block, kv_heads), 127, dtype=torch.uint8,
                          device=cuda).view(E8M0) for _ in range(2)]
    g = torch.Generator().manual_seed(1)
    x = torch.randn(40, 4, dim, generator=g).bfloat16()
    pages = torch.tensor([blocks - 1, 3, blocks - 7], dtype=torch.int32)
    j = torch.arange(40)
    slots = pages.long()[j // block] * block + j % block
    q, k, v = (t.contiguous().to(cuda) for t in x.split([2, 1, 1], 1))
    svllm_ops.rope_cache_fp8(q, k, v, torch.zeros(40, dtype=torch.long, device=cuda),
                             slots.to(cuda), *caches, THETA)
    codes, scale, _ = ref.quantise(x[:, 2:].double())  # position 0: nothing turns
    held = ref.values(codes, scale)
    n = torch.tensor([40], dtype=torch.int32, device=cuda)
    k_read, v_read = svllm_ops.cache_read_fp8(*caches, pages[None].to(cuda), n)
    assert torch.equal(k_read[0, :40, 0].cpu().double(), held[:, 0])
    assert torch.equal(v_read[0, :40, 0].cpu().double(), held[:, 1])
    for wide in (3, 2000):  # by items, by lines
        t = torch.zeros(1, wide, dtype=torch.int32)
        t[0, :3] = pages
        out = svllm_ops.decode_attention_fp8(q[-1:], *caches, t.to(cuda), n).cpu()
        small = [c.cpu()[:, None] for c in (codes[:, :1], codes[:, 1:], scale[:, :1], scale[:, 1:])]
        want, bound = ref.attention(q[-1:].cpu(), *small, torch.arange(40)[None].int(), [40],
                                    dim ** -0.5)
        assert ((out.double() - want).abs() <= bound).all()
    # nothing else was written: the rows beside them, and those 4 GB below
    for c, fill in zip(caches, (0, 0, 127, 127)):
        flat = c.view(torch.uint8).flatten(0, 1)
        near = torch.cat([slots - 16, slots + 32 * block, slots - (1 << 32) // dim])
        near = near[(near >= 0) & (near < len(flat))]
        near = near[~torch.isin(near, slots)]
        assert (flat[near.to(cuda)] == fill).all()


@pytest.mark.gpu
@pytest.mark.parametrize("width", [None, 700], ids=["by items", "by lines"])
def test_c_abi_gives_the_same_bits(cuda, width):
    """The entry points without LibTorch, a workspace that holds anything and serves calls in turn."""
    lens, block = [5000, 33, 0], 16
    tables, total = ref.make_tables(3, lens, block, width=width)
    caches = [t.to(cuda) for t in ref.make_cache(4, total, block, 2, 128)]
    t, n = tables.to(cuda), torch.tensor(lens, dtype=torch.int32, device=cuda)
    g = torch.Generator().manual_seed(5)
    size = capi.decode_attention_fp8_workspace_bytes(3, 6, 2, 128, t.shape[1], block)
    assert (size > 0) == (width is not None)
    workspace = torch.full((size,), 255, dtype=torch.uint8, device=cuda) if size else None
    for _ in range(3):
        q = torch.randn(3, 6, 128, generator=g).bfloat16().to(cuda)
        out = torch.empty_like(q)
        capi.decode_attention_fp8(out, q, *caches, t, n, 128 ** -0.5, workspace)
        assert torch.equal(out, svllm_ops.decode_attention_fp8(q, *caches, t, n))
    if size:
        for few in (workspace[: size - 1], None):
            with pytest.raises(capi.CapiError):
                capi.decode_attention_fp8(out, q, *caches, t, n, 128 ** -0.5, few)
    k, v = (torch.empty(3, t.shape[1] * block, 2, 128, dtype=torch.bfloat16, device=cuda)
            for _ in range(2))
    capi.cache_read_fp8(k, v, *caches, t, n)
    assert all(torch.equal(a, b) for a, b in
               zip((k, v), svllm_ops.cache_read_fp8(*caches, t, n)))
    c = write_case(4, 40, 6, 2, 128)
    inv = svllm_ops.rope_inv_freq(THETA, 128, None).tolist()
    for norm in (True, False):
        want = call_write(c, cuda, 6, 2, 128, norm)
        q, k, v = split(c["qkv"].to(cuda).clone(), 6, 2, 128)
        own = [x.clone().to(cuda) for x in c["caches"]]
        w, pos, slots = c["weights"].to(cuda), c["positions"].to(cuda), c["slots"].to(cuda)
        if norm:
            capi.qk_norm_rope_cache_fp8(q, k, v, w[0], w[1], pos, slots, *own, EPS, inv)
        else:
            capi.rope_cache_fp8(q, k, v, pos, slots, *own, inv)
        assert torch.equal(q.cpu(), want[0])
        assert all(torch.equal(bits(a), bits(b)) for a, b in zip(own, want[1]))


@pytest.mark.gpu
def test_bad_pages_and_lengths_on_cuda(cuda):
    """Entries outside the cache and lengths past the table are cut to what there is; the error word
    tells, and the other requests are exact."""
    lens, block = [40, 40, 40], 16
    tables, total = ref.make_tables(3, lens, block)
    caches = ref.make_cache(4, total, block, 2, 64)
    dev = [t.to(cuda) for t in caches]
    q = torch.randn(3, 4, 64, generator=torch.Generator().manual_seed(5)).bfloat16()
    want, bound = ref.attention(q, *caches, tables, lens, 64 ** -0.5)
    svllm_ops.read_device_error(0, True)

    def both(t, n):
        t, n = t.to(cuda), torch.tensor(n, dtype=torch.int32, device=cuda)
        out = svllm_ops.decode_attention_fp8(q.to(cuda), *dev, t, n).cpu()
        flag = svllm_ops.read_device_error(0, True)
        k, v = svllm_ops.cache_read_fp8(*dev, t, n)
        return out, k.cpu(), flag, svllm_ops.read_device_error(0, True)

    bad = tables.clone()
    bad[1, 1], bad[1, 2] = total, -5
    out, k, f1, f2 = both(bad, lens)
    assert f1 & 1 and f2 & 1
    zero = tables.clone()
    zero[1, 1] = zero[1, 2] = 0
    good, _ = ref.attention(q, *caches, zero, lens, 64 ** -0.5)
    assert ((out.double() - good).abs() <= 2 * bound + 2.0 ** -6).all()
    assert torch.equal(k[1, :40].double(), ref.rows_of(caches[0], caches[2], zero[1], 40))
    out, k, f1, f2 = both(tables, [40, 1000, -3])
    assert f1 & 1 and f2 & 1
    assert ((out[0].double() - want[0]).abs() <= bound[0]).all()
    assert (out[2] == 0).all() and (k[2] == 0).all()
    full, fb = ref.attention(q, *caches, tables, [40, 48, 0], 64 ** -0.5)
    assert ((out.double() - full).abs() <= fb).all()
    _, _, f1, f2 = both(tables, lens)
    assert f1 == 0 and f2 == 0
    # a slot past the cache writes nothing
    c = write_case(9, 3, 4, 2, 64)
    c["slots"][1] = c["caches"][0].shape[0] * 16
    got = call_write(c, cuda, 4, 2, 64, True)
    assert svllm_ops.read_device_error(0, True) & 1
    c["slots"][1] = -1
    check_write(c, got, 4, 2, 64, True)


def with_scales(caches, rows, byte):
    """The caches with the scales of the given (block, slot, head) rows of K and of V set."""
    out = list(caches)
    for i, at in zip((2, 3), rows):
        scale = caches[i].view(torch.uint8).clone()
        scale[at] = byte
        out[i] = scale.view(E8M0)
    return out


@pytest.mark.parametrize("byte", [0, 66, 188, 254, 255])
def test_scales_out_of_range_are_refused(byte):
    """The writer leaves 2^-60 to 2^60, bytes 67 to 187; others among the rows that are read."""
    lens = [40, 20]
    tables, total = ref.make_tables(3, lens, 16)
    caches = ref.make_cache(4, total, 16, 2, 64)
    q = torch.randn(2, 4, 64, generator=torch.Generator().manual_seed(5)).bfloat16()
    t = tables.tolist()
    seen, behind = (t[1][1], 3, 1), (t[1][1], 4, 1)  # rows 19 and 20 of the second request
    n = torch.tensor(lens, dtype=torch.int32)
    for rows in [(seen, behind), (behind, seen)]:
        bad = with_scales(caches, rows, byte)
        with pytest.raises(RuntimeError, match="scale"):
            svllm_ops.decode_attention_fp8(q, *bad, tables, n)
        with pytest.raises(RuntimeError, match="scale"):
            svllm_ops.cache_read_fp8(*bad, tables, n)
    unseen = with_scales(caches, (behind, behind), byte)
    want, bound = ref.attention(q, *caches, tables, lens, 64 ** -0.5)
    assert ((run_attention("cpu", q, unseen, tables, lens).double() - want).abs() <= bound).all()
    svllm_ops.cache_read_fp8(*unseen, tables, n)


@pytest.mark.gpu
@pytest.mark.parametrize("byte", [0, 66, 188, 254, 255])
@pytest.mark.parametrize("width", [None, 2000], ids=["by items", "by lines"])
@pytest.mark.parametrize("dim", [64, 128])
def test_scales_out_of_range_on_cuda(cuda, byte, width, dim):
    """They raise the error word and count as the nearest in range; a scale behind a request's end is
    not looked at."""
    lens = [40, 20]
    tables, total = ref.make_tables(3, lens, 16, width=width)
    caches = ref.make_cache(4, total, 16, 2, dim)
    q = torch.randn(2, 4, dim, generator=torch.Generator().manual_seed(5)).bfloat16()
    t = tables.tolist()
    seen, behind = (t[1][1], 3, 1), (t[1][1], 4, 1)
    n = torch.tensor(lens, dtype=torch.int32)
    svllm_ops.read_device_error(0, True)
    for rows, flag in [((seen, behind), 1), ((behind, seen), 1), ((behind, behind), 0)]:
        bad = with_scales(caches, rows, byte)
        near = with_scales(caches, rows, min(max(byte, 67), 187))
        got = run_attention(cuda, q, bad, tables, lens)
        assert svllm_ops.read_device_error(0, True) == flag
        assert torch.equal(got, run_attention(cuda, q, near, tables, lens))
        read = svllm_ops.cache_read_fp8(*(c.to(cuda) for c in bad), tables.to(cuda), n.to(cuda))
        assert svllm_ops.read_device_error(0, True) == flag
        want = svllm_ops.cache_read_fp8(*(c.to(cuda) for c in near), tables.to(cuda), n.to(cuda))
        assert torch.equal(read[0], want[0]) and torch.equal(read[1], want[1])
        assert svllm_ops.read_device_error(0, True) == 0


# ------------------------------------------------------------------------------------ refusals

def test_write_refuses():
    c = write_case(1, 4, 4, 2, 64)
    q, k, v = split(c["qkv"].clone(), 4, 2, 64)
    base = dict(q=q, k=k, v=v, q_weight=c["weights"][0], k_weight=c["weights"][1],
                positions=c["positions"], slot_mapping=c["slots"], k_cache=c["caches"][0],
                v_cache=c["caches"][1], k_scale=c["caches"][2], v_scale=c["caches"][3], eps=EPS,
                theta=THETA)

    def refused(match, **change):
        with pytest.raises(RuntimeError, match=match):
            svllm_ops.qk_norm_rope_cache_fp8(**{**base, **change})

    refused("float8_e4m3fn", k_cache=c["caches"][0].float())
    refused("float8_e8m0fnu", k_scale=c["caches"][2].float())
    refused("expected bf16", q=q.float(), k=k.float())
    refused("expected bf16 v", v=v.float())
    refused("contiguous", k_cache=c["caches"][0].transpose(0, 1))
    refused("scales of shape", k_scale=c["caches"][2][:, :, :1].contiguous())
    refused("v of shape", v=v[:, :1])
    refused("slot_mapping", slot_mapping=c["slots"].int())
    refused("slot_mapping", slot_mapping=c["slots"][:3])
    refused("positions", positions=c["positions"][:3])
    refused("does not match|must be contiguous", k_cache=ref.make_cache(1, 3, 16, 3, 64)[0],
            v_cache=ref.make_cache(1, 3, 16, 3, 64)[1], k_scale=ref.make_cache(1, 3, 16, 3, 64)[2],
            v_scale=ref.make_cache(1, 3, 16, 3, 64)[3])
    refused("past the cache", slot_mapping=c["slots"] + 1000)
    wide = ref.make_cache(1, 3, 16, 2, 32)
    with pytest.raises(RuntimeError, match="64 or 128"):
        svllm_ops.rope_cache_fp8(q[..., :32].contiguous(), k[..., :32].contiguous(),
                                 v[..., :32].contiguous(), c["positions"], c["slots"], *wide,
                                 THETA)


def test_read_and_attention_refuse():
    tables, total = ref.make_tables(1, [20, 3], 16)
    caches = ref.make_cache(1, total, 16, 2, 64)
    lens = torch.tensor([20, 3], dtype=torch.int32)
    q = torch.randn(2, 4, 64).bfloat16()
    base = dict(q=q, k_cache=caches[0], v_cache=caches[1], k_scale=caches[2], v_scale=caches[3],
                block_tables=tables, seq_lens=lens)

    def refused(match, **change):
        a = {**base, **change}
        with pytest.raises(RuntimeError, match=match):
            svllm_ops.decode_attention_fp8(**a)
        if not {"q", "scale"} & change.keys():
            del a["q"]
            with pytest.raises(RuntimeError, match=match):
                svllm_ops.cache_read_fp8(**a)

    refused("float8_e4m3fn", v_cache=caches[1].float())
    refused("float8_e8m0fnu", v_scale=caches[3].view(torch.uint8))
    refused("num_blocks, block_size", k_cache=caches[0].flatten(0, 1),
            v_cache=caches[1].flatten(0, 1), k_scale=caches[2].flatten(0, 1),
            v_scale=caches[3].flatten(0, 1))
    refused("int32", block_tables=tables.long())
    refused("int32", seq_lens=lens.long())
    refused("must be", seq_lens=lens[:1])
    refused("does not fit", seq_lens=lens + 40)
    refused("does not fit", seq_lens=-lens)
    refused("outside the cache", block_tables=tables + total)
    refused("expected bf16 q", q=q.float())
    refused("does not match", q=q[:, :3])
    refused("does not match", q=torch.randn(2, 4, 128).bfloat16())
    refused("heads must be contiguous", q=torch.randn(2, 64, 4).bfloat16().transpose(1, 2))
    refused("requests", q=q[:1])
    refused("scale", scale=0.0)
    refused("scale", scale=math.inf)
    refused("scale", scale=3e38)  # past fp32 in base 2


def test_empty_batches(device):
    tables = torch.zeros(0, 3, dtype=torch.int32, device=device)
    caches = [t.to(device) for t in ref.make_cache(1, 3, 16, 2, 64)]
    lens = torch.zeros(0, dtype=torch.int32, device=device)
    q = torch.zeros(0, 4, 64, dtype=torch.bfloat16, device=device)
    assert svllm_ops.decode_attention_fp8(q, *caches, tables, lens).shape == (0, 4, 64)
    k, v = svllm_ops.cache_read_fp8(*caches, tables, lens)
    assert k.shape == v.shape == (0, 48, 2, 64)
    # a table without columns serves requests without rows
    tables = torch.zeros(2, 0, dtype=torch.int32, device=device)
    lens = torch.zeros(2, dtype=torch.int32, device=device)
    q = torch.ones(2, 4, 64, dtype=torch.bfloat16, device=device)
    assert (svllm_ops.decode_attention_fp8(q, *caches, tables, lens) == 0).all()
    assert svllm_ops.cache_read_fp8(*caches, tables, lens)[0].shape == (2, 0, 2, 64)
