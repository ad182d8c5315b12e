"""Lists that contradict the cache, on CUDA: the requests that they do not name are as before, to the
bit where the batch is cut in the same places, and the one that they do is what the replaced entry or
the cut length gives."""

from __future__ import annotations

import pytest
import torch

import fp8_reference as ref
import svllm_ops

LENS = [40, 45, 33]


def run(cuda, q, caches, tables, lens):
    dev = [c.to(cuda) for c in caches]
    t, n = tables.to(cuda), torch.tensor(lens, dtype=torch.int32, device=cuda)
    svllm_ops.read_device_error(0, True)
    out = svllm_ops.decode_attention_fp8(q.to(cuda), *dev, t, n).cpu()
    first = svllm_ops.read_device_error(0, True)
    k, v = svllm_ops.cache_read_fp8(*dev, t, n)
    return out, k.cpu(), v.cpu(), (first, svllm_ops.read_device_error(0, True))


@pytest.mark.gpu
@pytest.mark.parametrize("width", [None, 3000], ids=["by items", "by lines"])
@pytest.mark.parametrize("heads, kv_heads, dim", [(4, 2, 64), (6, 2, 128)])
@pytest.mark.parametrize("entry", ["past", "far past", "negative"])
def test_blocks_outside_the_cache(cuda, width, heads, kv_heads, dim, entry):
    tables, total = ref.make_tables(3, LENS, 16, width=width)
    caches = ref.make_cache(4, total, 16, kv_heads, dim)
    q = torch.randn(3, heads, dim, generator=torch.Generator().manual_seed(5)).bfloat16()
    good = run(cuda, q, caches, tables, LENS)
    assert good[3] == (0, 0)
    bad, zero = tables.clone(), tables.clone()
    bad[1, 1] = {"past": total, "far past": 2 ** 31 - 1, "negative": -2 ** 31}[entry]
    zero[1, 1] = 0
    out, k, v, flags = run(cuda, q, caches, bad, LENS)
    assert flags == (1, 1)
    for s in (0, 2):
        assert torch.equal(out[s], good[0][s])
        assert torch.equal(k[s], good[1][s]) and torch.equal(v[s], good[2][s])
    want, bound = ref.attention(q, *caches, zero, LENS, dim ** -0.5)
    assert ((out.double() - want).abs() <= bound).all()
    n = LENS[1]
    assert torch.equal(k[1, :n].double(), ref.rows_of(caches[0], caches[2], zero[1], n))
    assert torch.equal(v[1, :n].double(), ref.rows_of(caches[1], caches[3], zero[1], n))
    # behind the request's end nothing is looked at
    behind = tables.clone()
    behind[2, 3:] = -7
    if behind.shape[1] > 3:
        assert run(cuda, q, caches, behind, LENS)[3] == (0, 0)


@pytest.mark.gpu
@pytest.mark.parametrize("width", [3, 3000], ids=["by items", "by lines"])
@pytest.mark.parametrize("length, cut", [(-1, 0), (-2 ** 31, 0), (2 ** 31 - 1, None)])
def test_lengths_outside_the_table(cuda, width, length, cut):
    tables, total = ref.make_tables(3, LENS, 16, width=width)
    caches = ref.make_cache(4, total, 16, 2, 64)
    q = torch.randn(3, 4, 64, generator=torch.Generator().manual_seed(5)).bfloat16()
    good = run(cuda, q, caches, tables, LENS)
    lens = [LENS[0], length, LENS[2]]
    out, k, v, flags = run(cuda, q, caches, tables, lens)
    assert flags == (1, 1)
    # By lines each warp takes an equal share of the steps of the whole batch, 2 at least: 2 heads times
    # (2 + 2 + 2) steps, or (2 + 1 + 2), are cut at every second one, which is where items end; with
    # 1500 steps in the middle the cuts lie elsewhere, also inside requests 0 and 2, whose fp32 sums are
    # then formed in another order. That is within `bound`, not to the bit.
    same_cuts = cut is not None or width == 3
    for s in (0, 2):
        assert not same_cuts or torch.equal(out[s], good[0][s])
        assert torch.equal(k[s], good[1][s]) and torch.equal(v[s], good[2][s])
    whole = [LENS[0], width * 16 if cut is None else cut, LENS[2]]
    want, bound = ref.attention(q, *caches, tables, whole, 64 ** -0.5)
    assert ((out.double() - want).abs() <= bound).all()
    assert torch.equal(k[1, : whole[1]].double(),
                       ref.rows_of(caches[0], caches[2], tables[1], whole[1]))
    assert (k[1, whole[1]:] == 0).all() and (v[1, whole[1]:] == 0).all()
