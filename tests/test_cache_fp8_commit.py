"""tree_commit over 8-bit caches: codes and scales move together or not at all."""

from __future__ import annotations

import pytest
import torch

import fp8_reference as ref
import svllm_ops

BLOCKS, BLOCK, HEADS, DIM = 4, 4, 2, 64


def caches(device, layers=2):
    """Planes of every layer, K codes, V codes, K scales and V scales, and the step's lists: request 0
    accepts nodes 0 and 3 of 4, request 1 node 0 of 2."""
    made = [ref.make_cache(i, BLOCKS, BLOCK, HEADS, DIM) for i in range(layers)]
    planes = [[layer[p].to(device) for layer in made] for p in range(4)]
    lists = (torch.tensor([[0, 3], [0, -1]], dtype=torch.int32, device=device),
             torch.tensor([2, 1], dtype=torch.int32, device=device),
             torch.tensor([5, 6, 7, 9, 1, 2], device=device),
             torch.tensor([0, 4, 6], dtype=torch.int32, device=device))
    return planes, lists


def rows(t):
    return t.view(torch.uint8).flatten(0, 1).cpu()


def held(planes):
    return [rows(t).clone() for p in planes for t in p]


def moved(state):
    want = [t.clone() for t in state]
    for t in want:
        t[6] = t[9]
    return want


def equal(a, b):
    return all(torch.equal(x, y) for x, y in zip(a, b, strict=True))


def test_codes_and_scales_move(device):
    (k, v, ks, vs), lists = caches(device)
    before = held((k, v, ks, vs))
    svllm_ops.tree_commit(k, v, *lists, ks, vs)
    assert equal(held((k, v, ks, vs)), moved(before))


def test_codes_without_scales_are_refused(device):
    """The call of a bf16 cache would leave the rows under the scales of others."""
    (k, v, ks, vs), lists = caches(device)
    before = held((k, v, ks, vs))
    for scales in ((), (None, None), ([], [])):
        with pytest.raises(RuntimeError, match="move with their scales"):
            svllm_ops.tree_commit(k, v, *lists, *scales)
    assert equal(held((k, v, ks, vs)), before)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.uint8])
def test_scales_of_a_cache_without_are_refused(device, dtype):
    (k, v, ks, vs), lists = caches(device)
    if dtype == torch.bfloat16:
        k, v = ([t.float().bfloat16() for t in p] for p in (k, v))
    else:
        k, v = ([t.view(dtype) for t in p] for p in (k, v))
    before = held((ks, vs)) + [t.clone() for p in (k, v) for t in p]
    with pytest.raises(RuntimeError, match="only of float8_e4m3fn caches"):
        svllm_ops.tree_commit(k, v, *lists, ks, vs)
    assert equal(held((ks, vs)) + [t for p in (k, v) for t in p], before)


def test_eight_bit_caches_of_another_kind_move_as_bytes(device):
    """Rows without scales of their own: seen as bytes, they move alone."""
    (k, v, ks, vs), lists = caches(device)
    codes, scales = held((k, v)), held((ks, vs))
    svllm_ops.tree_commit([t.view(torch.uint8) for t in k], [t.view(torch.uint8) for t in v], *lists)
    assert equal(held((k, v)), moved(codes)) and equal(held((ks, vs)), scales)
