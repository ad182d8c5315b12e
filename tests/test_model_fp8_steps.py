"""Steps of the model over the 8-bit KV cache at the edges of what a scheduler asks for."""

from __future__ import annotations

import pytest
import torch

import test_model as tm

pytest.importorskip("transformers")


def lists(device, requests, width):
    def zeros(*shape, dtype=torch.int64):
        return torch.zeros(*shape, dtype=dtype, device=device)

    i32 = torch.int32
    return (zeros(0), zeros(0), zeros(0), zeros(requests, width, dtype=i32),
            zeros(requests, dtype=i32), zeros(requests + 1, dtype=i32))


@pytest.mark.parametrize("requests, width", [(0, 0), (0, 3), (2, 0), (2, 3)])
def test_steps_without_tokens(device, requests, width):
    """A scheduler's empty step gives empty outputs and leaves the cache as it was."""
    _, model = tm.tiny("qwen3", device)
    model.allocate_kv_cache(8, tm.BLOCK, fp8=True)
    before = [t.clone() for t in (*model.k_cache, *model.v_cache)]
    ids, positions, slots, tables, lens, starts = lists(device, requests, width)
    assert model.forward(ids, positions, slots, tables, lens, starts).shape[0] == 0
    if width > 0:
        assert model.verify(ids, positions, slots, tables, lens, starts).shape == (0,)
    if requests == 0 and width > 0:
        assert model.decode(ids, positions, slots, tables, lens).shape == (0,)
    for t, old in zip((*model.k_cache, *model.v_cache), before):
        assert torch.equal(t.view(torch.uint8), old.view(torch.uint8))
