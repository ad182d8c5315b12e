"""The model over the 8-bit KV cache: its logits against a model that quantises in 64 bits, and steps at
the edges of what a scheduler asks for."""

from __future__ import annotations

import pytest
import torch

import fp8_reference as ref
import test_model as tm

transformers = pytest.importorskip("transformers")


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


class QuantisedCache(transformers.DynamicCache):
    """Hugging Face's cache with every K and V row put through the 8-bit format in 64 bits. `spoil`: a
    (layer, KV head, 0 for K or 1 for V) whose rows are read at twice their scale."""

    def __init__(self, spoil=None):
        super().__init__()
        self.spoil = spoil

    def update(self, key_states, value_states, layer_idx, *args, **kwargs):
        held = []
        for i, x in enumerate((key_states, value_states)):  # [1, KV heads, tokens, head_dim]
            y = ref.values(*ref.quantise(x.double().cpu())[:2])
            if self.spoil is not None and self.spoil[0] == layer_idx and self.spoil[2] == i:
                y[:, self.spoil[1]] *= 2
            held.append(y.to(x))  # exact: a code times its scale is a bf16 value
        return super().update(*held, layer_idx, *args, **kwargs)


def hf_logits(hf, tokens, count, device, spoil=None):
    with torch.no_grad():
        out = hf(tokens.to(device)[None], past_key_values=QuantisedCache(spoil), use_cache=True)
    return out.logits[0, -count:].float()


def off(a, b):
    return ((a - b).abs().max() / b.abs().max()).item()


# As test_model_fp8.py's bar between two ways of reading the same codes: bf16 noise of 2%, and a code's
# step, 2^-3, in the one value of sixteen that bf16 noise moves over a rounding border.
BAR = 0.03


@pytest.mark.parametrize("arch", ["qwen3", "llama"])
def test_logits_equal_a_model_that_quantises_in_64_bits(device, arch):
    """Prefill of a packed batch and decode steps against Hugging Face's model over the same format."""
    hf, model = tm.tiny(arch, device)
    model.allocate_kv_cache(64, tm.BLOCK, fp8=True)
    g = torch.Generator().manual_seed(12)
    prompts = [torch.randint(0, tm.VOCAB, (n,), generator=g) for n in (41, 17, 2)]
    reqs = tm.Requests(prompts, device)
    inputs = reqs.step_inputs(prompts)
    logits = model.logits(model.forward(**inputs)).float()
    ends = inputs["query_start_loc"].tolist()
    for s, p in enumerate(prompts):
        assert off(logits[ends[s]: ends[s + 1]], hf_logits(hf, p, len(p), device)) <= BAR
    for i in range(3):
        new = [torch.tensor([9 + 5 * s + i]) for s in range(3)]
        for s in range(3):
            reqs.tokens[s] = torch.cat([reqs.tokens[s], new[s]])
        inputs = reqs.step_inputs(new)
        inputs.pop("query_start_loc")
        got = model.decode(**inputs).cpu()
        want = torch.cat([hf_logits(hf, t, 1, device) for t in reqs.tokens])
        top2 = want.topk(2, dim=-1).values
        clear = (top2[:, 0] - top2[:, 1] > 2 * BAR * want.abs().max()).cpu()
        assert torch.equal(got[clear], want.argmax(-1).cpu()[clear])


@pytest.mark.parametrize("arch", ["qwen3", "llama"])
@pytest.mark.parametrize("layer", [0, 1])
def test_a_scale_off_by_one_binade_in_one_head_would_show(arch, layer):
    """The mistake that the test above is for, planted in its oracle: V's scales doubled in one KV head
    of one layer move the logits past the bar."""
    hf, _ = tm.tiny(arch, torch.device("cpu"))
    tokens = torch.randint(0, tm.VOCAB, (41,), generator=torch.Generator().manual_seed(12))
    want = hf_logits(hf, tokens, 41, "cpu")
    for head in range(tm.KV_HEADS):
        assert off(hf_logits(hf, tokens, 41, "cpu", spoil=(layer, head, 1)), want) > 2 * BAR
