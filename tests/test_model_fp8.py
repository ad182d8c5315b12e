"""The model forward over the 8-bit KV cache: prefill, decode steps, verification steps and their
graphs.

Against Hugging Face's bf16 forward: every cached value is off by at most 2^-4 of itself (e4m3's
rounding), which through two layers bounds what the logits move by 2 * 2^-4 of the largest. Against
the same cache read another way (a prefill of the same tokens, whose attention runs over the
read-back) the codes are the same but for values that bf16 noise moves over a rounding border, and
the bar is the 2% of test_model.py plus one e4m3 step, 2^-3, of one value in sixteen: 3%."""

from __future__ import annotations

import pytest
import torch

import fp8_reference as ref
import svllm_ops
import test_model as tm
from test_tree_decoding import Pool, drafted, make_model

transformers = pytest.importorskip("transformers")

HF_BAR = 0.125
SELF_BAR = 0.03


def close(a, b, bar):
    assert (a.float() - b.float()).abs().max() <= bar * b.float().abs().max()


@pytest.mark.parametrize("arch", ["qwen3", "llama"])
def test_prefill_then_decode(device, arch):
    hf, model = tm.tiny(arch, device)
    model.allocate_kv_cache(64, tm.BLOCK, fp8=True)
    assert model.k_cache[0].dtype == ref.E4M3 and model.v_scale[1].dtype == ref.E8M0
    g = torch.Generator().manual_seed(11)
    prompts = [torch.randint(0, tm.VOCAB, (n,), generator=g) for n in (37, 20, 1)]
    reqs = tm.Requests(prompts, device)
    inputs = reqs.step_inputs(prompts)
    logits = model.logits(model.forward(**inputs))
    ends = inputs["query_start_loc"].tolist()
    for s, p in enumerate(prompts):
        close(logits[ends[s]: ends[s + 1]], tm.hf_last_logits(hf, p, len(p), device), HF_BAR)
    last = [torch.tensor([5 + s]) for s in range(3)]
    for _ in range(3):
        for s in range(3):
            reqs.tokens[s] = torch.cat([reqs.tokens[s], last[s]])
        inputs = reqs.step_inputs(last)
        qsl = inputs.pop("query_start_loc")
        # one new token each: through forward (read-back) and through decode (8-bit attention)
        logits = model.logits(model.forward(query_start_loc=qsl, **inputs))
        want = torch.cat([tm.hf_last_logits(hf, reqs.tokens[s], 1, device) for s in range(3)])
        close(logits, want, HF_BAR)
        got = model.decode(**inputs).cpu()
        top2 = logits.float().topk(2, dim=-1).values
        clear = ((top2[:, 0] - top2[:, 1]) > SELF_BAR * logits.float().abs().max()).cpu()
        assert torch.equal(got[clear], logits.float().argmax(-1).cpu()[clear])
        last = [got[s: s + 1] for s in range(3)]
    # the same tokens in one prefill over fresh pages leave the same rows, but for borders
    kept = [c.clone() for c in (*model.k_cache, *model.v_cache, *model.k_scale, *model.v_scale)]
    model.allocate_kv_cache(64, tm.BLOCK, fp8=True)
    again = tm.Requests(reqs.tokens, device)
    model.forward(**again.step_inputs(reqs.tokens))
    fresh = [*model.k_cache, *model.v_cache, *model.k_scale, *model.v_scale]
    for i in range(2 * tm.LAYERS):
        for s in range(3):
            n = len(reqs.tokens[s])
            a = ref.rows_of(kept[i].cpu(), kept[i + 2 * tm.LAYERS].cpu(), reqs.tables[s], n)
            b = ref.rows_of(fresh[i].cpu(), fresh[i + 2 * tm.LAYERS].cpu(), again.tables[s], n)
            assert (a - b).norm() <= SELF_BAR * b.norm()


def test_verified_chain_equals_decoding(device):
    """A chain fed through verify gives the targets of the same tokens decoded one at a time."""
    model = make_model(device, True)
    model.allocate_kv_cache(64, 4, fp8=True)
    g = torch.Generator().manual_seed(21)
    prompts = [torch.randint(0, 500, (n,), generator=g) for n in (9, 3)]
    chain = torch.randint(0, 500, (2, 6), generator=g).to(device)
    lens = torch.tensor([9, 3], dtype=torch.int32, device=device)
    pools = [Pool(2, device), Pool(2, device)]
    outs = []
    for pool in pools:
        for c in (*model.k_cache, *model.v_cache):
            c.view(torch.uint8).zero_()
        starts, seq, slots, positions, _ = pool.plan(lens, 12)
        model.forward(torch.cat(prompts).to(device), positions, slots, pool.tables, seq, starts)
        pool.context = pool.context + lens
        if not outs:
            starts, seq, slots, positions, _ = pool.plan(6 * torch.ones_like(lens), 12)
            meta = (positions, slots, pool.tables, seq, starts)
            logits = model.logits(model.forward(chain.flatten(), *meta)).view(2, 6, -1).float()
            outs.append(model.verify(chain.flatten(), *meta).view(2, 6))
        else:
            one = []
            for i in range(6):
                starts, seq, slots, positions, _ = pool.plan(torch.ones_like(lens), 2)
                one.append(model.decode(chain[:, i].contiguous(), positions, slots, pool.tables,
                                        seq))
                pool.context = pool.context + 1
            outs.append(torch.stack(one, 1))
    top2 = logits.topk(2, dim=-1).values
    clear = top2[..., 0] - top2[..., 1] > SELF_BAR * logits.abs().max()
    assert clear.sum() >= 6
    assert torch.equal(outs[0][clear], outs[1][clear])


def test_accepted_rows_and_scales_move(device):
    """A tree's step over the 8-bit cache: after tree_commit the front rows hold the accepted
    nodes' codes and scales, in every layer."""
    model = make_model(device, True)
    model.allocate_kv_cache(64, 4, fp8=True)
    g = torch.Generator().manual_seed(7)
    pool = Pool(2, device)
    lens = torch.tensor([9, 3], dtype=torch.int32, device=device)
    prompts = torch.randint(0, 500, (12,), generator=g).to(device)
    starts, seq, slots, positions, _ = pool.plan(lens, 12)
    model.forward(prompts, positions, slots, pool.tables, seq, starts)
    pool.context = pool.context + lens
    trees = [drafted(3, torch.randint(0, 500, (9,), generator=g), 1, g) for _ in range(2)]
    counts = [len(t[0]) for t in trees]
    ids = torch.tensor(trees[0][0] + trees[1][0]).to(device)
    parents = torch.tensor(trees[0][1] + trees[1][1], dtype=torch.int32, device=device)
    starts, seq, slots, positions, mask = pool.plan(
        torch.tensor(counts, dtype=torch.int32, device=device), sum(counts), parents, max(counts))
    targets = model.verify(ids, positions, slots, pool.tables, seq, starts, mask)
    # make the model's targets follow a path to the last node of each tree
    at = starts.tolist()
    for s in range(2):
        node = counts[s] - 1
        while trees[s][1][node] >= 0:
            targets[at[s] + trees[s][1][node]] = ids[at[s] + node]
            node = trees[s][1][node]
    path, _, accepted, _ = svllm_ops.tree_accept(ids, targets, parents, starts, seq, pool.context,
                                                 max(counts))
    assert (accepted >= 3).all()
    planes = (model.k_cache, model.v_cache, model.k_scale, model.v_scale)
    before = [[t.view(torch.uint8).flatten(0, 1).cpu().clone() for t in p] for p in planes]
    svllm_ops.tree_commit(model.k_cache, model.v_cache, path, accepted, slots, starts,
                          model.k_scale, model.v_scale)
    slot = slots.cpu()
    for p, olds in zip(planes, before):
        for t, want in zip(p, olds):
            source = want.clone()
            for s in range(2):
                for i in range(1, int(accepted[s])):
                    want[slot[at[s] + i]] = source[slot[at[s] + int(path[s, i])]]
            assert torch.equal(t.view(torch.uint8).flatten(0, 1).cpu(), want)
    with pytest.raises(RuntimeError, match="k_scales and v_scales"):
        svllm_ops.tree_commit(model.k_scale, model.v_scale, path, accepted, slots, starts)
    with pytest.raises(RuntimeError, match="scales"):
        svllm_ops.tree_commit(model.k_cache, model.v_cache, path, accepted, slots, starts,
                              model.k_scale)
    with pytest.raises(RuntimeError, match="float8_e8m0fnu"):
        svllm_ops.tree_commit(model.k_cache, model.v_cache, path, accepted, slots, starts,
                              [t.view(torch.uint8) for t in model.k_scale], model.v_scale)
    # a refused call moves nothing: the codes neither
    state = [t.view(torch.uint8).clone() for p in planes for t in p]
    with pytest.raises(RuntimeError, match="given twice"):
        svllm_ops.tree_commit(model.k_cache, model.v_cache, path, accepted, slots, starts,
                              model.k_scale, model.k_scale)
    assert all(torch.equal(t.view(torch.uint8), old)
               for t, old in zip([t for p in planes for t in p], state))


@pytest.mark.gpu
def test_decode_graphs(cuda):
    """Graph replays equal the eager step at the same padded batch bit for bit, cache included."""
    _, model = tm.tiny("qwen3", cuda)
    model.allocate_kv_cache(64, tm.BLOCK, fp8=True)
    filled = [ref.make_cache(i, 64, tm.BLOCK, tm.KV_HEADS, tm.HEAD_DIM) for i in range(tm.LAYERS)]
    planes = (model.k_cache, model.v_cache, model.k_scale, model.v_scale)
    for i in range(tm.LAYERS):
        for p, t in zip(planes, filled[i]):
            p[i].copy_(t)
    graphs = svllm_ops.DecodeGraphs(model, max_num_seqs=24, max_blocks_per_seq=8)
    for n, seed in [(1, 1), (3, 2), (8, 3), (13, 4), (24, 5)]:
        batch = tm.decode_batch(n, cuda, seed)
        b = min(s for s in graphs.batch_sizes if s >= n)
        start = [[t.clone() for t in p] for p in planes]
        got = graphs.step(**batch)
        after = [[t.clone() for t in p] for p in planes]
        for p, old in zip(planes, start):
            for t, o in zip(p, old):
                t.copy_(o)
        assert torch.equal(got, model.decode(**tm.padded(batch, b))[:n])
        for p, new in zip(planes, after):
            for t, x in zip(p, new):
                assert torch.equal(t.view(torch.uint8), x.view(torch.uint8))


def test_cache_kinds(device):
    _, model = tm.tiny("qwen3", device)
    assert model.k_scale == [] and model.k_cache[0].dtype == torch.bfloat16
    model.allocate_kv_cache(8, 16, fp8=True)
    assert len(model.k_scale) == len(model.v_scale) == tm.LAYERS
    assert model.k_scale[0].shape == (8, 16, tm.KV_HEADS)
    model.allocate_kv_cache(8, 16)
    assert model.k_scale == [] and model.v_cache[0].dtype == torch.bfloat16
