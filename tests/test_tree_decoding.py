"""The drafted-tree operators in a run together, as a serving loop uses them: paged_plan, the rotary
+ cache-write ops and tree_attention inside Model.verify, tree_accept and tree_commit, step after
step, against the same model decoding one token at a time.

The model's logits in a verification step and in a decode step differ by bf16 rounding noise (other
GEMM shapes, another attention kernel), as in test_model.py: logits are held to 2% of the largest, so
a token may differ where the top two logits are closer than that, and the comparison of tokens stops
at such a place."""

from __future__ import annotations

import pytest
import torch

import svllm_ops
from tree_reference import masks_of, walk_reference

VOCAB, HIDDEN, INTER, LAYERS, HEADS, KV_HEADS, HEAD_DIM = 500, 256, 512, 3, 4, 2, 64
BLOCK, BLOCKS, WIDTH = 4, 64, 12
REL_BAR = 0.02


def make_model(device, qk_norm):
    g = torch.Generator().manual_seed(3)

    def w(*shape, scale=None):
        t = torch.randn(shape, generator=g) * (scale if scale else shape[-1] ** -0.5)
        return t.to(device, torch.bfloat16)

    weights = {"model.embed_tokens.weight": w(VOCAB, HIDDEN, scale=1.0),
               "model.norm.weight": 1 + w(HIDDEN, scale=0.1)}
    for layer in range(LAYERS):
        p = f"model.layers.{layer}."
        weights |= {p + "input_layernorm.weight": 1 + w(HIDDEN, scale=0.1),
                    p + "post_attention_layernorm.weight": 1 + w(HIDDEN, scale=0.1),
                    p + "self_attn.q_proj.weight": w(HEADS * HEAD_DIM, HIDDEN),
                    p + "self_attn.k_proj.weight": w(KV_HEADS * HEAD_DIM, HIDDEN),
                    p + "self_attn.v_proj.weight": w(KV_HEADS * HEAD_DIM, HIDDEN),
                    p + "self_attn.o_proj.weight": w(HIDDEN, HEADS * HEAD_DIM),
                    p + "self_attn.q_norm.weight": 1 + w(HEAD_DIM, scale=0.1),
                    p + "self_attn.k_norm.weight": 1 + w(HEAD_DIM, scale=0.1),
                    p + "mlp.gate_proj.weight": w(INTER, HIDDEN),
                    p + "mlp.up_proj.weight": w(INTER, HIDDEN),
                    p + "mlp.down_proj.weight": w(HIDDEN, INTER)}
    cfg = svllm_ops.ModelConfig(vocab_size=VOCAB, hidden_size=HIDDEN, intermediate_size=INTER,
                                num_layers=LAYERS, num_heads=HEADS, num_kv_heads=KV_HEADS,
                                head_dim=HEAD_DIM, rms_norm_eps=1e-6, rope_theta=1e6,
                                tie_word_embeddings=True, qk_norm=qk_norm)
    model = svllm_ops.Model(cfg, weights)
    model.allocate_kv_cache(BLOCKS, BLOCK)
    return model


class Pool:
    """The paging state of a batch, kept on the device."""

    def __init__(self, requests, device):
        self.tables = torch.zeros(requests, WIDTH, dtype=torch.int32, device=device)
        self.owned = torch.zeros(requests, dtype=torch.int32, device=device)
        g = torch.Generator().manual_seed(9)
        self.stack = torch.randperm(BLOCKS, generator=g).to(device, torch.int32)
        self.count = torch.tensor([BLOCKS], dtype=torch.int32, device=device)
        self.context = torch.zeros(requests, dtype=torch.int32, device=device)

    def plan(self, query, tokens, parents=None, width=1):
        starts, seq, slots, positions, mask, self.owned, self.count = svllm_ops.paged_plan(
            self.context, query, self.tables, self.owned, self.stack, self.count, tokens, BLOCK,
            parents, width)
        return starts, seq, slots, positions, mask


def sequential(model, prompts, steps, device):
    """Greedy decoding one token a step: per request the tokens, and whether each was clear."""
    pool = Pool(len(prompts), device)
    lens = torch.tensor([len(p) for p in prompts], dtype=torch.int32, device=device)
    tokens = int(lens.sum())
    starts, seq, slots, positions, _ = pool.plan(lens, tokens)
    hidden = model.forward(torch.cat(prompts).to(device), positions, slots, pool.tables, seq,
                           starts)
    pool.context = pool.context + lens
    logits = model.logits(hidden[starts[1:].long() - 1])
    one = torch.ones_like(lens)
    out, clear = [], []
    for _ in range(steps):
        top = logits.float().topk(2, dim=-1)
        clear.append(top.values[:, 0] - top.values[:, 1] > 2 * REL_BAR * logits.abs().max())
        out.append(top.indices[:, 0].contiguous())
        starts, seq, slots, positions, _ = pool.plan(one, len(prompts))
        hidden = model.forward(out[-1], positions, slots, pool.tables, seq, starts)
        pool.context = pool.context + 1
        logits = model.logits(hidden)
    return torch.stack(out, 1).cpu(), torch.stack(clear, 1).cpu()


def drafted(step, truth, at, g):
    """A tree around the continuation truth[at], truth[at + 1], ...: node 0 holds truth[at - 1]
    (fed again), the true tokens hang in it among wrong ones, cut short at a different depth for
    every step."""
    ids, parents = [int(truth[at - 1])], [-1]
    cur = 0
    for d in range(1 + step % 4):
        right = int(truth[at + d])
        kids = [right] + [int(x) for x in torch.randint(0, VOCAB, (2,), generator=g)]
        order = torch.randperm(3, generator=g).tolist()
        nxt = None
        for k in order:
            ids.append(kids[k])
            parents.append(cur)
            if k == 0:
                nxt = len(ids) - 1
        cur = nxt
    return ids, parents


@pytest.mark.parametrize("qk_norm", [True, False], ids=["qk_norm", "plain"])
def test_verified_trees_emit_the_sequential_tokens(device, qk_norm):
    model = make_model(device, qk_norm)
    g = torch.Generator().manual_seed(21)
    prompts = [torch.randint(0, VOCAB, (n,), generator=g) for n in (9, 3, 14)]
    truth, clear = sequential(model, prompts, 24, device)
    for c in model.k_cache + model.v_cache:
        c.zero_()

    pool = Pool(3, device)
    lens = torch.tensor([9, 3, 14], dtype=torch.int32, device=device)
    starts, seq, slots, positions, _ = pool.plan(lens, 26)
    # the prompt as chains, through the same step
    targets = model.verify(torch.cat(prompts).to(device), positions, slots, pool.tables, seq,
                           starts)
    pool.context = pool.context + lens
    firsts = targets[starts[1:].long() - 1].cpu()
    emitted = [[int(x)] for x in firsts]
    blocks = pool.count.item() + pool.owned.sum().item()
    for step in range(6):
        trees = []
        for s in range(3):
            base = torch.tensor(emitted[s] + truth[s, len(emitted[s]):].tolist())
            trees.append(drafted(step + s, base, len(emitted[s]), g))
        counts = [len(t[0]) for t in trees]
        ids = torch.tensor(sum((t[0] for t in trees), []))
        parents = torch.tensor(sum((t[1] for t in trees), []), dtype=torch.int32)
        starts, seq, slots, positions, mask = pool.plan(
            torch.tensor(counts, dtype=torch.int32, device=device), sum(counts),
            parents.to(device), max(counts))
        assert torch.equal(mask.cpu(), masks_of(parents.tolist(), counts))
        targets = model.verify(ids.to(device), positions, slots, pool.tables, seq, starts, mask)
        path, tokens, accepted, context = svllm_ops.tree_accept(
            ids.to(device), targets, parents.to(device), starts, seq, pool.context, max(counts))
        want = walk_reference(ids.tolist(), targets.tolist(), parents.tolist(), starts.tolist(),
                              seq.tolist(), pool.context.tolist(), max(counts))
        for a, b in zip((path, tokens, accepted, context), want):
            assert torch.equal(a.cpu(), b)
        svllm_ops.tree_commit(model.k_cache, model.v_cache, path, accepted, slots, starts)
        pool.context = context
        for s in range(3):
            emitted[s] += tokens[s, : accepted[s]].tolist()
        assert pool.count.item() + pool.owned.sum().item() == blocks  # no block lost

    for s in range(3):
        n = min(len(emitted[s]), truth.shape[1])
        assert n >= 13  # the drafts were accepted, not just one token a step
        stop = next((i for i in range(n) if not clear[s, i]), n)
        assert emitted[s][:stop] == truth[s, :stop].tolist()
    # at least one request was compared over several steps
    assert max(next((i for i in range(24) if not clear[s, i]), 24) for s in range(3)) >= 8

    # the cache holds what a prefill of the accepted tokens writes: rows of the sequence in order
    kept = [c.clone() for c in model.k_cache + model.v_cache]
    tables, context = pool.tables.cpu().long(), pool.context.tolist()
    fresh = Pool(3, device)
    full = [torch.cat([p, torch.tensor(e)])[: c] for p, e, c in zip(prompts, emitted, context)]
    lens = torch.tensor(context, dtype=torch.int32, device=device)
    starts, seq, slots, positions, _ = fresh.plan(lens, sum(context))
    model.forward(torch.cat(full).to(device), positions, slots, fresh.tables, seq, starts)
    for old, new in zip(kept, model.k_cache + model.v_cache):
        for s in range(3):
            j = torch.arange(context[s])
            a = old.cpu().view(-1, KV_HEADS, HEAD_DIM)[tables[s][j // BLOCK] * BLOCK + j % BLOCK]
            b = new.cpu().view(-1, KV_HEADS, HEAD_DIM)[
                fresh.tables.cpu().long()[s][j // BLOCK] * BLOCK + j % BLOCK]
            # bf16 noise of three layers, against rows of other tokens that differ by their size
            bar = 4 * REL_BAR * b.float().abs().max()
            assert ((a.float() - b.float()).abs() <= bar).all()

    # a finished request gives its blocks back
    before = pool.count.item()
    pool.plan(torch.tensor([-1, 0, -1], dtype=torch.int32, device=device), 0)
    assert pool.count.item() + pool.owned.sum().item() == blocks and pool.count.item() > before
    assert pool.owned[0].item() == 0 and pool.owned[2].item() == 0


@pytest.mark.gpu
def test_a_verification_step_replays_from_a_graph(cuda):
    """Plan, forward, walk and move of one step captured and replayed: the replay's outputs equal
    the eager step's from the same state."""
    model = make_model(cuda, True)
    g = torch.Generator().manual_seed(5)
    prompts = [torch.randint(0, VOCAB, (n,), generator=g) for n in (9, 3)]
    pool = Pool(2, cuda)
    lens = torch.tensor([9, 3], dtype=torch.int32, device=cuda)
    starts, seq, slots, positions, _ = pool.plan(lens, 12)
    model.forward(torch.cat(prompts).to(cuda), positions, slots, pool.tables, seq, starts)
    context = pool.context + lens
    ids = torch.randint(0, VOCAB, (10,), generator=g).to(cuda)
    parents = torch.tensor([-1, 0, 0, 1, 2, 4, -1, 0, 1, 0], dtype=torch.int32, device=cuda)
    query = torch.tensor([6, 4], dtype=torch.int32, device=cuda)
    owned, count = pool.owned.clone(), pool.count.clone()

    def step():
        starts, seq, slots, positions, mask, o, c = svllm_ops.paged_plan(
            context, query, pool.tables, owned, pool.stack, count, 10, BLOCK, parents, 6)
        targets = model.verify(ids, positions, slots, pool.tables, seq, starts, mask)
        path, tokens, accepted, after = svllm_ops.tree_accept(ids, targets, parents, starts, seq,
                                                              context, 6)
        svllm_ops.tree_commit(model.k_cache, model.v_cache, path, accepted, slots, starts)
        return targets, path, tokens, accepted, after, o, c

    kept = [c.clone() for c in model.k_cache + model.v_cache]
    want = [t.clone() for t in step()]
    caches = [c.clone() for c in model.k_cache + model.v_cache]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step()
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for c, k in zip(model.k_cache + model.v_cache, kept):
        c.copy_(k)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(out, want))
    assert all(torch.equal(a, b) for a, b in zip(model.k_cache + model.v_cache, caches))


def test_verify_refuses_what_tree_attention_refuses():
    model = make_model(torch.device("cpu"), True)
    with pytest.raises(RuntimeError, match="tree_mask"):
        model.verify(torch.tensor([1]), torch.tensor([0]), torch.tensor([0]),
                     torch.zeros(1, 1, dtype=torch.int32), torch.tensor([1], dtype=torch.int32),
                     torch.tensor([0, 1], dtype=torch.int32), torch.ones(2, 1, dtype=torch.int64))
