"""Workloads of the operators that check a tree of drafted tokens against the paged KV cache:
the step's plan (block tables, slots, positions and ancestor masks from request lengths),
attention of the tree's nodes over the cache, the greedy acceptance walk, and the move of the
accepted nodes' K and V to the front of the step's rows.

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
VOCAB = 151936  # the vocabulary of the repository's default configuration
_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _ops():
    path = os.path.join(_ROOT, "small-vllm_b200", "python")
    if path not in sys.path:
        sys.path.insert(0, path)
    import svllm_ops

    return svllm_ops


# ------------------------------------------------------------------------------------- cases

def _attn(name, requests, nodes_lo, nodes, ctx_lo, ctx, heads, kv_heads, dim, block=16,
          shape="tree", pad=0):
    return {"name": name, "op": "attention", "requests": requests, "nodes_lo": nodes_lo,
            "nodes": nodes, "ctx_lo": ctx_lo, "ctx": ctx, "heads": heads, "kv_heads": kv_heads,
            "dim": dim, "block": block, "shape": shape, "pad": pad}


def _plan(name, requests, nodes_lo, nodes, ctx_lo, ctx, block=16, shape="tree", short=False):
    return {"name": name, "op": "plan", "requests": requests, "nodes_lo": nodes_lo,
            "nodes": nodes, "ctx_lo": ctx_lo, "ctx": ctx, "block": block, "shape": shape,
            "short": short}


def _accept(name, requests, nodes_lo, nodes):
    return {"name": name, "op": "accept", "requests": requests, "nodes_lo": nodes_lo,
            "nodes": nodes}


def _commit(name, requests, nodes_lo, nodes, ctx_lo, ctx, layers, kv_heads, dim, block=16):
    return {"name": name, "op": "commit", "requests": requests, "nodes_lo": nodes_lo,
            "nodes": nodes, "ctx_lo": ctx_lo, "ctx": ctx, "layers": layers,
            "kv_heads": kv_heads, "dim": dim, "block": block}


def listed():
    return [
        # one user, a small tree right after a short prompt: latency is everything
        _attn("attn 1x8 over 128", 1, 8, 8, 120, 120, 16, 8, 128),
        # one user, a full tree over a long document: the cache has to be split over the GPU
        _attn("attn 1x32 over 32k", 1, 32, 32, 32736, 32736, 16, 8, 128),
        # a batch whose draft model proposes chains of a few tokens (no tree mask)
        _attn("attn chains 32x5 over 2k", 32, 3, 5, 512, 2048, 32, 8, 64, shape="chain"),
        # a full serving batch with full trees over ordinary contexts: the largest
        _attn("attn 64x64 over 4k", 64, 48, 64, 2048, 4096, 16, 8, 128),
        # odd everything: 5 query heads per KV head, 12-token pages, contexts from zero on,
        # padding rows behind the last request
        _attn("attn odd 13x37", 13, 1, 37, 0, 777, 20, 4, 128, block=12, pad=5),
        # large trees and 8 query heads per KV head: arithmetic counts as much as the cache
        _attn("attn wide 8x128 over 4k", 8, 100, 128, 1024, 4096, 32, 4, 128),
        # the plan of a small step
        _plan("plan 4x8", 4, 8, 8, 16, 700),
        # the plan of a very large batch whose pool runs out of blocks part way
        _plan("plan 1024x64", 1024, 1, 64, 0, 4096, short=True),
        # the acceptance walk of a small step, and of a very large one
        _accept("accept 4x8", 4, 8, 8),
        _accept("accept 1024x64", 1024, 32, 64),
        # moving one user's accepted rows in every layer, and a batch's
        _commit("commit 1x16", 1, 16, 16, 100, 100, 28, 8, 128),
        _commit("commit 128x24", 128, 12, 24, 16, 48, 28, 8, 128),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["attention", "attention", "attention", "plan", "accept", "commit"])
    if op == "attention":
        heads, kv_heads, dim = rng.choice([(16, 8, 128), (32, 8, 64), (8, 8, 128), (24, 8, 64),
                                           (28, 4, 128), (20, 4, 128), (32, 4, 128), (8, 1, 64),
                                           (6, 2, 64)])
        nodes = _log_int(rng, 1, 128)
        ctx = _log_int(rng, 1, 32768)
        # no more cached rows, nor more products, than the largest listed case
        requests = _log_int(rng, 1, 64)
        per = (ctx + nodes) * kv_heads
        requests = max(1, min(requests, 64 * 4096 * 8 // per,
                              64 * 64 * 4096 * 16 * 128 // (nodes * heads * dim * (ctx + nodes))))
        nodes_lo = rng.randint(1, nodes)
        return {"op": op, "requests": requests, "nodes_lo": nodes_lo, "nodes": nodes,
                "ctx_lo": rng.randint(0, ctx), "ctx": ctx, "heads": heads, "kv_heads": kv_heads,
                "dim": dim, "block": rng.choice([1, 8, 12, 16, 16, 32, 64, 256]),
                "shape": rng.choice(["tree", "tree", "chain"]), "pad": rng.choice([0, 0, 3])}
    if op == "plan":
        nodes = _log_int(rng, 1, 64)
        ctx = _log_int(rng, 1, 4096)
        return {"op": op, "requests": _log_int(rng, 1, 1000), "nodes_lo": rng.randint(0, nodes),
                "nodes": nodes, "ctx_lo": rng.randint(0, ctx), "ctx": ctx,
                "block": rng.choice([1, 8, 12, 16, 16, 32, 64]),
                "shape": rng.choice(["tree", "tree", "chain"]),
                "short": rng.choice([False, False, True])}
    if op == "accept":
        nodes = _log_int(rng, 1, 200)
        return {"op": op, "requests": _log_int(rng, 1, 65536 // max(64, nodes)),
                "nodes_lo": rng.randint(0, nodes), "nodes": nodes}
    nodes = _log_int(rng, 2, 48)
    ctx = _log_int(rng, 1, 64)
    kv_heads, dim, layers = rng.choice([(8, 128, 28), (8, 64, 16), (4, 128, 16), (1, 64, 5)])
    return {"op": op, "requests": _log_int(rng, 1, 64), "nodes_lo": rng.randint(1, nodes),
            "nodes": nodes, "ctx_lo": rng.randint(0, ctx), "ctx": ctx, "layers": layers,
            "kv_heads": kv_heads, "dim": dim, "block": rng.choice([1, 8, 12, 16, 32])}


def lengths(case):
    """Nodes and cached tokens of every request: spread over the case's ranges, the first request
    at the top of both."""
    s = np.arange(case["requests"], dtype=np.int64)
    q = case["nodes"] - (s * 7919) % (case["nodes"] - case["nodes_lo"] + 1)
    c = s * 0
    if "ctx" in case:
        c = case["ctx"] - (s * 6151) % (case["ctx"] - case["ctx_lo"] + 1)
    return q, c


def _starts(q):
    return np.concatenate([[0], np.cumsum(q)]).astype(np.int64)


def _draft_parents(rng, q):
    """Random trees: node 0 of a request is the root, every other hangs on one of the up to
    six nodes before it. Request-local indices, packed."""
    start = _starts(q)
    i = np.arange(start[-1]) - np.repeat(start[:-1], q)
    back = 1 + rng.integers(0, 6, size=i.shape)
    return np.where(i == 0, -1, np.maximum(i - back, 0)).astype(np.int32)


def _masks(parents, q):
    """Ancestor-or-self bits of every node, [T, W] int64 words of 64 nodes."""
    words = max(1, -(-int(q.max(initial=1)) // 64))
    out = np.zeros((len(parents), words), np.uint64)
    start = _starts(q)
    for s in range(len(q)):
        seen = []
        for i in range(q[s]):
            p = parents[start[s] + i]
            m = (seen[p] if p >= 0 else 0) | (1 << i)
            seen.append(m)
            for w in range(words):
                out[start[s] + i, w] = (m >> (64 * w)) & 0xFFFFFFFFFFFFFFFF
    return out.view(np.int64)


def _dev(a, dtype=None):
    t = torch.from_numpy(np.ascontiguousarray(a))
    return t.to(DEV, dtype=dtype) if dtype else t.to(DEV)


def _pages(rng, q, c, block):
    """Random pages for every request's cached tokens and nodes: tables, number of blocks, slots
    of the nodes."""
    need = -(-(q + c) // block)
    num_blocks = int(need.sum()) + 3
    order = rng.permutation(num_blocks)[: need.sum()]
    width = max(1, int(need.max(initial=1)))
    tables = np.zeros((len(q), width), np.int32)
    first = _starts(need)
    for s in range(len(q)):
        tables[s, : need[s]] = order[first[s]: first[s + 1]]
    start = _starts(q)
    slots = np.empty(start[-1], np.int64)
    for s in range(len(q)):
        r = c[s] + np.arange(q[s])
        slots[start[s]: start[s + 1]] = tables[s][r // block].astype(np.int64) * block + r % block
    return tables, num_blocks, slots


def prepare(case, seed):
    rng = np.random.default_rng(seed)
    gen = torch.Generator(device=DEV).manual_seed(seed)
    q, c = lengths(case)
    start = _starts(q)
    tokens = int(start[-1])
    if case["op"] == "attention":
        tables, num_blocks, _ = _pages(rng, q, c, case["block"])
        heads, kv, dim = case["heads"], case["kv_heads"], case["dim"]
        rows = tokens + case["pad"]
        qkv = torch.randn(rows, (heads + 2 * kv) * dim, device=DEV, generator=gen).bfloat16()
        shape = (num_blocks, case["block"], kv, dim)
        state = {"q": qkv[:, : heads * dim].view(rows, heads, dim),
                 "k_cache": torch.randn(shape, device=DEV, generator=gen).bfloat16(),
                 "v_cache": torch.randn(shape, device=DEV, generator=gen).bfloat16(),
                 "block_tables": _dev(tables), "seq_lens": _dev(q + c, torch.int32),
                 "query_start_loc": _dev(start, torch.int32), "tree_mask": None,
                 "scale": dim ** -0.5, "max_nodes": int(q.max())}
        if case["shape"] == "tree":
            m = _masks(_draft_parents(rng, q), q)
            state["tree_mask"] = _dev(np.concatenate(
                [m, np.zeros((case["pad"], m.shape[1]), np.int64)]))
        return {"case": case, **state}
    if case["op"] == "plan":
        block = case["block"]
        owned = -(-c // block) + np.arange(len(q)) % 2  # some own a spare one
        need = np.maximum(0, -(-(q + c) // block) - owned)
        width = int((owned + need).max(initial=1)) + 1
        pool = int(need.sum()) + 7
        have = int(need.sum()) * 3 // 4 if case["short"] else pool
        ids = rng.permutation(int(owned.sum()) + pool).astype(np.int32)
        tables = np.zeros((len(q), width), np.int32)
        first = _starts(owned)
        for s in range(len(q)):
            tables[s, : owned[s]] = ids[first[s]: first[s + 1]]
        q = q.copy()
        if case["short"]:
            q[5::97] = -1  # finished requests, whose blocks come back
        pad = 0 if case["shape"] == "tree" else 3
        q0 = np.maximum(q, 0)
        parents = _draft_parents(rng, q0) if case["shape"] == "tree" else None
        room = np.zeros(pool + int(owned.sum()), np.int32)
        room[:pool] = ids[int(owned.sum()):]
        return {"case": case, "context_lens": _dev(c, torch.int32),
                "query_lens": _dev(q, torch.int32), "block_tables": _dev(tables),
                "blocks_owned": _dev(owned, torch.int32), "free_blocks": _dev(room),
                "free_count": _dev(np.array([have]), torch.int32),
                "num_tokens": int(q0.sum()) + pad, "block_size": block,
                "parents": None if parents is None else _dev(parents),
                "max_query_len": max(1, case["nodes"])}
    parents = _draft_parents(rng, q)
    if case["op"] == "accept":
        ids = rng.integers(0, VOCAB, size=tokens)
        targets = rng.integers(0, VOCAB, size=tokens)
        # the model agrees with one child of most nodes
        i = np.arange(tokens)
        base = np.repeat(start[:-1], q)
        child = i[parents >= 0]
        kept = child[rng.random(child.shape) < 0.5]
        targets[base[kept] + parents[kept]] = ids[kept]
        return {"case": case, "ids": _dev(ids), "targets": _dev(targets),
                "parents": _dev(parents), "query_start_loc": _dev(start, torch.int32),
                "context_lens": _dev(np.arange(len(q)) % 977, torch.int32),
                "seq_lens": _dev(np.arange(len(q)) % 977 + q, torch.int32),
                "max_query_len": max(1, int(q.max(initial=1)))}
    # commit: the path from every request's root to one of its last nodes
    tables, num_blocks, slots = _pages(rng, q, c, case["block"])
    width = max(1, int(q.max(initial=1)))
    path = np.full((len(q), width), -1, np.int32)
    count = np.zeros(len(q), np.int32)
    for s in range(len(q)):
        node, back = int(rng.integers(q[s] * 3 // 4, q[s])), []
        while node >= 0:
            back.append(node)
            node = int(parents[start[s] + node])
        count[s] = len(back)
        path[s, : len(back)] = back[::-1]
    caches = torch.randn(2, case["layers"], num_blocks, case["block"], case["kv_heads"],
                         case["dim"], device=DEV, generator=gen, dtype=torch.bfloat16)
    return {"case": case, "caches": caches, "k_caches": list(caches[0]),
            "v_caches": list(caches[1]), "path": _dev(path), "num_accepted": _dev(count),
            "slot_mapping": _dev(slots), "query_start_loc": _dev(start, torch.int32)}


# ------------------------------------------------------------------------------- plain forms

def _plain_attention(s):
    """softmax(scale q k^T + mask) v over the gathered pages, in fp32."""
    q, tables = s["q"], s["block_tables"].long()
    rows, heads, dim = q.shape
    _, block, kv, _ = s["k_cache"].shape
    qsl, seq = s["query_start_loc"].long(), s["seq_lens"].long()
    count = qsl[1:] - qsl[:-1]
    ctx = seq - count
    n, group = s["max_nodes"], heads // kv
    node = torch.arange(n, device=q.device)
    valid = node < count[:, None]                                   # [S, n]
    at = (qsl[:-1, None] + node).clamp(max=rows - 1)
    k = s["k_cache"][tables].float().flatten(1, 2)                  # [S, L, Hk, D]
    v = s["v_cache"][tables].float().flatten(1, 2)
    length = k.shape[1]
    j = torch.arange(length, device=q.device)
    tree = j - ctx[:, None]                                         # node index of key j
    if s["tree_mask"] is None:
        sees = tree[:, None, :] <= node[:, None]
    else:
        words = s["tree_mask"][at]                                  # [S, n, W]
        inside = tree.clamp(0, 64 * words.shape[2] - 1)[:, None, :].expand(-1, n, -1)
        sees = ((words.gather(2, inside // 64) >> (inside % 64)) & 1).bool()
        sees = sees | (tree < 0)[:, None, :]
    sees = sees & (j < seq[:, None])[:, None, :]                    # [S, n, L]
    qf = q[at].float().view(-1, n, kv, group, dim)
    scores = torch.einsum("snhgd,slhd->shgnl", qf, k) * s["scale"]
    scores = scores.masked_fill(~sees[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    p = torch.where(total > 0, p / total, torch.zeros_like(p))
    o = torch.einsum("shgnl,slhd->snhgd", p, v).reshape(-1, n, heads, dim)
    out = torch.zeros(rows, heads, dim, device=q.device, dtype=q.dtype)
    out[at[valid]] = o[valid].to(q.dtype)
    return out


def _closure(parents, qsl, n):
    """Ancestor-or-self matrices [S, n, n] of packed trees, and which nodes exist."""
    node = torch.arange(n, device=parents.device)
    count = qsl[1:] - qsl[:-1]
    valid = node < count[:, None]
    at = (qsl[:-1, None] + node).clamp(max=max(0, parents.shape[0] - 1))
    parent = torch.where(valid, parents.long()[at], torch.full_like(at, -1))
    step = (parent[:, :, None] == node).float()
    seen = step + torch.eye(n, device=parents.device)
    for _ in range(max(1, (n - 1).bit_length())):
        seen = (seen @ seen).clamp(max=1)
    return seen.bool() & valid[:, :, None], parent, valid, at


def _plain_plan(s):
    dev = s["query_lens"].device
    q, c = s["query_lens"].long(), s["context_lens"].long()
    owned, block, tokens = s["blocks_owned"].long(), s["block_size"], s["num_tokens"]
    tables, stack, have = s["block_tables"], s["free_blocks"], s["free_count"].long()
    width = tables.shape[1]
    col = torch.arange(width, device=dev)
    # blocks of finished requests go back on the free list
    gone = q < 0
    back = torch.where(gone, owned, 0)
    place = have + (back.cumsum(0) - back)[:, None] + col
    give = gone[:, None] & (col < owned[:, None])
    stack[place[give]] = tables[give]
    have = have + back.sum()
    # new blocks from its end, in the order of the requests, while it lasts
    q0 = q.clamp(min=0)
    need = torch.where(gone | (q == 0), 0, ((c + q0 + block - 1) // block - owned).clamp(min=0))
    end = need.cumsum(0)
    served = ~gone & ((need == 0) | (end <= have))
    take = served[:, None] & (col >= owned[:, None]) & (col < (owned + need)[:, None])
    rank = (end - need)[:, None] + col - owned[:, None]
    tables[take] = stack[(have - 1 - rank)[take]]
    used = torch.where(served & (need > 0), end, 0).amax()
    qsl = torch.cat([q0.new_zeros(1), q0.cumsum(0)])
    # tokens
    t = torch.arange(tokens, device=dev)
    r = torch.searchsorted(qsl[1:], t, right=True)
    inside = r < q.shape[0]
    r = r.clamp(max=q.shape[0] - 1)
    i = t - qsl[r]
    live = inside & served[r]
    if s["parents"] is None:
        depth, mask = i, None
    else:
        n = s["max_query_len"]
        seen, _, valid, at = _closure(s["parents"], qsl, n)
        flat = seen.sum(-1) - 1
        depth = torch.zeros(tokens, dtype=torch.long, device=dev)
        depth[at[valid]] = flat[valid]
        words = -(-n // 64)
        bits = torch.nn.functional.pad(seen, (0, 64 * words - n)).view(-1, n, words, 64)
        weight = torch.ones(64, dtype=torch.long, device=dev) << torch.arange(64, device=dev)
        packed = (bits * weight).sum(-1)
        mask = torch.zeros(tokens, words, dtype=torch.long, device=dev)
        mask[at[valid]] = packed[valid]
        mask = torch.where(live[:, None], mask, 0)
    row = c[r] + i
    page = tables[r, (row // block).clamp(0, width - 1)].long()
    slots = torch.where(live, page * block + row % block, -1)
    positions = torch.where(live, c[r] + depth, 0)
    seq = torch.where(served, c + q0, 0)
    owned = torch.where(gone, 0, torch.where(served, owned + need, owned))
    out = [qsl.int(), seq.int(), slots, positions, mask, owned.int(), (have - used).int(),
           tables, stack]
    return [x for x in out if x is not None]


def _plain_accept(s):
    qsl, n = s["query_start_loc"].long(), s["max_query_len"]
    ids, targets = s["ids"], s["targets"]
    seen, parent, valid, at = _closure(s["parents"], qsl, n)
    node = torch.arange(n, device=ids.device)
    up = parent.clamp(min=0)
    fits = (parent >= 0) & (ids[at] == targets[at].gather(1, up))
    # of several children with the wanted token the first counts
    first = torch.full(up.shape, n, device=ids.device).scatter_reduce(
        1, up, torch.where(fits, node.expand_as(up), n), "amin")
    good = (fits & (first.gather(1, up) == node)) | ((node == 0) & valid)
    taken = valid & ~(seen & ~good[:, None, :]).any(-1)
    count = taken.sum(-1)
    order = torch.where(taken, node, n).sort(-1).values
    have = order < n
    path = torch.where(have, order, -1)
    tokens = torch.where(have, targets[at].gather(1, order.clamp(max=n - 1)), -1)
    return path.int(), tokens, count.int(), (s["context_lens"] + count).int()


def _plain_commit(s):
    path, count = s["path"].long(), s["num_accepted"].long()
    i = torch.arange(path.shape[1], device=path.device)
    start = s["query_start_loc"].long()[:-1, None]
    moved = (i >= 1) & (i < count[:, None]) & (path != i)
    src = s["slot_mapping"][(start + path)[moved]]
    dst = s["slot_mapping"][(start + i)[moved]]
    rows = s["caches"].flatten(2, 3)
    rows[:, :, dst] = rows[:, :, src]
    return s["caches"]


def run(s):
    op = s["case"]["op"]
    if not own:
        return {"attention": _plain_attention, "plan": _plain_plan, "accept": _plain_accept,
                "commit": _plain_commit}[op](s)
    ops = _ops()
    if op == "attention":
        return ops.tree_attention(s["q"], s["k_cache"], s["v_cache"], s["block_tables"],
                                  s["seq_lens"], s["query_start_loc"], s["tree_mask"],
                                  s["scale"])
    if op == "plan":
        out = ops.paged_plan(s["context_lens"], s["query_lens"], s["block_tables"],
                             s["blocks_owned"], s["free_blocks"], s["free_count"],
                             s["num_tokens"], s["block_size"], s["parents"],
                             s["max_query_len"])
        return [x for x in out if x is not None] + [s["block_tables"], s["free_blocks"]]
    if op == "accept":
        return ops.tree_accept(s["ids"], s["targets"], s["parents"], s["query_start_loc"],
                               s["seq_lens"], s["context_lens"], s["max_query_len"])
    ops.tree_commit(s["k_caches"], s["v_caches"], s["path"], s["num_accepted"],
                    s["slot_mapping"], s["query_start_loc"])
    return s["caches"]


# ------------------------------------------------------------------------------ work, 64 bits

def work(case):
    q, c = lengths(case)
    tokens, n = int(q.sum()), int(case["requests"])
    if case["op"] == "attention":
        heads, kv, dim = case["heads"], case["kv_heads"], case["dim"]
        cached = int((q + c).sum())
        words = max(1, -(-int(q.max()) // 64)) if case["shape"] == "tree" else 0
        pages = int((-(-(q + c) // case["block"])).sum())
        return {"bytes": 4 * cached * kv * dim + 4 * tokens * heads * dim + 8 * tokens * words +
                4 * pages + 8 * n,
                "flops": 4 * heads * dim * int((q * (c + 1)).sum())}
    if case["op"] == "plan":
        words = -(-case["nodes"] // 64) if case["shape"] == "tree" else 0
        # lengths, owned counts and ends in and out; slots, positions, parents and masks; one
        # table entry per page that a node falls in
        return {"bytes": 24 * n + tokens * (16 + (4 + 8 * words if words else 0)) +
                4 * int((q // case["block"] + 1).sum()), "flops": 0}
    if case["op"] == "accept":
        return {"bytes": tokens * 20 + n * (20 + 12 * max(1, int(q.max()))), "flops": 0}
    # one of a tree's last nodes lies at a depth of about its index over 3.5, the mean step back
    # to a parent, and nearly every accepted node but the root moves
    moved = int(np.ceil(q * 0.875 / 3.5).sum())
    return {"bytes": 4 * moved * case["layers"] * 2 * case["kv_heads"] * case["dim"], "flops": 0}


def exact(case, seed):
    """The definition in 64 bits, request by request."""
    if case["op"] == "attention":
        s = prepare(case, seed)
        q, c = lengths(case)
        start = _starts(q)
        heads, kv, dim = case["heads"], case["kv_heads"], case["dim"]
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
        mask = None if s["tree_mask"] is None else s["tree_mask"].cpu().numpy().view(np.uint64)
        tables = s["block_tables"].cpu().numpy()
        flat_k = s["k_cache"].view(-1, kv, dim)
        flat_v = s["v_cache"].view(-1, kv, dim)
        for b in range(len(q)):
            rows = np.arange(q[b] + c[b])
            slot = _dev(tables[b][rows // case["block"]].astype(np.int64) * case["block"] +
                        rows % case["block"])
            see = np.ones((q[b], q[b] + c[b]), bool)
            for i in range(q[b]):
                for x in range(q[b]):
                    see[i, c[b] + x] = x <= i if mask is None else bool(
                        (int(mask[start[b] + i, x // 64]) >> (x % 64)) & 1)
            hide = _dev(~see)
            k, v = flat_k[slot].double(), flat_v[slot].double()
            for h in range(heads):
                g = h * kv // heads
                x = s["q"][start[b]: start[b + 1], h].double() @ k[:, g].T * s["scale"]
                x = x.masked_fill(hide, -math.inf)
                out[start[b]: start[b + 1], h] = torch.softmax(x, -1) @ v[:, g]
        return out
    if case["op"] == "commit":
        s = prepare(case, seed)
        rows = s["caches"].double().flatten(2, 3)
        path, count = s["path"].tolist(), s["num_accepted"].tolist()
        slots, start = s["slot_mapping"].tolist(), s["query_start_loc"].tolist()
        old = rows.clone()
        for b, n in enumerate(count):
            for i in range(1, n):
                rows[:, :, slots[start[b] + i]] = old[:, :, slots[start[b] + path[b][i]]]
        return rows.view(s["caches"].shape)
    return None  # whole numbers only
