"""The operators that check trees of drafted tokens, on CPU and GPU: paged_plan, tree_accept and
tree_commit (whole numbers and moved rows: exact), tree_attention against the definition in 64
bits, and their refusals. The sizes here are small; the GPU kernel's tiles and splits are covered
in test_gpu_tree_attention.py."""

from __future__ import annotations

import pytest
import torch

import svllm_ops
from tree_reference import (attention_bound, attention_reference, make_pages, masks_of,
                            pack_lists, plan_reference, random_parents, walk_reference)


def i32(values, device):
    return torch.tensor(values, dtype=torch.int32, device=device)


# -------------------------------------------------------------------------------- paged_plan

def run_plan(device, case):
    t = {k: i32(case[k], device) for k in ("context_lens", "query_lens", "blocks_owned",
                                           "free_blocks")}
    tables = i32(case["block_tables"], device)
    parents = None if case["parents"] is None else i32(case["parents"], device)
    stack = t["free_blocks"]
    out = svllm_ops.paged_plan(t["context_lens"], t["query_lens"], tables, t["blocks_owned"],
                               stack, i32([case["free_count"]], device), case["num_tokens"],
                               case["block_size"], parents, case["max_query_len"])
    return out, tables, stack


def make_plan_case(seed, requests, nodes, context, bs, *, tree, short, finish, pad=0):
    g = torch.Generator().manual_seed(seed)

    def rand(lo, hi, n=requests):
        return torch.randint(lo, hi + 1, (n,), generator=g).tolist()

    ctx = rand(0, context)
    query = rand(0, nodes)
    query[0] = nodes
    for s in range(1, requests, finish) if finish else ():
        query[s] = -1
    owned = [-(-c // bs) + e for c, e in zip(ctx, rand(0, 1))]
    need = [max(0, -(-(c + max(q, 0)) // bs) - o) for c, q, o in zip(ctx, query, owned)]
    width = max(o + n for o, n in zip(owned, need)) + 1
    total = sum(owned) + sum(need) + 3
    ids = torch.randperm(total, generator=g).tolist()
    tables, at = [], 0
    for o in owned:
        tables.append(ids[at: at + o] + [0] * (width - o))
        at += o
    count = sum(need) * 2 // 3 if short else sum(need) + 3
    q0 = [max(q, 0) for q in query]
    return {"context_lens": ctx, "query_lens": query, "block_tables": tables,
            "blocks_owned": owned, "free_blocks": ids[at:] + [0] * sum(owned),
            "free_count": count, "num_tokens": sum(q0) + pad, "block_size": bs,
            "parents": random_parents(seed, q0) + [-1] * pad if tree else None,
            "max_query_len": max(1, nodes)}


@pytest.mark.parametrize("requests, nodes, context, bs, tree, short, finish, pad", [
    (1, 1, 0, 16, True, False, 0, 0),         # the first token of one request
    (4, 8, 100, 16, True, False, 0, 0),
    (5, 64, 300, 16, True, False, 0, 0),      # a full mask word
    (5, 65, 300, 1, True, False, 0, 0),       # one node in a second word; one row per page
    (7, 130, 50, 12, True, True, 3, 0),       # three words, a pool that runs out, finished ones
    (40, 9, 500, 16, False, True, 4, 5),      # chains, padding tokens
    (33, 0, 64, 16, False, False, 2, 2),      # nobody has a token
    (1030, 3, 40, 16, True, True, 7, 0),      # more requests than one pass of a CTA takes
    (1500, 7, 64, 8, True, False, 5, 0),      # many tokens: the second kernel
    (2100, 4, 64, 8, False, True, 0, 9),
    (300, 64, 100, 16, True, True, 5, 7),     # full mask words, the second kernel
    (4200, 2, 20, 16, True, False, 0, 3),     # more starts than that one keeps
    (64, 40, 30, 1, True, False, 0, 0),       # long runs of blocks
    (1100, 0, 64, 16, False, False, 2, 0),    # nobody has a token, nor is there any
], ids=str)
def test_paged_plan(device, requests, nodes, context, bs, tree, short, finish, pad):
    case = make_plan_case(requests * 31 + nodes, requests, nodes, context, bs, tree=tree,
                          short=short, finish=finish, pad=pad)
    want, want_tables, want_stack = plan_reference(case)
    for _ in range(2):  # the second call, on the same inputs, writes the same
        out, tables, stack = run_plan(device, case)
        for name, got in zip(("query_start_loc", "seq_lens", "slot_mapping", "positions",
                              "tree_mask", "blocks_owned", "free_count"), out):
            if name == "tree_mask" and not tree:
                assert got is None
            else:
                assert torch.equal(got.cpu(), want[name]), name
        assert torch.equal(tables.cpu(), want_tables) and torch.equal(stack.cpu(), want_stack)
    if short:
        assert (want["seq_lens"] == 0).any()  # the case means what it says


@pytest.mark.parametrize("requests, nodes, tree, finish", [
    (7, 130, True, 3), (40, 9, False, 4), (300, 64, True, 5), (1030, 3, True, 7),
    (4200, 2, True, 2),
], ids=str)
def test_paged_plan_again_on_its_own_lists(device, requests, nodes, tree, finish):
    """A second call with the same lengths and counts, on the tables and the free list that the first
    has written, gives and writes the same: blocks that came back are where they were put, and those
    taken are taken again."""
    case = make_plan_case(requests + nodes, requests, nodes, 60, 8, tree=tree, short=True,
                          finish=finish, pad=3)
    want, want_tables, want_stack = plan_reference(case)
    lists = [i32(case[k], device) for k in ("context_lens", "query_lens", "block_tables",
                                            "blocks_owned", "free_blocks")]
    count = i32([case["free_count"]], device)
    parents = i32(case["parents"], device) if tree else None
    for _ in range(3):
        out = svllm_ops.paged_plan(*lists, count, case["num_tokens"], case["block_size"], parents,
                                   case["max_query_len"])
        for name, got in zip(("query_start_loc", "seq_lens", "slot_mapping", "positions",
                              "tree_mask", "blocks_owned", "free_count"), out):
            assert got is None if name == "tree_mask" and not tree else torch.equal(
                got.cpu(), want[name]), name
        assert torch.equal(lists[2].cpu(), want_tables)
        assert torch.equal(lists[4].cpu(), want_stack)
    assert (want["seq_lens"] == 0).any() and want_stack.tolist() != case["free_blocks"]


def test_paged_plan_without_requests(device):
    e = i32([], device)
    out = svllm_ops.paged_plan(e, e, torch.zeros(0, 3, dtype=torch.int32, device=device), e,
                               i32([4, 5], device), i32([2], device), 3, 16)
    assert out[0].tolist() == [0] and out[2].tolist() == [-1] * 3 and out[3].tolist() == [0] * 3
    assert out[6].tolist() == [2]


def test_paged_plan_rejects_bad_inputs():
    def call(**change):
        a = dict(context_lens=i32([4], "cpu"), query_lens=i32([2], "cpu"),
                 block_tables=torch.zeros(1, 4, dtype=torch.int32), blocks_owned=i32([1], "cpu"),
                 free_blocks=i32([1, 2, 3], "cpu"), free_count=i32([3], "cpu"), num_tokens=2,
                 block_size=4, parents=i32([-1, 0], "cpu"), max_query_len=2)
        a.update(change)
        return svllm_ops.paged_plan(**a)

    call()
    for change, what in [
        ({"query_lens": torch.tensor([2])}, "int32"),
        ({"query_lens": i32([2, 2], "cpu")}, "does not match"),
        ({"block_tables": torch.zeros(4, 1, dtype=torch.int32).t()[:, ::2]}, "contiguous"),
        ({"block_tables": torch.zeros(1, 0, dtype=torch.int32)}, "no room"),
        ({"block_size": 0}, "positive"),
        ({"num_tokens": 1, "parents": i32([-1], "cpu")}, "num_tokens"),
        ({"parents": i32([-1], "cpu")}, "does not match"),
        ({"max_query_len": 0}, "max_query_len"),
        ({"max_query_len": 1025}, "max_query_len"),
        ({"max_query_len": 1}, "max_query_len"),
        ({"parents": i32([-1, 1], "cpu")}, "does not come before"),
        ({"free_count": i32([4], "cpu")}, "free_count"),
        ({"context_lens": i32([15], "cpu")}, "does not fit"),
        ({"context_lens": i32([-1], "cpu")}, "does not fit"),
        ({"blocks_owned": i32([5], "cpu")}, "owns"),
        ({"query_lens": i32([-1], "cpu"), "free_count": i32([3], "cpu")}, "come back"),
        ({"context_lens": i32([4], "cpu").to("meta")}, "context_lens is on"),
    ]:
        with pytest.raises(RuntimeError, match=what):
            call(**change)


def test_paged_plan_refusals_write_nothing():
    """What a refused call was given is as it was: the tables and the free list, to which a finished
    request's blocks would have come back and from which two more would have been taken."""
    def lists():
        return dict(context_lens=i32([4, 8, 4, 4], "cpu"), query_lens=i32([2, -1, 3, 4], "cpu"),
                    block_tables=i32([[1, 0, 0, 0], [2, 3, 0, 0], [4, 0, 0, 0], [5, 0, 0, 0]],
                                     "cpu"),
                    blocks_owned=i32([1, 2, 1, 1], "cpu"),
                    free_blocks=i32([6, 0, 0, 0], "cpu"), free_count=i32([0], "cpu"),
                    num_tokens=9, block_size=4, parents=i32([-1, 0, -1, 0, 1, -1, 0, 1, 2], "cpu"),
                    max_query_len=4)

    served = lists()
    assert svllm_ops.paged_plan(**served)[1].tolist() == [6, 0, 7, 0]
    assert served["block_tables"][0, 1] == 3 and served["free_blocks"].tolist() == [2, 3, 0, 0]
    for change in [
        {"parents": i32([-1, 1, -1, 0, 1, -1, 0, 1, 2], "cpu")},   # of the first request
        {"parents": i32([-1, 0, -1, 0, -2, -1, 0, 1, 2], "cpu")},  # of the last that is served
        {"parents": i32([-1, 0, -1, 0, 1, -1, 0, 1, 7], "cpu")},   # of one that is not
        {"max_query_len": 3}, {"context_lens": i32([4, 8, 14, 4], "cpu")},
        {"blocks_owned": i32([1, 2, 1, 5], "cpu")}, {"free_count": i32([3], "cpu")},
        {"num_tokens": 8, "parents": i32([-1, 0, -1, 0, 1, -1, 0, 1], "cpu")},
    ]:
        a = {**lists(), **change}
        with pytest.raises(RuntimeError, match="paged_plan"):
            svllm_ops.paged_plan(**a)
        assert torch.equal(a["block_tables"], lists()["block_tables"]), change
        assert torch.equal(a["free_blocks"], lists()["free_blocks"]), change


@pytest.mark.gpu
def test_paged_plan_bad_lengths_on_cuda(cuda):
    """What the CPU refuses raises the bad-index bit, and only the request it concerns goes
    without."""
    case = {"context_lens": [4, -1, 4, 4, 15, 4], "query_lens": [2, 2, 2, 2, 2, 3],
            "block_tables": [[0, 0, 0, 0]] * 6, "blocks_owned": [1, 1, -1, 5, 4, 1],
            "free_blocks": list(range(10, 30)), "free_count": 20, "num_tokens": 13,
            "block_size": 4, "parents": [-1, 0] * 5 + [-1, 5, 0], "max_query_len": 8}
    svllm_ops.read_device_error(0, True)
    out, tables, _ = run_plan(cuda, case)
    assert svllm_ops.read_device_error(0, True) == 1
    assert out[1].tolist() == [6, 0, 0, 0, 0, 7]
    assert out[2].tolist() == [29 * 4, 29 * 4 + 1] + [-1] * 8 + [28 * 4, 28 * 4 + 1, 28 * 4 + 2]
    assert out[3].tolist() == [4, 5] + [0] * 8 + [4, 4, 5]  # node 1 counts as a root
    assert out[4].flatten().tolist() == [1, 3] + [0] * 8 + [1, 2, 5]
    assert out[5].tolist() == [2, 1, -1, 5, 4, 2] and out[6].tolist() == [18]
    # more tokens than room: the request that reaches past it is not served
    case["num_tokens"] = 12
    case["parents"] = case["parents"][:12]
    out, _, _ = run_plan(cuda, case)
    assert svllm_ops.read_device_error(0, True) == 1
    assert out[1].tolist() == [6, 0, 0, 0, 0, 0] and out[0].tolist()[-1] == 12


@pytest.mark.gpu
def test_paged_plan_bad_lengths_of_many_tokens_on_cuda(cuda):
    """The same where the tokens have a kernel of their own: a length of 2^31 - 1 in the middle,
    with which sums of lengths stop short of wrapping."""
    requests, at = 600, 400
    query = [3] * requests
    query[7], query[at] = 9, 2 ** 31 - 1   # wider than the mask; past every token
    case = {"context_lens": [4] * requests, "query_lens": query,
            "block_tables": [[0, 0, 0, 0]] * requests, "blocks_owned": [4] * requests,
            "free_blocks": [0], "free_count": 0, "num_tokens": 3 * requests + 6, "block_size": 4,
            "parents": ([-1, 0, 0] * 7 + [-1] * 9 + [-1, 0, 5] + [-1, 0, 1] * requests)[
                : 3 * requests + 6], "max_query_len": 8}
    svllm_ops.read_device_error(0, True)
    out, _, _ = run_plan(cuda, case)
    assert svllm_ops.read_device_error(0, True) == 1
    start = [0]
    for q in query:
        start.append(min(start[-1] + q, case["num_tokens"]))
    assert out[0].tolist() == start
    served = [7 if s != 7 and s < at else 0 for s in range(requests)]
    assert out[1].tolist() == served
    live = torch.tensor([s != 7 for s, q in enumerate(query[:at]) for _ in range(q)] +
                        [False] * (case["num_tokens"] - start[at]))
    masks, positions = out[4].flatten().cpu(), out[3].cpu()
    assert ((masks != 0) == live).all() and ((out[2].cpu() >= 0) == live).all()
    assert masks[:6].tolist() == [1, 3, 5, 1, 3, 5]
    assert masks[30:36].tolist() == [1, 3, 4, 1, 3, 7]  # a parent that comes later: a root
    assert positions[30:36].tolist() == [4, 5, 4, 4, 5, 6]


@pytest.mark.gpu
@pytest.mark.parametrize("more", [0, 300, 5000], ids=["one launch", "two", "two, many starts"])
@pytest.mark.parametrize("fault", ["parent", "width"])
def test_paged_plan_requests_that_are_not_served_on_cuda(cuda, more, fault):
    """A parent of a request that finds no blocks is checked like any other, and one whose tree has
    more nodes than the words of the mask has none of them written: both go without a slot, a
    position and a mask, and nobody else does."""
    nodes = [3, 70 if fault == "width" else 3, 3] + [3] * more
    case = {"context_lens": [4] * len(nodes), "query_lens": nodes,
            "block_tables": [[5] + [0] * 19] * len(nodes),
            "blocks_owned": [2] + [1 if fault == "parent" else 20] + [2] * (1 + more),
            "free_blocks": [9], "free_count": 0, "num_tokens": sum(nodes), "block_size": 4,
            "parents": [-1, 0, 1] + ([-1, 2, 0] if fault == "parent" else [-1] + [0] * 69) +
            [-1, 0, 0] * (1 + more), "max_query_len": 40}
    svllm_ops.read_device_error(0, True)
    out, tables, _ = run_plan(cuda, case)
    assert svllm_ops.read_device_error(0, True) == 1
    first, end = 3, 3 + nodes[1]
    assert out[1].tolist() == [7, 0] + [7] * (1 + more)
    assert out[2][first:end].tolist() == [-1] * nodes[1]
    assert out[3][first:end].tolist() == [0] * nodes[1]
    assert out[4][first:end].flatten().tolist() == [0] * nodes[1]
    assert out[2][:3].tolist() == [0, 1, 2] and out[4][:3].flatten().tolist() == [1, 3, 7]
    assert out[2][end:].tolist() == [0, 1, 2] * (1 + more)
    assert out[3][end:].tolist() == [4, 5, 5] * (1 + more)
    assert out[4][end:].flatten().tolist() == [1, 3, 5] * (1 + more)
    assert torch.equal(tables.cpu(), torch.tensor(case["block_tables"], dtype=torch.int32))


@pytest.mark.gpu
@pytest.mark.parametrize("requests", [40, 300, 4200])
def test_paged_plan_behind_the_kernel_that_makes_its_lengths(cuda, requests):
    """The lists of a plan come from the kernels right before it, and the tables it fills lie in one
    buffer with the parents it reads, in the same 32 bytes where they meet: captured, and replayed
    with other lists."""
    nodes, bs = 40, 4
    width = (64 + nodes) // bs + 1
    g = torch.Generator().manual_seed(requests)
    starts = i32([nodes * s for s in range(requests + 1)], cuda)
    ones = i32([1] * requests, cuda)
    targets = torch.ones(requests * nodes, dtype=torch.int64, device=cuda)
    tokens = requests * nodes
    buffer = torch.zeros(requests * width + tokens, dtype=torch.int32, device=cuda)
    tables = buffer[: requests * width].view(requests, width)
    parents = buffer[requests * width:]
    new_parents = torch.zeros_like(parents)
    ids, context = torch.zeros_like(targets), i32([0] * requests, cuda)
    owned = i32([0] * requests, cuda)
    stack = torch.arange(requests * width, dtype=torch.int32, device=cuda)
    count = i32([requests * width], cuda)

    def step():
        tables.zero_()
        parents.copy_(new_parents)
        # chains of which every request accepts as many as its ids say
        _, _, query, after = svllm_ops.tree_accept(ids, targets, None, starts, ones, context,
                                                   nodes)
        return (query, after) + svllm_ops.paged_plan(after, query, tables, owned, stack, count,
                                                     tokens, bs, parents, nodes)

    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for _ in range(4):
        length = torch.randint(1, nodes + 1, (requests,), generator=g)
        before = torch.randint(0, 24, (requests,), generator=g)
        packed = random_parents(requests, length.tolist())
        ids.copy_((torch.arange(nodes) < length[:, None]).long().flatten())
        context.copy_(before)
        new_parents.copy_(i32(packed + [-1] * (tokens - len(packed)), "cpu"))
        graph.replay()
        case = {"context_lens": (before + length).tolist(), "query_lens": length.tolist(),
                "block_tables": [[0] * width] * requests, "blocks_owned": [0] * requests,
                "free_blocks": list(range(requests * width)), "free_count": requests * width,
                "num_tokens": tokens, "block_size": bs,
                "parents": packed + [-1] * (tokens - len(packed)), "max_query_len": nodes}
        want, want_tables, _ = plan_reference(case)
        assert out[0].tolist() == case["query_lens"] and out[1].tolist() == case["context_lens"]
        for name, got in zip(("query_start_loc", "seq_lens", "slot_mapping", "positions",
                              "tree_mask", "blocks_owned", "free_count"), out[2:]):
            assert torch.equal(got.cpu(), want[name]), name
        assert torch.equal(tables.cpu(), want_tables)
        assert parents.tolist() == case["parents"]


# ------------------------------------------------------------------------------ tree_accept

@pytest.mark.parametrize("counts", [[1], [8], [0, 3, 0, 17], [64, 65, 33, 1], [200, 31, 0, 128],
                                    [1024]], ids=str)
@pytest.mark.parametrize("ids_dtype", [torch.int32, torch.int64])
@pytest.mark.parametrize("tree", [True, False], ids=["tree", "chain"])
def test_tree_accept(device, counts, ids_dtype, tree):
    g = torch.Generator().manual_seed(sum(counts))
    tokens = sum(counts)
    parents = random_parents(7, counts)
    ids = torch.randint(0, 4, (tokens,), generator=g)      # few ids: many equal siblings
    targets = torch.randint(0, 4, (tokens,), generator=g)
    if not tree:
        ids[:] = 1  # long walks
        targets[:] = (torch.rand(tokens, generator=g) < 0.9).long()
    starts, _ = pack_lists(counts)
    context = list(range(5, 5 + len(counts)))
    seq = [c + n for c, n in zip(context, counts)]
    if len(seq) > 2:
        seq[1] = 0  # not served
    width = max(1, max(counts)) + 2
    want = walk_reference(ids.tolist(), targets.tolist(), parents if tree else None, starts, seq,
                          context, width)
    got = svllm_ops.tree_accept(ids.to(device, ids_dtype), targets.to(device),
                                i32(parents, device) if tree else None, i32(starts, device),
                                i32(seq, device), i32(context, device), min(width, 1024))
    for name, a, b in zip(("path", "tokens", "num_accepted", "context"), got, want):
        b = b[:, :1024] if b.dim() == 2 else b
        assert torch.equal(a.cpu(), b), name


def test_tree_accept_rejects_bad_inputs():
    def call(**change):
        a = dict(ids=torch.tensor([1, 2]), targets=torch.tensor([2, 3]),
                 parents=i32([-1, 0], "cpu"), query_start_loc=i32([0, 2], "cpu"),
                 seq_lens=i32([6], "cpu"), context_lens=i32([4], "cpu"), max_query_len=2)
        a.update(change)
        return svllm_ops.tree_accept(**a)

    assert call()[2].tolist() == [2]
    for change, what in [
        ({"ids": torch.tensor([1.0, 2.0])}, "int32 or int64"),
        ({"targets": i32([2, 3], "cpu")}, "targets"),
        ({"parents": i32([-1], "cpu")}, "parents"),
        ({"query_start_loc": i32([0], "cpu")}, "query_start_loc"),
        ({"query_start_loc": i32([0, 3], "cpu")}, "query_start_loc"),
        ({"query_start_loc": i32([2, 0], "cpu")}, "query_start_loc"),
        ({"context_lens": torch.tensor([4])}, "context_lens"),
        ({"max_query_len": 0}, "max_query_len"),
        ({"max_query_len": 1025}, "max_query_len"),
        ({"max_query_len": 1}, "max_query_len"),
        ({"seq_lens": i32([6], "cpu").to("meta")}, "is on"),
    ]:
        with pytest.raises(RuntimeError, match=what):
            call(**change)


@pytest.mark.gpu
def test_tree_accept_bad_starts_on_cuda(cuda):
    """Requests whose tokens are out of range or too many accept nothing; the others do."""
    svllm_ops.read_device_error(0, True)
    out = svllm_ops.tree_accept(torch.ones(8, dtype=torch.int64, device=cuda),
                                torch.ones(8, dtype=torch.int64, device=cuda), None,
                                i32([0, 2, 1, 3, 9], cuda), i32([9] * 4, cuda), i32([3] * 4, cuda),
                                4)
    assert svllm_ops.read_device_error(0, True) == 1
    assert out[2].tolist() == [2, 0, 2, 0] and out[3].tolist() == [5, 3, 5, 3]
    assert out[0].tolist() == [[0, 1, -1, -1], [-1] * 4, [0, 1, -1, -1], [-1] * 4]


# ------------------------------------------------------------------------------ tree_commit

def random_paths(seed, counts, parents, starts, width):
    g = torch.Generator().manual_seed(seed)
    paths, accepted = [], []
    for s, n in enumerate(counts):
        node = int(torch.randint(0, n, (1,), generator=g)) if n else -1
        back = []
        while node >= 0:
            back.append(node)
            node = parents[starts[s] + node]
        accepted.append(len(back))
        paths.append(back[::-1] + [-1] * (width - len(back)))
    return paths, accepted


@pytest.mark.parametrize("counts, layers, kv_heads, dim, dtype", [
    ([9], 1, 1, 8, torch.bfloat16),               # one 16-byte vector per row
    ([40, 0, 33, 1], 3, 8, 128, torch.bfloat16),
    ([64, 200, 17], 2, 2, 64, torch.float32),
    ([12, 30], 70, 2, 8, torch.bfloat16),         # more planes than one launch takes
    ([20] * 9, 2, 5, 24, torch.bfloat16),         # rows that no power of two divides
    ([300], 1, 24, 128, torch.bfloat16),          # rows longer than the CTA
], ids=str)
def test_tree_commit(device, counts, layers, kv_heads, dim, dtype):
    bs = 4
    g = torch.Generator().manual_seed(len(counts) + layers)
    context = [3 * s + 1 for s in range(len(counts))]
    _, blocks, slots = make_pages(5, counts, context, bs)
    starts, _ = pack_lists(counts)
    parents = random_parents(11, counts)
    width = max(counts)
    paths, accepted = random_paths(3, counts, parents, starts, width)
    if len(counts) == 9:
        slots[starts[4]: starts[5]] = [-1] * 20  # a request without slots
    shape = (blocks, bs, kv_heads, dim)
    k = [torch.randn(shape, generator=g).to(dtype) for _ in range(layers)]
    v = [torch.randn(shape, generator=g).to(dtype) for _ in range(layers)]
    want = [c.clone() for c in k + v]
    for c, old in zip(want, k + v):
        for s, n in enumerate(accepted):
            for i in range(1, n):
                src, dst = slots[starts[s] + paths[s][i]], slots[starts[s] + i]
                if src >= 0 and dst >= 0:
                    c.view(-1, kv_heads, dim)[dst] = old.view(-1, kv_heads, dim)[src]
    k, v = [c.to(device) for c in k], [c.to(device) for c in v]
    svllm_ops.tree_commit(k, v, i32(paths, device).view(len(counts), width), i32(accepted, device),
                          torch.tensor(slots, device=device), i32(starts, device))
    for got, w in zip(k + v, want):
        assert torch.equal(got.cpu(), w)


def test_tree_commit_rejects_bad_inputs():
    def call(**change):
        a = dict(k_caches=[torch.zeros(2, 4, 1, 8)], v_caches=[torch.zeros(2, 4, 1, 8)],
                 path=i32([[0, 2, -1]], "cpu"), num_accepted=i32([2], "cpu"),
                 slot_mapping=torch.tensor([0, 1, 2]), query_start_loc=i32([0, 3], "cpu"))
        a.update(change)
        return svllm_ops.tree_commit(**a)

    call()
    cache = torch.zeros(2, 4, 1, 8)
    for change, what in [
        ({"k_caches": []}, "0 K caches"),
        ({"v_caches": [cache, cache]}, "2 V caches"),
        ({"v_caches": [cache.bfloat16()]}, "one shape"),
        ({"v_caches": [torch.zeros(2, 4, 8, 2).transpose(2, 3)[:, :, :1]]}, "one shape"),
        ({"k_caches": [torch.zeros(8, 8)], "v_caches": [torch.zeros(8, 8)]}, "caches must be"),
        ({"path": torch.tensor([[0, 2, -1]])}, "path"),
        ({"path": i32([0, 2, -1], "cpu")}, "path"),
        ({"slot_mapping": i32([0, 1, 2], "cpu")}, "slot_mapping"),
        ({"num_accepted": i32([4], "cpu")}, "accepts"),
        ({"num_accepted": i32([-1], "cpu")}, "accepts"),
        ({"path": i32([[0, 0, -1]], "cpu")}, "rise"),
        ({"path": i32([[0, 3, -1]], "cpu")}, "rise"),
        ({"slot_mapping": torch.tensor([0, 1, 8])}, "past the cache"),
        ({"query_start_loc": i32([0, 4], "cpu")}, "query_start_loc"),
        ({"path": i32([[0, 2, -1]], "cpu").to("meta")}, "is on"),
    ]:
        with pytest.raises(RuntimeError, match=what):
            call(**change)


def test_tree_commit_takes_lists_and_tuples_of_tensors():
    lists = (i32([[0, 2, -1]], "cpu"), i32([2], "cpu"), torch.tensor([0, 1, 2]), i32([0, 3], "cpu"))
    k = torch.arange(64, dtype=torch.float32).view(2, 4, 1, 8)
    v = torch.nn.Parameter(-k, requires_grad=False)
    svllm_ops.tree_commit((k,), [v], *lists)
    assert torch.equal(k[0, 1], k[0, 2]) and torch.equal(v[0, 1], v[0, 2])
    for bad in (k, None, [None], [[k]], (k, 1)):
        with pytest.raises(TypeError, match="k_caches"):
            svllm_ops.tree_commit(bad, [v], *lists)


def test_tree_commit_refuses_a_cache_given_twice(device):
    """Its rows would move twice. 1 to 300 layers: a table of the caches seen, then all pairs."""
    small = [torch.zeros(2, 4, 1, 8, device=device) for _ in range(600)]
    lists = (i32([[0, 2, -1]], device), i32([2], device),
             torch.tensor([0, 1, 2], device=device), i32([0, 3], device))
    for layers in (1, 2, 36, 256, 257, 300):
        k, v = small[:layers], small[300: 300 + layers]
        svllm_ops.tree_commit(k, v, *lists)
        for bad in (v[:-1] + k[:1], v[:-1] + v[:1] if layers > 1 else k):
            with pytest.raises(RuntimeError, match="invalid argument"):
                svllm_ops.tree_commit(k, bad, *lists)


@pytest.mark.gpu
def test_tree_commit_bad_paths_on_cuda(cuda):
    """A path that does not rise moves no row from there on, a slot past the cache leaves its
    row; the other requests' rows move."""
    cache = torch.arange(32, device=cuda, dtype=torch.float32).view(32, 1, 1).repeat(1, 1, 8)
    k, v = [cache.clone()], [cache.clone()]
    svllm_ops.read_device_error(0, True)
    svllm_ops.tree_commit(k, v, i32([[0, 2, 2, 3], [0, 3, -1, -1], [0, 2, 3, -1], [0, 1, 2, 3]],
                                    cuda),
                          i32([4, 2, 3, 9], cuda),
                          torch.tensor([0, 1, 2, 3, 4, 5, 6, 7, 8, 9, 99, 11, 12, 13, 14, 15],
                                       device=cuda),
                          i32([0, 4, 8, 12, 16], cuda))
    assert svllm_ops.read_device_error(0, True) == 1
    want = list(range(32))
    want[1] = 2          # request 0: up to the step that does not rise
    want[5] = 7          # request 1
    # request 2: its step 1 reads slot 99, its step 2 writes it; request 3 counts past its nodes
    for c in k + v:
        assert c[:, 0, 0].tolist() == want


# --------------------------------------------------------------------------- tree_attention

def check_attention(device, counts, context, heads, kv_heads, dim, bs, *, tree=True, pad=0,
                    dtype=torch.bfloat16, seed=0):
    g = torch.Generator().manual_seed(seed)
    tables, blocks, _ = make_pages(seed, counts, context, bs)
    starts, tokens = pack_lists(counts)
    rows = tokens + pad
    qkv = torch.randn(rows, (heads + 2) * dim, generator=g).to(dtype)
    q = qkv[:, : heads * dim].view(rows, heads, dim)
    k, v = (torch.randn(blocks, bs, kv_heads, dim, generator=g).to(dtype) for _ in range(2))
    seq = [c + n for c, n in zip(context, counts)]
    mask = None
    if tree:
        mask = torch.cat([masks_of(random_parents(seed, counts), counts),
                          torch.zeros(pad, max(1, -(-max(counts) // 64)), dtype=torch.long)])
    got = svllm_ops.tree_attention(
        q.to(device) if device.type == "cpu" else
        qkv.to(device)[:, : heads * dim].view(rows, heads, dim),
        k.to(device), v.to(device), i32(tables, device), i32(seq, device), i32(starts, device),
        None if mask is None else mask.to(device))
    assert got.shape == (rows, heads, dim) and got.dtype == dtype
    ref, size = attention_reference(q, k, v, tables, seq, starts, mask, dim ** -0.5)
    assert ((got.cpu().double() - ref).abs() <= attention_bound(ref, size, dtype)).all()


@pytest.mark.parametrize("counts, context, heads, kv_heads, dim, bs, tree, pad", [
    ([1], [0], 2, 1, 64, 16, True, 0),               # one token, nothing cached
    ([3], [5], 4, 2, 128, 4, True, 0),
    ([7, 0, 2], [20, 9, 0], 6, 2, 64, 12, True, 2),  # a request that sits out, padding rows
    ([65, 4], [31, 70], 8, 8, 64, 16, True, 0),      # two mask words
    ([5, 9], [40, 3], 5, 1, 128, 1, False, 1),       # causal, one row per page
], ids=str)
def test_tree_attention(device, counts, context, heads, kv_heads, dim, bs, tree, pad):
    check_attention(device, counts, context, heads, kv_heads, dim, bs, tree=tree, pad=pad)


def test_tree_attention_fp32_and_other_head_dims_on_cpu():
    cpu = torch.device("cpu")
    check_attention(cpu, [4, 2], [11, 0], 4, 2, 24, 8, dtype=torch.float32)
    check_attention(cpu, [4, 2], [11, 0], 3, 3, 40, 8)


def test_tree_attention_rejects_bad_inputs():
    def call(**change):
        a = dict(q=torch.zeros(3, 4, 8, dtype=torch.bfloat16),
                 k_cache=torch.zeros(4, 2, 2, 8, dtype=torch.bfloat16),
                 v_cache=torch.zeros(4, 2, 2, 8, dtype=torch.bfloat16),
                 block_tables=torch.zeros(1, 3, dtype=torch.int32), seq_lens=i32([5], "cpu"),
                 query_start_loc=i32([0, 3], "cpu"), tree_mask=torch.ones(3, 1, dtype=torch.int64))
        a.update(change)
        return svllm_ops.tree_attention(**a)

    call()
    cache = torch.zeros(4, 2, 2, 8, dtype=torch.bfloat16)
    for change, what in [
        ({"q": torch.zeros(3, 4, 8, dtype=torch.float16)}, "bf16"),
        ({"q": torch.zeros(3, 4, 8)}, "caches are"),
        ({"q": torch.zeros(4, 3, 8, dtype=torch.bfloat16).transpose(0, 1)}, "contiguous"),
        ({"q": torch.zeros(3, 32, dtype=torch.bfloat16)}, r"\[tokens, heads, head_dim\]"),
        ({"q": torch.zeros(3, 3, 8, dtype=torch.bfloat16)}, "caches of shape"),
        ({"v_cache": cache[:2]}, "caches of shape"),
        ({"k_cache": cache.transpose(1, 2)}, "caches of shape"),
        ({"seq_lens": torch.tensor([5])}, "int32"),
        ({"block_tables": torch.zeros(2, 3, dtype=torch.int32)}, "block_tables"),
        ({"query_start_loc": i32([0], "cpu")}, "query_start_loc"),
        ({"query_start_loc": i32([1, 3], "cpu")}, "starts at"),
        ({"query_start_loc": i32([0, 4], "cpu")}, "falls or ends"),
        ({"tree_mask": torch.ones(3, 1, dtype=torch.int32)}, "tree_mask"),
        ({"tree_mask": torch.ones(2, 1, dtype=torch.int64)}, "tree_mask"),
        ({"tree_mask": torch.ones(3, 17, dtype=torch.int64)}, "tree_mask"),
        ({"seq_lens": i32([2], "cpu")}, "does not fit"),
        ({"seq_lens": i32([7], "cpu")}, "does not fit"),
        ({"block_tables": i32([[0, 4, 0]], "cpu")}, "outside the cache"),
        ({"scale": 0.0}, "scale"),
        ({"scale": float("inf")}, "scale"),
        ({"seq_lens": i32([5], "cpu").to("meta")}, "elsewhere"),
    ]:
        with pytest.raises(RuntimeError, match=what):
            call(**change)
