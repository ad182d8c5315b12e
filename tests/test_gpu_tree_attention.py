"""Tree attention on the GPU against the definition in 64 bits, at the sizes where a tiled kernel
that splits long contexts can go wrong, and what a caller may do with it: strided q, other streams,
captured graphs, values that must not leak out of masked places."""

from __future__ import annotations

import pytest
import torch

import svllm_capi
import svllm_ops
from tree_reference import (attention_bound, attention_reference, make_pages, masks_of, pack_lists,
                            random_parents)

pytestmark = pytest.mark.gpu


def build(cuda, counts, context, heads, kv_heads, dim, bs, *, shape="tree", pad=0, seed=0,
          spare=0):
    g = torch.Generator(device=cuda).manual_seed(seed)
    tables, blocks, _ = make_pages(seed, counts, context, bs)
    starts, tokens = pack_lists(counts)
    rows = tokens + pad
    qkv = torch.randn(rows, (heads + 2 * kv_heads) * dim, device=cuda, generator=g).bfloat16()
    mask = None
    if shape == "tree":
        m = masks_of(random_parents(seed, counts), counts)
        mask = torch.cat([m, torch.zeros(pad, m.shape[1], dtype=torch.long)]).to(cuda)
    return {"q": qkv[:, : heads * dim].view(rows, heads, dim),
            "k": torch.randn(blocks + spare, bs, kv_heads, dim, device=cuda,
                             generator=g).bfloat16(),
            "v": torch.randn(blocks + spare, bs, kv_heads, dim, device=cuda,
                             generator=g).bfloat16(),
            "tables": torch.tensor(tables, dtype=torch.int32, device=cuda),
            "seq": torch.tensor([c + n for c, n in zip(context, counts)], dtype=torch.int32,
                                device=cuda),
            "starts": torch.tensor(starts, dtype=torch.int32, device=cuda), "mask": mask,
            "scale": dim ** -0.5}


def run(s):
    return svllm_ops.tree_attention(s["q"], s["k"], s["v"], s["tables"], s["seq"], s["starts"],
                                    s["mask"], s["scale"])


def reference(s):
    return attention_reference(s["q"], s["k"], s["v"], s["tables"].tolist(), s["seq"].tolist(),
                               s["starts"].tolist(), s["mask"], s["scale"])


def check(s, out=None):
    svllm_ops.read_device_error(0, True)
    out = run(s) if out is None else out
    torch.cuda.synchronize()
    assert svllm_ops.read_device_error(0, True) == 0
    ref, size = reference(s)
    assert ((out.double() - ref).abs() <= attention_bound(ref, size, torch.bfloat16)).all()


@pytest.mark.parametrize("counts, context, heads, kv_heads, dim, bs, shape", [
    ([8], [120], 16, 8, 128, 16, "tree"),
    ([1], [127], 2, 2, 128, 16, "tree"),            # a length of exactly one tile of 128 rows
    ([1], [128], 2, 2, 128, 16, "tree"),            # and one past it
    ([64], [64], 2, 1, 64, 16, "tree"),             # 128 query rows per KV head
    ([65], [63], 2, 1, 64, 16, "tree"),             # 130
    ([128], [400], 2, 1, 128, 16, "tree"),          # 256
    ([129, 3], [400, 200], 2, 1, 128, 16, "tree"),  # 258
    ([200], [900], 5, 1, 128, 16, "tree"),          # 1000 query rows, odd grouping
    ([1024], [100], 1, 1, 64, 16, "tree"),          # the widest mask
    ([31, 1, 0, 64, 17], [5000, 3, 70, 0, 1024], 28, 4, 128, 16, "tree"),
    ([7] * 33, [50 * s for s in range(33)], 16, 8, 128, 16, "tree"),
    ([16] * 9, [611] * 9, 32, 8, 64, 64, "tree"),
    ([3], [20000], 16, 8, 128, 16, "tree"),         # one long request over the whole GPU
    ([40], [9000], 8, 1, 128, 256, "tree"),         # a single KV head
    ([37, 9], [777, 130], 20, 4, 128, 12, "tree"),  # pages that end inside a tile
    ([37, 9], [777, 130], 6, 2, 64, 1, "tree"),
    ([12, 12], [301, 40], 3, 3, 64, 3, "tree"),
    ([5] * 32, [64 * s for s in range(32)], 32, 8, 64, 16, "chain"),
    ([300, 1, 90], [1000, 250, 0], 4, 2, 128, 16, "chain"),
    ([2000], [0], 2, 1, 64, 16, "chain"),           # a causal prompt
    ([9], [200], 16, 8, 128, 16, "tree"),           # tables of two tiles: items stay whole
    ([130, 2, 0, 33], [110, 0, 7, 215], 6, 3, 64, 16, "tree"),
    ([8] * 40, [11 * s for s in range(40)], 16, 8, 128, 16, "tree"),  # of four, enough for all
    ([40, 7, 99] * 11, [400, 0, 313] * 11, 21, 3, 128, 12, "tree"),
    ([6] * 60, [7 * s for s in range(60)], 9, 9, 64, 32, "chain"),
], ids=str)
def test_matches_the_definition(cuda, counts, context, heads, kv_heads, dim, bs, shape):
    check(build(cuda, counts, context, heads, kv_heads, dim, bs, shape=shape,
                seed=sum(counts) + sum(context)))


def test_the_same_inputs_give_the_same_bits(cuda):
    s = build(cuda, [33, 64, 9], [4000, 100, 2500], 16, 8, 128, 16)
    first = run(s)
    for _ in range(3):
        assert torch.equal(run(s), first)


def test_rows_that_see_nothing_are_zero(cuda):
    """Empty masks with nothing cached, requests that were not served, padding rows."""
    s = build(cuda, [5, 4, 6], [0, 30, 300], 16, 8, 128, 16, pad=3)
    s["mask"][2] = 0
    s["seq"][1] = 0
    out = run(s)
    check(s, out)
    assert (out[2] == 0).all() and (out[5:9] == 0).all() and (out[15:] == 0).all()
    assert (out[3] != 0).any() and (out[9:15] != 0).any()
    # a batch without requests, and one whose requests have no token
    none = dict(s, tables=s["tables"][:0], seq=s["seq"][:0], starts=s["starts"][:1])
    assert (run(none) == 0).all()
    idle = dict(s, starts=torch.zeros_like(s["starts"]))
    idle["seq"] = torch.tensor([0, 30, 300], dtype=torch.int32, device=cuda)
    assert (run(idle) == 0).all()


@pytest.mark.parametrize("counts, context, heads, kv_heads, dim", [
    ([9, 70], [20, 300], 16, 8, 128),
    ([140], [1000], 8, 2, 64),
], ids=str)
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")], ids=str)
def test_masked_values_do_not_leak(cuda, counts, context, heads, kv_heads, dim, bad):
    """K and V of a node that is NaN or infinite reach only the nodes that see it; rows of a page
    behind the request's length reach nobody."""
    s = build(cuda, counts, context, heads, kv_heads, dim, 16, spare=1)
    clean = run(s)
    last = len(counts) - 1
    n, ctx = counts[last], context[last]
    first = s["starts"][last].item()
    node = 3
    row = ctx + node
    table = s["tables"][last].tolist()
    sees = ((s["mask"][first: first + n, 0] >> node) & 1).bool()
    assert sees.any() and not sees.all()
    for which in ("k", "v"):
        t = dict(s)
        t[which] = s[which].clone()
        t[which][table[row // 16], row % 16, :, 1] = bad
        end = ctx + n
        if end % 16:  # the rest of the last page
            t[which][table[end // 16], end % 16:] = bad
        out = run(t)
        blind = torch.ones(out.shape[0], dtype=torch.bool, device=cuda)
        blind[first: first + n] = ~sees
        assert torch.equal(out[blind], clean[blind])
        if which == "v":
            assert torch.equal(out[~blind][..., 2:], clean[~blind][..., 2:])
            got = out[~blind][..., 1]
            assert (got.isnan() if bad != bad else got == bad).all()
        elif bad != bad:
            assert out[~blind].isnan().all()


def test_large_scores_and_a_row_that_outweighs_the_rest(cuda):
    """Scores far apart and rising along the context: the running maximum moves in every tile, and
    the early rows' weights underflow against the last ones'."""
    s = build(cuda, [20], [1500], 8, 2, 128, 16)
    flat = torch.zeros_like(s["k"])
    table = s["tables"][0].long()
    j = torch.arange(1520, device=cuda)
    rows = table[j // 16] * 16 + j % 16
    ramp = (j.float() / 8)[:, None, None] * torch.ones(1, 2, 128, device=cuda)
    flat.view(-1, 2, 128)[rows] = ramp.bfloat16()
    s["k"] = flat
    s["q"] = torch.ones_like(s["q"])
    check(s)
    s["q"] = -s["q"]  # falling
    check(s)


def test_tables_past_int32_offsets(cuda):
    """Pages beyond 2^31 elements of the cache."""
    dim, kv, bs, blocks = 128, 8, 16, 140_000  # 2.3e9 elements
    free, _ = torch.cuda.mem_get_info()
    if free < 4 * blocks * bs * kv * dim + (4 << 30):
        pytest.skip("needs 14 GB of free device memory")
    s = build(cuda, [10, 3], [200, 90], 16, kv, dim, bs)
    small_k, small_v, small = s["k"], s["v"], s["tables"].clone()
    want = run(s)
    s["k"] = torch.zeros(blocks, bs, kv, dim, dtype=torch.bfloat16, device=cuda)
    s["v"] = torch.zeros_like(s["k"])
    shift = blocks - small_k.shape[0]
    s["k"][shift:] = small_k
    s["v"][shift:] = small_v
    s["tables"] = small + shift
    assert torch.equal(run(s), want)


def test_bad_lengths_and_blocks_raise_the_error_word(cuda):
    s = build(cuda, [4, 4, 4, 4], [30, 30, 30, 30], 16, 8, 128, 16)
    good = run(s)
    svllm_ops.read_device_error(0, True)
    s["seq"][0] = 3                                  # fewer rows than nodes
    s["seq"][1] = s["tables"].shape[1] * 16 + 1      # past the table
    s["tables"][2, 1] = s["k"].shape[0]              # a block outside the cache: block 0 is read
    out = run(s)
    torch.cuda.synchronize()
    assert svllm_ops.read_device_error(0, True) == 1
    assert (out[:8] == 0).all() and torch.equal(out[12:], good[12:])
    s["tables"][2, 1] = 0
    assert torch.equal(run(s)[8:12], out[8:12])
    # starts that fall: that request gets nothing, the device word says so
    s = build(cuda, [4, 4, 4], [30, 30, 30], 16, 8, 128, 16)
    svllm_ops.read_device_error(0, True)
    s["starts"] = torch.tensor([0, 4, 3, 40], dtype=torch.int32, device=cuda)
    run(s)
    torch.cuda.synchronize()
    assert svllm_ops.read_device_error(0, True) == 1


def test_requests_that_overlap_do_no_more_than_they_could(cuda):
    """Starts that rise and fall 10000 times: 10000 requests of the same 4096 tokens over 32768
    rows, 262144 steps each. Counted in 32 bits their sum would wrap; nothing of them runs."""
    requests, tokens, bs = 20001, 4096, 32768
    q = torch.ones(tokens, 64, 64, dtype=torch.bfloat16, device=cuda)
    cache = torch.ones(1, bs, 8, 64, dtype=torch.bfloat16, device=cuda)
    starts = torch.zeros(requests + 1, dtype=torch.int32, device=cuda)
    starts[1::2] = tokens
    seq = torch.full((requests,), bs, dtype=torch.int32, device=cuda)
    tables = torch.zeros(requests, 1, dtype=torch.int32, device=cuda)
    svllm_ops.read_device_error(0, True)
    svllm_ops.tree_attention(q, cache, cache, tables, seq, starts)
    torch.cuda.synchronize()
    assert svllm_ops.read_device_error(0, True) == 1


def test_on_another_stream_and_two_at_once(cuda):
    a = build(cuda, [33, 64, 9], [4000, 100, 2500], 16, 8, 128, 16, seed=1)
    b = build(cuda, [64] * 4, [3000] * 4, 16, 8, 128, 16, seed=2)
    want = run(a), run(b)
    torch.cuda.synchronize()
    streams = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(5):
        got = []
        for s, st in zip((a, b), streams):
            with torch.cuda.stream(st):
                got.append(run(s))
        torch.cuda.synchronize()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_captured_graphs_do_not_share_a_workspace(cuda):
    """Two graphs replayed at once on two streams, their lengths changed between replays."""
    states = [build(cuda, [33, 64], [4000, 100], 16, 8, 128, 16, seed=1),
              build(cuda, [20, 64], [3000, 800], 16, 8, 128, 16, seed=2)]
    want = [run(s) for s in states]
    graphs, outs = [], []
    for s in states:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(run(s))
        graphs.append(g)
    streams = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(4):
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o, w) for o, w in zip(outs, want))
    states[0]["seq"] -= torch.tensor([1000, 10], dtype=torch.int32, device=cuda)
    graphs[0].replay()
    check(states[0], outs[0])


def test_refusals(cuda):
    s = build(cuda, [3], [5], 4, 2, 64, 16)
    with pytest.raises(RuntimeError, match="no kernel"):  # head_dim 32
        svllm_ops.tree_attention(s["q"][..., :32].contiguous(), s["k"][..., :32].contiguous(),
                                 s["v"][..., :32].contiguous(), s["tables"], s["seq"],
                                 s["starts"], s["mask"])
    with pytest.raises(RuntimeError, match="bf16"):
        svllm_ops.tree_attention(s["q"].float(), s["k"].float(), s["v"].float(), s["tables"],
                                 s["seq"], s["starts"], s["mask"])
    odd = torch.zeros(3 * 260 + 8, dtype=torch.bfloat16, device=cuda)
    with pytest.raises(RuntimeError, match="no kernel"):  # a token stride of 260
        q = odd[: 3 * 260].view(3, 260)[:, :256].view(3, 4, 64)
        svllm_ops.tree_attention(q, s["k"], s["v"], s["tables"], s["seq"], s["starts"], s["mask"])
    with pytest.raises(RuntimeError, match="no kernel"):  # not 16-byte aligned
        q = odd[4: 4 + 3 * 256].view(3, 4, 64)
        svllm_ops.tree_attention(q, s["k"], s["v"], s["tables"], s["seq"], s["starts"], s["mask"])
    with pytest.raises(RuntimeError, match="elsewhere"):
        svllm_ops.tree_attention(s["q"], s["k"], s["v"], s["tables"].cpu(), s["seq"], s["starts"],
                                 s["mask"])


@pytest.mark.parametrize("starts", [
    [2, 4, 8, 12],    # rises, but not from 0
    [0, 4, 3, 12],    # falls
    [0, 12, 4, 12],   # falls, and the requests left overlap
    [0, 4, 8, 40],    # ends past the tokens
    [-1, 4, 8, 12],
    [3],              # no request, and yet a first token
], ids=str)
@pytest.mark.parametrize("repeat", [1, 17], ids=["few", "many"])  # 3 or 51 requests
def test_starts_that_contradict_themselves_leave_nothing_unwritten(cuda, starts, repeat):
    """query_start_loc has to rise from 0 to at most the number of tokens. Where it does not the
    error word says so, and all of the output is zero: nothing of what its memory held before, and
    no row that depends on which of two requests wrote it last."""
    s = build(cuda, [4, 4, 4] * repeat, [30, 200, 30] * repeat, 16, 8, 128, 16)
    if len(starts) > 1:
        good = s["starts"].tolist()
        starts = starts[:-1] + good[3:-1] + [starts[-1] + 12 * (repeat - 1)]
    else:
        s["tables"], s["seq"] = s["tables"][:0], s["seq"][:0]
    s["starts"] = torch.tensor(starts, dtype=torch.int32, device=cuda)
    workspace = torch.empty(svllm_capi.tree_attention_workspace_bytes(128), dtype=torch.uint8,
                            device=cuda)
    for mask in (s["mask"], None):
        svllm_ops.read_device_error(0, True)
        out = torch.full(s["q"].shape, 7.0, dtype=torch.bfloat16, device=cuda)
        svllm_capi.tree_attention(out, s["q"], s["k"], s["v"], s["tables"], s["seq"], s["starts"],
                                  mask, s["scale"], workspace)
        torch.cuda.synchronize()
        assert svllm_ops.read_device_error(0, True) == 1
        assert (out == 0).all()


@pytest.mark.parametrize("counts, context, heads, kv_heads, dim, bs, shape", [
    ([8, 60], [120, 500], 16, 8, 128, 8, "tree"),      # boxes of 8 rows: two loaders
    ([37, 9, 1], [777, 130, 2], 20, 4, 128, 24, "tree"),
    ([130, 6], [300, 900], 4, 2, 64, 40, "tree"),
    ([8, 60], [120, 500], 16, 8, 128, 4, "tree"),      # of 4: four
    ([5] * 9, [100 * s for s in range(9)], 32, 8, 64, 20, "chain"),
    ([37, 9, 1], [777, 130, 2], 20, 4, 128, 1, "tree"),  # gathered rows, over several tiles
    ([130, 6], [300, 900], 8, 1, 128, 3, "tree"),
    ([200], [0], 4, 2, 128, 6, "chain"),
], ids=str)
def test_page_sizes_on_both_sides_of_each_way_to_load(cuda, counts, context, heads, kv_heads, dim,
                                                      bs, shape):
    check(build(cuda, counts, context, heads, kv_heads, dim, bs, shape=shape, seed=bs))


@pytest.mark.parametrize("bs", [1, 3, 4, 8, 12, 16])
@pytest.mark.parametrize("node", [0, 3, 30, 69, 101])  # rows that different helper warps check
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")], ids=str)
def test_masked_values_do_not_leak_from_pages_of_any_size(cuda, bs, node, bad):
    """As above, for each way to load pages and both numbers of helper warps: a V that is not
    finite in one column reaches that column of the nodes that see it and nothing else."""
    s = build(cuda, [7, 110], [20, 300], 16, 8, 128, bs, seed=node)
    clean = run(s)
    row, table = 300 + node, s["tables"][1].tolist()
    sees = ((s["mask"][7:, node // 64] >> (node % 64)) & 1).bool()
    assert sees.any() and (node == 0 or not sees.all())
    s["v"] = s["v"].clone()
    s["v"][table[row // bs], row % bs, :, 70] = bad
    if 410 % bs:  # the rest of the last page
        s["v"][table[410 // bs], 410 % bs:] = bad
    out = run(s)
    seeing = torch.zeros(117, dtype=torch.bool, device=cuda)
    seeing[7:] = sees
    assert torch.equal(out[~seeing], clean[~seeing])
    other = [d for d in range(128) if d != 70]
    assert torch.equal(out[seeing][..., other], clean[seeing][..., other])
    got = out[seeing][..., 70]
    assert (got.isnan() if bad != bad else got == bad).all()


@pytest.mark.parametrize("counts, context, heads, kv_heads, dim, bs", [
    ([8], [120], 16, 8, 128, 16),
    ([40] * 64, [200] * 64, 16, 8, 128, 16),
    ([31, 1, 0, 64, 17], [500, 3, 70, 0, 102], 28, 4, 128, 12),
    ([200, 7], [90, 300], 5, 1, 64, 1),
], ids=str)
def test_tables_wider_than_any_request(cuda, counts, context, heads, kv_heads, dim, bs):
    """A table of a fixed width, as a captured step has: what stands behind a request's pages is not
    read, and the items of short requests may be cut, which those over a fitted table are not."""
    s = build(cuda, counts, context, heads, kv_heads, dim, bs, seed=7)
    wide = torch.full((len(counts), 4096 // bs), 2 ** 31 - 1, dtype=torch.int32, device=cuda)
    for i, (n, c) in enumerate(zip(counts, context)):
        pages = -(-(n + c) // bs)
        wide[i, :pages] = s["tables"][i, :pages]
    out = run(dict(s, tables=wide))
    check(s, out)
