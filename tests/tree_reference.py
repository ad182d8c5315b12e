"""Plain implementations of the drafted-tree operators for the tests: Python loops over requests
and nodes, 64-bit arithmetic."""

from __future__ import annotations

import torch


def pack_lists(counts):
    starts = [0]
    for n in counts:
        starts.append(starts[-1] + n)
    return starts, starts[-1]


def random_parents(seed, counts, reach=5):
    """Per request a random tree: node 0 the root, node i on one of the `reach` nodes before it."""
    g = torch.Generator().manual_seed(seed)
    out = []
    for n in counts:
        for i in range(n):
            out.append(-1 if i == 0 else
                       max(0, i - 1 - int(torch.randint(0, reach, (1,), generator=g))))
    return out


def masks_of(parents, counts):
    """[T, W] int64 ancestor-or-self masks."""
    words = max(1, -(-max(counts, default=1) // 64))
    rows, at = [], 0
    for n in counts:
        seen = []
        for i in range(n):
            p = parents[at + i]
            seen.append((seen[p] if p >= 0 else 0) | (1 << i))
        for m in seen:
            row = [(m >> (64 * w)) & (2 ** 64 - 1) for w in range(words)]
            rows.append([x - 2 ** 64 if x >= 2 ** 63 else x for x in row])
        at += n
    return torch.tensor(rows, dtype=torch.int64).view(-1, words)


def make_pages(seed, counts, context, bs):
    """Random pages: tables [S][B], the number of blocks (two spare), the nodes' slots."""
    g = torch.Generator().manual_seed(seed + 1)
    need = [-(-(c + n) // bs) for c, n in zip(context, counts)]
    blocks = sum(need) + 2
    order = torch.randperm(blocks, generator=g).tolist()
    width, at = max(1, max(need, default=1)), 0
    tables, slots = [], []
    for c, n, b in zip(context, counts, need):
        table = order[at: at + b]
        at += b
        tables.append(table + [0] * (width - b))
        slots += [table[r // bs] * bs + r % bs for r in range(c, c + n)]
    return tables, blocks, slots


def plan_reference(case):
    bs = case["block_size"]
    tables = [list(r) for r in case["block_tables"]]
    stack, have = list(case["free_blocks"]), case["free_count"]
    for s, q in enumerate(case["query_lens"]):
        if q < 0:
            for b in tables[s][: case["blocks_owned"][s]]:
                stack[have] = b
                have += 1
    top, needed, used = have, 0, 0
    starts, seq, owned_out = [0], [], []
    slots, positions, masks = [], [], []
    words = -(-case["max_query_len"] // 64)
    for s, (c, q, owned) in enumerate(zip(case["context_lens"], case["query_lens"],
                                          case["blocks_owned"])):
        starts.append(starts[-1] + max(q, 0))
        need = max(0, -(-(c + q) // bs) - owned) if q > 0 else 0
        served = q >= 0 and (need == 0 or needed + need <= top)
        if served:
            for i in range(need):
                tables[s][owned + i] = stack[top - 1 - needed - i]
            used += need
        needed += need
        seq.append(c + q if served else 0)
        owned_out.append(0 if q < 0 else owned + (need if served else 0))
        bits, depths = [], []
        for i in range(max(q, 0)):
            p = i - 1 if case["parents"] is None else case["parents"][starts[s] + i]
            bits.append((bits[p] if p >= 0 else 0) | (1 << i))
            depths.append(depths[p] + 1 if p >= 0 else 0)
            row = c + i
            slots.append(tables[s][row // bs] * bs + row % bs if served else -1)
            positions.append(c + depths[i] if served else 0)
            m = bits[i] if served else 0
            row = [(m >> (64 * w)) & (2 ** 64 - 1) for w in range(words)]
            masks.append([x - 2 ** 64 if x >= 2 ** 63 else x for x in row])
    pad = case["num_tokens"] - starts[-1]
    slots += [-1] * pad
    positions += [0] * pad
    masks += [[0] * words] * pad

    def i32(x):
        return torch.tensor(x, dtype=torch.int32)

    return ({"query_start_loc": i32(starts), "seq_lens": i32(seq),
             "slot_mapping": torch.tensor(slots, dtype=torch.int64),
             "positions": torch.tensor(positions, dtype=torch.int64),
             "tree_mask": torch.tensor(masks, dtype=torch.int64).view(-1, words),
             "blocks_owned": i32(owned_out), "free_count": i32([have - used])},
            i32(tables), i32(stack))


def walk_reference(ids, targets, parents, starts, seq, context, width):
    path, tokens, counts = [], [], []
    for s in range(len(seq)):
        a, n = starts[s], starts[s + 1] - starts[s]
        nodes = []
        cur = 0 if n and seq[s] > 0 else None
        while cur is not None:
            nodes.append(cur)
            cur = next((i for i in range(cur + 1, n)
                        if (i - 1 if parents is None else parents[a + i]) == cur and
                        ids[a + i] == targets[a + cur]), None)
        path.append(nodes + [-1] * (width - len(nodes)))
        tokens.append([targets[a + i] for i in nodes] + [-1] * (width - len(nodes)))
        counts.append(len(nodes))
    return (torch.tensor(path, dtype=torch.int32), torch.tensor(tokens),
            torch.tensor(counts, dtype=torch.int32),
            torch.tensor([c + n for c, n in zip(context, counts)], dtype=torch.int32))


def attention_reference(q, k_cache, v_cache, tables, seq, starts, mask, scale):
    """The definition in 64 bits, on q's device: out [T, H, D], and sum_j p_j |v_j|, the size that
    the roundings of the p_j are relative to."""
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    size = torch.zeros_like(out)
    heads, (bs, kv, dim) = q.shape[1], k_cache.shape[1:]
    group = heads // kv
    tables = torch.as_tensor(tables, device=q.device).long()
    for s, length in enumerate(seq):
        a, b = starts[s], starts[s + 1]
        if length == 0 or a == b:
            continue
        j = torch.arange(length, device=q.device)
        rows = tables[s][j // bs] * bs + j % bs
        k = k_cache.reshape(-1, kv, dim)[rows].double()
        v = v_cache.reshape(-1, kv, dim)[rows].double()
        node = j - (length - (b - a))
        if mask is None:
            sees = node <= torch.arange(b - a, device=q.device)[:, None]
        else:
            x = node.clamp(min=0)
            sees = ((mask[a:b].to(q.device)[:, x // 64] >> (x % 64)) & 1).bool() | (node < 0)
        for h in range(heads):
            w = q[a:b, h].double() @ k[:, h // group].T * scale
            w = w.masked_fill(~sees, float("-inf"))
            p = torch.softmax(w, -1)
            p = torch.where(sees.any(-1, keepdim=True), p, 0.0)
            # a row that is not seen has no part in the sum, whatever it holds
            if torch.isfinite(v).all():
                out[a:b, h] = p @ v[:, h // group]
                size[a:b, h] = p @ v[:, h // group].abs()
            else:
                for i in range(b - a):
                    at = sees[i]
                    out[a + i, h] = p[i, at] @ v[at, h // group]
                    size[a + i, h] = p[i, at] @ v[at, h // group].abs()
    return out, size


def attention_bound(ref, size, dtype):
    """How far an output may be off: with u half a step of dtype relative to the value (2^-8 for
    bf16, 2^-24 for fp32), u of sum p |v| where the softmax numerators are rounded to dtype, u of
    the output for its own rounding, and for the fp32 arithmetic 2^-11 of sum p |v|: a score of up
    to 128 products of normal values times scale, about sqrt(128) 2^-24 |q| |k| scale off, moves
    its weight by the same relative amount (|q| |k| scale < 40: below 2^-15), the base-2 exponent's
    argument of size below 64 is rounded once more (64 * 2^-24 = 2^-18), the approximate
    exponential is 2^-22 off, and a running sum of n terms is below n 2^-24 off, 2^-11 at 8192."""
    u = torch.finfo(dtype).eps / 2
    return (u + 2.0 ** -11) * size + u * ref.abs() + 1e-30
