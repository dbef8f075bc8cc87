"""The page operators as one thread would run them, in plain Python on the CPU, and inputs for their tests."""

from __future__ import annotations

import torch


def fork(table, lengths, parents, refs, bs):
    """-> (rows, lengths) of the forks; refs (a list) is counted up."""
    span = len(table[0]) * bs if table else 0
    rows, out = [], []
    for b in parents:
        n = min(max(lengths[b], 0), span) if 0 <= b < len(table) else 0
        row = []
        for j in range(len(table[0]) if table else 0):
            p = table[b][j] if j * bs < n else -1
            if not 0 <= p < len(refs):
                p = -1
            if p >= 0:
                refs[p] += 1
            row.append(p)
        rows.append(row)
        out.append(n)
    return rows, out


def free(table, keep, refs, bs):
    for row, n in zip(table, keep):
        for j in range(len(row)):
            if j * bs >= n:
                if 0 <= row[j] < len(refs) and refs[row[j]] > 0:
                    refs[row[j]] -= 1
                row[j] = -1


def reserve(table, seq, refs, bs, new):
    """-> (granted, [(source page, target page, rows copied)])."""
    granted, moves = [], []
    unused = [p for p, n in enumerate(refs) if n <= 0]
    for row, n in zip(table, seq):
        span = len(row) * bs
        n = min(n, span)
        if n < 0:
            granted.append(0)
            continue
        end = min(n + new, span)
        good = end - n
        for j in range(n // bs, -(-end // bs) if end > n else n // bs):
            p = row[j]
            held = 0 <= p < len(refs)
            if held and refs[p] <= 1:
                continue
            if not unused:
                good = min(good, max(j * bs - n, 0))
                continue
            row[j] = unused.pop(0)
            refs[row[j]] = 1
            if held:
                refs[p] -= 1
                if n > j * bs:
                    moves.append((p, row[j], n - j * bs))
        granted.append(good)
    return granted, moves


def compact(table, refs):
    """-> (moved, live, [(source page, target page)])."""
    used = [p for p, n in enumerate(refs) if n > 0]
    live = len(used)
    holes = [p for p in range(live) if refs[p] <= 0]
    pairs = list(zip([p for p in used if p >= live], holes))
    moved = [p if n > 0 else -1 for p, n in enumerate(refs)]
    for p, h in pairs:
        refs[h], refs[p], moved[p] = refs[p], 0, h
    for row in table:
        for j, p in enumerate(row):
            if 0 <= p < len(refs) and moved[p] >= 0:
                row[j] = moved[p]
    return moved, live, pairs


def copy(caches, scales, moves):
    """(source, target, rows) in every cache [blocks, Hkv, 1, bs, D] and scales [blocks, Hkv], in place."""
    for c in caches:
        bits = c.view(torch.uint8)
        for p, h, rows in moves:
            bits[h, :, :, :rows] = bits[p, :, :, :rows]
    for s in scales:
        for p, h, _ in moves:
            s[h] = s[p]


def caches(layers, blocks, Hkv, bs, D, dtype, heads_outermost=False):
    """Random bytes: every bit pattern, NaN among them, in each layer's cache."""
    out = []
    for _ in range(layers):
        size = torch.empty([], dtype=dtype).element_size()
        shape = [Hkv, blocks, 1, bs, D * size] if heads_outermost else [blocks, Hkv, 1, bs, D * size]
        c = torch.randint(0, 256, shape, dtype=torch.uint8).view(dtype)
        out.append(c.transpose(0, 1) if heads_outermost else c)
    return out


def pool(B, width, lengths, bs, extra, dtype=torch.int32):
    """A table whose rows hold the pages of their lengths, in shuffled order, and the counts."""
    need = [-(-n // bs) for n in lengths]
    blocks = sum(need) + extra
    ids = torch.randperm(blocks).tolist()
    table = [[ids.pop() if j < need[b] else -1 for j in range(width)] for b in range(B)]
    refs = [0] * blocks
    for row in table:
        for p in row:
            if p >= 0:
                refs[p] += 1
    return table, refs
