"""paged_causal_attn_decode_shared in float64 on the CPU, inputs for its tests, and the error that its rounding steps
allow."""

from __future__ import annotations

import math

import torch

from tests.operator_refs import half_step


def groups_of(starts, lens, B, span):
    """Per row: (positions read through another table, whose)."""
    cut, last = [], 0
    for s in starts:
        last = max(last, min(max(s, 0), B))
        cut.append(last)
    out = [(0, b) for b in range(B)]
    for g, n in enumerate(lens):
        for b in range(cut[g], cut[g + 1]):
            out[b] = (min(max(n, 0), span), cut[g])
    return out


def inputs(D, bs, dtype, Hkv, G, rows, starts, lens, own, extra_width=0, std=1.0, poison=True, index=torch.int32):
    """rows: number of sequences. own[b]: positions behind the shared ones, the new one among them (None: no
    sequence). Pages of a group's shared positions stand in all of its rows, a partly shared page as a copy; all cells
    that no row reads are NaN."""
    where = groups_of(starts, lens, rows, 1 << 30)
    total = [0 if m is None else n + m for (n, _), m in zip(where, own)]
    width = max(1, max(-(-n // bs) for n in total)) + extra_width
    need = sum(-(-n // bs) for n in total) + 2
    ids = torch.randperm(need).tolist()
    cell = torch.full([need, Hkv, 1, bs, D], float("nan") if poison else 3.0)
    kc, vc = cell.clone(), cell.clone()
    table = torch.full([rows, width], -1, dtype=torch.int64)
    for b in range(rows):
        n, lead = where[b]
        if own[b] is None:
            continue
        for j in range(-(-total[b] // bs)):
            if lead != b and (j + 1) * bs <= n and table[lead, j] >= 0:
                table[b, j] = table[lead, j]
                continue
            p = table[b, j] = ids.pop()
            lo, hi = j * bs, min((j + 1) * bs, total[b] - 1)  # the new position is written by the call
            if hi > lo:
                kc[p, :, 0, : hi - lo] = torch.randn(Hkv, hi - lo, D) * std
                vc[p, :, 0, : hi - lo] = torch.randn(Hkv, hi - lo, D)
    seq = torch.tensor([-1 if m is None else n - 1 for n, m in zip(total, own)], dtype=torch.int32)
    return {"q": (torch.randn(rows, Hkv, G, 1, D) * std).to(dtype), "k": (torch.randn(rows, Hkv, 1, 1, D) * std).to(dtype),
            "v": torch.randn(rows, Hkv, 1, 1, D).to(dtype), "kcache": kc.to(dtype), "vcache": vc.to(dtype), "seq": seq,
            "scale": torch.tensor(1.0 / math.sqrt(D)), "block_table": table.to(index), "block_size": bs,
            "group_starts": torch.tensor(starts, dtype=torch.int32), "shared_lens": torch.tensor(lens, dtype=torch.int32)}


def decode(x):
    """-> (out, bound) [B, Hkv, G, 1, D] in float64; the caches of x are written."""
    q, kc, vc, bs = x["q"], x["kcache"], x["vcache"], x["block_size"]
    B, Hkv, G, _, D = q.shape
    table = x["block_table"].long().expand(B, -1)
    span, blocks = table.shape[1] * bs, kc.shape[0]
    seq, scale = x["seq"].reshape(-1).tolist(), float(x["scale"])
    for b, n in enumerate(seq):
        if 0 <= n < span and 0 <= table[b, n // bs] < blocks and x["k"] is not None:
            p = table[b, n // bs]
            kc[p, :, 0, n % bs, :D], vc[p, :, 0, n % bs, :D] = x["k"][b, :, 0, 0], x["v"][b, :, 0, 0]
    out = torch.full([B, Hkv, G, 1, D], float("nan"), dtype=torch.float64)
    bound = torch.zeros_like(out)
    where = groups_of(x["group_starts"].tolist(), x["shared_lens"].tolist(), B, span)
    rounding = torch.finfo(q.dtype).eps / 2
    for b, n in enumerate(seq):
        L = 0 if n < 0 else min(n + 1, span)
        shared, lead = where[b] if n >= where[b][0] else (0, b)
        at = torch.arange(L)
        page = torch.where(at < shared, table[lead, at // bs], table[b, at // bs])
        at, page = at[(page >= 0) & (page < blocks)], page[(page >= 0) & (page < blocks)]
        if len(at) == 0:
            continue
        K, V = (c[page, :, 0, at % bs, :D].transpose(0, 1).double() for c in (kc, vc))  # [Hkv, T, D]
        Q = q[b, :, :, 0].double()
        p = torch.softmax(Q @ K.transpose(1, 2) * scale, dim=-1)
        e = (Q.abs() @ K.abs().transpose(1, 2) * abs(scale)).amax(-1, keepdim=True)
        o, size, T = p @ V, p @ V.abs(), len(at)
        # A probability is rounded once to the inputs' type. Its exponential is off by under 2^-20 (the function 2^-22,
        # and the parts' weights), a score by under 2^-20 of e, which moves numerator and denominator. The product is
        # summed in float32 sixteen keys at a time, each step off by a unit at most.
        inner = size * (rounding + 2.0 ** -20 + 2 * e * 2.0 ** -20 + (T / 16 + 40) * 2.0 ** -23)
        if q.dtype == torch.float16:  # below 2^-14 of the largest, half a subnormal step
            inner = inner + T * 2.0 ** -25 * V.abs().amax()
        out[b, :, :, 0] = o
        bound[b, :, :, 0] = inner + half_step(o.abs() + inner, q.dtype)
    return out, bound


ORDER = ("q", "k", "v", "kcache", "vcache", "seq", "scale", "block_table", "block_size", "group_starts", "shared_lens")


def gpu(x):
    return {n: v.cuda() if isinstance(v, torch.Tensor) and n != "scale" else v for n, v in x.items()}


def call(x):
    import torch_rbln_b200

    return torch_rbln_b200.paged_causal_attn_decode_shared(*[x[n] for n in ORDER])


def within(got, want, bound, what=""):
    got = got.double().cpu()
    assert torch.equal(torch.isnan(got), torch.isnan(want)), f"{what}: NaN where there should be none, or none where there should"
    over = ((got - want).abs() - bound).nan_to_num(0.0)
    worst = over.max().item() if over.numel() else 0.0
    assert worst <= 0.0, f"{what}: off by {worst:.3g} more than the bound allows"


def check(x, what=""):
    """One call against float64: the output within its bound, the caches to the bit."""
    y = gpu(x)
    got = call(y)
    want, bound = decode(x)
    within(got, want, bound, what)
    for n in ("kcache", "vcache"):
        assert torch.equal(y[n].cpu().view(torch.int16), x[n].view(torch.int16)), f"{what}: {n}"
    return y, got
