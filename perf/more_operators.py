"""Cases, plain forms and exact values of the operators around pages that several sequences share.

Operators of a serving step in which one prompt has several continuations, measured one pass at a time:

  branch    the continuations of the last step are dropped (torch.ops.rbln_attn.paged_kv_free), sequences are forked,
            their full pages shared (paged_kv_fork), and every fork gets pages of its own for its next tokens, partly
            filled ones copied in every layer (paged_kv_reserve)
  compact   the pages in use moved to the front of the pool, in every layer, and the table after them
            (paged_kv_compact)
  attend    one new token a sequence over a paged cache in which groups of sequences share their first positions,
            which are read once for all (torch_rbln_b200.paged_causal_attn_decode_shared)

A page's count says how many table entries hold it; a page with a count of zero is free. Where `own` is false, run()
computes the operators with elementary torch operations, in 32 bits and rounded once at the end; where it is true, it
makes the calls that a user of the package makes.
"""

import math
import os
import sys

import torch

own = False

_FP8 = torch.float8_e4m3fn
_TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "fp8": _FP8}
_BYTES = {"bf16": 2, "f16": 2, "fp8": 1}


def listed():
    return [
        # two continuations of one short sequence, in the cache of one layer: the latency of the calls
        {"name": "branch one", "op": "branch", "layers": 1, "B": 1, "N": 2, "Hkv": 8, "D": 128, "bs": 16, "lo": 100,
         "hi": 100, "new": 1, "cache": "bf16"},
        # a decode step of 16 prompts with 4 continuations each, through all layers of a model
        {"name": "branch step", "op": "branch", "layers": 24, "B": 16, "N": 64, "Hkv": 8, "D": 128, "bs": 16,
         "lo": 200, "hi": 1500, "new": 1, "cache": "bf16"},
        # drafted tokens of many continuations over a quantised cache with longer pages
        {"name": "branch drafts fp8", "op": "branch", "layers": 8, "B": 40, "N": 200, "Hkv": 4, "D": 64, "bs": 64,
         "lo": 1, "hi": 900, "new": 70, "cache": "fp8"},
        # one long prompt and many continuations: the table is the work
        {"name": "branch long prompt", "op": "branch", "layers": 2, "B": 1, "N": 256, "Hkv": 2, "D": 128, "bs": 16,
         "lo": 32765, "hi": 32765, "new": 5, "cache": "f16"},
        # a small pool
        {"name": "compact small", "op": "compact", "layers": 1, "pages": 100, "live": 37, "moved": 20, "Hkv": 4,
         "D": 64, "bs": 16, "B": 5, "cache": "bf16"},
        # a quantised pool, half of it in use
        {"name": "compact fp8", "op": "compact", "layers": 12, "pages": 1500, "live": 700, "moved": 333, "Hkv": 8,
         "D": 128, "bs": 32, "B": 48, "cache": "fp8"},
        # the pool of a model after many sequences have ended
        {"name": "compact large", "op": "compact", "layers": 16, "pages": 4096, "live": 1640, "moved": 980, "Hkv": 8,
         "D": 128, "bs": 16, "B": 64, "cache": "bf16"},
        # four continuations of a short prompt: the latency of a call
        {"name": "attend four", "op": "attend", "B": 4, "groups": 1, "Hkv": 8, "G": 4, "D": 128, "bs": 16,
         "lo": 500, "hi": 500, "own_lo": 1, "own_hi": 60, "type": "bf16"},
        # a batch behind one system prompt
        {"name": "attend one prompt", "op": "attend", "B": 64, "groups": 1, "Hkv": 8, "G": 4, "D": 128, "bs": 16,
         "lo": 4096, "hi": 4096, "own_lo": 16, "own_hi": 512, "type": "bf16"},
        # several prompts of odd lengths, groups of unequal sizes
        {"name": "attend several prompts", "op": "attend", "B": 96, "groups": 6, "Hkv": 4, "G": 7, "D": 64, "bs": 32,
         "lo": 701, "hi": 6001, "own_lo": 1, "own_hi": 700, "type": "f16"},
        # many continuations of a long document
        {"name": "attend long prompt", "op": "attend", "B": 256, "groups": 1, "Hkv": 8, "G": 8, "D": 128, "bs": 16,
         "lo": 32768, "hi": 32768, "own_lo": 1, "own_hi": 1024, "type": "bf16"},
        # few rows behind a very long document, a query head for each KV head
        {"name": "attend few rows", "op": "attend", "B": 8, "groups": 1, "Hkv": 8, "G": 1, "D": 128, "bs": 64,
         "lo": 65536, "hi": 65536, "own_lo": 1, "own_hi": 100, "type": "bf16"},
    ]


def _log(rng, lo, hi):
    """A whole number of [lo, hi], spread over its logarithm."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["branch", "compact", "attend", "attend"])
    D = rng.choice([64, 128])
    bs = rng.choice([8, 16, 16, 32, 64, 128])
    Hkv = rng.choice([1, 2, 4, 8])
    if op == "attend":
        G = rng.choice([1, 2, 4, 5, 7, 8, 16])
        groups = _log(rng, 1, 8)
        hi = _log(rng, 16, 65536)
        most = min(256, 5 * 10 ** 8 // (Hkv * G * hi))
        B = max(groups, _log(rng, 1, max(1, most)))
        return {"op": op, "B": B, "groups": groups, "Hkv": Hkv, "G": G, "D": D, "bs": bs,
                "lo": _log(rng, 1, hi), "hi": hi, "own_lo": 1, "own_hi": _log(rng, 2, 1000),
                "type": rng.choice(["bf16", "bf16", "f16"])}
    layers = _log(rng, 1, 24)
    cache = rng.choice(["bf16", "f16", "fp8"])
    most = 4 * 10 ** 9 // (layers * Hkv * bs * D * 4)  # pages of the pool
    if op == "compact":
        pages = _log(rng, 20, max(20, min(4096, most)))
        live = rng.randint(pages // 8, pages - pages // 8)
        return {"op": op, "layers": layers, "pages": pages, "live": live,
                "moved": rng.randint(0, min(live, pages - live)), "Hkv": Hkv, "D": D, "bs": bs,
                "B": _log(rng, 1, 64), "cache": cache}
    B = _log(rng, 1, 64)
    new = _log(rng, 1, 100)
    N = _log(rng, 1, 256)
    room = max(bs, (most - 2 * N * (new // bs + 2)) * bs // (2 * B))
    hi = _log(rng, 2, min(32768, max(2, room)))
    return {"op": op, "layers": layers, "B": B, "N": N, "Hkv": Hkv, "D": D, "bs": bs, "lo": rng.randint(1, hi),
            "hi": hi, "new": new, "cache": cache}


# ---------------------------------------------------------------------------------------------------------- inputs


def _spread(n, lo, hi):
    """n whole numbers evenly spread over [lo, hi]: the same for every seed."""
    return [lo + (hi - lo) * (2 * i + 1) // (2 * n) for i in range(n)]


def _sizes(B, groups):
    """B rows in groups of unequal sizes, one row at least each."""
    rest = B - groups
    total = groups * (groups + 1) // 2
    sizes = [1 + rest * (i + 1) // total for i in range(groups)]
    sizes[-1] += B - sum(sizes)
    return sizes


def _pools(gen, layers, pages, Hkv, bs, D, kind, std, device):
    """The caches of all layers [layers, pages, Hkv, 1, bs, D] as a model fills them: normal values of a size of its
    own in each head and channel, and the scales of a quantised one."""
    out = torch.empty([layers, pages, Hkv, 1, bs, D], dtype=_TYPES[kind], device=device)
    scales = torch.empty([layers, pages, Hkv], device=device) if kind == "fp8" else None
    for i in range(layers):
        x = torch.randn([pages, Hkv, 1, bs, D], generator=gen, device=device)
        x *= torch.exp(0.3 * torch.randn([1, Hkv, 1, 1, D], generator=gen, device=device)) * std
        if kind == "fp8":
            scales[i] = x.abs().amax(dim=(2, 3, 4)).clamp_min(1e-6) / 448.0
            x = (x / scales[i][:, :, None, None, None]).clamp(-448, 448)
        out[i] = x.to(_TYPES[kind])
    return out, scales


def _pages(case):
    """Pages that a branch case's parents hold and that its forks need, at most."""
    bs = case["bs"]
    held = [-(-n // bs) for n in _spread(case["B"], case["lo"], case["hi"])]
    return held, case["N"] * ((case["new"] - 1) // bs + 2)


def prepare(case, seed):
    dev = torch.device("cuda" if torch.cuda.is_available() else "cpu")
    gen = torch.Generator(device=dev).manual_seed(int(seed))
    op, bs, Hkv, D = (case[n] for n in ("op", "bs", "Hkv", "D"))
    s = {"case": case}
    if own:
        _package()

    def shuffled(n):
        return torch.randperm(n, generator=gen, device=dev).to(torch.int32)

    if op == "branch":
        B, N, new = case["B"], case["N"], case["new"]
        held, needed = _pages(case)
        lens = _spread(B, case["lo"], case["hi"])
        width = (max(lens) + new - 1) // bs + 1
        pages = sum(held) + needed + 7
        ids = shuffled(pages)
        s["table"] = torch.full([B, width], -1, dtype=torch.int32, device=dev)
        s["refs"] = torch.zeros([pages], dtype=torch.int32, device=dev)
        at = 0
        for b, n in enumerate(held):
            s["table"][b, :n] = ids[at: at + n]
            at += n
        s["refs"][ids[:at].long()] = 1
        s["seq"] = torch.tensor(lens, dtype=torch.int32, device=dev)
        s["parents"] = torch.randint(0, B, [N], generator=gen, device=dev, dtype=torch.int32)
        s["none"] = torch.zeros([N], dtype=torch.int32, device=dev)
        # the step before left its own continuations behind
        before = torch.randint(0, B, [N], generator=gen, device=dev, dtype=torch.int32)
        s["held"], length = _fork(s["table"], s["seq"], before, s["refs"], bs)
        _reserve([], s["held"], length, s["refs"], bs, new)
        _layers(s, gen, case["layers"], pages, dev)
        return s
    if op == "compact":
        B, pages, live, moved = (case[n] for n in ("B", "pages", "live", "moved"))
        used = torch.cat([shuffled(live)[: live - moved], live + shuffled(pages - live)[:moved]])
        used = used[shuffled(live).long()]
        # every page in use stands in the table once, some twice
        width = -(-live // B) + 3
        flat = torch.full([B * width], -1, dtype=torch.int32, device=dev)
        flat[:live] = used
        more = min(live // 4, B * width - live)
        flat[live: live + more] = used[:more]
        s["table"] = flat[shuffled(B * width).long()].reshape(B, width)
        s["refs"] = torch.zeros([pages], dtype=torch.int32, device=dev)
        s["refs"][used.long()] = 1
        s["refs"][used[:more].long()] = 2
        _layers(s, gen, case["layers"], pages, dev)
        return s
    B, G, kind = case["B"], case["G"], _TYPES[case["type"]]
    sizes = _sizes(B, case["groups"])
    shared = _spread(case["groups"], case["lo"], case["hi"])
    row_shared = [n for n, size in zip(shared, sizes) for _ in range(size)]
    own_lens = torch.tensor(_spread(B, case["own_lo"], case["own_hi"]))
    own_lens = own_lens[torch.randperm(B, generator=torch.Generator().manual_seed(int(seed)))].tolist()
    last = [n + m for n, m in zip(row_shared, own_lens)]  # positions, the new one among them
    width = -(-(max(shared) + max(own_lens)) // bs)
    full = [n // bs for n in shared]
    pages = sum(full) + sum(-(-n // bs) + 1 for n in own_lens) + 3  # the same number for every seed
    ids = shuffled(pages)
    s["kc"], _ = _pools(gen, 1, pages, Hkv, bs, D, case["type"], 1.0, dev)
    s["vc"], _ = _pools(gen, 1, pages, Hkv, bs, D, case["type"], 0.5, dev)
    s["kc"], s["vc"] = s["kc"][0], s["vc"][0]
    s["table"] = torch.full([B, width], -1, dtype=torch.int32, device=dev)
    at = b = 0
    for n, size in zip(shared, sizes):
        first = b
        common = ids[at: at + n // bs]
        at += n // bs
        for b in range(first, first + size):
            mine = -(-last[b] // bs) - n // bs
            s["table"][b, : n // bs] = common
            s["table"][b, n // bs: n // bs + mine] = ids[at: at + mine]
            at += mine
            if n % bs and b > first:  # a fork holds a copy of the page that the prompt ends in
                for c in (s["kc"], s["vc"]):
                    c[s["table"][b, n // bs], :, :, : n % bs] = c[s["table"][first, n // bs], :, :, : n % bs]
        b = first + size
    s["seq"] = torch.tensor([n - 1 for n in last], dtype=torch.int32, device=dev)
    s["starts"] = torch.tensor([sum(sizes[:i]) for i in range(len(sizes) + 1)], dtype=torch.int32, device=dev)
    s["shared"] = torch.tensor(shared, dtype=torch.int32, device=dev)
    s["row_shared"] = torch.tensor(row_shared, device=dev)
    s["groups"] = [(sum(sizes[:i]), sizes[i], shared[i]) for i in range(len(sizes))]
    s["own_pages"] = max(-(-n // bs) - m // bs for n, m in zip(last, row_shared))
    s["q"] = torch.randn([B, Hkv, G, 1, D], generator=gen, device=dev).to(kind)
    s["k"] = torch.randn([B, Hkv, 1, 1, D], generator=gen, device=dev).to(kind)
    s["v"] = (torch.randn([B, Hkv, 1, 1, D], generator=gen, device=dev) * 0.5).to(kind)
    s["scale"] = torch.tensor(1.0 / math.sqrt(D))
    return s


def _layers(s, gen, layers, pages, dev):
    """The caches of all layers, and a view of each as a program passes them."""
    case = s["case"]
    for name, std in (("k", 1.0), ("v", 0.5)):
        pool, scales = _pools(gen, layers, pages, case["Hkv"], case["bs"], case["D"], case["cache"], std, dev)
        s[name], s[name + "_scale"] = pool, scales
        s[name + "_list"] = list(pool.unbind(0))
        s[name + "_scale_list"] = None if scales is None else list(scales.unbind(0))


# ------------------------------------------------------------------------------------------------------ plain forms


def _count(refs, ids, valid, by):
    """refs[ids] += by where valid."""
    n = refs.numel()
    more = torch.zeros([n + 1], dtype=refs.dtype, device=refs.device)
    at = torch.where(valid, ids, torch.full_like(ids, n)).long().reshape(-1)
    more.scatter_add_(0, at, torch.full_like(at, by, dtype=refs.dtype))
    refs += more[:n]


def _inside(ids, refs):
    return (ids >= 0) & (ids < refs.numel())


def _fork(table, lengths, parents, refs, bs):
    B, width = table.shape
    known = (parents >= 0) & (parents < B)
    at = parents.clamp(0, B - 1).long()
    length = torch.where(known, lengths[at].clamp(0, width * bs), torch.zeros_like(lengths[at]))
    rows = table[at]
    valid = (torch.arange(width, device=table.device) * bs < length[:, None]) & _inside(rows, refs)
    _count(refs, rows, valid, 1)
    return torch.where(valid, rows, torch.full_like(rows, -1)), length


def _free(table, keep, refs, bs):
    gone = torch.arange(table.shape[1], device=table.device) * bs >= keep[:, None]
    _count(refs, table, gone & _inside(table, refs), -1)
    refs.clamp_min_(0)
    table.masked_fill_(gone, -1)


def _reserve(caches, table, seq, refs, bs, new):
    """caches: the caches [layers, pages, Hkv, 1, bs, D] and scales [layers, pages, Hkv] of all layers."""
    B, width = table.shape
    dev = table.device
    slots = (new - 1) // bs + 2
    seq = seq.long()
    end = (seq + new).clamp_max(width * bs)
    j = (seq // bs)[:, None] + torch.arange(slots, device=dev)
    want = (j * bs < end[:, None]) & (seq >= 0)[:, None]
    j = j.clamp(0, width - 1)
    page = table.gather(1, j)
    valid = want & _inside(page, refs)
    flat = torch.where(valid, page, torch.full_like(page, refs.numel())).long().reshape(-1)
    order = torch.arange(flat.numel(), device=dev)
    count = torch.cat([refs, refs.new_zeros([1])])[flat]
    here = torch.zeros([refs.numel() + 1], dtype=torch.int64, device=dev)
    last = here.clone()
    here.scatter_add_(0, flat, torch.ones_like(flat))
    last.scatter_reduce_(0, flat, order, "amax")
    # of a page that only this call's entries hold, the last one keeps it
    keeps = (here[flat] >= count) & (last[flat] == order)
    shared = valid.reshape(-1) & (count > 1) & ~keeps
    need = (want & ~valid).reshape(-1) | shared
    unused, at = torch.sort((refs > 0).to(torch.int8), stable=True)
    rank = torch.cumsum(need.long(), 0) - 1
    got = need & (rank < (unused == 0).sum())
    fresh = at[rank.clamp(0, at.numel() - 1)].to(table.dtype).reshape(B, slots)
    got = got.reshape(B, slots)
    moved = got & shared.reshape(B, slots)
    copied = moved & (j * bs < seq[:, None])
    b, i = copied.nonzero(as_tuple=True)
    src, dst = page[b, i].long(), fresh[b, i].long()
    held = torch.arange(bs, device=dev) < (seq % bs)[b][:, None]
    for cache in caches:
        for layer in cache:
            if layer.dim() == 2:
                layer[dst] = layer[src]
            else:
                bits = layer.view(torch.uint8)
                bits[dst] = torch.where(held[:, None, None, :, None], bits[src], bits[dst])
    _count(refs, page, moved, -1)
    _count(refs, fresh, got, 1)
    page = torch.where(got, fresh, page)
    wide = torch.cat([table, table.new_zeros([B, 1])], dim=1)
    wide.scatter_(1, torch.where(want, j, torch.full_like(j, width)), page)
    table.copy_(wide[:, :width])
    # an entry may be written when nothing else holds its page
    good = want & _inside(page, refs) & (refs[page.clamp(0, refs.numel() - 1).long()] <= 1)
    first = torch.where(want & ~good, j * bs, torch.full_like(j, width * bs)).amin(1)
    granted = torch.minimum(first, end) - seq
    return torch.where(seq >= 0, granted.clamp_min(0), torch.zeros_like(granted)).to(torch.int32)


def _compact(caches, table, refs):
    pages = refs.numel()
    used = refs > 0
    live = used.sum()
    at = torch.arange(pages, device=refs.device)
    src = (used & (at >= live)).nonzero()[:, 0]
    dst = (~used & (at < live)).nonzero()[:, 0]
    moved = torch.where(used, at, torch.full_like(at, -1)).to(torch.int32)
    moved[src] = dst.to(torch.int32)
    for cache in caches:
        for layer in cache:
            bits = layer.view(torch.uint8)
            bits[dst] = bits[src]
    refs[dst] = refs[src]
    refs[src] = 0
    now = moved[table.clamp(0, pages - 1).long()]
    table.copy_(torch.where(_inside(table, refs) & (now >= 0), now, table))
    return moved, live.to(torch.int32).reshape(1)


def _attend(s):
    case = s["case"]
    bs, D = case["bs"], case["D"]
    B, Hkv, G = s["q"].shape[:3]
    dev = s["q"].device
    seq, table = s["seq"].long(), s["table"].long()
    page = table.gather(1, (seq // bs)[:, None])[:, 0]
    s["kc"][page, :, 0, seq % bs] = s["k"][:, :, 0, 0]
    s["vc"][page, :, 0, seq % bs] = s["v"][:, :, 0, 0]
    q = s["q"][:, :, :, 0].float() * s["scale"].item()
    j = (s["row_shared"] // bs)[:, None] + torch.arange(s["own_pages"], device=dev)
    pages = table.gather(1, j.clamp_max(table.shape[1] - 1)).clamp_min(0)

    def rows(cache, ids):  # [.., Hkv, tokens, D] in 32 bits
        x = cache[ids][..., 0, :, :].transpose(-4, -3)
        return x.reshape(*x.shape[:-3], -1, D).float()

    at = (j[:, :, None] * bs + torch.arange(bs, device=dev)).reshape(B, -1)
    seen = (at >= s["row_shared"][:, None]) & (at <= seq[:, None])
    score = (q @ rows(s["kc"], pages).transpose(-1, -2)).masked_fill_(~seen[:, None, None], -math.inf)
    most = score.amax(dim=-1, keepdim=True)
    p = torch.exp(score - most)
    total, out = p.sum(dim=-1, keepdim=True), p @ rows(s["vc"], pages)
    for first, size, n in s["groups"]:
        ids = table[first, : -(-n // bs)]
        mine = q[first: first + size].transpose(0, 1).reshape(Hkv, size * G, D)

        def back(x):
            return x.reshape(Hkv, size, G, -1).transpose(0, 1)

        score = mine @ rows(s["kc"], ids)[:, :n].transpose(-1, -2)
        top = score.amax(dim=-1, keepdim=True)
        score = score.sub_(top).exp_()
        part, value = back(score.sum(dim=-1, keepdim=True)), back(score @ rows(s["vc"], ids)[:, :n])
        top = back(top)
        this = slice(first, first + size)
        now = torch.maximum(most[this], top)
        a, c = torch.exp(most[this] - now), torch.exp(top - now)
        total[this] = total[this] * a + part * c
        out[this] = out[this] * a + value * c
    return (out / total).to(s["q"].dtype)[:, :, :, None]


def _package():
    at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "torch-rbln_b200")
    if at not in sys.path:
        sys.path.insert(0, at)
    import torch_rbln_b200

    return torch_rbln_b200


def _held(s):
    return [x for x in (s["k"], s["v"], s["k_scale"], s["v_scale"]) if x is not None]


def run(state):
    s, case = state, state["case"]
    op, bs = case["op"], case["bs"]
    if op == "branch":
        if own:
            ops = torch.ops.rbln_attn
            ops.paged_kv_free(s["held"], s["none"], s["refs"], bs)
            table, length = ops.paged_kv_fork(s["table"], s["seq"], s["parents"], s["refs"], bs)
            granted = ops.paged_kv_reserve(s["k_list"], s["v_list"], table, length, s["refs"], bs, case["new"],
                                           s["k_scale_list"], s["v_scale_list"])
        else:
            _free(s["held"], s["none"], s["refs"], bs)
            table, length = _fork(s["table"], s["seq"], s["parents"], s["refs"], bs)
            granted = _reserve(_held(s), table, length, s["refs"], bs, case["new"])
        s["held"] = table  # the next pass drops them
        return [table, length, granted, s["refs"]] + _held(s)
    if op == "compact":
        table, refs = s["table"].clone(), s["refs"].clone()  # so that every pass has the same pages to move
        if own:
            moved, live = torch.ops.rbln_attn.paged_kv_compact(s["k_list"], s["v_list"], table, refs,
                                                               s["k_scale_list"], s["v_scale_list"])
        else:
            moved, live = _compact(_held(s), table, refs)
        return [table, refs, moved, live] + _held(s)
    if own:
        out = _package().paged_causal_attn_decode_shared(s["q"], s["k"], s["v"], s["kc"], s["vc"], s["seq"],
                                                         s["scale"], s["table"], bs, s["starts"], s["shared"])
    else:
        out = _attend(s)
    return [out, s["kc"], s["vc"]]


# ------------------------------------------------------------------------------------------------------------- work


def work(case):
    op, bs, Hkv, D = (case[n] for n in ("op", "bs", "Hkv", "D"))
    if op == "attend":
        size = _BYTES[case["type"]]
        B, G = case["B"], case["G"]
        sizes = _sizes(B, case["groups"])
        shared = _spread(case["groups"], case["lo"], case["hi"])
        mine = sum(_spread(B, case["own_lo"], case["own_hi"]))
        cached = (sum(shared) + mine - B) * Hkv * 2 * D * size
        new = B * Hkv * D * size * (2 * G + 4)  # queries, output, the new rows read and written
        table = 4 * (sum(-(-n // bs) for n in shared) + -(-mine // bs)) + 8 * B
        pairs = sum(n * m for n, m in zip(shared, sizes)) + mine
        return {"bytes": cached + new + table, "flops": 4 * Hkv * G * D * pairs}
    cell = _BYTES[case["cache"]]
    layers = case["layers"]
    if op == "compact":
        page = layers * 2 * Hkv * (bs * D * cell + 4 * (cell == 1))
        entries = case["B"] * (-(-case["live"] // case["B"]) + 3)
        return {"bytes": 2 * case["moved"] * page + 12 * case["pages"] + 8 * entries, "flops": 0}
    B, N = case["B"], case["N"]
    lens = _spread(B, case["lo"], case["hi"])
    # on average: a fork holds its parent's pages, and has a copy of the rows in the last one
    row = layers * 2 * Hkv * D * cell
    held = sum(n % bs for n in lens) / B
    part = sum(n % bs > 0 for n in lens) / B
    copied = N * (held * row + part * layers * 2 * Hkv * 4 * (cell == 1))
    width = (max(lens) + case["new"] - 1) // bs + 1
    # the tables: the parents' read, the dropped forks' read and cleared, the new ones written; the counts both ways
    tables = 4 * width * (B + 3 * N) + 8 * (sum(_pages(case)[0]) + _pages(case)[1]) + 8 * N
    return {"bytes": int(2 * copied + tables), "flops": 0}


# ------------------------------------------------------------------------------------------------------------ exact


def exact(case, seed):
    s = prepare(case, seed)
    op, bs = case["op"], case["bs"]
    if op == "branch":
        return _exact_branch(s, case, bs)
    if op == "compact":
        table, refs = s["table"].tolist(), s["refs"].tolist()
        used = [p for p, n in enumerate(refs) if n > 0]
        live = len(used)
        holes = (p for p in range(live) if refs[p] <= 0)
        goes = {p: p if p < live else next(holes) for p in used}
        pairs = [(p, h) for p, h in goes.items() if p != h]
        for p, h in pairs:
            refs[h], refs[p] = refs[p], 0
        if pairs:
            src, dst = (torch.tensor(x, device=s["k"].device) for x in zip(*pairs))
            for pool in _held(s):
                bits = pool.view(torch.uint8)
                bits[:, dst] = bits[:, src]
        table = [[goes.get(p, p) for p in row] for row in table]
        moved = [goes.get(p, -1) for p in range(len(refs))]
        return [torch.tensor(x, dtype=torch.int32) for x in (table, refs, moved, [live])] + _held(s)
    B, Hkv, G, _, D = s["q"].shape
    kc, vc = s["kc"].double(), s["vc"].double()
    for b, n in enumerate(s["seq"].tolist()):
        p = int(s["table"][b, n // bs])
        kc[p, :, 0, n % bs], vc[p, :, 0, n % bs] = s["k"][b, :, 0, 0].double(), s["v"][b, :, 0, 0].double()
    out = torch.empty([B, Hkv, G, 1, D], dtype=torch.float64, device=kc.device)
    seq = s["seq"].tolist()

    def rows(cache, b, lo, hi):
        x = cache[s["table"][b, lo // bs: -(-hi // bs)].long()][:, :, 0].transpose(0, 1).reshape(Hkv, -1, D)
        return x[:, lo - lo // bs * bs:][:, : hi - lo]

    for first, size, n in s["groups"]:
        K, V = rows(kc, first, 0, n), rows(vc, first, 0, n)
        for b in range(first, first + size):
            q = s["q"][b, :, :, 0].double() * float(s["scale"])
            score = torch.cat([torch.einsum("hgd,htd->hgt", q, x) for x in (K, rows(kc, b, n, seq[b] + 1))], dim=-1)
            p = torch.softmax(score, dim=-1)
            out[b, :, :, 0] = (torch.einsum("hgt,htd->hgd", p[..., :n], V)
                               + torch.einsum("hgt,htd->hgd", p[..., n:], rows(vc, b, n, seq[b] + 1)))
    return [out, kc, vc]


def _exact_branch(s, case, bs):
    """One entry after the other, as the operators are defined."""
    refs, new = s["refs"].tolist(), case["new"]
    for row in s["held"].tolist():
        for p in row:
            if p >= 0:
                refs[p] -= 1
    seq, parent = s["seq"].tolist(), s["table"].tolist()
    table, length, granted, pairs = [], [], [], []
    for b in s["parents"].tolist():
        n = -(-seq[b] // bs)
        table.append(parent[b][:n] + [-1] * (len(parent[b]) - n))
        length.append(seq[b])
        for p in table[-1][:n]:
            refs[p] += 1
    unused = (p for p, n in enumerate(list(refs)) if n <= 0)
    for row, n in zip(table, length):
        for j in range(n // bs, (n + new - 1) // bs + 1):
            p = row[j]
            if p >= 0 and refs[p] == 1:
                continue
            row[j] = next(unused)
            refs[row[j]] = 1
            if p >= 0:
                refs[p] -= 1
                if n > j * bs:
                    pairs.append((p, row[j], n - j * bs))
        granted.append(new)
    for held in sorted({n for _, _, n in pairs}):
        src, dst = (torch.tensor(x, device=s["k"].device) for x in zip(*[(p, h) for p, h, n in pairs if n == held]))
        for pool in (s["k"], s["v"]):
            bits = pool.view(torch.uint8)
            bits[:, dst, :, :, :held] = bits[:, src, :, :, :held]
        for scale in (s["k_scale"], s["v_scale"]):
            if scale is not None:
                scale[:, dst] = scale[:, src]
    return [torch.tensor(x, dtype=torch.int32) for x in (table, length, granted, refs)] + _held(s)
