"""Cases, plain forms and exact values of the operators around a quantised paged KV cache.

Four operators of a serving or training step, measured one pass at a time:

  rotary    rotary positions of queries and keys [B, H, S, D], forward, or forward and gradient
            (torch.ops.rbln_attn.rotary)
  write     rotary positions of a step's queries and keys, the keys and values written into the paged cache,
            quantised where the cache is float8_e4m3fn (torch.ops.rbln_attn.rotary_paged_kv_write)
  attend    attention of S new tokens a sequence over a float8_e4m3fn paged cache with one scale for each block and
            KV head, the new rows written first (torch_rbln_b200.paged_causal_attn_prefill_kvfp8)
  read      the cache read back into dense rows (torch.ops.rbln_attn.paged_kv_read)

Where `own` is false, run() computes them with elementary torch operations in 32 bits (angles in 64), rounded once at
the end; where it is true, it makes the calls that a user of the package makes.
"""

import math
import os
import sys

import torch

own = False

_FP8 = torch.float8_e4m3fn
_TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32, "fp8": _FP8}
_BYTES = {"bf16": 2, "f16": 2, "f32": 4, "fp8": 1}


def listed():
    return [
        # one token of one sequence: the latency of a call
        {"name": "rotary one token", "op": "rotary", "B": 1, "S": 1, "H": 32, "Hkv": 8, "D": 128, "R": 128,
         "type": "bf16", "interleaved": False, "heads_first": False, "train": False, "base": 10000.0, "stretch": 1.0,
         "mscale": 1.0, "far": 4096},
        # a training step's queries and keys, as a projection leaves them ([B, S, H, D] seen as [B, H, S, D])
        {"name": "rotary training", "op": "rotary", "B": 4, "S": 4096, "H": 32, "Hkv": 8, "D": 128, "R": 128,
         "type": "bf16", "interleaved": False, "heads_first": False, "train": True, "base": 500000.0, "stretch": 1.0,
         "mscale": 1.0, "far": 0},
        # part of the head, interleaved, fp32, an odd length, positions stretched for a long context
        {"name": "rotary part of the head", "op": "rotary", "B": 3, "S": 777, "H": 12, "Hkv": 12, "D": 64, "R": 32,
         "type": "f32", "interleaved": True, "heads_first": True, "train": True, "base": 10000.0, "stretch": 8.0,
         "mscale": 1.2, "far": 1000000},
        # one decode step of a large batch
        {"name": "write decode fp8", "op": "write", "B": 256, "Hkv": 8, "G": 4, "S": 1, "D": 128, "R": 128, "bs": 16,
         "lo": 16, "hi": 500, "type": "bf16", "cache": "fp8", "interleaved": False},
        # chunked prefill, 512 new tokens for each of 8 sequences
        {"name": "write chunk fp8", "op": "write", "B": 8, "Hkv": 8, "G": 4, "S": 512, "D": 128, "R": 128, "bs": 16,
         "lo": 0, "hi": 8192, "type": "bf16", "cache": "fp8", "interleaved": False},
        # a ragged chunk into an unquantised cache, half the head rotated
        {"name": "write ragged f16", "op": "write", "B": 5, "Hkv": 4, "G": 7, "S": 333, "D": 64, "R": 32, "bs": 32,
         "lo": 0, "hi": 1000, "type": "f16", "cache": "f16", "interleaved": True},
        # four tokens a sequence: drafted tokens attended at once
        {"name": "attend 4 tokens", "op": "attend", "B": 64, "Hkv": 8, "G": 4, "S": 4, "D": 128, "bs": 16, "lo": 128,
         "hi": 4096, "type": "bf16", "both": False, "mask": False},
        # chunked prefill over 0 to 8192 cached tokens
        {"name": "attend chunk", "op": "attend", "B": 8, "Hkv": 8, "G": 4, "S": 512, "D": 128, "bs": 16, "lo": 0,
         "hi": 8192, "type": "bf16", "both": False, "mask": False},
        # few new tokens behind a long context
        {"name": "attend long context", "op": "attend", "B": 4, "Hkv": 8, "G": 8, "S": 48, "D": 128, "bs": 16,
         "lo": 16384, "hi": 32768, "type": "bf16", "both": False, "mask": False},
        # small and ragged, with a mask over positions
        {"name": "attend ragged mask", "op": "attend", "B": 3, "Hkv": 2, "G": 5, "S": 77, "D": 64, "bs": 32, "lo": 0,
         "hi": 300, "type": "f16", "both": True, "mask": True},
        # a batch of caches read back whole
        {"name": "read back fp8", "op": "read", "B": 16, "Hkv": 8, "D": 128, "bs": 16, "lo": 512, "hi": 8192,
         "cache": "fp8", "type": "bf16"},
        # one short sequence
        {"name": "read back one", "op": "read", "B": 1, "Hkv": 8, "D": 128, "bs": 16, "lo": 333, "hi": 333,
         "cache": "fp8", "type": "f16"},
    ]


def _log(rng, lo, hi):
    """A whole number of [lo, hi], spread over its logarithm."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rotary", "write", "attend", "read"])
    D = rng.choice([64, 128])
    bs = rng.choice([8, 16, 16, 32, 64, 128])
    kind = rng.choice(["bf16", "bf16", "f16"])
    if op == "rotary":
        Hkv = rng.choice([1, 2, 8, 12])
        H = Hkv * rng.choice([1, 3, 4])
        S = _log(rng, 1, 8192)
        return {"op": op, "B": _log(rng, 1, max(1, min(64, 4 * 4096 * 20 // (S * (H + Hkv))))), "S": S, "H": H,
                "Hkv": Hkv, "D": D, "R": rng.choice([D, D, D // 2, D // 4]), "type": rng.choice(["bf16", "f16", "f32"]),
                "interleaved": rng.random() < 0.5, "heads_first": rng.random() < 0.5, "train": rng.random() < 0.5,
                "base": rng.choice([10000.0, 500000.0]), "stretch": rng.choice([1.0, 4.0, 32.0]),
                "mscale": rng.choice([1.0, 1.3]), "far": _log(rng, 1, 1000000)}
    Hkv = rng.choice([1, 2, 4, 8])
    if op == "write":
        S = _log(rng, 1, 1024)
        B = _log(rng, 1, max(1, min(256, 4096 // S)))
        lo = _log(rng, 1, 200)
        return {"op": op, "B": B, "Hkv": Hkv, "G": rng.choice([1, 4, 7]), "S": S, "D": D,
                "R": rng.choice([D, D, D // 2]), "bs": bs, "lo": lo, "hi": lo + _log(rng, 1, 300), "type": kind,
                "cache": rng.choice(["fp8", "fp8", kind]), "interleaved": rng.random() < 0.5}
    if op == "read":
        lo = _log(rng, 1, 8000)
        hi = lo + _log(rng, 1, 8192 - lo + 1)
        return {"op": op, "B": _log(rng, 1, max(1, 16 * 4096 // hi)), "Hkv": Hkv, "D": D, "bs": bs, "lo": lo,
                "hi": hi, "cache": rng.choice(["fp8", kind]), "type": kind}
    G = rng.choice([1, 4, 5, 8])
    S = _log(rng, 1, 1000)
    hi = _log(rng, 16, 16384)
    most = min(64 * 2048 // (hi + S), 5 * 10 ** 8 // (Hkv * G * S * (hi + S)))
    return {"op": op, "B": _log(rng, 1, max(1, min(64, most))), "Hkv": Hkv, "G": G, "S": S, "D": D, "bs": bs,
            "lo": rng.randint(0, hi), "hi": hi, "type": kind, "both": rng.random() < 0.25, "mask": rng.random() < 0.3}


# ---------------------------------------------------------------------------------------------------------- inputs


def _lengths(case):
    """The batch's lengths, evenly spread over [lo, hi]: the same set for every seed."""
    B, lo, hi = case["B"], case["lo"], case["hi"]
    return [lo + (hi - lo) * (2 * b + 1) // (2 * B) for b in range(B)]


def _inv_freq(R, base, stretch, device):
    i = torch.arange(R // 2, dtype=torch.float64, device=device)
    return (base ** (-2.0 * i / R) / stretch).float()


def _pool(gen, blocks, Hkv, bs, D, kind, std, device):
    """A cache [blocks, Hkv, 1, bs, D] as a model fills it: normal values of a size of its own in each head, a few
    channels larger, and the scales of a quantised one."""
    x = torch.randn([blocks, Hkv, 1, bs, D], generator=gen, device=device)
    size = torch.exp(0.3 * torch.randn([1, Hkv, 1, 1, D], generator=gen, device=device)) * std
    x = x * size
    if kind != "fp8":
        return x.to(_TYPES[kind]), None
    scale = x.abs().amax(dim=(2, 3, 4)).clamp_min(1e-6) / 448.0
    return (x / scale[:, :, None, None, None]).clamp(-448, 448).to(_FP8), scale


def prepare(case, seed):
    dev = torch.device("cuda" if torch.cuda.is_available() else "cpu")
    gen = torch.Generator(device=dev).manual_seed(int(seed))
    op, kind = case["op"], _TYPES[case["type"]]
    s = {"case": case}
    if own:
        _package()

    def normal(*shape, std=1.0):
        return (torch.randn(list(shape), generator=gen, device=dev) * std).to(kind)

    if op == "rotary":
        B, S, H, Hkv, D = (case[n] for n in ("B", "S", "H", "Hkv", "D"))

        def rows(heads):
            return normal(B, heads, S, D) if case["heads_first"] else normal(B, S, heads, D).transpose(1, 2)

        s["q"], s["k"] = rows(H), rows(Hkv)
        if case["train"]:
            s["q"].requires_grad_(True), s["k"].requires_grad_(True)
            s["dq"], s["dk"] = rows(H), rows(Hkv)
        first = torch.randint(0, case["far"] + 1, [B, 1], generator=gen, device=dev)
        s["positions"] = first + torch.arange(S, device=dev)
        s["inv_freq"] = _inv_freq(case["R"], case["base"], case["stretch"], dev)
        return s
    B, Hkv, D, bs = (case[n] for n in ("B", "Hkv", "D", "bs"))
    S = case.get("S", 0)
    lens = _lengths(case)
    width = max(1, -(-(max(lens) + S) // bs))
    blocks = B * width + 3
    order = torch.randperm(B, generator=gen, device=dev)
    s["seq"] = torch.tensor(lens, dtype=torch.int32, device=dev)[order]
    s["table"] = torch.randperm(blocks, generator=gen, device=dev)[: B * width].reshape(B, width).to(torch.int32)
    cache = case.get("cache", "fp8")
    s["kc"], s["ks"] = _pool(gen, blocks, Hkv, bs, D, cache, 1.0, dev)
    s["vc"], s["vs"] = _pool(gen, blocks, Hkv, bs, D, cache, 0.5, dev)
    if op == "read":
        s["most"] = max(lens)
        return s
    G = case["G"]
    s["q"] = normal(B, Hkv, G, S, D)
    s["k"] = normal(B, Hkv, 1, S, D)
    s["v"] = normal(B, Hkv, 1, S, D, std=0.5)
    if op == "write":
        s["inv_freq"] = _inv_freq(case["R"], 10000.0, 1.0, dev)
        return s
    s["scale"] = torch.tensor(1.0 / math.sqrt(D))
    s["mask"] = None
    if case["mask"]:  # a few positions are dropped, the first never
        keep = torch.rand([B, width * bs], generator=gen, device=dev) > 0.1
        keep[:, 0] = True
        s["mask"] = keep.to(kind)
    return s


# ------------------------------------------------------------------------------------------------------ plain forms


def _cos_sin(positions, inv_freq, mscale):
    """[B, 1, S, R/2] each, in 32 bits from angles in 64."""
    angle = (positions.double()[:, :, None] * inv_freq.double())[:, None]
    return (torch.cos(angle) * mscale).float(), (torch.sin(angle) * mscale).float()


def _turn(x, cos, sin, interleaved):
    """Rows x [B, H, S, D] in 32 bits, the first R = 2 * cos.size(-1) dimensions turned."""
    R = 2 * cos.shape[-1]
    x = x.float()
    head, rest = x[..., :R], x[..., R:]
    if interleaved:
        a, b = head[..., 0::2], head[..., 1::2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], dim=-1).flatten(-2)
    else:
        a, b = head[..., : R // 2], head[..., R // 2:]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)
    return torch.cat([turned, rest], dim=-1)


def _write(cache, scales, rows, seq, table, bs):
    """rows [B, Hkv, S, D] in 32 bits written at [seq[b], seq[b] + S); a quantised cache's scales are found anew for
    the blocks that are touched."""
    B, Hkv, S, D = rows.shape
    seq, table = seq.long(), table.long()
    if scales is None:
        at = seq[:, None] + torch.arange(S, device=rows.device)
        cache[table.gather(1, at // bs), :, 0, at % bs] = rows.transpose(1, 2).to(cache.dtype)
        return
    slots = (S + bs - 1) // bs + 1
    block = (seq // bs)[:, None] + torch.arange(slots, device=rows.device)
    block = torch.minimum(block, ((seq + S - 1) // bs)[:, None])  # one past the last: the last again, alike
    phys = table.gather(1, block)
    at = block[:, :, None] * bs + torch.arange(bs, device=rows.device)  # [B, slots, bs]
    new = (at >= seq[:, None, None]) & (at < seq[:, None, None] + S)
    held = at < seq[:, None, None]
    bits = cache.view(torch.uint8)
    was = bits[phys][:, :, :, 0]  # [B, slots, Hkv, bs, D]
    old = scales[phys]  # [B, slots, Hkv]
    index = (at - seq[:, None, None]).clamp(0, S - 1).reshape(B, 1, slots * bs, 1)
    fresh = rows.gather(2, index.expand(B, Hkv, slots * bs, D)).reshape(B, Hkv, slots, bs, D).transpose(1, 2)
    new, held = new[:, :, None, :, None], held[:, :, None, :, None]
    value = torch.where(new, fresh, was.view(_FP8).float() * old[..., None, None])
    most = torch.where(new | held, value.abs(), torch.zeros_like(value)).amax(dim=(-1, -2))
    scale = most.clamp_min(1e-6) / 448.0
    codes = (value * (1.0 / scale)[..., None, None]).clamp(-448, 448).to(_FP8).view(torch.uint8)
    put = new | (held & (scale != old)[..., None, None])
    bits[phys] = torch.where(put, codes, was)[:, :, :, None]
    scales[phys] = scale


def _rows(cache, scales, table, bs):
    """The sequences' rows [B, Hkv, width * bs, D] in 32 bits."""
    table = table.long()
    if scales is None:
        x = cache[table].float()
    else:
        x = cache.view(torch.uint8)[table].view(_FP8).float() * scales[table][..., None, None, None]
    B, width, Hkv, _, _, D = x.shape
    return x[:, :, :, 0].transpose(1, 2).reshape(B, Hkv, width * bs, D)


def _attend(s):
    case = s["case"]
    S, bs = case["S"], case["bs"]
    _write(s["kc"], s["ks"], s["k"][:, :, 0].float(), s["seq"], s["table"], bs)
    _write(s["vc"], s["vs"], s["v"][:, :, 0].float(), s["seq"], s["table"], bs)
    K, V = _rows(s["kc"], s["ks"], s["table"], bs), _rows(s["vc"], s["vs"], s["table"], bs)
    B, Hkv, T, D = K.shape
    q = s["q"].float().reshape(B, Hkv, -1, D)
    score = (q @ K.transpose(-1, -2)).reshape(B, Hkv, -1, S, T) * s["scale"].item()
    t = torch.arange(T, device=q.device)
    last = s["seq"].long()[:, None] + (S - 1 if case["both"] else torch.arange(S, device=q.device))
    keep = t <= last[:, :, None] if not case["both"] else (t <= last[:, :, None]).expand(B, S, T)
    if s["mask"] is not None:
        keep = keep & (s["mask"] > 0)[:, None]
    score = score.masked_fill_(~keep[:, None, None], -math.inf)
    score = score.sub_(score.amax(dim=-1, keepdim=True)).exp_()
    total = score.sum(dim=-1, keepdim=True)
    out = (score.reshape(B, Hkv, -1, T) @ V).reshape(B, Hkv, -1, S, D) / total
    return out.to(s["q"].dtype)


def _package():
    at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "torch-rbln_b200")
    if at not in sys.path:
        sys.path.insert(0, at)
    import torch_rbln_b200

    return torch_rbln_b200


def _caches(s):
    return [s["kc"], s["vc"]] + ([] if s["ks"] is None else [s["ks"], s["vs"]])


def run(state):
    s, case = state, state["case"]
    op, bs = case["op"], case.get("bs")
    if own:
        ops = torch.ops.rbln_attn
        if op == "rotary":
            q, k = ops.rotary(s["q"], s["k"], s["positions"], s["inv_freq"], case["interleaved"], case["mscale"])
            if not case["train"]:
                return q, k
            dq, dk = torch.autograd.grad((q, k), (s["q"], s["k"]), (s["dq"], s["dk"]))
            return q, k, dq, dk
        if op == "write":
            q = ops.rotary_paged_kv_write(s["q"], s["k"], s["v"], s["kc"], s["vc"], s["seq"], s["table"], bs,
                                          s["inv_freq"], case["interleaved"], 1.0, s["ks"], s["vs"])
            return [q] + _caches(s)
        if op == "attend":
            out = _package().paged_causal_attn_prefill_kvfp8(
                s["q"], s["k"], s["v"], s["kc"], s["vc"], s["ks"], s["vs"], s["seq"], s["scale"], s["table"], bs,
                case["both"], s["mask"])
            return [out] + _caches(s)
        return ops.paged_kv_read(s["kc"], s["vc"], s["seq"], s["table"], bs, s["most"], s["ks"], s["vs"],
                                 _TYPES[case["type"]])
    if op == "rotary":
        with torch.no_grad():
            cos, sin = _cos_sin(s["positions"], s["inv_freq"], case["mscale"])
            got = [_turn(s[n], cos, sin, case["interleaved"]).to(s[n].dtype) for n in ("q", "k")]
            if case["train"]:  # the transposed map turns back
                got += [_turn(s[n], cos, -sin, case["interleaved"]).to(s[n].dtype) for n in ("dq", "dk")]
            return got
    if op == "write":
        at = s["seq"].long()[:, None] + torch.arange(case["S"], device=s["q"].device)
        cos, sin = _cos_sin(at, s["inv_freq"], 1.0)
        B, Hkv, G, S, D = s["q"].shape
        q = _turn(s["q"].reshape(B, Hkv * G, S, D), cos, sin, case["interleaved"]).to(s["q"].dtype)
        _write(s["kc"], s["ks"], _turn(s["k"][:, :, 0], cos, sin, case["interleaved"]), s["seq"], s["table"], bs)
        _write(s["vc"], s["vs"], s["v"][:, :, 0].float(), s["seq"], s["table"], bs)
        return [q.reshape(B, Hkv, G, S, D)] + _caches(s)
    if op == "attend":
        out = _attend(s)
        return [out] + _caches(s)
    got = []
    for cache, scales in ((s["kc"], s["ks"]), (s["vc"], s["vs"])):
        x = _rows(cache, scales, s["table"], bs)[:, :, : s["most"]]
        inside = torch.arange(s["most"], device=x.device) < s["seq"].long()[:, None]
        x = torch.where(inside[:, None, :, None], x, torch.zeros_like(x))
        got.append(x.to(_TYPES[case["type"]])[:, :, None])
    return tuple(got)


# ------------------------------------------------------------------------------------------------------------- work


def work(case):
    op, D = case["op"], case["D"]
    size = _BYTES[case["type"]]
    if op == "rotary":
        rows = case["B"] * case["S"] * (case["H"] + case["Hkv"])
        ways = 2 if case["train"] else 1
        return {"bytes": ways * 2 * rows * D * size + 8 * case["B"] * case["S"] + 2 * case["R"],
                "flops": ways * 3 * rows * case["R"]}
    B, Hkv = case["B"], case["Hkv"]
    lens = _lengths(case)
    cell = _BYTES[case.get("cache", "fp8")]
    bs = case["bs"]
    if op == "read":
        blocks = sum(-(-n // bs) for n in lens)
        rows = 2 * Hkv * sum(lens)
        return {"bytes": rows * D * cell + 2 * Hkv * B * max(lens) * D * size + blocks * (4 + 8 * Hkv * (cell == 1)),
                "flops": rows * D}
    S, G = case["S"], case["G"]
    new = B * S * Hkv
    touched = sum((n + S - 1) // bs - n // bs + 1 for n in lens)
    # a quantised cache's first block holds rows that set its scale too
    held = sum(n % bs for n in lens) * Hkv * 2 * D * (cell == 1)
    wrote = 2 * new * D * (size + cell) + held + touched * (4 + 16 * Hkv * (cell == 1))
    if op == "write":
        return {"bytes": wrote + 2 * new * G * D * size + 2 * case["R"], "flops": 3 * new * (G + 1) * case["R"] + 2 * new * D}
    seen = sum(n + S for n in lens)
    pairs = sum(S * (n + S) if case["both"] else S * n + S * (S + 1) // 2 for n in lens)
    cached = 2 * Hkv * sum(lens) * D + 8 * Hkv * sum(-(-n // bs) for n in lens)
    return {"bytes": wrote + cached + 2 * new * G * D * size + (seen * size if case["mask"] else 0),
            "flops": 4 * Hkv * G * D * pairs}


# ------------------------------------------------------------------------------------------------------------ exact


def _exact_turn(x, positions, inv_freq, interleaved, mscale, back=False):
    """x [B, H, S, D] turned in 64 bits, pair by pair as complex numbers."""
    x = x.detach().double()
    R = 2 * inv_freq.numel()
    angle = positions.double()[:, None, :, None] * inv_freq.double()
    unit = torch.polar(torch.full_like(angle, mscale), -angle if back else angle)
    y = x.clone()
    if interleaved:
        z = torch.complex(x[..., 0:R:2], x[..., 1:R:2]) * unit
        y[..., 0:R:2], y[..., 1:R:2] = z.real, z.imag
    else:
        z = torch.complex(x[..., : R // 2], x[..., R // 2: R]) * unit
        y[..., : R // 2], y[..., R // 2: R] = z.real, z.imag
    return y


def _exact_write(cache, scales, rows, seq, table, bs, coded):
    """The cache's values in 64 bits and its scales after rows [B, Hkv, S, D] are written. `coded`: a quantised cache
    holds the 8-bit codes; else the values that these round, in units of the scale."""
    x = cache.double()
    sc = None if scales is None else scales.double()
    S = rows.shape[2]
    for b, n in enumerate(seq.tolist()):
        for j in range(n // bs, (n + S - 1) // bs + 1):
            lo, hi = max(n, j * bs), min(n + S, (j + 1) * bs)
            p = int(table[b, j])
            held, part = max(0, min(n - j * bs, bs)), rows[b, :, lo - n: hi - n]
            if scales is None:
                x[p, :, 0, lo - j * bs: hi - j * bs] = part
                continue
            old = x[p, :, 0, :held] * sc[p][:, None, None]
            most = part.abs().amax(dim=(1, 2))
            if held:
                most = torch.maximum(most, old.abs().amax(dim=(1, 2)))
            now = most.clamp_min(1e-6) / 448.0
            both = torch.cat([old, part], dim=1) / now[:, None, None]
            if coded:  # the codes are defined in 32 bits: x * (1 / scale), each of the three rounded
                now = (most.float().clamp_min(1e-6) / 448.0)
                both = (torch.cat([old, part], dim=1).float() * (1.0 / now)[:, None, None]).clamp(-448, 448).to(_FP8)
                both, now = both.double(), now.double()
            x[p, :, 0, :held] = both[:, :held]
            x[p, :, 0, lo - j * bs: hi - j * bs] = both[:, held:]
            sc[p] = now
    return x, sc


def exact(case, seed):
    s = prepare(case, seed)
    op, bs = case["op"], case.get("bs")
    if op == "rotary":
        turn = (s["positions"], s["inv_freq"], case["interleaved"], case["mscale"])
        got = [_exact_turn(s["q"], *turn), _exact_turn(s["k"], *turn)]
        if case["train"]:
            got += [_exact_turn(s["dq"], *turn, back=True), _exact_turn(s["dk"], *turn, back=True)]
        return got
    table = s["table"].cpu()
    if op == "read":
        B, Hkv, D = case["B"], case["Hkv"], case["D"]
        got = []
        for cache, scales in ((s["kc"], s["ks"]), (s["vc"], s["vs"])):
            x = torch.zeros([B, Hkv, 1, s["most"], D], dtype=torch.float64, device=cache.device)
            for b, n in enumerate(s["seq"].tolist()):
                at = s["table"][b, : -(-n // bs)].long()
                rows = cache.view(torch.uint8)[at].view(cache.dtype).double() if scales is not None else cache[at].double()
                if scales is not None:
                    rows = rows * scales[at].double()[:, :, None, None, None]
                x[b, :, 0, :n] = rows[:, :, 0].transpose(0, 1).reshape(Hkv, -1, D)[:, :n]
            got.append(x)
        return tuple(got)
    B, Hkv, G, S, D = s["q"].shape
    k, v = s["k"][:, :, 0].double(), s["v"][:, :, 0].double()
    if op == "write":
        at = s["seq"].long()[:, None] + torch.arange(S, device=s["q"].device)
        turn = (at, s["inv_freq"], case["interleaved"], 1.0)
        q = _exact_turn(s["q"].reshape(B, Hkv * G, S, D), *turn).reshape(B, Hkv, G, S, D)
        kc, ks = _exact_write(s["kc"], s["ks"], _exact_turn(s["k"][:, :, 0], *turn), s["seq"], table, bs, False)
        vc, vs = _exact_write(s["vc"], s["vs"], v, s["seq"], table, bs, False)
        return [q, kc, vc] + ([] if ks is None else [ks, vs])
    # the attention reads the cache as it is held, in 8 bits
    kc, ks = _exact_write(s["kc"], s["ks"], k, s["seq"], table, bs, True)
    vc, vs = _exact_write(s["vc"], s["vs"], v, s["seq"], table, bs, True)
    out = torch.empty([B, Hkv, G, S, D], dtype=torch.float64, device=k.device)
    scale = float(s["scale"])
    for b, n in enumerate(s["seq"].tolist()):
        T = n + S
        at = s["table"][b, : -(-T // bs)].long()
        K, V = (((c[at] * z[at][:, :, None, None, None])[:, :, 0].transpose(0, 1).reshape(Hkv, -1, D)[:, :T])
                for c, z in ((kc, ks), (vc, vs)))
        score = torch.einsum("hgsd,htd->hgst", s["q"][b].double(), K) * scale
        t = torch.arange(T, device=k.device)
        seen = (t[None] < T) if case["both"] else (t[None] <= n + torch.arange(S, device=k.device)[:, None])
        if s["mask"] is not None:
            seen = seen & (s["mask"][b, :T] > 0)[None]
        score = torch.where(seen, score, torch.full_like(score, -math.inf))
        out[b] = torch.einsum("hgst,htd->hgsd", torch.softmax(score, dim=-1), V)
    return [out, kc, vc, ks, vs]
