"""Plain float64 forms of the rotary and quantised-cache operators, with the
error bounds that their rounding steps allow (shared by their tests).

A rounding to a type t is off by at most half a step, eps(t) / 2 of the
value, or half the smallest subnormal. The float32 work before it is bounded
term by term beside each bound.
"""

from __future__ import annotations

import torch


def half_step(x: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    """Largest error of rounding values near x to dtype."""
    f = torch.finfo(dtype)
    return x.abs() * (f.eps / 2) + f.smallest_normal * f.eps / 2


def rotary(x, positions, inv_freq, interleaved, mscale=1.0, inverse=False):
    """x [B, H, S, D], positions [B, S] -> (y, |x1| + |x2| of each element's pair), both float64."""
    x = x.double()
    R = 2 * inv_freq.numel()
    ang = positions.double()[:, None, :, None] * inv_freq.double()
    c, s = ang.cos() * mscale, ang.sin() * mscale * (-1 if inverse else 1)
    i = torch.arange(R // 2)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + R // 2)
    y, size = x.clone(), x.abs()
    y[..., a] = x[..., a] * c - x[..., b] * s
    y[..., b] = x[..., b] * c + x[..., a] * s
    size[..., a] = size[..., b] = (x[..., a].abs() + x[..., b].abs()) * abs(mscale)
    return y, size


def rotary_bound(y, size, dtype):
    """cos and sin are off by at most 2^-22 (angle 2^-23, the function two
    steps of 2^-24 and more), their factor, the two products and the sum by
    2^-24 each: under 2^-21 of (|x1| + |x2|) m together; then one rounding."""
    f32 = size * 2.0 ** -21
    return f32 + half_step(y.abs() + f32, dtype)


def attention(q, K, V, keep, scale):
    """q [Hkv, G, S, D], K / V [Hkv, T, D], keep [S, T] (float64 but keep) ->
    out, A = sum p |v| / sum p, and the scores' error scale
    e = max_t scale sum_d |q_d k_d| over the kept keys."""
    q, K, V = q.double(), K.double(), V.double()
    w = torch.einsum("hgsd,htd->hgst", q, K) * scale
    size = torch.einsum("hgsd,htd->hgst", q.abs(), K.abs()) * abs(scale)
    w = w.masked_fill(~keep, -float("inf"))
    p = torch.softmax(w, dim=-1)
    Vz = V.masked_fill(~keep.any(0)[:, None], 0.0)  # what no row sees may hold anything
    Vz = torch.nan_to_num(Vz, nan=0.0) if torch.isnan(Vz).any() else Vz
    return (torch.einsum("hgst,htd->hgsd", p, Vz), torch.einsum("hgst,htd->hgsd", p, Vz.abs()),
            size.masked_fill(~keep, 0.0).nan_to_num(0.0).amax(-1, keepdim=True))


def attention_bound(out, A, e, T, vmax, dtype):
    """The probabilities are rounded to f16 (2^-11 of each); exp2 and the
    float32 sums are off by under 2^-18; a score by under 2^-20 e (products
    of up to 128 terms summed in float32), which moves numerator and
    denominator by that much each. Probabilities far below 2^-14 keep 2^-25
    of the largest: T 2^-25 times twice the largest value."""
    rel = 2.0 ** -11 + 2.0 ** -18 + 2 * e * 2.0 ** -20
    inner = A * rel + T * 2.0 ** -24 * vmax
    return inner + half_step(out.abs() + inner, dtype)


def assert_within(got, ref, bound, what=""):
    got = got.double().cpu()
    nan = torch.isnan(ref)
    assert torch.equal(torch.isnan(got), nan), f"{what}: NaN where there should be none, or none where there should"
    over = ((got - ref).abs() - bound).masked_fill(nan, 0.0)
    worst = over.max().item() if over.numel() else 0.0
    assert worst <= 0.0, f"{what}: off by {worst:.3g} more than the bound allows"


def fp8_values(cache, scale):
    """Codes times scales, float64, [num_blocks, Hkv, 1, bs, D]."""
    return cache.double() * scale.double()[:, :, None, None, None]


def write_reciprocal(k, v, kcache, vcache, seq, table, bs, k_scale, v_scale):
    """The fp8 write of paged_causal_attn_prefill_kvfp8, in place: oracle.paged_attention.kv_write with
    scale = max(amax, 1e-6) * (1 / 448), the reciprocal rounded to float32 (what torch computes on the GPU for
    amax / 448.0). A sequence whose start is negative or whose rows pass the span is left."""
    B, Hkv, _, S, D = k.shape
    third = torch.tensor(1.0) / torch.tensor(448.0)
    for b in range(B):
        n = int(seq.reshape(-1)[b])
        if n < 0 or n + S > table.shape[1] * bs:
            continue
        for j in range(n // bs, (n + S - 1) // bs + 1):
            p = int(table[b, j])
            if not 0 <= p < kcache.shape[0]:
                continue
            lo, hi = max(n, j * bs), min(n + S, (j + 1) * bs)
            held = max(0, min(n - j * bs, bs))
            for cache, new, scales in ((kcache, k, k_scale), (vcache, v, v_scale)):
                rows = new[b, :, 0, lo - n: hi - n].float()  # [Hkv, rows, D]
                old = scales[p].clone()
                was = cache[p, :, 0, :held, :D].float() * old[:, None, None]
                amax = torch.cat([was, rows], 1).abs().amax((1, 2))
                scale = amax.clamp_min(1e-6) * third
                inv = (1.0 / scale)[:, None, None]

                def codes(x):
                    return (x * inv).clamp(-448, 448).to(torch.float8_e4m3fn)

                moved = (scale != old)[:, None, None]
                if held:
                    keep = cache[p, :, 0, :held, :D].view(torch.uint8)
                    cache.view(torch.uint8)[p, :, 0, :held, :D] = torch.where(moved, codes(was).view(torch.uint8), keep)
                cache.view(torch.uint8)[p, :, 0, lo - j * bs: hi - j * bs, :D] = codes(rows).view(torch.uint8)
                scales[p] = scale
