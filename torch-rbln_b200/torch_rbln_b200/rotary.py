"""Frequencies for rotary positions, plain or stretched for long contexts.

torch.ops.rbln_attn.rotary and rotary_paged_kv_write take one inverse frequency a pair and one factor for cosine and
sine; every scheme below is a choice of those two, made once for a model.
"""

from __future__ import annotations

import math
from typing import Optional, Tuple

import torch


def rotary_frequencies(rotary_dim: int, base: float = 10000.0, scaling: Optional[str] = None, factor: float = 1.0,
                       original_length: int = 0, low: float = 1.0, high: Optional[float] = None,
                       device=None) -> Tuple[torch.Tensor, float]:
    """(inv_freq, mscale) of rotary positions: inv_freq fp32 [rotary_dim / 2], inv_freq[i] = base^(-2 i / rotary_dim).

    scaling stretches a model trained on `original_length` positions by `factor` (at least 1):
      None      as it is (factor must be 1);
      "linear"  every frequency divided by factor;
      "ntk"     the base raised to base * factor^(R / (R - 2)), which leaves the fastest pair and divides the slowest
                by factor;
      "yarn"    by the turns r a pair makes over original_length: r >= high as it is, r <= low divided by factor, in
                between the two blended linearly in the pair's index (between the indices where r = high, rounded
                down, and r = low, rounded up); mscale = 0.1 ln(factor) + 1;
      "llama3"  the same with the blend linear in r.
    low is 1 turn unless given, high 32 for yarn and 4 for llama3. The values are computed in float64 and rounded once.
    """
    R = int(rotary_dim)
    if R <= 0 or R % 2:
        raise ValueError(f"rotary_frequencies: rotary_dim must be positive and even, got {rotary_dim}")
    if not base > 1.0:
        raise ValueError(f"rotary_frequencies: base must be above 1, got {base}")
    if not factor >= 1.0:
        raise ValueError(f"rotary_frequencies: factor must be at least 1, got {factor}")
    i = torch.arange(R // 2, dtype=torch.float64)
    if scaling == "ntk":
        if R < 4:
            raise ValueError("rotary_frequencies: ntk needs rotary_dim of at least 4")
        base = base * factor ** (R / (R - 2))
    inv = base ** (-2.0 * i / R)
    mscale = 1.0
    if scaling is None:
        if factor != 1.0:
            raise ValueError("rotary_frequencies: a factor needs a scaling")
    elif scaling == "linear":
        inv = inv / factor
    elif scaling in ("yarn", "llama3"):
        if high is None:
            high = 32.0 if scaling == "yarn" else 4.0
        if original_length <= 0 or not 0 < low < high:
            raise ValueError(f"rotary_frequencies: {scaling} needs original_length > 0 and 0 < low < high")
        if scaling == "llama3":
            keep = ((original_length * inv / (2 * math.pi) - low) / (high - low)).clamp(0.0, 1.0)
        else:
            def index(turns):  # the (fractional) pair that makes `turns` turns over original_length
                return R * math.log(original_length / (turns * 2 * math.pi)) / (2 * math.log(base))

            first, last = max(math.floor(index(high)), 0), min(math.ceil(index(low)), R - 1)
            keep = 1.0 - ((i - first) / max(last - first, 1e-3)).clamp(0.0, 1.0)
            mscale = 0.1 * math.log(factor) + 1.0
        inv = keep * inv + (1.0 - keep) * inv / factor
    elif scaling != "ntk":
        raise ValueError(f"rotary_frequencies: scaling must be None, linear, ntk, yarn or llama3, got {scaling!r}")
    return inv.to(torch.float32).to(device), mscale
