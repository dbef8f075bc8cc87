"""The two rules that find a block's scale from its largest value, held against each other in float32 (no GPU):
max(amax, 1e-6) / 448, and the product with the rounded reciprocal."""

import torch

FP8 = torch.float8_e4m3fn


def rules():
    third = torch.tensor(1.0) / torch.tensor(448.0)
    return (lambda m: m * third), (lambda m: m / torch.tensor(448.0))


def units(a, b):
    return a.view(torch.int32) - b.view(torch.int32)


def test_how_far_a_scale_moves():
    """Every mantissa: one write's scales differ by a unit at most; found again from 448 times itself, a scale rests
    after 6 steps of a unit up (reciprocal) or one of a unit (division)."""
    first = torch.arange(1 << 23, dtype=torch.int32).add_(127 << 23).view(torch.float32)
    product, quotient = rules()
    assert units(product(first), quotient(first)).abs().max() == 1
    for rule, lo, hi, steps in ((product, 0, 6, 6), (quotient, -1, 1, 1)):
        s = first
        for _ in range(steps):
            now = rule(448.0 * s)
            assert units(now, s).abs().max() == 1
            s = now
        assert torch.equal(rule(448.0 * s), s)
        moved = units(s, first)
        assert int(moved.min()) == lo and int(moved.max()) == hi


def test_codes_do_not_move_with_a_scale_that_rounds():
    """All finite codes, decoded by a scale and coded by one that differs by up to 2^-20 of it: the same codes."""
    code = torch.arange(256, dtype=torch.uint8)
    code = code[~torch.isnan(code.view(FP8).float())]
    old = torch.exp2(torch.rand(4000, 1, generator=torch.Generator().manual_seed(0)) * 60 - 28)
    for d in (-(2.0 ** -20), -(2.0 ** -23), 0.0, 2.0 ** -23, 2.0 ** -20):
        new = old * (1.0 + d)
        again = (code.view(FP8).float() * old * (1.0 / new)).clamp(-448, 448).to(FP8).view(torch.uint8)
        assert torch.equal(again, code.expand_as(again))
