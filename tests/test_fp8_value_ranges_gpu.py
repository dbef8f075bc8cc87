"""paged_causal_attn_prefill_kvfp8 where the scales of the blocks differ by much: zero, not numbers, at the ends of
float32, or of other sizes before and behind a row's limit. Bounds as in tests/operator_refs.py, but each row's own:
the largest value is taken over the blocks that the row sees."""

import pytest
import torch

from tests import operator_refs as R
from tests import test_prefill_kvfp8_gpu as P

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(scope="module", autouse=True)
def _ext():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    import torch_rbln_b200  # noqa: F401


def reference(d, mask=None, rows=True):
    """(out, bound) in float64; a probability is rounded relative to a power of two at most twice the largest V scale
    that its row sees, so 448 of that scale stands for the bound's largest value."""
    B, Hkv, G, S, D = d["q"].shape
    bs, bt = d["bs"], d["bt"].long()
    if rows:
        R.write_reciprocal(d["k"], d["v"], d["kc"], d["vc"], d["seq"], bt, bs, d["ks"], d["vs"])
    t = torch.arange(bt.shape[1] * bs)
    outs, bounds = [], []
    for b in range(B):
        blk = bt[b][t // bs]
        K, V = ((c[blk, :, 0, t % bs].double() * s[blk].double()[:, :, None]).transpose(0, 1)
                for c, s in ((d["kc"], d["ks"]), (d["vc"], d["vs"])))
        keep = t < int(d["seq"][b]) + 1 + torch.arange(S)[:, None]
        if mask is not None:
            keep = keep & mask[b, : t.numel()]
        out, A, e = R.attention(d["q"][b], K, V, keep, float(d["scale"]))
        seen = d["vs"][blk].double().t()[:, None].expand(Hkv, S, -1).masked_fill(~keep, 0.0)
        vmax = 448 * seen.amax(-1)[:, None, :, None]
        outs.append(out)
        bounds.append(R.attention_bound(out, A, e, t.numel(), vmax, d["q"].dtype))
    return torch.stack(outs), torch.stack(bounds)


def check(d, mask=None, rows=True):
    out = P.run(P.dev(d), mask=None if mask is None else mask.to(DEV), rows=rows)
    torch.cuda.synchronize()
    ref, bound = reference(d, mask, rows)
    R.assert_within(out, ref, bound)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("S", [4, 40, 200])
def test_key_scales_of_zero(S, dtype):
    """A block whose keys are all zeros, its scale too, and only some of its keys kept: scores of zero, no NaN."""
    d = P.setup([200, 90], S, 2, 4, 64, 16, dtype)
    for b, j in ((0, 2), (0, 5), (1, 1)):
        d["ks"][d["bt"][b, j].item()] = 0.0
    mask = torch.ones([2, d["bt"].shape[1] * 16], dtype=torch.bool)
    mask[0, 33:45:2] = False
    mask[1, 18:21] = False
    check(d, mask, rows=False)


@pytest.mark.parametrize("name", ["ks", "vs"])
@pytest.mark.parametrize("S,D", [(4, 128), (40, 128), (150, 64)])
def test_parts_of_a_split_that_hold_no_number(S, D, name):
    """NaN scales of a long run of blocks, so that some part of a split sequence holds nothing else (and, for one
    start of the run, no part holds NaN and numbers): NaN all the same."""
    for starts, first, n in (([6000], 8, 22), ([6000], 9, 21), ([6000], 10, 21), ([5000, 3], 8, 22)):
        d = P.setup(starts, S, 1, 4, D, 128)
        for j in range(first, first + n):
            d[name][d["bt"][0, j].item()] = float("nan")
        out = P.run(P.dev(d))
        assert torch.isnan(out[0]).all() and not torch.isnan(out[1:]).any()


@pytest.mark.parametrize("S,G,bs,first", [(16, 1, 8, 8), (8, 2, 8, 4), (4, 4, 16, 2), (24, 1, 8, 12), (64, 2, 16, 32),
                                          (200, 1, 8, 96), (100, 4, 16, 20)])
@pytest.mark.parametrize("binades", [16, 20, 26, 90])
def test_values_behind_a_row_cost_it_nothing(S, G, bs, first, binades):
    """The chunk's tokens from `first` on, a block's first row, hold values 2^16 and more times the earlier ones': a
    row that does not see them keeps its bits."""
    for vstd in (0.5, 1e-5):
        d = P.setup([(-first) % bs, (-first) % bs + 2 * bs], S, 2, G, 64, bs, vstd=vstd)
        d["v"][:, :, :, first:] *= 2.0 ** binades
        check(d)


@pytest.mark.parametrize("S,G,bs,first", [(4, 4, 16, 2), (40, 4, 64, 20), (40, 1, 128, 20), (100, 2, 32, 28)])
def test_values_behind_a_row_under_a_mask(S, G, bs, first):
    """A block of which the mask drops the chunk's earlier tokens; its kept ones, from `first` on, hold large values.
    A row before them sees nothing of that block, and its bits are those of the blocks before."""
    start = 2 * bs
    d = P.setup([start, start], S, 2, G, 64, bs)
    d["v"][:, :, :, first:] *= 2.0 ** 20
    mask = torch.ones([2, d["bt"].shape[1] * bs], dtype=torch.bool)
    mask[:, start: start + first] = False
    check(d, mask)


@pytest.mark.parametrize("S", [1, 4, 40])
@pytest.mark.parametrize("starts", [[300, 11], [5000]])
def test_values_near_the_largest(S, starts):
    """bf16 values up to 3e38, V scales up to 7e35: a mean of finite values is finite."""
    check(P.setup(starts, S, 2, 4, 128, 16, vstd=6e37))


@pytest.mark.parametrize("S", [1, 4, 40])
@pytest.mark.parametrize("starts", [[300, 11], [5000]])
def test_value_scales_far_below_one(S, starts):
    """V scales of 2^-123, as a caller may make them."""
    d = P.setup(starts, S, 2, 4, 128, 16)
    d["vs"] *= 2.0 ** -115
    check(d, rows=False)


@pytest.mark.parametrize("S", [1, 4, 40])
@pytest.mark.parametrize("small,large", [(-99, 60), (-120, 118), (-40, 100)])
@pytest.mark.parametrize("turned", [False, True])
def test_value_scales_from_end_to_end(S, small, large, turned):
    """Half of a sequence's blocks with V scales of one end of float32, half of the other: what is too small to count
    is lost, nothing else is."""
    d = P.setup([1200], S, 2, 4, 64, 16)
    half = d["bt"][0, :38].long()
    rest = d["bt"][0, 38:].long()
    d["vs"][half if not turned else rest] = 2.0 ** small
    d["vs"][rest if not turned else half] = 2.0 ** large
    check(d, rows=False)
