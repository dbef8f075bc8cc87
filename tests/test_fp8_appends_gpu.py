"""A block of an fp8 cache filled one token a call, by paged_causal_attn_prefill_kvfp8 and by paged_kv_write."""

import pytest
import torch

from tests import test_prefill_kvfp8_gpu as P

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(scope="module", autouse=True)
def _ext():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    import torch_rbln_b200  # noqa: F401


@pytest.mark.parametrize("D,bs", [(64, 16), (128, 16), (128, 64)])
def test_one_token_a_call(D, bs):
    """The first token holds the block's largest values. The scale moves by no more than its rule's rounding, the held
    codes not at all: a NaN code keeps its sign, which finding it anew would clear."""
    d = P.setup([0] * 4, 1, 8, 2, D, bs)
    x, y = P.dev(d), P.dev(d)
    g = torch.Generator().manual_seed(7)
    first = None
    for n in range(bs):
        for n_, std in (("k", 1.0), ("v", 0.5)):
            rows = torch.randn(d[n_].shape, generator=g) * std
            rows = rows.clamp(-std, std) * 0.9 if n else rows + 3 * std  # later tokens stay below the first
            x[n_] = y[n_] = rows.to(torch.bfloat16).to(DEV)
        for t in (x, y):
            t["seq"] = torch.full_like(t["seq"], n)
        P.run(x)
        torch.ops.rbln_attn.paged_kv_write(y["k"], y["v"], y["kc"], y["vc"], y["seq"], y["bt"], bs, y["ks"], y["vs"])
        at = x["bt"][:, 0].long()
        if n == 0:
            for c, new in (("kc", "k"), ("vc", "v")):  # over the row's smallest value, so that the largest stays
                codes = x[c].view(torch.uint8)
                codes[at, :, :, 0] = codes[at, :, :, 0].scatter(-1, x[new][:, :, :, 0].abs().argmin(-1, True), 0xFF)
            first = {c: x[c].view(torch.uint8)[at, :, :, 0].clone() for c in ("kc", "vc")}
            scale = {c: x[c][at].clone() for c in ("ks", "vs")}
            for c in ("ks", "vs"):
                assert (x[c][at].view(torch.int32) - y[c][at].view(torch.int32)).abs().max() <= 1
        for c in ("kc", "vc"):
            assert torch.equal(x[c].view(torch.uint8)[at, :, :, 0], first[c]), (n, c)
            same = x[c].view(torch.uint8)[at, :, :, 1: n + 1] == y[c].view(torch.uint8)[at, :, :, 1: n + 1]
            assert n == 0 or same.float().mean() > 0.99  # ties fall as the last bit of a scale does
        for c in ("ks", "vs"):
            up = x[c][at].view(torch.int32) - scale[c].view(torch.int32)
            assert 0 <= int(up.min()) and int(up.max()) <= 6
            # 6 up, the first write's unit, and the division's own
            assert (x[c][at].view(torch.int32) - y[c][at].view(torch.int32)).abs().max() <= 8
