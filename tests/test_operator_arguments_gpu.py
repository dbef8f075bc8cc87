"""Calls of the paged and rotary operators that are refused, or that take an unusual argument, on the GPU."""

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


def freqs(rot):
    return (10000.0 ** (-2.0 * torch.arange(rot // 2, dtype=torch.float64) / rot)).float()


@pytest.mark.parametrize("name", ["k", "v", "vc"])
def test_tensors_of_another_device(name):
    """Keys, values or one of the caches left on the host: refused by every paged op, before any launch."""
    import torch_rbln_b200 as tr

    f = freqs(64).to(DEV)
    for S in (1, 5):
        x = P.dev(P.setup([20, 3], S, 2, 4, 64, 16))
        wide = {n: x[n].to(torch.bfloat16) for n in ("kc", "vc")}  # a 16-bit cache
        x[name] = x[name].cpu()
        if name == "vc":
            wide["vc"] = wide["vc"].cpu()
        new, at = (x["q"], x["k"], x["v"]), (x["seq"], x["scale"], x["bt"], x["bs"])
        fp8, scales = (x["kc"], x["vc"]), (x["ks"], x["vs"])
        b16 = (wide["kc"], wide["vc"])
        calls = [lambda: tr.paged_causal_attn_prefill_kvfp8(*new, *fp8, *scales, *at, False),
                 lambda: tr.paged_causal_attn_prefill(*new, *b16, *at, False),
                 lambda: torch.ops.rbln_attn.rotary_paged_kv_write(*new, *fp8, x["seq"], x["bt"], x["bs"], f, False, 1.0,
                                                                   *scales),
                 lambda: torch.ops.rbln_attn.paged_kv_write(*new[1:], *fp8, x["seq"], x["bt"], x["bs"], *scales)]
        if S == 1:
            calls += [lambda: tr.paged_causal_attn_decode_kvfp8(*new, *fp8, *scales, *at),
                      lambda: tr.paged_causal_attn_decode(*new, *b16, *at)]
        if name == "vc":
            calls.append(lambda: torch.ops.rbln_attn.paged_kv_read(*fp8, x["seq"], x["bt"], x["bs"], 20, *scales))
        for i, call in enumerate(calls):
            with pytest.raises(RuntimeError, match="device|must be"):
                call()
                pytest.fail(f"call {i} was taken")
    torch.cuda.synchronize()


@pytest.mark.parametrize("S", [1, 5, 40])
def test_masks_over_no_position(S):
    """A position mask [B, 0] keeps nothing; it is refused, not taken for no mask."""
    import torch_rbln_b200 as tr

    x = P.dev(P.setup([20, 3], S, 2, 4, 64, 16))
    mask = torch.ones([2, 0], dtype=torch.bool, device=DEV)
    with pytest.raises(RuntimeError, match="mask covers no position"):
        P.run(x, mask=mask)
    new, at = (x["q"], x["k"], x["v"]), (x["seq"], x["scale"], x["bt"], x["bs"])
    wide = [x[n].to(torch.bfloat16) for n in ("kc", "vc")]
    with pytest.raises(RuntimeError, match="mask covers no position"):
        tr.paged_causal_attn_prefill(*new, *wide, *at, False, mask)
    if S == 1:
        with pytest.raises(RuntimeError, match="mask covers no position"):
            tr.paged_causal_attn_decode(*new, *wide, *at, mask)


@pytest.mark.parametrize("S", [1, 4, 40])
def test_rows_that_are_there_cost_no_copies(S):
    """k and v None: the call allocates its output and its workspace, nothing that would stand in for the rows."""
    x = P.dev(P.setup([200, 90], S, 2, 4, 64, 16))
    P.run(x)
    for _ in range(2):
        before = torch.cuda.memory_stats()["allocation.all.allocated"]
        out = P.run(x, rows=False)
        assert torch.cuda.memory_stats()["allocation.all.allocated"] - before == 2
    assert out.shape == x["q"].shape


@pytest.mark.parametrize("which", ["key", "value", "grad_out", "out", "logsumexp"])
def test_sdpa_backward_of_another_device(which):
    """A tensor of the backward call left on the host: refused before any launch."""
    q, k, v = (torch.randn(1, 2, 16, 64, device=DEV, dtype=torch.bfloat16) for _ in range(3))
    out, lse, cq, ck, mq, mk, seed, off, _ = torch.ops.aten._scaled_dot_product_fused_attention_overrideable(
        q, k, v, None, 0.0, True)
    t = dict(grad_out=torch.ones_like(out), query=q, key=k, value=v, out=out, logsumexp=lse)
    t[which] = t[which].cpu()
    with pytest.raises(RuntimeError, match="must be on query's device"):
        torch.ops.aten._scaled_dot_product_fused_attention_overrideable_backward(
            t["grad_out"], t["query"], t["key"], t["value"], torch.empty(0, device=DEV), [True, True, True, False],
            t["out"], t["logsumexp"], cq, ck, mq, mk, 0.0, True, seed, off)
