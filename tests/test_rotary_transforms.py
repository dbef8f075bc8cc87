"""Derivatives of torch.ops.rbln_attn.rotary as the tracer sees them: fake CUDA tensors, no GPU."""

import pytest
import torch
import torch.autograd.forward_ad as fwd
from torch._subclasses.fake_tensor import FakeTensorMode


@pytest.fixture(scope="module", autouse=True)
def _ext():
    import torch_rbln_b200  # noqa: F401


def inputs():
    q, k = (torch.empty(2, h, 3, 64, device="cuda", dtype=torch.bfloat16) for h in (4, 2))
    return q, k, torch.empty(2, 3, device="cuda", dtype=torch.int64), torch.empty(32, device="cuda")


def op(*args):
    return torch.ops.rbln_attn.rotary(*args)


def test_forward_mode_tangents():
    """A dual input gives a dual output, on either side alone too; the other side has none."""
    with FakeTensorMode():
        q, k, p, f = inputs()
        with fwd.dual_level():
            dq, dk = (fwd.make_dual(x, torch.empty_like(x)) for x in (q, k))
            for a, b in ((dq, dk), (dq, k), (q, dk), (q, k)):
                for x, y in zip((a, b), op(a, b, p, f)):
                    t = fwd.unpack_dual(y).tangent
                    assert (t is None) == (fwd.unpack_dual(x).tangent is None)
                    assert t is None or (t.shape == x.shape and t.dtype == x.dtype)
            with pytest.raises(RuntimeError, match="inv_freq has no gradient"):
                op(q, k, p, fwd.make_dual(f, torch.empty_like(f)))


def test_a_training_step_is_traced():
    """The forward pass with gradients, leaves used once and twice: no CUDA runtime is asked for anything."""
    with FakeTensorMode():
        q, k, p, f = inputs()
        q.requires_grad_(), k.requires_grad_()
        for _ in range(2):
            a, b = op(q, k, p, f)
            assert a.requires_grad and b.requires_grad and a.shape == q.shape and b.shape == k.shape


def test_symbolic_sizes_are_traced():
    """A sequence length that is a symbol, with and without gradients."""
    from torch._dynamo.source import ConstantSource
    from torch.fx.experimental.symbolic_shapes import ShapeEnv

    env = ShapeEnv()
    symbol = env.create_symbol(7, source=ConstantSource("S"))
    with FakeTensorMode(shape_env=env):
        S = env.create_symintnode(symbol, hint=7)
        q, k = (torch.empty(2, h, S, 64, device="cuda") for h in (4, 2))
        p, f = torch.empty(2, S, device="cuda", dtype=torch.int64), torch.empty(32, device="cuda")
        for grad in (False, True):
            a, b = op(q.requires_grad_(grad), k, p, f)
            assert a.shape == q.shape and b.shape == k.shape and a.requires_grad == grad
            assert not env.guards, f"the length was made a constant: {env.guards}"


def test_frequencies_that_are_a_parameter():
    """Taken where no gradient is asked for, refused where one is."""
    with FakeTensorMode():
        q, k, p, f = inputs()
        f.requires_grad_()
        with torch.no_grad():
            assert op(q, k, p, f)[0].shape == q.shape
        with torch.inference_mode():
            assert op(q, k, p, f)[0].shape == q.shape
        assert op(q, k, p, f.detach())[0].shape == q.shape
        with pytest.raises(RuntimeError, match="inv_freq has no gradient"):
            op(q, k, p, f)
