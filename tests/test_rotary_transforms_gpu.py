"""torch.ops.rbln_attn.rotary under forward mode and torch.func, against the plain map of tests/operator_refs.py."""

import pytest
import torch
import torch.autograd.forward_ad as fwd

from tests import operator_refs as R
from tests.test_rotary_gpu import freqs, inputs, op

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(scope="module", autouse=True)
def _ext():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    import torch_rbln_b200  # noqa: F401


def case(seed=0, dtype=torch.float32):
    """q, k, their tangents (or cotangents), positions and frequencies, on the host."""
    q, k, pos = inputs(2, 4, 2, 5, 64, dtype, "bshd", seed)
    tq, tk, _ = inputs(2, 4, 2, 5, 64, dtype, "bhsd", seed + 1)
    return q, k, tq, tk, pos, freqs(32)


def near(got, x, pos, f, *args, **kw):
    ref, size = R.rotary(x, pos, f, *args, **kw)
    R.assert_within(got.detach(), ref, R.rotary_bound(ref, size, x.dtype))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("interleaved", [False, True])
def test_forward_mode(dtype, interleaved):
    """The tangents are the same map of the inputs' tangents, through dual numbers and through torch.func.jvp."""
    q, k, tq, tk, pos, f = case(dtype=dtype)
    x = [t.to(DEV) for t in (q, k, tq, tk, pos, f)]
    with fwd.dual_level():
        out = op(fwd.make_dual(x[0], x[2]), fwd.make_dual(x[1], x[3]), x[4], x[5], interleaved, 1.25)
        got = [fwd.unpack_dual(y) for y in out]
        for g, a, t in zip(got, (q, k), (tq, tk)):
            near(g.primal, a, pos, f, interleaved, 1.25)
            near(g.tangent, t, pos, f, interleaved, 1.25)
        half = op(fwd.make_dual(x[0], x[2]), x[1], x[4], x[5], interleaved, 1.25)
        near(fwd.unpack_dual(half[0]).tangent, tq, pos, f, interleaved, 1.25)
        assert fwd.unpack_dual(half[1]).tangent is None
    out, tan = torch.func.jvp(lambda a, b: op(a, b, x[4], x[5], interleaved, 1.25), (x[0], x[1]), (x[2], x[3]))
    for y, t, a, da in zip(out, tan, (q, k), (tq, tk)):
        near(y, a, pos, f, interleaved, 1.25)
        near(t, da, pos, f, interleaved, 1.25)


def test_forward_over_reverse():
    """The tangent of a gradient: the transposed map of the cotangent's tangent, zero along the inputs."""
    q, k, tq, tk, pos, f = case(3)
    x = [t.to(DEV) for t in (q, k, tq, tk, pos, f)]

    def grad(a, up):
        return torch.func.vjp(lambda a: op(a, x[1], x[4], x[5])[0], a)[1](up)[0]

    d, t = torch.func.jvp(grad, (x[0], x[2]), (x[2], x[0]))
    near(d, tq, pos, f, False, 1.0, inverse=True)
    near(t, q, pos, f, False, 1.0, inverse=True)


def test_functional_gradient():
    """torch.func.grad, and under vmap a gradient for each of several cotangents."""
    q, k, tq, tk, pos, f = case(5)
    x = [t.to(DEV) for t in (q, k, tq, tk, pos, f)]
    got = torch.func.grad(lambda a, b: sum((y * t).sum() for y, t in zip(op(a, b, x[4], x[5]), (x[2], x[3]))),
                          argnums=(0, 1))(x[0], x[1])
    near(got[0], tq, pos, f, False, 1.0, inverse=True)
    near(got[1], tk, pos, f, False, 1.0, inverse=True)
    _, pull = torch.func.vjp(lambda a: op(a, x[1], x[4], x[5])[0], x[0])
    many = torch.func.vmap(pull)(torch.stack([x[2], x[0]]))[0]
    near(many[0], tq, pos, f, False, 1.0, inverse=True)
    near(many[1], q, pos, f, False, 1.0, inverse=True)


def test_compiled_for_any_length():
    """A function traced once for every length, gradients with it."""
    f = freqs(32)
    seen = []

    def backend(gm, args):
        from torch._dynamo.backends.common import aot_autograd

        seen.append(1)
        return aot_autograd(fw_compiler=lambda g, _: g, bw_compiler=lambda g, _: g)(gm, args)

    @torch.compile(backend=backend, dynamic=True, fullgraph=True)
    def turn(q, k, pos, f):
        a, b = op(q * 1.0, k * 1.0, pos, f)
        return a, b

    for S in (5, 9, 17):
        q, k, pos = inputs(2, 4, 2, S, 64, torch.float32, seed=S)
        x = [q.to(DEV).requires_grad_(), k.to(DEV).requires_grad_()]
        a, b = turn(*x, pos.to(DEV), f.to(DEV))
        near(a, q, pos, f, False)
        near(b, k, pos, f, False)
        dq, dk = torch.autograd.grad((a, b), x, (torch.ones_like(a), torch.ones_like(b)))
        near(dq, torch.ones_like(q), pos, f, False, 1.0, inverse=True)
        near(dk, torch.ones_like(k), pos, f, False, 1.0, inverse=True)
    assert len(seen) == 1
