"""torch.ops.rbln_attn.rotary: forward, gradient, layouts, strides and types
against float64, with the bounds of tests/operator_refs.py."""

import pytest
import torch

from tests import operator_refs as R

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(scope="module", autouse=True)
def _ext():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    import torch_rbln_b200  # noqa: F401


def op(*args, **kw):
    return torch.ops.rbln_attn.rotary(*args, **kw)


def inputs(B, H, Hk, S, D, dtype, layout="bhsd", seed=0, far=5000):
    g = torch.Generator().manual_seed(seed)
    shape = (lambda h: [B, h, S, D]) if layout == "bhsd" else (lambda h: [B, S, h, D])
    q, k = torch.randn(shape(H), generator=g).to(dtype), torch.randn(shape(Hk), generator=g).to(dtype)
    if layout != "bhsd":
        q, k = q.transpose(1, 2), k.transpose(1, 2)
    pos = torch.randint(0, far, [B, 1], generator=g) + torch.arange(S)
    return q, k, pos


def freqs(rot, base=10000.0):
    return (base ** (-2.0 * torch.arange(rot // 2, dtype=torch.float64) / rot)).float()


def check(q, k, pos, f, interleaved, mscale=1.0, inverse=False, what=""):
    got = op(q.to(DEV) if not q.is_cuda else q, k.to(DEV) if not k.is_cuda else k, pos.to(DEV), f.to(DEV), interleaved,
             mscale, inverse)
    p = pos if pos.dim() == 2 else pos[None]
    for x, y in zip((q.cpu(), k.cpu()), got):
        ref, size = R.rotary(x, p, f, interleaved, mscale, inverse)
        assert y.dtype == x.dtype and y.shape == x.shape
        R.assert_within(y, ref, R.rotary_bound(ref, size, x.dtype), what)
    return got


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("layout", ["bhsd", "bshd"])
@pytest.mark.parametrize("S,D,rot", [(1, 128, 128), (7, 64, 32), (130, 128, 64), (5, 96, 96), (3, 80, 20), (2, 7, 2)])
def test_types_layouts_and_sizes(dtype, interleaved, layout, S, D, rot):
    """Vector sizes, and head dimensions and rotary parts that only the scalar kernel takes (80 / 20, 7 / 2)."""
    q, k, pos = inputs(2, 6, 2, S, D, dtype, layout, seed=S + D)
    check(q, k, pos, freqs(rot), interleaved, mscale=1.25)


@pytest.mark.parametrize("B,S", [(1, 1), (64, 1), (3, 1000), (1, 5000)])
def test_few_and_many_tokens(B, S):
    """Both sides of the rule that puts four tokens in a CTA, and a last CTA that is not full."""
    q, k, pos = inputs(B, 5, 1, S, 128, torch.bfloat16, "bshd", seed=B)
    check(q, k, pos, freqs(128), False)


def test_far_positions():
    """The angle of a far position is many turns: a float32 product would lose it."""
    q, k, _ = inputs(1, 2, 2, 4, 64, torch.float32)
    pos = torch.tensor([[1 << 20, 999_999_937, (1 << 31) + 12345, -77]])
    check(q, k, pos, freqs(64, 500000.0), False)
    check(q, k, pos[:, :1].expand(1, 4).contiguous(), freqs(64), True)


def test_position_forms():
    q, k, pos = inputs(3, 4, 2, 9, 64, torch.bfloat16)
    f = freqs(64)
    check(q, k, pos.to(torch.int32), f, False)
    check(q, k, pos[0], f, False)                       # [S]
    check(q, k, pos[:1], f, False)                      # [1, S]
    check(q, k, pos.t().contiguous().t(), f, False)     # strided


def test_strided_inputs():
    """Slices of a fused projection, a strided head dimension, an unaligned start, a broadcast head."""
    g = torch.Generator().manual_seed(3)
    f, pos = freqs(64), torch.arange(6)[None].expand(2, 6)
    qkv = torch.randn([2, 6, (4 + 1 + 1) * 64], generator=g).to(torch.bfloat16).to(DEV)
    q = qkv[..., : 4 * 64].view(2, 6, 4, 64).transpose(1, 2)
    k = qkv[..., 4 * 64: 5 * 64].view(2, 6, 1, 64).transpose(1, 2)
    check(q, k, pos, f, False, what="projection")
    w = torch.randn([2, 4, 64, 6], generator=g).to(DEV)
    check(w.transpose(2, 3), w.transpose(2, 3)[:, :2], pos, f, True, what="strided head dimension")
    flat = torch.randn([2 * 4 * 6 * 64 + 1], generator=g).to(torch.float16).to(DEV)
    u = flat[1:].view(2, 4, 6, 64)
    check(u, u[:, 1:3], pos, f, False, what="unaligned")
    one = torch.randn([2, 1, 6, 64], generator=g).to(torch.bfloat16).to(DEV)
    check(one.expand(2, 4, 6, 64), one, pos, f, False, what="broadcast")


def test_output_keeps_the_layout():
    q, k, pos = inputs(2, 4, 2, 5, 64, torch.bfloat16, "bshd")
    a, b = op(q.to(DEV), k.to(DEV), pos.to(DEV), freqs(64).to(DEV))
    assert a.stride() == q.stride() and b.stride() == k.stride()


@pytest.mark.parametrize("B,H,Hk,S", [(0, 2, 2, 3), (2, 2, 2, 0), (2, 0, 2, 3), (2, 2, 0, 3)])
def test_empty(B, H, Hk, S):
    q, k = torch.zeros([B, H, S, 64], device=DEV), torch.ones([B, Hk, S, 64], device=DEV)
    a, b = op(q, k, torch.zeros([B, S], dtype=torch.int64, device=DEV), freqs(64).to(DEV))
    assert a.shape == q.shape and b.shape == k.shape
    if b.numel():
        assert torch.equal(b, k)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("interleaved", [False, True])
def test_gradient_is_the_transposed_map(dtype, interleaved):
    q, k, pos = inputs(2, 3, 1, 11, 64, dtype, "bshd", seed=9)
    f = freqs(32)
    qd, kd = q.to(DEV).requires_grad_(), k.to(DEV).requires_grad_()
    g = torch.Generator().manual_seed(1)
    gq, gk = torch.randn(q.shape, generator=g).to(dtype), torch.randn(k.shape, generator=g).to(dtype)
    a, b = op(qd, kd, pos.to(DEV), f.to(DEV), interleaved, 1.5)
    dq, dk = torch.autograd.grad((a, b), (qd, kd), (gq.to(DEV), gk.to(DEV)))
    for d, up in ((dq, gq), (dk, gk)):
        ref, size = R.rotary(up, pos, f, interleaved, 1.5, inverse=True)
        R.assert_within(d, ref, R.rotary_bound(ref, size, dtype))
    # only k's output used; a broadcast leaf sums over its copies
    leaf = torch.randn([2, 1, 11, 64], generator=g).to(dtype).to(DEV).requires_grad_()
    a, b = op(leaf.expand(2, 3, 11, 64), kd, pos.to(DEV), f.to(DEV), interleaved)
    (only,) = torch.autograd.grad(b, kd, gk.to(DEV), retain_graph=True)
    ref, size = R.rotary(gk, pos, f, interleaved, 1.0, inverse=True)
    R.assert_within(only, ref, R.rotary_bound(ref, size, dtype))
    (dl,) = torch.autograd.grad(a, leaf, gq.to(DEV))
    ref, size = R.rotary(gq, pos, f, interleaved, 1.0, inverse=True)
    bound = R.rotary_bound(ref, size, dtype).sum(1, keepdim=True)
    total = ref.sum(1, keepdim=True)
    # the sum over copies is torch's: three terms, each partial sum rounded at most once more
    bound = bound + 3 * R.half_step(ref.abs().sum(1, keepdim=True), dtype)
    R.assert_within(dl, total, bound)


def test_gradient_against_differences():
    """float32, a central difference of a random projection of the output."""
    q, k, pos = inputs(1, 2, 1, 5, 32, torch.float32, seed=4)
    f = freqs(32).to(DEV)
    qd, kd, pd = q.to(DEV).requires_grad_(), k.to(DEV), pos.to(DEV)
    w = torch.randn(q.shape, generator=torch.Generator().manual_seed(2)).to(DEV)
    (dq,) = torch.autograd.grad((op(qd, kd, pd, f)[0] * w).sum(), qd)
    step = torch.randn(q.shape, generator=torch.Generator().manual_seed(5)).to(DEV)
    with torch.no_grad():
        # the map is linear: a difference of any step is exact but for rounding
        up, down = (op(q.to(DEV) + s * step, kd, pd, f)[0].double() for s in (0.5, -0.5))
    diff = ((up - down) * w.double()).sum().item()
    want = (dq.double() * step.double()).sum().item()
    # 320 terms, each off by under 2^-20 of (|x| + |step|) |w| twice over
    scale = ((q.to(DEV).abs() + step.abs()).double() * w.abs().double()).sum().item() * 4
    assert abs(diff - want) <= scale * 2.0 ** -20


def test_second_derivative():
    q, k, pos = inputs(1, 1, 1, 3, 32, torch.float32)
    qd, up = q.to(DEV).requires_grad_(), torch.ones(q.shape, device=DEV, requires_grad=True)
    f = freqs(32).to(DEV)
    a, _ = op(qd, k.to(DEV), pos.to(DEV), f)
    (d,) = torch.autograd.grad(a, qd, up, create_graph=True)
    (dd,) = torch.autograd.grad(d, up, qd.detach())
    assert torch.equal(dd, op(qd.detach(), k.to(DEV), pos.to(DEV), f)[0])


def test_captured_and_on_another_stream():
    """Forward and gradient captured into a graph and replayed on new values. While an eager graph of the same leaves
    lives the capture is refused, and nothing is broken by that."""
    q, k, pos = inputs(2, 4, 2, 33, 64, torch.bfloat16, "bshd")
    f, pd = freqs(64).to(DEV), pos.to(DEV)
    qd, kd = q.to(DEV).requires_grad_(), k.to(DEV).requires_grad_()
    gq, gk = torch.ones_like(qd), torch.ones_like(kd)
    eager = op(qd, kd, pd, f)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for _ in range(2):
            torch.autograd.grad(op(qd, kd, pd, f), (qd, kd), (gq, gk))
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="lives on another stream"):
        with torch.cuda.graph(graph):
            op(qd, kd, pd, f)
    torch.autograd.grad(eager, (qd, kd), (gq, gk))  # the eager graph is still good
    del eager
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = op(qd, kd, pd, f)
        grads = torch.autograd.grad(out, (qd, kd), (gq, gk))
    with torch.no_grad():
        qd.copy_(qd * 2)
        gq.fill_(3.0)
        pd.add_(7)
    graph.replay()
    torch.cuda.synchronize()
    for x, y in zip((qd, kd), out):
        ref, size = R.rotary(x.detach().cpu(), pd.cpu(), f.cpu(), False)
        R.assert_within(y.detach(), ref, R.rotary_bound(ref, size, x.dtype))
    ref, size = R.rotary(gq.cpu(), pd.cpu(), f.cpu(), False, inverse=True)
    R.assert_within(grads[0], ref, R.rotary_bound(ref, size, qd.dtype))


def test_through_sdpa():
    """Rotary, then this package's causal SDPA, forward and gradient, as an attention layer runs them."""
    g = torch.Generator().manual_seed(8)
    x = [torch.randn([1, 70, h, 64], generator=g).to(torch.bfloat16).to(DEV).transpose(1, 2).requires_grad_()
         for h in (4, 2, 2)]
    pos, f = torch.arange(70, device=DEV), freqs(64).to(DEV)

    def layer(q, k, v):
        q, k = op(q, k, pos, f)
        return torch.nn.functional.scaled_dot_product_attention(q, k, v, is_causal=True, enable_gqa=True)

    up = torch.randn([1, 4, 70, 64], generator=g).to(torch.bfloat16).to(DEV)
    out = layer(*x)
    grads = torch.autograd.grad(out, x, up)
    y = [t.detach().cpu().double().requires_grad_() for t in x]
    rq, rk = (R.rotary(t, pos.cpu()[None], f.cpu(), False)[0] for t in y[:2])
    rk, rv = (t.repeat_interleave(2, 1) for t in (rk, y[2]))
    w = (rq @ rk.transpose(-1, -2)) / 8.0
    w = w.masked_fill(~torch.ones(70, 70).tril().bool(), -float("inf"))
    ref = torch.softmax(w, -1) @ rv
    want = torch.autograd.grad(ref, y, up.cpu().double())
    # bf16 in four places on the way (turned q and k, P, dS): 2^-8 each of the tensors' largest values
    for a, b in zip((out,) + grads, (ref,) + want):
        assert (a.detach().cpu().double() - b).abs().max() <= 4 * 2.0 ** -8 * b.abs().max()


@pytest.mark.parametrize("dtype,H,D", [(torch.bfloat16, 40, 128), (torch.float32, 3, 1024)])
@pytest.mark.parametrize("tokens", [147, 149, 295, 296, 601, 1183, 1187])
def test_tokens_around_the_choice_of_tokens_a_cta(dtype, H, D, tokens):
    q, k, pos = inputs(1, H, 1, tokens, D, dtype, seed=tokens)
    check(q, k, pos, freqs(D), False)


def test_one_tensor_as_queries_and_keys():
    """The gradient of a leaf that is both is the sum; an expanded gradient of a sum too."""
    g = torch.Generator().manual_seed(2)
    x = torch.randn([2, 3, 9, 64], generator=g)
    pos, f = torch.arange(9), freqs(64)
    leaf = x.to(DEV).requires_grad_()
    a, b = op(leaf, leaf, pos.to(DEV), f.to(DEV))
    assert torch.equal(a, b)
    (d,) = torch.autograd.grad(a.sum() + b.sum(), leaf)
    ref, size = R.rotary(torch.ones_like(x), pos[None], f, False, 1.0, inverse=True)
    bound = R.rotary_bound(ref, size, torch.float32)
    # twice one gradient: the sum of two equal floats is exact
    R.assert_within(d, 2 * ref, 2 * bound)
