"""torch.ops.rbln_attn.rotary_paged_kv_write and paged_kv_read: the write
against paged_kv_write (bit for bit where no angle turns) and float64, the
read-back bit for bit, and a run of both."""

import pytest
import torch

from tests import operator_refs as R

pytestmark = pytest.mark.gpu
DEV = "cuda"
FP8 = torch.float8_e4m3fn


@pytest.fixture(scope="module", autouse=True)
def _ext():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    import torch_rbln_b200  # noqa: F401


def setup(starts, S, Hkv, G, D, bs, dtype, cache, seed=0, bt_dtype=torch.int32, extra=1):
    g = torch.Generator().manual_seed(seed)
    B = len(starts)
    width = (max(starts) + S + bs - 1) // bs + extra
    nb = B * width + 3
    d = dict(B=B, S=S, Hkv=Hkv, G=G, D=D, bs=bs, dtype=dtype)
    d["bt"] = torch.randperm(nb, generator=g)[: B * width].reshape(B, width).to(bt_dtype)
    d["seq"] = torch.tensor(starts, dtype=torch.int32)
    d["q"] = torch.randn([B, Hkv, G, S, D], generator=g).to(dtype)
    d["k"] = (torch.randn([B, Hkv, 1, S, D], generator=g) * 2).to(dtype)
    d["v"] = (torch.randn([B, Hkv, 1, S, D], generator=g) * 0.3).to(dtype)
    if cache == FP8:
        d["kc"], d["vc"] = (torch.randn([nb, Hkv, 1, bs, D], generator=g).mul(100).clamp(-448, 448).to(FP8) for _ in "kv")
        d["ks"], d["vs"] = (torch.rand([nb, Hkv], generator=g) * 0.02 + 0.001 for _ in "kv")
    else:
        d["kc"], d["vc"] = (torch.randn([nb, Hkv, 1, bs, D], generator=g).to(cache) for _ in "kv")
        d["ks"] = d["vs"] = None
    return d


def dev(d):
    return {n: (x.to(DEV) if isinstance(x, torch.Tensor) else x) for n, x in d.items()}


def write(x, f, interleaved=False, mscale=1.0, q=None, k=None, v=None):
    return torch.ops.rbln_attn.rotary_paged_kv_write(
        x["q"] if q is None else q, x["k"] if k is None else k, x["v"] if v is None else v, x["kc"], x["vc"], x["seq"],
        x["bt"], x["bs"], f, interleaved, mscale, x["ks"], x["vs"])


def plain_write(x):
    torch.ops.rbln_attn.paged_kv_write(x["k"], x["v"], x["kc"], x["vc"], x["seq"], x["bt"], x["bs"], x["ks"], x["vs"])


def same(a, b, what):
    assert torch.equal(a.cpu().view(torch.uint8), b.cpu().view(torch.uint8)), what


def freqs(rot, base=10000.0):
    return (base ** (-2.0 * torch.arange(rot // 2, dtype=torch.float64) / rot)).float()


CASES = [  # starts, S, Hkv, G, D, bs, dtype, cache
    ([0, 5, 30], 41, 2, 3, 128, 16, torch.bfloat16, FP8),
    ([0, 5, 30], 41, 2, 3, 64, 16, torch.float16, FP8),
    ([15, 16, 17, 0], 1, 8, 4, 128, 16, torch.bfloat16, FP8),     # one token: ends, starts, joins a block
    ([7, 100], 300, 1, 1, 128, 128, torch.bfloat16, FP8),          # a block of eight 16-row tiles
    ([3], 700, 2, 2, 64, 256, torch.bfloat16, FP8),                # blocks past the angles a CTA keeps
    ([0, 8, 3], 20, 3, 5, 64, 8, torch.float16, FP8),
    ([0, 5, 30], 41, 2, 3, 128, 16, torch.bfloat16, torch.bfloat16),
    ([9, 64], 130, 2, 7, 64, 32, torch.float16, torch.float16),
    ([3], 700, 2, 2, 64, 256, torch.bfloat16, torch.bfloat16),
]


@pytest.mark.parametrize("case", CASES)
def test_no_angle_is_the_plain_write(case):
    """inv_freq 0: the caches and scales of paged_kv_write bit for bit, and q as it came."""
    d = setup(*case)
    a, b = dev(d), dev(d)
    out = write(a, torch.zeros(8, device=DEV))
    plain_write(b)
    assert torch.equal(out.cpu(), d["q"])
    for n in ("kc", "vc", "ks", "vs"):
        if d[n] is not None:
            same(a[n], b[n], n)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("case", CASES)
def test_turned_rows(case, interleaved):
    """q and a 16-bit cache's keys within one rounding; an fp8 cache's scales within float32 and its codes within half
    a step; values, untouched rows and untouched blocks as paged_kv_write leaves them."""
    d = setup(*case)
    B, Hkv, G, S, D, bs, dtype = (d[n] for n in ("B", "Hkv", "G", "S", "D", "bs", "dtype"))
    rot = D if interleaved else D // 2
    f, m = freqs(rot), 1.1
    x, p = dev(d), dev(d)
    out = write(x, f.to(DEV), interleaved, m)
    plain_write(p)
    pos = d["seq"].long()[:, None] + torch.arange(S)
    ref, size = R.rotary(d["q"].reshape(B, Hkv * G, S, D), pos, f, interleaved, m)
    R.assert_within(out.reshape(B, Hkv * G, S, D), ref, R.rotary_bound(ref, size, dtype), "q")
    same(x["vc"], p["vc"], "vcache")
    ref, size = R.rotary(d["k"][:, :, 0], pos, f, interleaved, m)
    kc, was = x["kc"].cpu(), d["kc"]
    touched = torch.zeros(was.shape[0], bs, dtype=torch.bool)
    scaled = torch.zeros(was.shape[0], dtype=torch.bool)
    for b in range(B):
        s0 = int(d["seq"][b])
        for j in range(s0 // bs, (s0 + S - 1) // bs + 1):
            n = int(d["bt"][b, j])
            lo, hi = max(s0, j * bs), min(s0 + S, (j + 1) * bs)
            held = max(0, min(s0 - j * bs, bs))
            rows, at = slice(lo - s0, hi - s0), slice(lo - j * bs, hi - j * bs)
            y, e = ref[b, :, rows], size[b, :, rows] * 2.0 ** -21
            touched[n, at] = True
            if d["ks"] is None:
                R.assert_within(kc[n, :, 0, at], y, R.rotary_bound(y, size[b, :, rows], dtype), "k")
                continue
            touched[n, :held] = True
            scaled[n] = True
            old = R.fp8_values(was[n:n + 1], d["ks"][n:n + 1])[0, :, 0, :held]
            amax = torch.cat([old, y], 1).abs().amax((1, 2)).clamp_min(1e-6)
            got = x["ks"][n].cpu().double()
            assert ((got * 448 - amax).abs() <= amax * 2.0 ** -20).all()
            both = torch.cat([old, y], 1) / got[:, None, None]
            codes = kc[n, :, 0, : held + y.shape[1]].double() if held else kc[n, :, 0, at].double()
            err = torch.cat([old.abs() * 2.0 ** -21, e], 1) / got[:, None, None]
            # half a step of e4m3 (2^-4 of a value, 2^-10 at least) around a value float32 has within err
            assert ((codes - both).abs() <= err + (both.abs() + err) * 2.0 ** -4 + 2.0 ** -10).all()
    keep = (~touched)[:, None, None, :, None].expand_as(was)
    assert torch.equal(kc.view(torch.uint8)[keep.expand_as(kc)] if d["ks"] is not None else kc[keep],
                       was.view(torch.uint8)[keep] if d["ks"] is not None else was[keep])
    if d["ks"] is not None:
        assert torch.equal(x["ks"].cpu()[~scaled], d["ks"][~scaled])
        same(x["vs"], p["vs"], "v scale")


@pytest.mark.parametrize("bt_dtype", [torch.int16, torch.int64])
def test_index_types_and_strided_inputs(bt_dtype):
    d = setup([0, 5], 19, 2, 2, 64, 16, torch.bfloat16, FP8, bt_dtype=bt_dtype)
    a, b = dev(d), dev(d)
    f = freqs(64).to(DEV)
    q, k, v = (torch.cat([b[n], b[n]], -1)[..., :64] for n in "qkv")  # every second 64 elements
    same(write(a, f), write(b, f, q=q, k=k, v=v), "q")
    for n in ("kc", "vc", "ks", "vs"):
        same(a[n], b[n], n)


def test_refused_rows_leave_the_cache():
    """A negative start, rows past the table's span, and a block outside the pool: q is turned, the cache left."""
    d = setup([0, 5, 3], 20, 2, 2, 64, 16, torch.bfloat16, FP8, extra=0)
    d["seq"] = torch.tensor([-4, 100, 3], dtype=torch.int32)
    d["bt"][2] = 10 ** 6
    x = dev(d)
    out = write(x, freqs(64).to(DEV))
    pos = d["seq"].long()[:, None] + torch.arange(20)
    ref, size = R.rotary(d["q"].reshape(3, 4, 20, 64), pos, freqs(64), False)
    R.assert_within(out.reshape(3, 4, 20, 64), ref, R.rotary_bound(ref, size, torch.bfloat16))
    for n in ("kc", "vc", "ks", "vs"):
        same(x[n], d[n], n)


def test_device_flags():
    import ctypes

    from torch_rbln_b200 import cabi

    for seq, block, want in ((-1, 0, cabi.DEVERR_SEQ_RANGE), (30, 0, cabi.DEVERR_SEQ_RANGE),
                             (0, 99, cabi.DEVERR_BLOCK_ID_RANGE), (0, 0, 0)):
        d = setup([0], 8, 1, 1, 64, 16, torch.bfloat16, FP8, extra=1)
        d["seq"][:] = seq
        d["bt"][:] = block
        x = dev(d)
        out, f = torch.empty_like(x["q"]), freqs(64).to(DEV)
        p, keep = cabi.paged_params(x["q"], x["k"], x["v"], x["kc"], x["vc"], x["seq"], x["bt"], 16, 1.0,
                                    k_scale=x["ks"], v_scale=x["vs"], out=out)
        r = cabi.RotaryParams()
        r.rotary_dim, r.inv_freq, r.mscale = 64, f.data_ptr(), 1.0
        err = torch.zeros(1, dtype=torch.int32, device=DEV)
        p.error_flags = err.data_ptr()
        stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
        assert cabi.lib().rbln_rotary_paged_kv_write(ctypes.byref(p), ctypes.byref(r), stream) == cabi.OK
        assert int(err.item()) == want


# ------------------------------------------------------------------ read-back


def read(x, lens, most, dtype=None):
    return torch.ops.rbln_attn.paged_kv_read(x["kc"], x["vc"], lens, x["bt"], x["bs"], most, x["ks"], x["vs"], dtype)


def plain_read(cache, scale, lens, bt, bs, most, dtype):
    B, Hkv, D = len(lens), cache.shape[1], cache.shape[-1]
    out = torch.zeros([B, Hkv, 1, most, D])
    for b in range(B):
        for t in range(max(0, min(int(lens[b]), most, bt.shape[1] * bs))):
            n = int(bt[b if bt.shape[0] > 1 else 0, t // bs])
            if 0 <= n < cache.shape[0]:
                row = cache[n, :, 0, t % bs].float()
                out[b, :, 0, t] = row if scale is None else row * scale[n][:, None]
    return out.to(dtype)


@pytest.mark.parametrize("cache", [FP8, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dtype", [None, torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("D,bs", [(64, 16), (128, 8), (128, 256)])
def test_read_back(cache, dtype, D, bs):
    """Lengths 0, 1, inside and at the ends of blocks, past max_len and past the span; bit for bit."""
    d = setup([150] * 6, 1, 2, 1, D, bs, torch.bfloat16, cache, seed=D + bs, extra=0)
    span = d["bt"].shape[1] * bs
    lens = torch.tensor([0, 1, bs, 77, 150, span + 9], dtype=torch.int32)
    most = 131
    x = dev(d)
    got = read(x, lens.to(DEV), most, dtype)
    want = dtype or (torch.bfloat16 if cache == FP8 else cache)
    for g, c, s in zip(got, (d["kc"], d["vc"]), (d["ks"], d["vs"])):
        assert torch.equal(g.cpu(), plain_read(c, s, lens, d["bt"], bs, most, want))


def test_read_back_bad_blocks_and_shared_table():
    d = setup([60, 60], 1, 2, 1, 64, 16, torch.bfloat16, FP8)
    d["bt"] = torch.tensor([[3, -1, 2, 999]], dtype=torch.int64)
    lens = torch.tensor([64, -5], dtype=torch.int32)
    x = dev(d)
    got = read(x, lens.to(DEV), 70)
    for g, c, s in zip(got, (d["kc"], d["vc"]), (d["ks"], d["vs"])):
        assert torch.equal(g.cpu(), plain_read(c, s, lens, d["bt"], 16, 70, torch.bfloat16))
    assert read(x, lens.to(DEV), 0)[0].shape == (2, 2, 1, 0, 64)
    k, v = read(x, lens[:0].to(DEV), 5)
    assert k.shape == (0, 2, 1, 5, 64)


def test_read_back_offsets_past_32_bits():
    """A pool of over 2^31 elements: the last block's rows come back."""
    bs, D, Hkv = 256, 128, 8
    nb = (1 << 31) // (bs * D * Hkv) + 2
    kc = torch.zeros([nb, Hkv, 1, bs, D], dtype=torch.uint8, device=DEV).view(FP8)
    vc = torch.zeros([nb, Hkv, 1, bs, D], dtype=torch.uint8, device=DEV).view(FP8)
    last = torch.randint(0, 120, [Hkv, 1, bs, D], dtype=torch.uint8, device=DEV)
    kc.view(torch.uint8)[-1] = last
    vc.view(torch.uint8)[-1] = last.flip(0)
    sc = torch.full([nb, Hkv], 0.5, device=DEV)
    bt = torch.tensor([[nb - 1]], dtype=torch.int32, device=DEV)
    k, v = torch.ops.rbln_attn.paged_kv_read(kc, vc, torch.tensor([bs], device=DEV), bt, bs, bs, sc, sc, torch.float32)
    assert torch.equal(k[0], last.view(FP8).float() * 0.5)
    assert torch.equal(v[0], last.flip(0).view(FP8).float() * 0.5)
    # the write reaches it too
    q = torch.ones([1, Hkv, 1, 3, D], dtype=torch.bfloat16, device=DEV)
    torch.ops.rbln_attn.rotary_paged_kv_write(q, q, q, kc, vc, torch.zeros(1, dtype=torch.int32, device=DEV), bt, bs,
                                              torch.zeros(32, device=DEV), False, 1.0, sc, sc)
    k, _ = torch.ops.rbln_attn.paged_kv_read(kc, vc, torch.tensor([3], device=DEV), bt, bs, 3, sc, sc, torch.float32)
    assert torch.equal(k, torch.ones_like(k))


def test_captured_step_on_another_stream():
    """A write and a read-back captured on a side stream, replayed with moved positions and new rows."""
    d = setup([5, 40], 1, 2, 2, 64, 16, torch.bfloat16, FP8, extra=1)
    x, e = dev(d), dev(d)
    f = freqs(64).to(DEV)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        write(dev(d), f), read(x, x["seq"] + 1, 50)
        graph = torch.cuda.CUDAGraph()
        s.synchronize()
        with torch.cuda.graph(graph, stream=s):
            out = write(x, f)
            got = read(x, x["seq"] + 1, 50)
    for step in range(3):
        for y in (x, e):
            y["seq"].copy_(d["seq"] + step)
            y["k"].copy_(d["k"].to(DEV) * (step + 1))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, write(e, f))
        for g, w in zip(got, read(e, e["seq"] + 1, 50)):
            assert torch.equal(g, w)
    for n in ("kc", "vc", "ks", "vs"):
        same(x[n], e[n], n)


@pytest.mark.parametrize("cache", [FP8, torch.bfloat16])
def test_nothing_to_write(cache):
    """No tokens, and no sequences: empty queries, the cache left."""
    d = setup([4, 9], 1, 2, 3, 64, 16, torch.bfloat16, cache)
    x = dev(d)
    for q, k, x["seq"], x["bt"] in ((x["q"][:, :, :, :0], x["k"][:, :, :, :0], x["seq"], x["bt"]),
                                    (x["q"][:0], x["k"][:0], x["seq"][:0], x["bt"][:0])):
        assert write(x, freqs(64).to(DEV), q=q, k=k, v=k).shape == q.shape
    for n in ("kc", "vc"):
        same(x[n], d[n], n)


@pytest.mark.parametrize("Hkv,G", [(1, 71), (5, 40), (17, 1)])
@pytest.mark.parametrize("S", [1, 37])
def test_odd_heads_are_the_rotation_and_the_write(Hkv, G, S):
    """Queries bit for bit the rotary op's; a 16-bit cache's rows those of its keys and the plain write."""
    d = setup([11, 0], S, Hkv, G, 64, 16, torch.bfloat16, torch.bfloat16)
    a, b = dev(d), dev(d)
    f = freqs(32).to(DEV)
    out = write(a, f)
    pos = b["seq"].long()[:, None] + torch.arange(S, device=DEV)
    q, k = torch.ops.rbln_attn.rotary(b["q"].flatten(1, 2), b["k"].flatten(1, 2), pos, f)
    assert torch.equal(out.flatten(1, 2), q)
    b["k"] = k.reshape(b["k"].shape)
    plain_write(b)
    for n in ("kc", "vc"):
        same(a[n], b[n], n)


def test_expanded_inputs_and_two_streams_at_once():
    """Inputs that broadcast one row, and two pools written and read on two streams: as one after the other."""
    f = freqs(128).to(DEV)
    pools = [setup([7, 300], 200, 2, 4, 128, 16, torch.bfloat16, FP8, seed=s) for s in (1, 2)]
    first, then = [dev(d) for d in pools], [dev(d) for d in pools]
    for x in first + then:
        x["q"] = x["q"][:, :, :1].expand(-1, -1, 4, -1, -1)
        x["v"] = x["v"][:, :1].expand(-1, 2, -1, -1, -1)
    lens = [x["seq"] + 200 for x in first]
    want = [(write(x, f), *read(x, n, 500)) for x, n in zip(first, lens)]
    streams = [torch.cuda.Stream() for _ in pools]
    torch.cuda.synchronize()
    got = []
    for x, n, s in zip(then, lens, streams):
        with torch.cuda.stream(s):
            got.append((write(x, f), *read(x, n, 500)))
    torch.cuda.synchronize()
    for w, g in zip(want, got):
        assert all(torch.equal(x, y) for x, y in zip(w, g))
