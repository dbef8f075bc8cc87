"""paged_causal_attn_prefill_kvfp8: caches and scales bit for bit the plain
write, the output within the bounds of tests/operator_refs.py of float64
attention over what the cache then holds."""

import math

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


def setup(starts, S, Hkv, G, D, bs, dtype=torch.bfloat16, seed=0, kstd=1.0, vstd=0.5, bt_dtype=torch.int32, extra=1,
          spread=0.0):
    """Random pool with scales a block and head; `spread`: the V scales' spread in binades between blocks."""
    g = torch.Generator().manual_seed(seed)
    B = len(starts)
    width = (max(max(starts), 0) + S + bs - 1) // bs + extra
    nb = B * width + 3
    d = dict(S=S, bs=bs)
    d["bt"] = torch.randperm(nb, generator=g)[: B * width].reshape(B, width).to(bt_dtype)
    d["seq"] = torch.tensor(starts, dtype=torch.int32).reshape(B, 1)
    d["q"] = torch.randn([B, Hkv, G, S, D], generator=g).to(dtype)
    d["k"] = (torch.randn([B, Hkv, 1, S, D], generator=g) * kstd).to(dtype)
    d["v"] = (torch.randn([B, Hkv, 1, S, D], generator=g) * vstd).to(dtype)

    def pool(std):
        x = torch.randn([nb, Hkv, 1, bs, D], generator=g) * std
        x = x * torch.exp2(spread * (torch.rand([nb, Hkv, 1, 1, 1], generator=g) - 0.5))
        sc = (x.abs().amax((2, 3, 4)).clamp_min(1e-6) / 448).contiguous()
        return (x / sc[:, :, None, None, None]).clamp(-448, 448).to(FP8), sc

    d["kc"], d["ks"] = pool(kstd)
    d["vc"], d["vs"] = pool(vstd)
    d["scale"] = torch.tensor(1.0 / math.sqrt(D))
    return d


def dev(d):
    return {n: (x.to(DEV) if isinstance(x, torch.Tensor) and n != "scale" else x) for n, x in d.items()}


def run(x, both=False, mask=None, rows=True):
    import torch_rbln_b200 as tr

    return tr.paged_causal_attn_prefill_kvfp8(
        x["q"], x["k"] if rows else None, x["v"] if rows else None, x["kc"], x["vc"], x["ks"], x["vs"], x["seq"],
        x["scale"], x["bt"], x["bs"], both, mask)


def reference(d, both=False, mask=None, rows=True):
    """(out, bound) in float64 from the oracle's cache; d's caches and scales are updated in place."""
    B, Hkv, G, S, D = d["q"].shape
    bs, bt = d["bs"], d["bt"].long()
    span = bt.shape[1] * bs
    if rows:
        R.write_reciprocal(d["k"], d["v"], d["kc"], d["vc"], d["seq"], bt, bs, d["ks"], d["vs"])
    outs, bounds = [], []
    t = torch.arange(span)
    for b in range(B):
        n = int(d["seq"][b])
        blk = bt[b][t // bs]
        ok = (blk >= 0) & (blk < d["kc"].shape[0])
        blk = blk.clamp(0, d["kc"].shape[0] - 1)
        K, V = ((c[blk, :, 0, t % bs].double() * s[blk].double()[:, :, None]).transpose(0, 1)
                for c, s in ((d["kc"], d["ks"]), (d["vc"], d["vs"])))
        end = torch.full([S, 1], n + S) if both else n + 1 + torch.arange(S)[:, None]
        keep = (t < end) & ok if n >= 0 else torch.zeros(S, span, dtype=torch.bool)
        if mask is not None:
            m = torch.zeros(span, dtype=torch.bool)
            row = mask[b if mask.shape[0] > 1 else 0]
            L = min(span, row.numel())
            m[:L] = row[:L] > 0
            keep = keep & m
        K = torch.where(keep.any(0)[:, None], K, torch.zeros_like(K))  # unseen keys may hold anything
        out, A, e = R.attention(d["q"][b], K, V, keep, float(d["scale"]))
        vmax = V[:, keep.any(0)].abs().max().item() if keep.any() else 0.0
        outs.append(out)
        bounds.append(R.attention_bound(out, A, e, span, vmax, d["q"].dtype))
    return torch.stack(outs), torch.stack(bounds)


def check(d, both=False, mask=None, rows=True, x=None):
    x = dev(d) if x is None else x
    out = run(x, both, None if mask is None else mask.to(DEV), rows)
    torch.cuda.synchronize()
    ref, bound = reference(d, both, mask, rows)
    R.assert_within(out, ref, bound)
    for n in ("kc", "vc", "ks", "vs"):
        assert torch.equal(x[n].cpu().view(torch.uint8), d[n].view(torch.uint8)), n
    return out


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("S,G", [(1, 1), (1, 8), (2, 4), (4, 4), (1, 16), (3, 5), (5, 4), (17, 3), (40, 8), (64, 4), (77, 1),
                                 (150, 4), (300, 2), (3, 128)])
def test_lengths_and_groups(dtype, D, S, G):
    """From one token to several row tiles, rows that do and do not fill a tile; contexts from none on."""
    check(setup([0, 1, 37, 200, 511], S, 2, G, D, 16, dtype, seed=S * G))


@pytest.mark.parametrize("bs", [8, 16, 32, 64, 128, 256])
@pytest.mark.parametrize("S", [1, 5, 70])
def test_block_sizes(bs, S):
    check(setup([0, bs - 1, bs, 3 * bs + 5], S, 2, 4, 128, bs, seed=bs))


@pytest.mark.parametrize("S", [1, 3, 33, 130])
def test_both_ways(S):
    check(setup([0, 5, 290], S, 2, 4, 64, 16), both=True)


@pytest.mark.parametrize("mdt", [torch.bool, torch.float32, torch.bfloat16])
@pytest.mark.parametrize("S", [1, 4, 50])
def test_position_mask(mdt, S):
    """Dropped keys, among them whole tiles and blocks; a mask shorter and longer than the span; a broadcast one."""
    d = setup([10, 200, 400], S, 2, 4, 128, 16)
    g = torch.Generator().manual_seed(S)
    for rows, L in ((3, 470), (3, 300), (1, 2000)):
        m = torch.rand([rows, L], generator=g) > 0.3
        m[:, 0] = True
        m[:, 16:180] = False
        mask = m if mdt == torch.bool else (m.to(mdt) * 2 - 1)
        check({n: (v.clone() if isinstance(v, torch.Tensor) else v) for n, v in d.items()}, mask=mask)


@pytest.mark.parametrize("S", [1, 4, 60])
def test_rows_that_see_nothing(S):
    """A mask that drops a sequence's every key: NaN there, the others untouched; a negative start likewise."""
    d = setup([30, 40, -1], S, 2, 4, 64, 16)
    mask = torch.ones([3, 120], dtype=torch.bool)
    mask[1] = False
    out = check(d, mask=mask)
    assert torch.isnan(out[1]).all() and torch.isnan(out[2]).all() and not torch.isnan(out[0]).any()


@pytest.mark.parametrize("low", [torch.finfo(torch.float32).min, -float("inf"), float("nan")])
def test_mask_values(low):
    """Any value that is not above zero drops a key: the type's lowest, -inf, NaN, zero."""
    d = setup([100], 9, 1, 4, 64, 16)
    mask = torch.ones([1, 112])
    mask[0, 3:40] = low
    mask[0, 50] = 0.0
    check(d, mask=mask)


@pytest.mark.parametrize("S", [1, 6, 70])
def test_bad_bytes_and_scales_in_unseen_places(S):
    """NaN codes behind the last row and at masked positions, NaN scales of blocks that are not in use, and blocks
    outside the pool: none is seen."""
    d = setup([100, 33], S, 2, 4, 128, 16, extra=2)
    used = torch.zeros(d["kc"].shape[0], dtype=torch.bool)
    mask = torch.ones([2, 400], dtype=torch.bool)
    mask[:, 20:27] = False
    for b in range(2):
        n = int(d["seq"][b])
        for j in range(d["bt"].shape[1]):
            p = int(d["bt"][b, j])
            rows = torch.arange(16) + 16 * j
            used[p] = 16 * j < n + S
            for c in (d["kc"], d["vc"]):
                bad = (rows >= n + S) | ((rows >= 20) & (rows < 27) & (rows < n))
                c.view(torch.uint8)[p][:, :, bad] = 0x7f
    d["ks"][~used] = float("nan")
    d["vs"][~used] = float("nan")
    # the write's amax over held rows skips NaN codes as fmaxf does; keep those out of the touched block
    first = 16 * (int(d["seq"][1]) // 16)
    assert first >= 27
    x = dev(d)
    out = run(x, mask=mask.to(DEV))
    for n in ("kc", "vc"):
        v = d[n].view(torch.uint8)
        v[v == 0x7f] = 0
    d["ks"][~used] = d["vs"][~used] = 1.0
    ref, bound = reference(d, mask=mask)
    R.assert_within(out, ref, bound)


@pytest.mark.parametrize("S", [1, 40])
def test_blocks_outside_the_pool_are_not_seen(S):
    d = setup([200, 90], S, 2, 4, 64, 16)
    d["bt"][0, 3], d["bt"][0, 7], d["bt"][1, 0] = -1, 10 ** 6, d["kc"].shape[0]
    check(d)


def test_writes_past_the_span_are_refused():
    """As paged_kv_write: nothing of that sequence is written; its queries see what the table holds."""
    d = setup([20, 4], 13, 1, 4, 64, 16, extra=0)
    d["seq"][0] = 30  # 30 + 13 is past the 3-block span
    d["bt"] = d["bt"][:, :2].contiguous()
    check(d)


@pytest.mark.parametrize("S", [1, 4, 50])
def test_rows_already_written(S):
    """k and v None: the rows are taken from the cache as they are, the same output as with them."""
    d = setup([0, 61, 200], S, 2, 4, 128, 16)
    x = dev(d)
    first = run(x)
    again = run(x, rows=False)
    assert torch.equal(first.view(torch.int16), again.view(torch.int16))
    reference(d)
    check(d, rows=False, x=x)


@pytest.mark.parametrize("S,G", [(1, 1), (4, 4), (3, 12), (48, 8), (100, 4)])
def test_long_contexts_are_split_and_joined(S, G):
    """One long sequence beside short ones: its keys are shared among many CTAs and the parts joined."""
    check(setup([6000, 3, 0, 700], S, 2, G, 128, 16, seed=5))
    check(setup([9000], S, 1, G, 64, 32, seed=6))


def test_many_sequences():
    """More (sequence, row tile) items than a CTA keeps a prefix of."""
    g = torch.Generator().manual_seed(1)
    starts = torch.randint(0, 40, [1100], generator=g).tolist()
    check(setup(starts, 9, 1, 8, 64, 8, extra=0))


@pytest.mark.parametrize("S", [1, 4, 40])
@pytest.mark.parametrize("vstd", [1e-4, 3e3])
def test_small_and_large_values(S, vstd):
    """V scales of 1e-6 and of 30: relative precision is kept."""
    check(setup([300, 11], S, 2, 4, 128, 16, vstd=vstd))


@pytest.mark.parametrize("S", [1, 4, 40])
def test_scales_that_differ_between_blocks(S):
    """V scales over 12 binades between blocks, growing and falling along a sequence."""
    check(setup([700, 300], S, 2, 4, 128, 16, spread=12.0))


@pytest.mark.parametrize("size", [2.0 ** -100, 2.0 ** 60])
@pytest.mark.parametrize("S", [2, 40])
def test_query_sizes(size, S):
    """bf16 queries far outside f16's range (the softmax scale brings the scores back)."""
    d = setup([90], S, 2, 4, 64, 16)
    d["q"] = (d["q"].float() * size).to(torch.bfloat16)
    d["scale"] = torch.tensor(1.0 / 8 / size)
    check(d)


def test_scale_forms():
    """A device tensor, a negative and a zero softmax scale."""
    for s in (0.3, -0.2, 0.0):
        for S in (2, 40):
            d = setup([150, 20], S, 2, 4, 64, 16)
            d["scale"] = torch.tensor(s)
            x = dev(d)
            x["scale"] = torch.tensor([s], device=DEV)
            check(d, x=x)


@pytest.mark.parametrize("bt_dtype", [torch.int16, torch.int64])
def test_index_types_and_strided_inputs(bt_dtype):
    d = setup([77, 5], 7, 2, 3, 64, 16, bt_dtype=bt_dtype)
    x = dev(d)
    for n in "qkv":
        x[n] = torch.cat([x[n], x[n]], -1)[..., :64]
    x["bt"] = torch.cat([x["bt"], x["bt"]], 1)[:, : d["bt"].shape[1]]
    wide = torch.empty([d["ks"].shape[0], 5], device=DEV)
    wide[:, 1:3] = x["ks"]
    x["ks"] = wide[:, 1:3]
    wide = torch.empty([d["ks"].shape[0], 5], device=DEV)
    wide[:, 1:3] = x["vs"]
    x["vs"] = wide[:, 1:3]
    out = run(x)
    ref, bound = reference(d)
    R.assert_within(out, ref, bound)
    assert torch.equal(x["ks"].cpu(), d["ks"])


def test_padded_head_dimension():
    """A cache whose rows are wider than head_dim, and views of a [2, ...] unified pool."""
    d = setup([50, 9], 6, 2, 4, 64, 16)
    x = dev(d)
    nb = d["kc"].shape[0]
    pool = torch.zeros([2, nb, 2, 1, 16, 128], dtype=torch.uint8, device=DEV).view(FP8)
    for i, n in enumerate(("kc", "vc")):
        pool.view(torch.uint8)[i, ..., :64] = x[n].view(torch.uint8)
    x["kc"], x["vc"] = pool[0], pool[1]
    out = run(x)
    ref, bound = reference(d)
    R.assert_within(out, ref, bound)
    assert torch.equal(pool[0][..., :64].cpu().float(), d["kc"].float())


def test_empty_batch():
    d = setup([5], 3, 2, 4, 64, 16)
    x = dev(d)
    for n in ("q", "k", "v", "seq", "bt"):
        x[n] = x[n][:0]
    assert run(x).shape == (0, 2, 4, 3, 64)


def test_two_streams_at_once():
    """Two calls on two streams, each with its own workspace."""
    ds = [setup([3000, 100], 4, 2, 4, 128, 16, seed=s) for s in (1, 2)]
    xs = [dev(d) for d in ds]
    streams = [torch.cuda.Stream() for _ in ds]
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(3):
        for i, (x, s) in enumerate(zip(xs, streams)):
            with torch.cuda.stream(s):
                outs[i].append(run(x))
    torch.cuda.synchronize()
    for d, o in zip(ds, outs):
        ref, bound = reference(d)
        for out in o:
            R.assert_within(out, ref, bound)


@pytest.mark.parametrize("S", [1, 4, 40])
def test_captured_and_replayed(S):
    """Two graphs of one step, replayed in turn as the sequences grow, the caches shared."""
    d = setup([100, 37, 0], S, 2, 4, 128, 16, extra=20)
    x = dev(d)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        run(dev(d))
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = run(x)
        graphs.append((graph, out))
    for step in range(4):
        x["seq"].copy_(d["seq"])
        x["k"].copy_(d["k"])
        torch.cuda.synchronize()
        graph, out = graphs[step % 2]
        graph.replay()
        torch.cuda.synchronize()
        ref, bound = reference(d)
        R.assert_within(out, ref, bound)
        for n in ("kc", "vc", "ks", "vs"):
            assert torch.equal(x[n].cpu().view(torch.uint8), d[n].view(torch.uint8)), n
        d["seq"] += S
        d["k"] = (d["k"].float() * 1.5).to(d["k"].dtype)


def test_a_served_prompt():
    """A prompt in chunks, then drafted tokens, then single tokens, through rotary_paged_kv_write and attention over
    the cache, beside float64 attention over the cache as it is read back."""
    from torch_rbln_b200 import rotary_frequencies

    g = torch.Generator().manual_seed(2)
    B, Hkv, G, D, bs = 2, 2, 4, 128, 16
    width = 20
    nb = B * width + 1
    kc, vc = (torch.zeros([nb, Hkv, 1, bs, D], dtype=torch.uint8, device=DEV).view(FP8) for _ in "kv")
    ks, vs = (torch.ones([nb, Hkv], device=DEV) for _ in "kv")
    bt = torch.randperm(nb, generator=g)[: B * width].reshape(B, width).to(torch.int32).to(DEV)
    f, m = rotary_frequencies(D, 10000.0, "yarn", 4.0, 128, device=DEV)
    seq = torch.zeros([B], dtype=torch.int32, device=DEV)
    scale = torch.tensor(D ** -0.5)
    for S in (100, 61, 5, 1, 1, 3, 1):
        q, k, v = (torch.randn([B, Hkv, h, S, D], generator=g).to(torch.bfloat16).to(DEV) for h in (G, 1, 1))
        rq = torch.ops.rbln_attn.rotary_paged_kv_write(q, k, v, kc, vc, seq, bt, bs, f, False, m, ks, vs)
        out = torch.ops.rbln_custom_ops.paged_causal_attn_prefill_kvfp8(rq, None, None, kc, vc, ks, vs, seq, scale, bt,
                                                                       bs, False)
        lens = seq + S
        K, V = torch.ops.rbln_attn.paged_kv_read(kc, vc, lens, bt, bs, int(lens.max()), ks, vs, torch.float32)
        for b in range(B):
            n = int(seq[b])
            t = torch.arange(n + S)
            keep = t <= n + torch.arange(S)[:, None]
            Kb, Vb = K[b, :, 0, : n + S].cpu(), V[b, :, 0, : n + S].cpu()
            ref, A, e = R.attention(rq[b].cpu(), Kb, Vb, keep, float(scale))
            # the read-back itself is rounded once to float32: 2^-24 of each key and value
            bound = R.attention_bound(ref, A, e, n + S, Vb.abs().max().item(), torch.bfloat16) + A * (1 + 2 * e) * 2.0 ** -23
            R.assert_within(out[b], ref, bound, f"S = {S}")
            pos = (n + torch.arange(S))[None]
            want, size = R.rotary(q[b].cpu().reshape(1, Hkv * G, S, D), pos, f.cpu(), False, m)
            R.assert_within(rq[b].reshape(1, Hkv * G, S, D), want, R.rotary_bound(want, size, torch.bfloat16))
        seq = seq + S


def test_scales_are_those_of_torch_and_near_the_cache_writes():
    """The scales are what torch computes on the GPU for amax / 448.0, and within one unit in the last place of
    paged_kv_write's, which divides."""
    d = setup([0, 0, 0], 64, 4, 2, 64, 16, seed=11)
    x, y = dev(d), dev(d)
    run(x)
    torch.ops.rbln_attn.paged_kv_write(y["k"], y["v"], y["kc"], y["vc"], y["seq"], y["bt"], y["bs"], y["ks"], y["vs"])
    differ = 0
    for b in range(3):
        for j in range(4):
            p = int(d["bt"][b, j])
            amax = x["k"][b, :, 0, 16 * j: 16 * j + 16].float().abs().amax((1, 2))
            assert torch.equal(x["ks"][p], amax.clamp_min(1e-6) / 448.0)
            bits = (x["ks"][p].view(torch.int32) - y["ks"][p].view(torch.int32)).abs()
            assert int(bits.max()) <= 1
            differ += int(bits.sum())
    assert differ > 0


@pytest.mark.parametrize("S", [1, 4, 40])
def test_scales_that_are_not_numbers(S):
    """A NaN scale of a block that is seen gives NaN, for K and for V; of a block that the mask drops, nothing."""
    for name in ("ks", "vs"):
        d = setup([200, 90], S, 2, 4, 64, 16)
        d[name][d["bt"][0, 2].item()] = float("nan")  # keys 32 to 47 of sequence 0
        x = dev(d)
        out = run(x)
        assert torch.isnan(out[0]).all() and not torch.isnan(out[1]).any()
        mask = torch.ones([2, 300], dtype=torch.bool)
        mask[0, 32:48] = False
        out = run(x, mask=mask.to(DEV), rows=False)
        assert not torch.isnan(out).any()


@pytest.mark.parametrize("S", [1, 4, 40])
def test_bad_query_rows_stay_alone(S):
    """Inf and NaN in one query row: NaN in its output, no other touched. And the largest finite bf16 queries."""
    d = setup([150], S, 2, 4, 64, 16)
    clean = run(dev(d))
    d["q"][0, 1, 2, S - 1, 5] = float("inf")
    d["q"][0, 0, 1, 0, 7] = float("nan")
    x = dev(d)
    out = run(x)
    assert torch.isnan(out[0, 0, 1, 0]).all()
    keep = torch.ones([1, 2, 4, S], dtype=torch.bool)
    keep[0, 1, 2, S - 1] = keep[0, 0, 1, 0] = False
    assert torch.equal(out[keep.to(DEV)], clean[keep.to(DEV)])
    d = setup([90], S, 2, 4, 64, 16)
    big = torch.finfo(torch.bfloat16).max
    d["q"] = (d["q"].float() / 8 * big).clamp(-big, big).to(torch.bfloat16)
    d["scale"] = torch.tensor(0.25 * 2.0 ** -126)
    assert not torch.isnan(run(dev(d))).any()


@pytest.mark.parametrize("S", [1, 4, 40])
def test_softmax_scales_at_the_ends(S):
    """NaN gives NaN; zero the mean of the keys, for the largest finite queries too."""
    d = setup([150], S, 2, 4, 64, 16)
    d["scale"] = torch.tensor(float("nan"))
    assert torch.isnan(run(dev(d))).all()
    for big in (False, True):
        d = setup([150], S, 2, 4, 64, 16)
        d["scale"] = torch.tensor(0.0)
        x = dev(d)
        if big:
            x["q"] = torch.full_like(x["q"], torch.finfo(torch.bfloat16).max)
        out = run(x)
        d["q"].zero_()
        want, bound = reference(d)
        assert ((out.double().cpu() - want).abs() <= bound).all()


@pytest.mark.parametrize("S", [1, 4, 40])
@pytest.mark.parametrize("both", [False, True])
def test_lengths_past_the_table(S, both):
    """Rows that are there already and a length of up to 2^31 - 1: every key of the table is seen, none behind it."""
    d = setup([100, 100], S, 2, 4, 64, 16)
    x = dev(d)
    span = x["bt"].shape[1] * 16
    x["seq"] = torch.full_like(x["seq"], span)
    want = run(x, both, rows=False)
    x["seq"] = torch.full_like(x["seq"], 2**31 - 1)
    assert torch.equal(run(x, both, rows=False), want)
