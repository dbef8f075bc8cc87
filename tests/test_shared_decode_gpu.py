"""Decode over a shared prefix on B200 against float64, with bounds counted in the roundings that its kernels make."""

import ctypes

import pytest
import torch

from tests import page_refs, shared_refs as ref

pytestmark = pytest.mark.gpu

BF, F16 = torch.bfloat16, torch.float16


@pytest.fixture(scope="module", autouse=True)
def _package():
    import torch_rbln_b200  # noqa: F401


SHAPES = [  # D, bs, type, Hkv, G
    (128, 16, BF, 2, 4), (64, 8, F16, 1, 7), (128, 128, F16, 3, 1), (64, 32, BF, 2, 16), (128, 64, BF, 1, 8),
    (128, 256, BF, 2, 5), (64, 16, BF, 4, 2),
]


@pytest.mark.parametrize("D,bs,dtype,Hkv,G", SHAPES)
@pytest.mark.parametrize("shared", [1, 127, 128, 129, 700])
def test_one_group(D, bs, dtype, Hkv, G, shared):
    own = [1, 2, 17, 128, 130, 5, 64, 300, 16]
    ref.check(ref.inputs(D, bs, dtype, Hkv, G, len(own), [0, len(own)], [shared], own))


@pytest.mark.parametrize("D,bs,dtype,Hkv,G", SHAPES)
def test_many_rows(D, bs, dtype, Hkv, G):
    """More rows than one, two and four tiles of 128 hold, and a last tile of one row."""
    n = 4 * (128 // G) + 1
    ref.check(ref.inputs(D, bs, dtype, Hkv, G, n, [0, n], [260], [1 + b % 19 for b in range(n)]))


@pytest.mark.parametrize("sizes", [[1], [1, 1, 1], [5, 0, 40, 1, 33], [70, 3, 64], [0, 0, 7]])
@pytest.mark.parametrize("D,bs,dtype,Hkv,G", SHAPES[:3])
def test_several_groups(D, bs, dtype, Hkv, G, sizes):
    B = sum(sizes)
    starts = [sum(sizes[:i]) for i in range(len(sizes) + 1)]
    lens = [(37 * i * i + 90 * i + 5) % 900 for i in range(len(sizes))]
    ref.check(ref.inputs(D, bs, dtype, Hkv, G, B, starts, lens, [1 + 13 * b % 50 for b in range(B)]))


def test_rows_outside_groups_and_missing_rows():
    own = [3, 40, None, 7, 1, None, 200, 12, 90, 4]
    ref.check(ref.inputs(128, 16, BF, 2, 4, 10, [2, 5, 8], [300, 33], own))
    ref.check(ref.inputs(128, 16, BF, 2, 4, 10, [0, 10], [130], [None] * 10))
    ref.check(ref.inputs(128, 16, BF, 2, 4, 10, [0], [], own))  # no groups at all


def test_new_position_below_the_shared_length():
    """Such a row is read through its own table alone, its new token included; the others are not disturbed."""
    x = ref.inputs(64, 16, BF, 2, 4, 6, [0, 6], [200], [10, 20, 30, 40, 50, 60], poison=False)
    free = x["kcache"].shape[0]
    more = torch.randn(4, *x["kcache"].shape[1:]).to(BF)
    x["kcache"], x["vcache"] = torch.cat([x["kcache"], more]), torch.cat([x["vcache"], more * 0.5])
    x["block_table"][3] = -1
    x["block_table"][3, :4] = torch.arange(free, free + 4)
    x["seq"][3] = 50
    ref.check(x)


def test_shared_length_zero_negative_and_past_the_span():
    for n, seq in ((0, None), (-7, None), (10 ** 6, None), (64, 64), (64, 900)):
        x = ref.inputs(128, 16, F16, 1, 4, 5, [0, 5], [40], [24] * 5, poison=False)
        x["shared_lens"][0] = n
        if seq is not None:  # past the span: nothing is written, all positions are shared
            x["seq"][:] = seq
        ref.check(x, f"{n} {seq}")


@pytest.mark.parametrize("D,bs,shared,B", [(64, 16, 200, 6), (128, 16, 700, 40), (128, 128, 6000, 70), (64, 8, 3000, 300)])
def test_new_positions_in_shared_pages(D, bs, shared, B):
    """New tokens that go to pages of the group's shared positions, the first sequence's own among them: all of its
    sequences see them, and so do those of a second group over the same pages."""
    for again in range(4):
        n = B - B // 4
        x = ref.inputs(D, bs, BF, 3, 4, B, [0, n, B], [shared, shared], [1 + b % 30 for b in range(B)], poison=False)
        whole = shared // bs
        x["block_table"][n:, :whole] = x["block_table"][0, :whole]
        x["seq"][0], x["seq"][2], x["seq"][n] = 50 + again, 16, whole * bs - 1
        ref.check(x, str(again))


@pytest.mark.parametrize("Hkv", [1, 5, 150])
def test_all_new_positions_in_shared_pages(Hkv):
    """Every sequence of a group below its shared length, over the same pages: each sees the new tokens of those before
    it, and none is read through another's table."""
    B, n = (60, 700) if Hkv < 100 else (9, 90)
    x = ref.inputs(64, 16, BF, Hkv, 2, B, [0, B], [n], [4] * B, poison=False)
    x["block_table"][:] = x["block_table"][0]
    x["seq"][:] = torch.randperm(n)[:B]
    ref.check(x)


@pytest.mark.parametrize("D,bs,dtype,Hkv,G", SHAPES[:3])
def test_the_largest_position(D, bs, dtype, Hkv, G):
    """A position of 2^31 - 1, past the span as any other: nothing is written, all positions are seen, and the rows
    beside it are as they were."""
    for starts, lens in (([0, 12], [300]), ([0], []), ([3, 8], [129])):
        x = ref.inputs(D, bs, dtype, Hkv, G, 12, starts, lens, [1 + 17 * b for b in range(12)], poison=False)
        x["seq"][[0, 4, 11]] = 2 ** 31 - 1
        t = x["block_table"]
        spare = next(p for p in range(len(x["kcache"])) if not (t == p).any())  # no row writes it
        x["block_table"] = torch.where(t < 0, spare, t)
        ref.check(x, str(starts))


def test_starts_that_do_not_ascend():
    for starts in ([0, 6, 3, 9], [5, 5, 5, 2], [-4, 3, 100, 7], [9, 0, 0, 0]):
        x = ref.inputs(128, 16, BF, 1, 4, 9, [0, 3, 6, 9], [64, 64, 64], [20] * 9)
        x["group_starts"] = torch.tensor(starts, dtype=torch.int32)
        ref.check(x, str(starts))


def test_pages_outside_the_pool():
    """A position in such a page is not seen: of the shared part, of a row's own, and of all that a row has."""
    for bs in (8, 16, 128, 256):
        x = ref.inputs(128, bs, BF, 2, 4, 7, [0, 6, 7], [5 * bs + 3, 2 * bs], [2 * bs + 5] * 7, poison=False)
        x["block_table"][0, 1] = 10 ** 6  # row 0 is the first of its group
        x["block_table"][0, 4] = -3
        x["block_table"][3, 6] = x["kcache"].shape[0]
        x["block_table"][6] = -1
        ref.check(x, str(bs))


def test_a_row_whose_shared_part_is_gone():
    x = ref.inputs(64, 16, BF, 1, 4, 3, [0, 3], [160], [5, 6, 7], poison=False)
    x["block_table"][0, :10] = -1
    ref.check(x)


@pytest.mark.parametrize("index", [torch.int16, torch.int64])
def test_index_types_and_scales(index):
    for scale in (torch.tensor(0.1).cuda(), torch.tensor(-0.3), torch.tensor(0.0)):
        x = ref.inputs(128, 16, BF, 2, 3, 20, [0, 12, 20], [150, 99], [9] * 20, index=index)
        x["scale"] = scale
        x["group_starts"], x["shared_lens"] = x["group_starts"].long(), x["shared_lens"].long()
        ref.check(x)


def test_far_apart_scores():
    """Scores of many thousands: the softmax is one key, in the shared part or in a row's own."""
    for std in (8.0, 60.0):
        ref.check(ref.inputs(128, 16, BF, 2, 4, 40, [0, 40], [1000], [1 + b for b in range(40)], std=std))


def test_nan_in_seen_places():
    """Scores that are all NaN in one CTA's part, or in a row's own, give that row NaN."""
    for D, bs, G, n in ((128, 16, 4, 40), (64, 64, 2, 5)):
        x = ref.inputs(D, bs, BF, 2, G, n, [0, n], [6000], [1 + 3 * b for b in range(n)], poison=False)
        y = {m: c.clone() if isinstance(c, torch.Tensor) else c for m, c in x.items()}
        x["k"][3] = float("nan")
        x["q"][n - 1, 1, 0] = float("nan")
        ref.check(x)
        y["kcache"][y["block_table"][0, 1024 // bs: 2048 // bs].long(), 1] = float("nan")
        ref.check(y)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("shared", [1, 100, 129])
@pytest.mark.parametrize("B", [1, 4])
@pytest.mark.parametrize("G", [1, 4, 8])
def test_nan_alone_in_a_part(D, shared, B, G):
    """One of few parts holds nothing but NaN: that of the new token, or those of the shared positions."""
    x = ref.inputs(D, 16, BF, 8, G, B, [0, B], [shared], [1] * B, poison=False)
    y = {m: c.clone() if isinstance(c, torch.Tensor) else c for m, c in x.items()}
    x["k"][B - 1] = float("nan")
    ref.check(x, "new key")
    y["kcache"][y["block_table"][0, : -(-shared // 16)].long(), 1] = float("nan")
    ref.check(y, "shared keys")


def test_groups_given_in_64_bits():
    x = ref.inputs(64, 16, BF, 1, 4, 6, [0, 6], [64], [16] * 6, poison=False)
    x["group_starts"], x["shared_lens"] = torch.tensor([-2 ** 40, 2 ** 40]), torch.tensor([2 ** 33])
    x["seq"][:] = 200  # past the span of 80: all 80 positions are shared
    y = ref.gpu(x)
    got = ref.call(y)
    x["group_starts"], x["shared_lens"] = torch.tensor([0, 6]), torch.tensor([10 ** 6])
    want, bound = ref.decode(x)
    ref.within(got, want, bound)


def test_long_context():
    """Prefixes whose parts are joined over many CTAs, with few rows and with many."""
    ref.check(ref.inputs(128, 16, BF, 1, 1, 2, [0, 2], [20001], [1, 90]))
    ref.check(ref.inputs(128, 64, BF, 2, 8, 33, [0, 33], [6000], [1 + b for b in range(33)]))
    ref.check(ref.inputs(64, 16, F16, 1, 16, 20, [0, 11, 20], [9000, 3000], [700] * 20))


def test_one_table_row_for_all():
    """A table [1, max_blocks] stands for every sequence."""
    x = ref.inputs(64, 16, BF, 2, 4, 5, [0, 5], [100], [1] * 5, poison=False)
    x["block_table"] = x["block_table"][:1].clone()
    x["k"], x["v"] = x["k"][:1].expand_as(x["k"]).clone(), x["v"][:1].expand_as(x["v"]).clone()
    ref.check(x)


def test_table_wider_than_the_lengths_need():
    """The batch's spans add up to more positions than 31 bits hold; the lengths do not."""
    x = ref.inputs(64, 16, BF, 2, 4, 40, [0, 40], [100], [1] * 40, poison=False)
    wide = torch.full([1, 2 ** 22], -1, dtype=torch.int32)
    wide[:, : x["block_table"].shape[1]] = x["block_table"][:1]
    x["block_table"] = wide
    x["k"], x["v"] = x["k"][:1].expand_as(x["k"]).clone(), x["v"][:1].expand_as(x["v"]).clone()
    ref.check(x)


def test_strided_inputs_and_heads_outermost_pools():
    x = ref.inputs(128, 16, BF, 3, 4, 18, [0, 18], [333], [1 + b for b in range(18)])
    y = ref.gpu(x)
    for n in ("kcache", "vcache"):
        c = y[n]
        y[n] = torch.empty(c.shape[1], c.shape[0], *c.shape[2:], dtype=BF, device="cuda").transpose(0, 1).copy_(c)
    y["q"] = y["q"].permute(0, 3, 1, 2, 4).contiguous().permute(0, 2, 3, 1, 4)
    y["q"] = torch.stack([y["q"], y["q"]], 1)[:, 0]
    got = ref.call(y).double().cpu()
    want, bound = ref.decode(x)
    ref.within(got, want, bound)
    assert torch.equal(y["kcache"].cpu().contiguous().view(torch.int16), x["kcache"].view(torch.int16))


def test_cache_rows_longer_than_the_head():
    """A cache whose last dimension is larger than the queries': its first D elements are the head."""
    x = ref.inputs(64, 16, BF, 2, 4, 40, [0, 33, 40], [300, 140], [1 + b for b in range(40)])
    for n in ("kcache", "vcache"):
        x[n] = torch.cat([x[n], torch.full_like(x[n], float("nan"))], dim=-1).contiguous()
    ref.check(x)


def test_the_most_sequences_and_groups():
    """4096 sequences in 1024 groups, some empty, some of one sequence, some of many."""
    sizes = [(i * 7) % 9 for i in range(1023)]
    sizes.append(4096 - sum(sizes))
    starts = [sum(sizes[:i]) for i in range(1025)]
    lens = [(i * 37) % 200 for i in range(1024)]
    own = [None if b % 11 == 3 else 1 + b % 21 for b in range(4096)]
    ref.check(ref.inputs(64, 16, BF, 1, 2, 4096, starts, lens, own))


def test_pool_beyond_32_bits():
    """Pages at byte offsets that 32 bits do not hold."""
    D, bs, Hkv = 128, 16, 8
    blocks = 5 * 2 ** 30 // (Hkv * bs * D * 2)
    x = ref.inputs(D, bs, BF, Hkv, 2, 9, [0, 9], [200], [1 + 5 * b for b in range(9)])
    used = x["kcache"].shape[0]
    y = ref.gpu(x)
    for n in ("kcache", "vcache"):
        big = torch.empty(blocks, Hkv, 1, bs, D, dtype=BF, device="cuda")
        big[blocks - used:] = y[n]
        y[n] = big
    y["block_table"] = torch.where(y["block_table"] >= 0, y["block_table"] + blocks - used, y["block_table"])
    got = ref.call(y)
    want, bound = ref.decode(x)
    ref.within(got, want, bound)
    assert torch.equal(y["kcache"][blocks - used:].cpu().view(torch.int16), x["kcache"].view(torch.int16))


def test_no_sequences():
    x = ref.gpu(ref.inputs(64, 16, BF, 1, 2, 1, [0, 1], [3], [4]))
    for n in ("q", "k", "v", "seq", "block_table"):
        x[n] = x[n][:0]
    assert ref.call(x).shape == (0, 1, 2, 1, 64)


def test_same_bits_every_time():
    x = ref.gpu(ref.inputs(128, 16, BF, 2, 4, 70, [0, 30, 70], [1500, 400], [1 + 7 * b % 300 for b in range(70)]))
    first = ref.call(x)
    for _ in range(5):
        assert torch.equal(ref.call(x).view(torch.int16), first.view(torch.int16))


def test_calls_back_to_back():
    """Many different calls without a pause, each over the workspace that another left behind: every one gives what
    it gives alone."""
    cases = []
    for i in range(24):
        D, bs, Hkv, G = (64, 128)[i % 2], (16, 64, 32)[i % 3], (1, 2, 4)[i // 2 % 3], (1, 4, 8, 2)[i // 3 % 4]
        sizes = [(13, 32, 5)[i % 3]] * (1 + i % 2)
        starts = [sum(sizes[:j]) for j in range(len(sizes) + 1)]
        x = ref.inputs(D, bs, BF if i % 4 else F16, Hkv, G, sum(sizes), starts, [(700, 128, 3001)[i // 4 % 3]] * len(sizes),
                       [1 + (b * 7 + i) % 60 for b in range(sum(sizes))])
        cases.append((ref.gpu(x), ref.decode(x)))
    for i in range(12):
        order = torch.randperm(24, generator=torch.Generator().manual_seed(i)).tolist()
        outs = [ref.call(cases[k][0]) for k in order]
        for k, got in zip(order, outs):
            ref.within(got, *cases[k][1], f"pass {i}, case {k}")


def test_graphs_and_streams():
    """Two captured graphs and eager calls on other streams, interleaved."""
    xs = [ref.inputs(128, 16, BF, 2, 4, 24, [0, 10, 24], [500, 130], [1 + (7 + i) * b % 90 for b in range(24)])
          for i in range(3)]
    ys = [ref.gpu(x) for x in xs]
    for y in ys:
        ref.call(y)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for y in ys[:2]:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(ref.call(y))
        graphs.append(g)
    side = torch.cuda.Stream()
    for _ in range(3):
        graphs[0].replay()
        with torch.cuda.stream(side):
            eager = ref.call(ys[2])
        graphs[1].replay()
    torch.cuda.synchronize()
    for x, got in zip(xs, outs + [eager]):
        want, bound = ref.decode(x)
        ref.within(got, want, bound)


def test_lengths_change_between_replays():
    """What a captured call read on the device is read again: one graph serves steps of other lengths and groups."""
    x = ref.inputs(64, 16, BF, 2, 4, 12, [0, 12], [200], [40] * 12, poison=False)
    y = ref.gpu(x)
    ref.call(y)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = ref.call(y)
    for starts, n, seq in (([0, 12], 200, 239), ([0, 5], 130, 205), ([3, 12], 0, 230), ([0, 12], 199, 199)):
        for z in (x, y):
            z["group_starts"].copy_(torch.tensor(starts))
            z["shared_lens"].fill_(n)
            z["seq"].fill_(seq)
        g.replay()
        want, bound = ref.decode(x)
        ref.within(out, want, bound, str((starts, n, seq)))


def test_pages_forked_reserved_attended_and_freed():
    """The operators as they are used: prompts forked, pages reserved, tokens decoded over the shared pages, forks
    dropped, the pool compacted, and decoding goes on; every step against float64 and the plain decode op."""
    import torch_rbln_b200 as pkg

    ops = torch.ops.rbln_attn
    bs, Hkv, G, D, layers = 16, 2, 4, 64, 2
    lengths, forks = [150, 61], [0, 0, 0, 1, 1, 1, 1]
    table, refs = page_refs.pool(2, 14, lengths, bs, 40)
    blocks = len(refs)
    kc, vc = ([torch.randn(blocks, Hkv, 1, bs, D).to(BF).cuda() for _ in range(layers)] for _ in range(2))
    t = torch.tensor(table, dtype=torch.int32).cuda()
    r, n = torch.tensor(refs, dtype=torch.int32).cuda(), torch.tensor(lengths, dtype=torch.int32).cuda()
    rows, seq = ops.paged_kv_fork(t, n, torch.tensor(forks).cuda(), r, bs)
    ops.paged_kv_free(t, torch.zeros_like(n), r, bs)  # the prompts' own rows are done
    starts, lens = torch.tensor([0, 3, 7]), torch.tensor(lengths)
    scale = torch.tensor(D ** -0.5)
    for step in range(40):
        granted = ops.paged_kv_reserve(kc, vc, rows, seq, r, bs, 1)
        assert granted.tolist() == [1] * 7
        if step == 20:
            _, live = ops.paged_kv_compact(kc, vc, rows, r)
            assert rows.max() < live.item() == (r > 0).sum().item()
        for layer in range(layers):
            q, k, v = (torch.randn(7, Hkv, g, 1, D).to(BF).cuda() for g in (G, 1, 1))
            x = {"q": q, "k": k, "v": v, "kcache": kc[layer], "vcache": vc[layer], "seq": seq, "scale": scale,
                 "block_table": rows, "block_size": bs, "group_starts": starts, "shared_lens": lens}
            plain = {m: c.cpu().clone() if isinstance(c, torch.Tensor) else c for m, c in x.items()}
            got = ref.call(x).double().cpu()
            want, bound = ref.decode(plain)
            ref.within(got, want, bound, str(step))
            assert torch.equal(kc[layer].cpu(), plain["kcache"]) and torch.equal(vc[layer].cpu(), plain["vcache"])
            alone = pkg.paged_causal_attn_decode(q, k, v, kc[layer], vc[layer], seq, scale, rows, bs).double().cpu()
            ref.within(alone, want, bound, str(step))
        seq += 1
    ops.paged_kv_free(rows, torch.zeros_like(seq), r, bs)
    assert (r == 0).all() and (rows == -1).all()


def test_schema_fake_and_trace():
    x = ref.gpu(ref.inputs(64, 16, BF, 2, 4, 4, [0, 4], [40], [3] * 4, poison=False))
    torch.library.opcheck(torch.ops.rbln_custom_ops.paged_causal_attn_decode_shared.default,
                          tuple(x[n] for n in ref.ORDER))


def test_no_groups_and_no_arrays_of_them():
    """Through the C entry point, as it may be called without any group: the arrays are NULL."""
    from torch_rbln_b200 import cabi

    x = ref.inputs(128, 16, BF, 2, 4, 6, [0], [], [3, 40, 300, 1, 17, 130])
    y = ref.gpu(x)
    p, keep = cabi.paged_params(y["q"], y["k"], y["v"], y["kcache"], y["vcache"], y["seq"], y["block_table"], 16,
                                float(x["scale"]))
    s, n = cabi.SharedPrefix(0, None, None), ctypes.c_size_t(0)
    assert cabi.lib().rbln_paged_decode_shared_workspace_size(ctypes.byref(p), ctypes.byref(s), ctypes.byref(n)) == 0
    ws = torch.empty(n.value, dtype=torch.uint8, device="cuda")
    p.workspace, p.workspace_bytes = ws.data_ptr(), n.value
    assert cabi.lib().rbln_paged_causal_attn_decode_shared(ctypes.byref(p), ctypes.byref(s),
                                                           ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)) == 0
    want, bound = ref.decode(x)
    ref.within(keep["out"], want, bound)
    assert torch.equal(y["kcache"].cpu().view(torch.int16), x["kcache"].view(torch.int16))


def test_error_flags():
    from torch_rbln_b200 import cabi

    x = ref.gpu(ref.inputs(128, 16, BF, 2, 4, 6, [0, 6], [100], [5] * 6, poison=False))
    for change, flag in ((None, 0), ("page", cabi.DEVERR_BLOCK_ID_RANGE), ("seq", cabi.DEVERR_SEQ_RANGE)):
        t, seq = x["block_table"].clone(), x["seq"].clone()
        if change == "page":
            t[0, 2] = 10 ** 7
        if change == "seq":
            seq[4] = -2
        p, keep = cabi.paged_params(x["q"], x["k"], x["v"], x["kcache"], x["vcache"], seq, t, 16, 0.1)
        err = torch.zeros(1, dtype=torch.int32, device="cuda")
        p.error_flags = err.data_ptr()
        s = cabi.SharedPrefix(1, x["group_starts"].data_ptr(), x["shared_lens"].data_ptr())
        n = ctypes.c_size_t(0)
        assert cabi.lib().rbln_paged_decode_shared_workspace_size(ctypes.byref(p), ctypes.byref(s), ctypes.byref(n)) == 0
        ws = torch.empty(n.value, dtype=torch.uint8, device="cuda")
        p.workspace, p.workspace_bytes = ws.data_ptr(), n.value
        rc = cabi.lib().rbln_paged_causal_attn_decode_shared(ctypes.byref(p), ctypes.byref(s),
                                                             ctypes.c_void_p(torch.cuda.current_stream().cuda_stream))
        assert rc == 0 and err.item() == flag


def test_refusals():
    x = ref.gpu(ref.inputs(64, 16, BF, 1, 4, 3, [0, 3], [20], [4] * 3))

    def refused(match, **changes):
        with pytest.raises(RuntimeError, match=match):
            ref.call({**x, **changes})

    refused("one entry more", group_starts=x["group_starts"][:1])
    refused("group_starts must be", group_starts=x["group_starts"].float())
    refused("shared_lens must be", shared_lens=x["shared_lens"].reshape(1, 1))
    refused("cache dtype", kcache=x["kcache"].half(), vcache=x["vcache"].half())
    refused("q's device", kcache=x["kcache"].cpu(), vcache=x["vcache"].cpu())
    refused("one query token", q=x["q"].expand(-1, -1, -1, 2, -1), k=x["k"].expand(-1, -1, -1, 2, -1),
            v=x["v"].expand(-1, -1, -1, 2, -1))
    refused("block_size", block_size=8)
    refused("unsupported", q=torch.zeros(3, 1, 17, 1, 64, dtype=BF).cuda())
    bad = torch.zeros(4, 1, 1, 24, 64, dtype=BF).cuda()
    refused("unsupported", kcache=bad, vcache=bad.clone(), block_size=24)
    many = torch.zeros(1026, dtype=torch.int32).cuda()
    refused("unsupported", group_starts=many, shared_lens=many[:1025])
    import torch_rbln_b200

    with pytest.raises(RuntimeError, match="takes 11 inputs"):
        torch_rbln_b200.paged_causal_attn_decode_shared(*[x[n] for n in ref.ORDER[:9]])
