"""Forking, reserving, freeing and compacting pages on B200, against the operators run one entry at a time on the CPU:
tables, counts, caches and scales equal to the bit."""

import copy

import pytest
import torch

from tests import page_refs as ref

pytestmark = pytest.mark.gpu

FP8 = torch.float8_e4m3fn


@pytest.fixture(scope="module")
def ops():
    import torch_rbln_b200  # noqa: F401

    return torch.ops.rbln_attn


def dev(x, dtype=torch.int32):
    return torch.tensor(x, dtype=dtype).cuda()


def table_of(rows, width, dtype=torch.int32):
    return torch.tensor(rows, dtype=dtype).reshape(len(rows), width).cuda()


def same_caches(got, want):
    for g, w in zip(got, want):
        assert torch.equal(g.cpu().contiguous().view(torch.uint8), w.contiguous().view(torch.uint8))


def to_gpu(cs):
    """Copies that keep the strides."""
    return [torch.empty_strided(c.shape, c.stride(), dtype=c.dtype, device="cuda").copy_(c) for c in cs]


CASES = [  # rows, forks, width, bs, lengths
    (1, 1, 1, 16, [1]),
    (1, 5, 3, 16, [33]),
    (3, 8, 7, 8, [0, 56, 17]),
    (4, 300, 300, 16, [4800, 1, 0, 3333]),
    (70, 40, 5, 24, None),
    (2, 0, 4, 16, [5, 64]),
]


@pytest.mark.parametrize("B,N,width,bs,lengths", CASES)
@pytest.mark.parametrize("index", [torch.int16, torch.int32, torch.int64])
def test_fork(ops, B, N, width, bs, lengths, index):
    lengths = lengths or torch.randint(0, width * bs + 1, [B]).tolist()
    table, refs = ref.pool(B, width, lengths, bs, 5)
    if B > 2:
        table[1][0] = len(refs) + 3  # not a page: the fork has none there either
        table[2][0] = -7
    parents = torch.randint(-1, B + 1, [N]).tolist()
    got_table, got_refs = table_of(table, width, index), dev(refs)
    rows, lens = ops.paged_kv_fork(got_table, dev(lengths, index), dev(parents, index), got_refs, bs)
    want_refs = list(refs)
    want, want_lens = ref.fork(table, lengths, parents, want_refs, bs)
    assert rows.dtype == index and lens.dtype == index
    assert rows.cpu().tolist() == want and lens.cpu().tolist() == want_lens
    assert got_refs.cpu().tolist() == want_refs
    assert got_table.cpu().tolist() == table  # as it was


def test_fork_lengths_outside_the_span(ops):
    table, refs = ref.pool(3, 4, [64, 64, 64], 16, 2)
    lengths = [-5, 10 ** 12, 64]
    t, r = table_of(table, 4), dev(refs)
    rows, lens = ops.paged_kv_fork(t, dev(lengths, torch.int64), dev([0, 1, 2, 1]), r, 16)
    want, want_lens = ref.fork(table, lengths, [0, 1, 2, 1], refs, 16)
    assert rows.cpu().tolist() == want and lens.cpu().tolist() == want_lens == [0, 64, 64, 64]
    assert r.cpu().tolist() == refs


@pytest.mark.parametrize("B,width,bs", [(1, 1, 16), (5, 9, 16), (33, 300, 8), (64, 17, 128)])
def test_free(ops, B, width, bs):
    lengths = torch.randint(0, width * bs + 1, [B]).tolist()
    table, refs = ref.pool(B, width, lengths, bs, 3)
    # some rows are forks of the row before, so that runs of equal entries and shared counts occur
    for b in range(1, B):
        if torch.rand([]) < 0.5:
            for j, p in enumerate(table[b]):
                if p >= 0:
                    refs[p] -= 1
            table[b] = list(table[b - 1])
            for p in table[b]:
                if p >= 0:
                    refs[p] += 1
    table[0][width - 1] = len(refs) + 1  # not a page: cleared, nothing counted
    keep = [int(torch.randint(-2, width * bs + 2, []).item()) for _ in range(B)]
    t, r = table_of(table, width), dev(refs)
    ops.paged_kv_free(t, dev(keep), r, bs)
    ref.free(table, keep, refs, bs)
    assert t.cpu().tolist() == table and r.cpu().tolist() == refs


def test_free_never_counts_below_zero(ops):
    """Counts that say less than the table holds stay at zero; a count below zero stays as it is."""
    table = [[0, 1, 2, 0], [0, 1, 2, 3]] * 20
    refs = [7, 0, -3, 20]
    t, r = table_of(table, 4), dev(refs)
    ops.paged_kv_free(t, dev([0] * 40), r, 16)
    assert r.cpu().tolist() == [0, 0, -3, 0] and (t.cpu() == -1).all()


def run_reserve(ops, table, refs, seq, bs, new, caches_k, caches_v, ks=None, vs=None, index=torch.int32, width=None):
    width = width or len(table[0])
    t, r = table_of(table, width, index), dev(refs)
    k, v = to_gpu(caches_k), to_gpu(caches_v)
    sk, sv = (None if s is None else [x.cuda() for x in s] for s in (ks, vs))
    granted = ops.paged_kv_reserve(k, v, t, dev(seq, index), r, bs, new, sk, sv)
    want_table, want_refs = copy.deepcopy(table), list(refs)
    want, moves = ref.reserve(want_table, seq, want_refs, bs, new)
    ref.copy(caches_k + caches_v, (ks or []) + (vs or []), moves)
    assert granted.cpu().tolist() == want
    assert t.cpu().tolist() == want_table and r.cpu().tolist() == want_refs
    same_caches(k + v, caches_k + caches_v)
    for got, s in zip((sk or []) + (sv or []), (ks or []) + (vs or [])):
        assert torch.equal(got.cpu(), s)
    return moves


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, FP8])
@pytest.mark.parametrize("bs,new,D,Hkv", [(16, 1, 128, 2), (8, 3, 64, 1), (32, 40, 64, 3), (128, 1, 128, 2),
                                          (24, 100, 192, 2)])
def test_reserve_after_fork(ops, dtype, bs, new, D, Hkv):
    """Forks of several rows: partly filled pages are copied for all holders but the last, in every layer."""
    B, N, layers = 5, 14, 3
    lengths = [1, bs, 2 * bs - 1, 3 * bs + 1, 0]
    width = 3 + (3 * bs + new) // bs + 1
    table, refs = ref.pool(B, width, lengths, bs, N * (new // bs + 2) + 4)
    parents = torch.randint(0, B, [N]).tolist()
    rows, seq = ref.fork(table, lengths, parents, refs, bs)
    # half of the parents are gone: their pages are held by forks of this call alone
    ref.free(table[:3], [0] * 3, refs, bs)
    k, v = (ref.caches(layers, len(refs), Hkv, bs, D, dtype) for _ in range(2))
    scales = [[torch.rand(len(refs), Hkv) for _ in range(layers)] for _ in range(2)] if dtype == FP8 else (None, None)
    moves = run_reserve(ops, rows, refs, seq, bs, new, k, v, *scales)
    assert moves, "the case copies nothing"


@pytest.mark.parametrize("free_pages", [0, 1, 3, 6])
def test_reserve_runs_out_of_pages(ops, free_pages):
    """Rows get pages in order; what is not granted stays as it was, and a page whose other holders could not move is
    not granted to the last of them."""
    bs, new = 16, 20
    table, refs = ref.pool(2, 6, [20, 40], bs, free_pages)
    rows, seq = ref.fork(table, [20, 40], [0, 1, 0, 1], refs, bs)
    ref.free(table, [0, 0], refs, bs)
    k, v = (ref.caches(1, len(refs), 2, bs, 64, torch.bfloat16) for _ in range(2))
    run_reserve(ops, rows, refs, seq, bs, new, k, v)


def test_reserve_edges(ops):
    """Rows that take no part, rows at and past the span's end, no new tokens, entries that are no pages."""
    bs = 16
    table, refs = ref.pool(6, 4, [64, 60, 16, 0, 33, 17], bs, 9)
    table[4][3] = 10 ** 6
    table[5][1] = -9
    for seq in ([-1, 60, 16, 0, 33, 17], [64, 64, 70, 1000, -5, 63]):
        for new in (0, 1, 17, 1000):
            k, v = (ref.caches(1, len(refs), 1, bs, 64, torch.float16) for _ in range(2))
            run_reserve(ops, table, refs, seq, bs, new, k, v, index=torch.int64)


def test_reserve_large(ops):
    """More entries and pages than one CTA takes, an int16 table, heads-outermost pools."""
    bs, B, width, new = 8, 600, 14, 25
    lengths = torch.randint(0, 80, [B // 2]).tolist()
    table, refs = ref.pool(B // 2, width, lengths, bs, 5000)
    rows, seq = ref.fork(table, lengths, torch.randint(0, B // 2, [B]).tolist(), refs, bs)
    k, v = (ref.caches(2, len(refs), 2, bs, 64, FP8, heads_outermost=True) for _ in range(2))
    ks, vs = ([torch.rand(2, len(refs)).t() for _ in range(2)] for _ in range(2))
    run_reserve(ops, rows, refs, seq, bs, new, k, v, [s.contiguous() for s in ks], [s.contiguous() for s in vs],
                index=torch.int16)


@pytest.mark.parametrize("B,new", [(7, 3), (600, 25)])
@pytest.mark.parametrize("order", ["heads outermost", "every second"])
def test_scales_of_other_strides(ops, B, new, order):
    """Scales that are not contiguous [blocks, heads], through both reservations and a compaction; what lies between
    them is left alone."""
    bs, width = 8, 14
    lengths = torch.randint(0, 80, [B]).tolist()
    table, refs = ref.pool(B, width, lengths, bs, 8 * B)
    rows, seq = ref.fork(table, lengths, torch.randint(0, B, [B]).tolist(), refs, bs)
    ref.free(table, [0] * B, refs, bs)
    n = len(refs)
    k, v = (ref.caches(2, n, 2, bs, 64, FP8) for _ in range(2))
    shape, view = ([2, n], torch.t) if order == "heads outermost" else ([n, 4], lambda c: c[:, ::2])
    cells = [torch.rand(shape) for _ in range(4)]
    on_gpu = [c.cuda() for c in cells]
    scales, got = [view(c) for c in cells], [view(c) for c in on_gpu]
    gk, gv, t, r = to_gpu(k), to_gpu(v), table_of(rows, width), dev(refs)
    granted = ops.paged_kv_reserve(gk, gv, t, dev(seq), r, bs, new, got[:2], got[2:])
    want, moves = ref.reserve(rows, seq, refs, bs, new)
    ref.copy(k + v, scales, moves)
    assert moves and granted.cpu().tolist() == want and t.cpu().tolist() == rows and r.cpu().tolist() == refs
    same_caches(gk + gv + on_gpu, k + v + cells)
    ops.paged_kv_compact(gk, gv, t, r, got[:2], got[2:])
    _, _, pairs = ref.compact(rows, refs)
    ref.copy(k + v, scales, [(p, h, bs) for p, h in pairs])
    assert pairs and t.cpu().tolist() == rows and r.cpu().tolist() == refs
    same_caches(gk + gv + on_gpu, k + v + cells)


def test_reserve_same_page_twice_in_a_row(ops):
    bs = 16
    table, refs = [[2, 2, 2], [2, 5, 2]], [0, 0, 5, 0, 0, 1, 0, 0, 0, 0]
    k, v = (ref.caches(1, 10, 1, bs, 64, torch.bfloat16) for _ in range(2))
    run_reserve(ops, table, refs, [3, 20], bs, 40, k, v)


def test_many_layers(ops):
    """More layers than one launch takes."""
    bs, layers = 16, 70
    table, refs = ref.pool(2, 3, [20, 5], bs, 8)
    rows, seq = ref.fork(table, [20, 5], [0, 0, 1, 1], refs, bs)
    k, v = (ref.caches(layers, len(refs), 1, bs, 64, torch.bfloat16) for _ in range(2))
    run_reserve(ops, rows, refs, seq, bs, 1, k, v)


def run_compact(ops, table, refs, k, v, ks=None, vs=None, index=torch.int32):
    t, r = table_of(table, len(table[0]), index), dev(refs)
    gk, gv = to_gpu(k), to_gpu(v)
    sk, sv = (None if s is None else [x.cuda() for x in s] for s in (ks, vs))
    moved, live = ops.paged_kv_compact(gk, gv, t, r, sk, sv)
    want_table, want_refs = copy.deepcopy(table), list(refs)
    want_moved, want_live, pairs = ref.compact(want_table, want_refs)
    ref.copy(k + v, (ks or []) + (vs or []), [(p, h, k[0].shape[3]) for p, h in pairs])
    assert moved.cpu().tolist() == want_moved and live.cpu().tolist() == [want_live]
    assert t.cpu().tolist() == want_table and r.cpu().tolist() == want_refs
    same_caches(gk + gv, k + v)
    for got, s in zip((sk or []) + (sv or []), (ks or []) + (vs or [])):
        assert torch.equal(got.cpu(), s)


@pytest.mark.parametrize("dtype", [torch.bfloat16, FP8])
@pytest.mark.parametrize("blocks,used", [(1, 0), (1, 1), (7, 3), (64, 64), (500, 130), (5000, 2600)])
def test_compact(ops, dtype, blocks, used):
    bs, Hkv, D, layers = 8, 2, 64, 2
    pages = torch.randperm(blocks)[:used].tolist()
    width = max(1, -(-used // 6)) + 2
    flat = pages + pages[: used // 3] + [-1, blocks, blocks + 9]
    flat = flat + [-1] * (6 * width * 2 - len(flat))
    flat = [flat[i] for i in torch.randperm(len(flat)).tolist()]
    table = [flat[i * width:(i + 1) * width] for i in range(12)]
    refs = [0] * blocks
    for p in flat:
        if 0 <= p < blocks:
            refs[p] += 1
    k, v = (ref.caches(layers, blocks, Hkv, bs, D, dtype, heads_outermost=blocks == 500) for _ in range(2))
    scales = [[torch.rand(blocks, Hkv) for _ in range(layers)] for _ in range(2)] if dtype == FP8 else (None, None)
    run_compact(ops, table, refs, k, v, *scales)
    run_compact(ops, table, [-n for n in refs], k, v, *scales)  # nothing in use


def test_life_of_pages_in_a_graph(ops):
    """Fork, reserve, free and compact captured once and replayed: each replay gives what a call gives, the counts
    come back, and a second graph that was captured in between does not disturb it."""
    bs, layers = 16, 2
    table, refs = ref.pool(3, 6, [40, 17, 3], bs, 30)
    seq, parents = [40, 17, 3], [0, 1, 0, 2, 0]
    t, r, n, p = table_of(table, 6), dev(refs), dev(seq), dev(parents)
    k, v = (to_gpu(ref.caches(layers, len(refs), 2, bs, 64, torch.bfloat16)) for _ in range(2))
    none = dev([0] * 5)

    def step():
        rows, lens = ops.paged_kv_fork(t, n, p, r, bs)
        granted = ops.paged_kv_reserve(k, v, rows, lens, r, bs, 4)
        held = rows.clone()
        ops.paged_kv_free(rows, none, r, bs)
        return held, lens, granted

    step()
    torch.cuda.synchronize()
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step())
        graphs.append(g)
    want_refs = list(refs)
    want, lens = ref.fork(table, seq, parents, want_refs, bs)
    granted, _ = ref.reserve(want, lens, want_refs, bs, 4)
    for i in (0, 1, 0):
        for x in outs[i]:
            x.zero_()
        graphs[i].replay()
        assert outs[i][0].cpu().tolist() == want and outs[i][2].cpu().tolist() == granted
        assert r.cpu().tolist() == refs
    moved, live = ops.paged_kv_compact(k, v, t, r)
    assert live.item() == sum(c > 0 for c in refs) and sorted(x for x in moved.tolist() if x >= 0) == list(range(live))


def test_two_streams(ops):
    """Calls on different pools run side by side on streams of their own."""
    bs = 16
    states = []
    for i in range(2):
        table, refs = ref.pool(8, 40, [600 - i * 7] * 8, bs, 100)
        states.append((table, refs, [600 - i * 7] * 8))
    streams = [torch.cuda.Stream() for _ in states]
    gpu = []
    for table, refs, seq in states:
        k, v = (to_gpu(ref.caches(1, len(refs), 2, bs, 64, torch.bfloat16)) for _ in range(2))
        gpu.append((table_of(table, 40), dev(refs), dev(seq), k, v))
    parents = dev([0, 1, 1, 2, 2, 2, 5] * 4)
    torch.cuda.synchronize()
    outs = []
    for s, (t, r, n, k, v) in zip(streams, gpu):
        with torch.cuda.stream(s):
            for _ in range(5):
                rows, lens = ops.paged_kv_fork(t, n, parents, r, bs)
                ops.paged_kv_reserve(k, v, rows, lens, r, bs, 2)
                held = rows.clone()
                ops.paged_kv_free(rows, torch.zeros_like(lens), r, bs)
            outs.append(held)
    torch.cuda.synchronize()
    for (table, refs, seq), held, (_, r, *_) in zip(states, outs, gpu):
        counts = list(refs)
        rows, lens = ref.fork(table, seq, parents.tolist(), counts, bs)
        ref.reserve(rows, lens, counts, bs, 2)
        assert held.cpu().tolist() == rows and r.cpu().tolist() == refs


def test_strided_table_and_lengths(ops):
    bs = 16
    table, refs = ref.pool(4, 5, [70, 3, 16, 80], bs, 12)
    wide = torch.full([5, 8], 77, dtype=torch.int32)
    wide[:, ::2] = torch.tensor(table, dtype=torch.int32).t()
    t = wide.cuda()[:, ::2].t()  # strides (2, 8)
    base = t._base
    n = torch.tensor([70, 0, 3, 0, 16, 0, 80, 0]).cuda()[::2]
    r = dev(refs)
    k, v = (ref.caches(1, len(refs), 1, bs, 64, torch.bfloat16) for _ in range(2))
    gk, gv = to_gpu(k), to_gpu(v)
    granted = ops.paged_kv_reserve(gk, gv, t, n, r, bs, 30)
    want, moves = ref.reserve(table, [70, 3, 16, 80], refs, bs, 30)
    assert t.cpu().tolist() == table and r.cpu().tolist() == refs and granted.cpu().tolist() == want
    ops.paged_kv_free(t, n, r, bs)
    ref.free(table, [70, 3, 16, 80], refs, bs)
    assert t.cpu().tolist() == table and r.cpu().tolist() == refs
    assert (base.cpu()[:, 1::2] == 77).all()


def test_pool_beyond_32_bits(ops):
    """Pages at byte offsets that 32 bits do not hold, and more pages than one CTA searches."""
    D, bs, Hkv = 128, 16, 8
    blocks = 5 * 2 ** 30 // (Hkv * bs * D * 2)
    k, v = (torch.empty(blocks, Hkv, 1, bs, D, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    last = blocks - 1
    k[last], v[last] = torch.randn_like(k[last]), torch.randn_like(v[last])
    refs = torch.ones(blocks, dtype=torch.int32, device="cuda")
    refs[last], refs[blocks - 5] = 2, 0
    k[blocks - 5], v[blocks - 5] = 0, 0
    t = torch.full([2, 2], last, dtype=torch.int32, device="cuda")
    t[:, 1] = -1
    assert ops.paged_kv_reserve([k], [v], t, dev([7, 7]), refs, bs, 1).tolist() == [1, 1]
    assert t[:, 0].tolist() == [blocks - 5, last] and refs[blocks - 5] == 1 and refs[last] == 1
    for c in (k, v):
        assert torch.equal(c[blocks - 5, :, :, :7], c[last, :, :, :7]) and (c[blocks - 5, :, :, 7:] == 0).all()
    refs.zero_()
    refs[last] = 3
    moved, live = ops.paged_kv_compact([k], [v], t, refs)
    assert live.item() == 1 and moved[last] == 0 and refs[0] == 3 and refs[last] == 0 and t[1, 0] == 0
    assert torch.equal(k[0], k[last]) and torch.equal(v[0], v[last])


def test_schemas_fakes_and_traces(ops):
    table, refs = ref.pool(3, 4, [30, 20, 50], 16, 9)
    t, r, n = table_of(table, 4), dev(refs), dev([30, 20, 50])
    k, v = ([torch.randn(len(refs), 1, 1, 16, 64).to(torch.bfloat16).cuda() for _ in range(2)] for _ in range(2))
    torch.library.opcheck(ops.paged_kv_fork.default, (t, n, dev([0, 2, 2]), r, 16))
    torch.library.opcheck(ops.paged_kv_free.default, (t, n, r, 16))
    torch.library.opcheck(ops.paged_kv_reserve.default, (k, v, t, n, r, 16, 3))
    torch.library.opcheck(ops.paged_kv_compact.default, (k, v, t, r))


def test_refusals(ops):
    bs = 16
    table, refs = ref.pool(2, 4, [30, 20], bs, 4)
    t, r, n = table_of(table, 4), dev(refs), dev([30, 20])
    k = to_gpu(ref.caches(2, len(refs), 1, bs, 64, torch.bfloat16))
    f8 = to_gpu(ref.caches(2, len(refs), 1, bs, 64, FP8))
    s = [torch.ones(len(refs), 1).cuda() for _ in range(2)]

    def refused(match, fn):
        with pytest.raises(RuntimeError, match=match):
            fn()

    refused("block_table must be", lambda: ops.paged_kv_fork(t[0], n, dev([0]), r, bs))
    refused("block_table must be", lambda: ops.paged_kv_fork(t.float(), n, dev([0]), r, bs))
    refused("refs must be", lambda: ops.paged_kv_fork(t, n, dev([0]), r.long(), bs))
    refused("refs must be", lambda: ops.paged_kv_fork(t, n, dev([0]), torch.stack([r, r], 1)[:, 0], bs))
    refused("refs must be on", lambda: ops.paged_kv_fork(t, n, dev([0]), r.cpu(), bs))
    refused("parents must be", lambda: ops.paged_kv_fork(t, n, dev([0.0], torch.float32), r, bs))
    refused("one entry per row", lambda: ops.paged_kv_fork(t, n[:1], dev([0]), r, bs))
    refused("block_size must be", lambda: ops.paged_kv_fork(t, n, dev([0]), r, 0))
    refused("2\\^31", lambda: ops.paged_kv_fork(t, n, dev([0]), r, 2 ** 30))
    refused("int16", lambda: ops.paged_kv_free(t.short(), n, torch.zeros(40000, dtype=torch.int32).cuda(), bs))
    refused("expanded", lambda: ops.paged_kv_free(t[:1].expand(2, 4), n, r, bs))
    refused("keep must be", lambda: ops.paged_kv_free(t, n.float(), r, bs))
    refused("one cache for each layer", lambda: ops.paged_kv_reserve([], [], t, n, r, bs, 1))
    refused("one cache for each layer", lambda: ops.paged_kv_reserve(k, k[:1], t, n, r, bs, 1))
    refused("alike|match", lambda: ops.paged_kv_reserve(k, [k[0], k[1][:, :, :, :8]], t, n, r, bs, 1))
    refused("match", lambda: ops.paged_kv_reserve(k, [k[0], k[1].half()], t, n, r, bs, 1))
    refused("on block_table's device", lambda: ops.paged_kv_reserve([c.cpu() for c in k], k, t, n, r, bs, 1))
    refused("does not match the cache's block", lambda: ops.paged_kv_reserve(k, k, t, n, r, 8, 1))
    refused("blocks, refs", lambda: ops.paged_kv_reserve(k, k, t, n, r[:-1], bs, 1))
    refused("new_tokens", lambda: ops.paged_kv_reserve(k, k, t, n, r, bs, -1))
    refused("k_scales and v_scales go with", lambda: ops.paged_kv_reserve(k, k, t, n, r, bs, 1, s, s))
    refused("k_scales and v_scales go with", lambda: ops.paged_kv_reserve(f8, f8, t, n, r, bs, 1))
    refused("one tensor for each layer", lambda: ops.paged_kv_reserve(f8, f8, t, n, r, bs, 1, s[:1], s))
    refused("k_scale/v_scale must be", lambda: ops.paged_kv_compact(f8, f8, t, r, [x[1:] for x in s], s))
    refused("contiguous last dim", lambda: ops.paged_kv_compact([c.transpose(3, 4) for c in k], k, t, r))
    refused("bfloat16, float16 or", lambda: ops.paged_kv_compact([c.float() for c in k], k, t, r))
    refused("expanded", lambda: ops.paged_kv_compact([c[:1].expand(len(refs), -1, -1, -1, -1) for c in k],
                                                     [c[:1].expand(len(refs), -1, -1, -1, -1) for c in k], t, r))
    assert t.cpu().tolist() == table and r.cpu().tolist() == refs  # a refused call changes nothing
