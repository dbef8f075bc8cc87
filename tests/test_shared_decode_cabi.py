"""Decode over a shared prefix on a host without a GPU: schema, fake kernel, the ctypes struct, refused calls."""

import ctypes

import pytest
import torch


def params(**changes):
    """A call in order (on host memory: nothing here may reach a launch), but for `changes`."""
    from torch_rbln_b200 import cabi

    q = torch.zeros(3, 2, 4, 1, 64, dtype=torch.bfloat16)
    k = torch.zeros(3, 2, 1, 1, 64, dtype=torch.bfloat16)
    c = torch.zeros(8, 2, 1, 16, 64, dtype=torch.bfloat16)
    seq, table = torch.zeros(3, dtype=torch.int32), torch.zeros(3, 4, dtype=torch.int32)
    starts, lens = torch.zeros(2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    p, keep = cabi.paged_params(q, k, k, c, c, seq, table, 16, 0.1)
    s = cabi.SharedPrefix(1, starts.data_ptr(), lens.data_ptr())
    for name, value in changes.items():
        setattr(s if name in ("num_groups", "group_starts", "shared_lens") else p, name, value)
    return p, s, (q, k, c, seq, table, starts, lens, keep)


def run(p, s):
    from torch_rbln_b200 import cabi

    return cabi.lib().rbln_paged_causal_attn_decode_shared(ctypes.byref(p), ctypes.byref(s), None)


@pytest.mark.parametrize("changes,rc", [
    ({"batch": -1}, -1), ({"num_kv_heads": 0}, -1), ({"group": 0}, -1), ({"max_blocks": 0}, -1), ({"num_blocks": 0}, -1),
    ({"q_len": 2}, -1), ({"num_groups": -1}, -1), ({"group_starts": None}, -1), ({"shared_lens": None}, -1),
    ({"q": None}, -1), ({"out": None}, -1), ({"kcache": None}, -1), ({"seq": None}, -1), ({"block_table": None}, -1),
    ({"k_new": None}, -1), ({"q": 8}, -1), ({"out": 4}, -1), ({"v_new": 2}, -1),
    ({"cache_stride": (ctypes.c_int64 * 3)(2048, 1024, 65)}, -1), ({"q_stride": (ctypes.c_int64 * 4)(1, 256, 64, 64)}, -1),
    ({"head_dim": 96}, -2), ({"group": 17}, -2), ({"block_size": 24}, -2), ({"block_size": 4}, -2), ({"batch": 4097}, -2),
    ({"num_groups": 1025}, -2), ({"mask": 256}, -2), ({"sinks": 256}, -2), ({"num_splits": 2}, -2), ({"q_dtype": 0}, -2),
    ({"kv_dtype": 3}, -2), ({"kv_dtype": 1}, -2), ({"block_table_dtype": 0}, -2), ({"max_blocks": 2 ** 27}, -2),
    ({}, -3),
])
def test_refused(changes, rc):
    p, s, keep = params(**changes)
    assert run(p, s) == rc


def test_workspace():
    from torch_rbln_b200 import cabi

    p, s, keep = params()
    n = ctypes.c_size_t(0)
    query = cabi.lib().rbln_paged_decode_shared_workspace_size
    assert query(ctypes.byref(p), ctypes.byref(s), None) == -1
    assert query(ctypes.byref(p), ctypes.byref(s), ctypes.byref(n)) == 0 and n.value > 0
    p.workspace, p.workspace_bytes = 256, n.value - 1
    assert run(p, s) == -3
    p.batch = 0
    assert run(p, s) == 0  # nothing to do
    assert cabi.lib().rbln_shared_prefix_sizeof() == ctypes.sizeof(cabi.SharedPrefix)


def test_schema_fake_and_argument_count():
    import torch_rbln_b200 as pkg
    from torch._subclasses.fake_tensor import FakeTensorMode

    assert str(torch.ops.rbln_custom_ops.paged_causal_attn_decode_shared.default._schema) == (
        "rbln_custom_ops::paged_causal_attn_decode_shared(Tensor q, Tensor k, Tensor v, Tensor(a3!) kcache, "
        "Tensor(a4!) vcache, Tensor seq, Tensor scale, Tensor block_table, SymInt block_size, Tensor group_starts, "
        "Tensor shared_lens) -> Tensor")
    for n in (10, 12):
        with pytest.raises(RuntimeError, match="takes 11 inputs"):
            pkg.paged_causal_attn_decode_shared(*([None] * n))
    with FakeTensorMode():
        q = torch.empty(2, 8, 4, 1, 64, dtype=torch.float16)
        k = torch.empty(2, 8, 1, 1, 64, dtype=torch.float16)
        c = torch.empty(4, 8, 1, 16, 64, dtype=torch.float16)
        i = torch.empty(2, dtype=torch.int32)
        out = pkg.paged_causal_attn_decode_shared(q, k, k, c, c, i, torch.empty(()), torch.empty(2, 3, dtype=torch.int32),
                                                  16, i, i[:1])
    assert out.shape == q.shape and out.dtype == q.dtype
    with pytest.raises(NotImplementedError):
        z, i = torch.zeros(1, 1, 1, 1, 64), torch.zeros(2, dtype=torch.int32)
        pkg.paged_causal_attn_decode_shared(z, z, z, z, z, i, z, z, 1, i, i)
