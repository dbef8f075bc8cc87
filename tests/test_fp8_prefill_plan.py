"""How rbln_paged_causal_attn_prefill plans a call over an fp8 cache, seen through its workspace size (no GPU)."""

import ctypes

import torch


def workspace(S, **stride):
    from torch_rbln_b200 import cabi

    q, k = torch.zeros(2, 2, 4, S, 64, dtype=torch.bfloat16), torch.zeros(2, 2, 1, S, 64, dtype=torch.bfloat16)
    kc, sc = torch.zeros(8, 2, 1, 16, 64, dtype=torch.float8_e4m3fn), torch.ones(8, 2)
    seq, bt = torch.zeros(2, dtype=torch.int32), torch.zeros(2, 4, dtype=torch.int32)
    p, keep = cabi.paged_params(q, k, k, kc, kc, seq, bt, 16, 1.0, k_scale=sc, v_scale=sc)
    for i, v in stride.items():
        p.cache_stride[int(i[1:])] = v
    n = ctypes.c_size_t(0)
    assert cabi.lib().rbln_paged_prefill_workspace_size(ctypes.byref(p), ctypes.byref(n)) == cabi.OK
    return n.value


def test_large_pools_leave_the_kernel_of_32_bit_offsets():
    """The kernel for few rows holds offsets of 16 bytes in 32 bits: a pool whose last row lies past that, by its
    blocks or by its heads, goes to the one that takes 64."""
    few, many = workspace(4), workspace(20)  # 16 and 80 rows of a KV head
    assert few != many
    limit = 16 << 32
    assert workspace(4, _0=limit // 8 - 1024, _1=1024, _2=64) == few
    assert workspace(4, _0=limit // 7, _1=1024, _2=64) == many
    assert workspace(4, _0=1024, _1=limit, _2=64) == many  # heads outermost
    assert workspace(4, _0=1024, _1=limit - 16384, _2=64) == few
