"""Fake (meta) kernels: output metadata equals q's, as in the reference's
register_fake functions (test/rbln/test_custom_kernel.py:95-135, 219-259,
346-385, 489-526, 597-645)."""

from __future__ import annotations

import torch

_NAMES = (
    "paged_attn_prefill",
    "paged_attn_decode",
    "paged_causal_attn_prefill",
    "paged_causal_attn_prefill_kvfp8",
    "paged_causal_attn_decode",
    "paged_causal_attn_decode_kvfp8",
    "flash_attention_naive_prefill",
    "flash_attention_naive_decode",
)


def _like_q(q, *args, **kwargs):
    return torch.empty_like(q)


for _name in _NAMES:
    if hasattr(torch.ops.rbln_custom_ops, _name):
        torch.library.register_fake(f"rbln_custom_ops::{_name}", _like_q)


def _writes_only(*args, **kwargs):
    """paged_kv_write mutates its caches (and scales) and returns nothing."""
    return None


torch.library.register_fake("rbln_attn::paged_kv_write", _writes_only)


@torch.library.register_fake("rbln_attn::rotary")
def _rotary(q, k, positions, inv_freq, interleaved=False, mscale=1.0, inverse=False):
    def like(x):  # x's layout, unless that would leave the head dimension strided
        y = torch.empty_like(x)
        return y if y.stride(-1) == 1 else torch.empty_like(x, memory_format=torch.contiguous_format)

    return like(q), like(k)


@torch.library.register_fake("rbln_attn::rotary_paged_kv_write")
def _rotary_paged_kv_write(q, *args, **kwargs):
    return torch.empty_like(q, memory_format=torch.contiguous_format)


@torch.library.register_fake("rbln_attn::paged_kv_read")
def _paged_kv_read(kcache, vcache, lengths, block_table, block_size, max_len, k_scale=None, v_scale=None, dtype=None):
    if dtype is None:
        dtype = torch.bfloat16 if kcache.dtype == torch.float8_e4m3fn else kcache.dtype
    shape = [lengths.numel(), kcache.shape[1], 1, max_len, kcache.shape[-1]]
    return kcache.new_empty(shape, dtype=dtype), kcache.new_empty(shape, dtype=dtype)
