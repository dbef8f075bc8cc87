"""The page operators' C entry points on a host without a GPU: the ctypes struct against the C layout, and calls that
are refused before anything is launched."""

import ctypes
import os
import subprocess

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_struct_field_offsets_match_c(tmp_path):
    from torch_rbln_b200 import cabi

    fields = [f for f, _ in cabi.PagesParams._fields_]
    src = "#include <stdio.h>\n#include <stddef.h>\n#include \"rbln_attn.h\"\nint main(void){\n"
    src += "".join(f'  printf("%zu\\n", offsetof(rbln_pages_params_t, {f}));\n' for f in fields)
    src += '  printf("%zu\\n", sizeof(rbln_pages_params_t));\n  return 0;\n}\n'
    (tmp_path / "off.c").write_text(src)
    cuda = os.path.join(os.environ.get("CUDA_HOME", "/usr/local/cuda"), "include")
    r = subprocess.run(["gcc", str(tmp_path / "off.c"), "-o", str(tmp_path / "off"), "-I",
                        os.path.join(ROOT, "include"), "-I", cuda], capture_output=True, text=True)
    if r.returncode != 0:
        pytest.skip("gcc or CUDA headers unavailable: " + r.stderr[-200:])
    offs = [int(x) for x in subprocess.run([str(tmp_path / "off")], capture_output=True, text=True).stdout.split()]
    assert offs == [getattr(cabi.PagesParams, f).offset for f in fields] + [ctypes.sizeof(cabi.PagesParams)]
    assert cabi.lib().rbln_pages_params_sizeof() == ctypes.sizeof(cabi.PagesParams)


def params(**changes):
    """A call that is in order (on host memory: nothing here may reach a launch), but for `changes`."""
    from torch_rbln_b200 import cabi

    t = {"table": torch.zeros(2, 4, dtype=torch.int32), "refs": torch.zeros(8, dtype=torch.int32),
         "lengths": torch.zeros(2, dtype=torch.int32), "cache": torch.zeros(8, 1, 1, 16, 64, dtype=torch.bfloat16)}
    p, keep = cabi.pages_params(t["table"], t["refs"], 16, t["lengths"], [t["cache"]], [t["cache"]])
    for name, value in changes.items():
        setattr(p, name, value)
    return p, (t, keep)


def reserve(p, new=1, granted=1):
    from torch_rbln_b200 import cabi

    return cabi.lib().rbln_paged_kv_reserve(ctypes.byref(p), new, granted, None)


@pytest.mark.parametrize("changes,rc", [
    ({"batch": -1}, -1), ({"max_blocks": -1}, -1), ({"num_blocks": -1}, -1), ({"block_size": 0}, -1),
    ({"block_table": None}, -1), ({"refs": None}, -1), ({"lengths": None}, -1),
    ({"block_table_dtype": 0}, -2), ({"lengths_dtype": 2}, -2),
    ({"block_table_dtype": 4, "num_blocks": 40000}, -2),
    ({"max_blocks": 2 ** 27}, -2),
])
def test_tables_are_refused(changes, rc):
    from torch_rbln_b200 import cabi

    p, keep = params(**changes)
    assert reserve(p) == rc
    assert cabi.lib().rbln_paged_kv_free(ctypes.byref(p), None) == rc
    assert cabi.lib().rbln_paged_kv_fork(ctypes.byref(p), 1, cabi.DT_I32, 1, 1, 1, 4, 1, None) == rc


@pytest.mark.parametrize("changes,rc", [
    ({"num_layers": 0}, -1), ({"num_kv_heads": 0}, -1), ({"head_dim": 0}, -1), ({"kv_dtype": 0}, -2),
    ({"kv_dtype": 3}, -1),  # fp8 without scales
    ({"head_dim": 65}, -1), ({"cache_stride": (ctypes.c_int64 * 3)(1024, 1024, 65)}, -1),
])
def test_caches_are_refused(changes, rc):
    from torch_rbln_b200 import cabi

    p, keep = params(**changes)
    assert reserve(p) == rc
    assert cabi.lib().rbln_paged_kv_compact(ctypes.byref(p), 1, 1, None) == rc


@pytest.mark.parametrize("head_dim,block_size,rc", [(128, 2 ** 27, -2), (64, 2 ** 28 - 1, -2), (128, 2 ** 27 - 17, -3),
                                                    (64, 2 ** 27, -3)])
def test_pages_whose_rows_pass_31_bits_are_refused(head_dim, block_size, rc):
    """A page is copied in 16-byte pieces, counted in 32 bits by lanes that step 256 at a time; -3: only the workspace is
    missing."""
    from torch_rbln_b200 import cabi

    p, keep = params(head_dim=head_dim, block_size=block_size, max_blocks=2)
    assert reserve(p) == rc
    assert cabi.lib().rbln_paged_kv_compact(ctypes.byref(p), 1, 1, None) == rc


def test_other_refusals():
    from torch_rbln_b200 import cabi

    L = cabi.lib()
    p, keep = params()
    assert reserve(p, new=-1) == -1 and reserve(p, granted=None) == -1
    assert reserve(p) == -3  # no workspace
    assert L.rbln_paged_kv_compact(ctypes.byref(p), 1, 1, None) == -3
    assert L.rbln_paged_kv_compact(ctypes.byref(p), 1, None, None) == -1
    assert L.rbln_paged_kv_fork(ctypes.byref(p), 1, cabi.DT_F32, 1, 1, 1, 4, 1, None) == -1
    assert L.rbln_paged_kv_fork(ctypes.byref(p), None, cabi.DT_I32, 1, 1, 1, 4, 1, None) == -1
    assert L.rbln_paged_kv_fork(ctypes.byref(p), None, cabi.DT_I32, 1, 0, None, 4, None, None) == 0  # nothing to do
    n = ctypes.c_size_t(0)
    assert L.rbln_paged_kv_pages_workspace_size(ctypes.byref(p), 1, None) == -1
    assert L.rbln_paged_kv_pages_workspace_size(ctypes.byref(p), 1, ctypes.byref(n)) == 0 and n.value > 0
    p.workspace, p.workspace_bytes = 256, n.value - 1
    assert reserve(p) == -3
    cache = keep[0]["cache"]
    ptr = (ctypes.c_void_p * 1)(cache.data_ptr() + 2)  # not on a 16-byte boundary
    p.kcaches = ctypes.cast(ptr, ctypes.POINTER(ctypes.c_void_p))
    assert reserve(p) == -1


def test_cpu_tensors_have_no_kernel():
    import torch_rbln_b200  # noqa: F401

    t, r, n = torch.zeros(2, 4, dtype=torch.int32), torch.zeros(8, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(NotImplementedError):
        torch.ops.rbln_attn.paged_kv_fork(t, n, n, r, 16)
    with pytest.raises(NotImplementedError):
        torch.ops.rbln_attn.paged_kv_free(t, n, r, 16)


def test_fake_kernels():
    import torch_rbln_b200  # noqa: F401
    from torch._subclasses.fake_tensor import FakeTensorMode

    ops = torch.ops.rbln_attn
    with FakeTensorMode():
        t = torch.empty(3, 5, dtype=torch.int64, device="cuda")
        r = torch.empty(9, dtype=torch.int32, device="cuda")
        n = torch.empty(3, dtype=torch.int32, device="cuda")
        c = [torch.empty(9, 2, 1, 16, 64, dtype=torch.bfloat16, device="cuda")]
        rows, lens = ops.paged_kv_fork(t, n, torch.empty(7, dtype=torch.int32, device="cuda"), r, 16)
        assert rows.shape == (7, 5) and rows.dtype == torch.int64 and lens.shape == (7,) and lens.dtype == torch.int32
        assert ops.paged_kv_free(t, n, r, 16) is None
        granted = ops.paged_kv_reserve(c, c, t, n, r, 16, 2)
        assert granted.shape == (3,) and granted.dtype == torch.int32
        moved, live = ops.paged_kv_compact(c, c, t, r)
        assert moved.shape == (9,) and live.shape == (1,)
