"""CPU checks of the rotary and quantised-cache operators: registration,
tracing, refusals that come before any launch, and the frequencies."""

import ctypes
import math

import pytest
import torch


@pytest.fixture(scope="module", autouse=True)
def _ext():
    import torch_rbln_b200  # noqa: F401


def test_argument_counts():
    import torch_rbln_b200 as tr

    with pytest.raises(RuntimeError, match="takes 12 or 13 inputs"):
        tr.paged_causal_attn_prefill_kvfp8(*([None] * 11))


def test_no_cpu_kernels():
    q = torch.zeros(1, 2, 3, 64)
    with pytest.raises(NotImplementedError):
        torch.ops.rbln_attn.rotary(q, q, torch.zeros(1, 3, dtype=torch.int64), torch.zeros(32))
    kc = torch.zeros(2, 1, 1, 16, 64, dtype=torch.bfloat16)
    with pytest.raises(NotImplementedError):
        torch.ops.rbln_attn.paged_kv_read(kc, kc, torch.zeros(1, dtype=torch.int32), torch.zeros(1, 1, dtype=torch.int32),
                                          16, 16)


def test_tracing():
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode():
        q = torch.empty(2, 5, 4, 64, dtype=torch.bfloat16).transpose(1, 2)
        a, b = torch.ops.rbln_attn.rotary(q, q[:, :2], torch.empty(2, 5, dtype=torch.int64), torch.empty(32))
        assert a.stride() == q.stride() and b.shape == (2, 2, 5, 64)
        q = torch.empty(2, 8, 4, 3, 64, dtype=torch.bfloat16)
        k = torch.empty(2, 8, 1, 3, 64, dtype=torch.bfloat16)
        kc = torch.empty(9, 8, 1, 16, 64, dtype=torch.float8_e4m3fn)
        sc = torch.empty(9, 8)
        seq, bt = torch.empty(2, dtype=torch.int32), torch.empty(2, 4, dtype=torch.int32)
        out = torch.ops.rbln_attn.rotary_paged_kv_write(q, k, k, kc, kc, seq, bt, 16, torch.empty(32), False, 1.0, sc, sc)
        assert out.shape == q.shape and out.dtype == q.dtype
        out = torch.ops.rbln_custom_ops.paged_causal_attn_prefill_kvfp8(q, None, None, kc, kc, sc, sc, seq, torch.empty(()),
                                                                       bt, 16, False)
        assert out.shape == q.shape
        k, v = torch.ops.rbln_attn.paged_kv_read(kc, kc, seq, bt, 16, 40, sc, sc)
        assert k.shape == (2, 8, 1, 40, 64) and v.dtype == torch.bfloat16


def _stream():
    return ctypes.c_void_p(None)


def test_rotary_refusals():
    from torch_rbln_b200 import cabi

    L = cabi.lib()
    assert L.rbln_rotary(None, None) == cabi.ERR_INVALID_ARGUMENT
    q, k = torch.zeros(2, 4, 3, 64, dtype=torch.bfloat16), torch.zeros(2, 2, 3, 64, dtype=torch.bfloat16)
    pos, f = torch.zeros(2, 3, dtype=torch.int64), torch.zeros(32)

    def rc(**change):
        p = cabi.rotary_params(q, k, q, k, pos, f)
        for n, v in change.items():
            setattr(p, n, v)
        return L.rbln_rotary(ctypes.byref(p), None)

    for bad in ({"rotary_dim": 0}, {"rotary_dim": 31}, {"rotary_dim": 66}, {"head_dim": 0}, {"batch": -1},
                {"q": None}, {"k_out": None}, {"positions": None}, {"inv_freq": None}):
        assert rc(**bad) == cabi.ERR_INVALID_ARGUMENT, bad
    for bad in ({"dtype": cabi.DT_FP8_E4M3}, {"positions_dtype": cabi.DT_I16}, {"head_dim": 2048}):
        assert rc(**bad) == cabi.ERR_UNSUPPORTED, bad
    assert rc(batch=0) == cabi.OK and rc(seq_len=0) == cabi.OK


def _paged(cabi, S=3, D=64, bs=16, cache=torch.float8_e4m3fn, dtype=torch.bfloat16):
    q = torch.zeros(2, 2, 4, S, D, dtype=dtype)
    k = torch.zeros(2, 2, 1, S, D, dtype=dtype)
    kc = torch.zeros(8, 2, 1, bs, D, dtype=cache)
    seq, bt = torch.zeros(2, dtype=torch.int32), torch.zeros(2, 4, dtype=torch.int32)
    sc = torch.ones(8, 2)
    p, keep = cabi.paged_params(q, k, k, kc, kc, seq, bt, bs, 1.0, k_scale=sc, v_scale=sc)
    keep["all"] = (q, k, kc, seq, bt, sc)
    return p, keep


def test_rotary_write_refusals():
    from torch_rbln_b200 import cabi

    L = cabi.lib()
    f = torch.zeros(32)

    def rc(rot=64, inv=True, **change):
        p, keep = _paged(cabi)
        r = cabi.RotaryParams()
        r.rotary_dim, r.inv_freq, r.mscale = rot, f.data_ptr() if inv else None, 1.0
        for n, v in change.items():
            setattr(p, n, v)
        return L.rbln_rotary_paged_kv_write(ctypes.byref(p), ctypes.byref(r), None)

    assert L.rbln_rotary_paged_kv_write(None, None, None) == cabi.ERR_INVALID_ARGUMENT
    for bad in ({"rot": 0}, {"rot": 80}, {"inv": False}, {"q": None}, {"k_new": None}, {"k_scale": None}, {"seq": None},
                {"kcache": 8 + 4}, {"block_size": 0}):
        assert rc(**bad) == cabi.ERR_INVALID_ARGUMENT, bad
    for bad in ({"rot": 24}, {"head_dim": 96}, {"q_dtype": cabi.DT_F32}, {"kv_dtype": cabi.DT_F16},
                {"block_table_dtype": cabi.DT_F32}, {"max_blocks": 1 << 28}):
        assert rc(**bad) == cabi.ERR_UNSUPPORTED, bad
    assert rc(batch=0) == cabi.OK and rc(q_len=0) == cabi.OK


def test_read_refusals():
    from torch_rbln_b200 import cabi

    L = cabi.lib()
    out = torch.zeros(2, 2, 3, 64, dtype=torch.bfloat16)
    stride = (ctypes.c_int64 * 3)(out.stride(0), out.stride(1), out.stride(2))

    def rc(to=out.data_ptr(), **change):
        p, keep = _paged(cabi)
        for n, v in change.items():
            setattr(p, n, v)
        return L.rbln_paged_kv_read(ctypes.byref(p), to, out.data_ptr(), stride, None)

    for bad in ({"to": None}, {"to": out.data_ptr() + 2}, {"kcache": None}, {"v_scale": None}, {"seq": None},
                {"num_blocks": 0}):
        assert rc(**bad) == cabi.ERR_INVALID_ARGUMENT, bad
    for bad in ({"head_dim": 96}, {"q_dtype": cabi.DT_FP8_E4M3}, {"kv_dtype": cabi.DT_F32},
                {"block_table_dtype": cabi.DT_BOOL}):
        assert rc(**bad) == cabi.ERR_UNSUPPORTED, bad
    assert rc(batch=0) == cabi.OK and rc(q_len=0) == cabi.OK


def test_fp8_prefill_refusals():
    from torch_rbln_b200 import cabi

    L = cabi.lib()

    def rc(S=3, **change):
        p, keep = _paged(cabi, S=S)
        n = ctypes.c_size_t(0)
        assert L.rbln_paged_prefill_workspace_size(ctypes.byref(p), ctypes.byref(n)) == cabi.OK
        ws = torch.empty(max(n.value, 1), dtype=torch.uint8)
        p.workspace, p.workspace_bytes = ws.data_ptr(), n.value
        for name, v in change.items():
            setattr(p, name, v)
        return L.rbln_paged_causal_attn_prefill(ctypes.byref(p), None)

    for S in (1, 3, 200):
        for bad in ({"q": None}, {"k_new": None}, {"k_scale": None}, {"block_table": None}, {"kcache": 16 + 8},
                    {"group": 0}):
            assert rc(S, **bad) == cabi.ERR_INVALID_ARGUMENT, bad
        for bad in ({"block_size": 12}, {"block_size": 192}, {"head_dim": 96}, {"q_dtype": cabi.DT_F32},
                    {"group": 129}, {"sinks": 16}, {"block_table_dtype": cabi.DT_F32}):
            assert rc(S, **bad) == cabi.ERR_UNSUPPORTED, bad
        assert rc(S, workspace=None) == cabi.ERR_WORKSPACE
        assert rc(S, workspace_bytes=16) == cabi.ERR_WORKSPACE
        assert rc(S, batch=0) == cabi.OK
    p, keep = _paged(cabi)
    assert L.rbln_paged_attn_prefill(ctypes.byref(p), None) == cabi.ERR_UNSUPPORTED  # keep-masks: 16-bit caches only


def test_frequencies():
    from torch_rbln_b200 import rotary_frequencies as rf

    f, m = rf(128)
    i = torch.arange(64, dtype=torch.float64)
    plain = 10000.0 ** (-2 * i / 128)
    assert f.dtype == torch.float32 and torch.equal(f, plain.float()) and m == 1.0
    f, m = rf(128, 500000.0, "linear", 8.0)
    assert torch.equal(f, (500000.0 ** (-2 * i / 128) / 8).float()) and m == 1.0
    f, m = rf(64, 10000.0, "ntk", 4.0)
    # the fastest pair stays, the slowest is divided by the factor
    assert f[0] == 1.0 and abs(float(f[-1]) * 4.0 * 10000.0 ** (62 / 64) - 1) < 1e-6
    f, m = rf(128, 10000.0, "yarn", 16.0, 4096)
    assert abs(m - (0.1 * math.log(16.0) + 1)) < 1e-12
    turns = 4096 * plain / (2 * math.pi)
    fast, slow = turns > 40, turns < 0.8
    assert torch.equal(f[fast], plain[fast].float()) and torch.equal(f[slow], (plain[slow] / 16).float())
    assert ((f.double() <= plain * (1 + 1e-6)) & (f.double() >= plain / 16 * (1 - 1e-6))).all()
    f, m = rf(128, 500000.0, "llama3", 8.0, 8192, 1.0, 4.0)
    plain = 500000.0 ** (-2 * i / 128)
    turns = 8192 * plain / (2 * math.pi)
    w = ((turns - 1) / 3).clamp(0, 1)
    torch.testing.assert_close(f.double(), w * plain + (1 - w) * plain / 8, rtol=2.0 ** -23, atol=0)
    assert m == 1.0
    for bad in ((7,), (0,), (64, 0.5), (64, 1e4, "linear", 0.5), (64, 1e4, None, 2.0), (64, 1e4, "yarn", 2.0),
                (64, 1e4, "other", 2.0), (64, 1e4, "llama3", 2.0, 100, 4.0, 1.0), (2, 1e4, "ntk", 2.0)):
        with pytest.raises(ValueError):
            rf(*bad)


def test_rotary_struct_matches_c():
    import os
    import subprocess
    import tempfile

    from torch_rbln_b200 import cabi

    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    fields = [f for f, _ in cabi.RotaryParams._fields_]
    src = "#include <stdio.h>\n#include <stddef.h>\n#include \"rbln_attn.h\"\nint main(void){\n"
    for f in fields:
        src += f'  printf("%zu\\n", offsetof(rbln_rotary_params_t, {f}));\n'
    src += '  printf("%zu\\n", sizeof(rbln_rotary_params_t));\n  return 0;\n}\n'
    with tempfile.TemporaryDirectory() as td:
        c, exe = os.path.join(td, "off.c"), os.path.join(td, "off")
        open(c, "w").write(src)
        inc = os.path.join(os.environ.get("CUDA_HOME", "/usr/local/cuda"), "include")
        r = subprocess.run(["gcc", c, "-o", exe, "-I", os.path.join(root, "include"), "-I", inc], capture_output=True,
                           text=True)
        if r.returncode != 0:
            pytest.skip("gcc or CUDA headers unavailable: " + r.stderr[-200:])
        want = [int(x) for x in subprocess.run([exe], capture_output=True, text=True).stdout.split()]
    assert want == [getattr(cabi.RotaryParams, f).offset for f in fields] + [ctypes.sizeof(cabi.RotaryParams)]
