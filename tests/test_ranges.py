"""csrc/ranges.cuh, compiled for the host with every overflow an error: arithmetic at the ends of its range."""

import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
MOST = 2 ** 31 - 1


def values(tmp_path, expressions):
    src = "#include <stdio.h>\n#include \"ranges.cuh\"\nint main() {\n"
    src += "".join(f'  printf("%lld\\n", (long long)({e}));\n' for e in expressions) + "}\n"
    (tmp_path / "r.cpp").write_text(src)
    # the arguments are kept from the compiler's constant folding by no optimisation
    r = subprocess.run(["g++", "-O0", "-std=c++17", "-fsanitize=undefined", "-fno-sanitize-recover", "-I",
                        os.path.join(ROOT, "torch-rbln_b200", "csrc"), str(tmp_path / "r.cpp"), "-o", str(tmp_path / "r")],
                       capture_output=True, text=True)
    if r.returncode != 0 and "ubsan" in r.stderr:
        pytest.skip("no sanitizer runtime: " + r.stderr[-200:])
    assert r.returncode == 0, r.stderr
    r = subprocess.run([str(tmp_path / "r")], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    return [int(x) for x in r.stdout.split()]


def test_positions_seen(tmp_path):
    cases = [(p, s) for s in (0, 1, 64, 2 ** 30, MOST)
             for p in (-MOST - 1, -1, 0, 1, 62, 63, 64, 65, 2 ** 30 - 1, 2 ** 30, MOST - 1, MOST)]
    got = values(tmp_path, [f"rbln::positions_seen({'-2147483647 - 1' if p == -MOST - 1 else p}, {s})" for p, s in cases])
    assert got == [0 if p < 0 else min(p + 1, s) for p, s in cases]


def test_share_start(tmp_path):
    lines = [(4, 0), (4, 1), (4, 590), (9, 1000), (7_300_000, 2 ** 30 - 1), (14_700_000, 14_700_000), (2 ** 29, 2 ** 30 - 1),
             (2 ** 30 - 1, 2 ** 30 - 1)]
    cases = [(c, share, line) for share, line in lines for c in (0, 1, 2, 100, 146, 147, 148)]
    got = values(tmp_path, [f"rbln::share_start({c}, {share}, {line})" for c, share, line in cases])
    assert got == [min(c * share, line) for c, share, line in cases]
