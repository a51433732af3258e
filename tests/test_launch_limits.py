"""Launches of the language-model operators at sizes near 2^32 threads, counted on the CPU against the device's limits: the library's own
host code with launches that are looked at instead of run (tests/launch_limits)."""
import os
import subprocess
from concurrent.futures import ThreadPoolExecutor

import pytest

from test_patch_kernel_addresses import CLANG, ROOT, WALK_DIR

DIR = os.path.join(ROOT, "tests", "launch_limits")
PARTS = ("GEMM", "NORM", "ACT", "EMBED", "SCAN", "CLIP")
B31 = (1 << 31) - 1


@pytest.fixture(scope="module")
def binaries():
    if not os.path.exists(CLANG):
        pytest.skip("no clang++ to build the host emulation with")
    out = os.path.join(WALK_DIR, "build")
    os.makedirs(out, exist_ok=True)

    def build(part):
        exe = os.path.join(out, "limits_" + part.lower())
        r = subprocess.run([CLANG, "-x", "c++", "-std=c++17", "-O1", "-I", DIR, "-DFX_HOST_EMULATION=1", "-DLIMITS_" + part, "-Wno-unknown-attributes",
                            "-Wno-unused-value", "-Wno-psabi", "-o", exe, os.path.join(DIR, "limits.cpp")], capture_output=True, text=True, cwd=DIR)
        assert r.returncode == 0, r.stderr[-4000:]
        return exe
    with ThreadPoolExecutor(len(PARTS)) as pool:
        return dict(zip(PARTS, pool.map(build, PARTS)))


def run(exe, cases):
    lines = "".join("%s %s %d %d %d\n" % c for c in cases)
    r = subprocess.run([exe], input=lines, capture_output=True, text=True, timeout=100)
    assert r.returncode == 0, r.stderr
    return r.stdout.splitlines()


# call, type, three sizes: (products) M N K, (rows) rows dim -, (lookup) tokens vocabulary dim, (recurrence) sequences steps dim, (clipping) tensors
# elements -.
TAKEN = {
    "GEMM": [("linear", t, m, n, k) for t in ("f32", "f64") for m, n, k in ((1, (1 << 26) - 4, 2), (1, (1 << 26) - 3, 2), (1, (1 << 26) - 1, 1), (1, 1 << 26, 2),
                                                                          (4, (1 << 26) - 1, 512), (2, 70000000, 513), (4000000, 1, 2), (1, 1, 1 << 20),
                                                                          (70000, 70000, 0), (1, 1 << 30, 0))],
    "NORM": [(c, t, r, d, 0) for t in ("f32", "f64") for c in ("norm", "norm_res", "norm_bwd")
             for r, d in ((B31, 1), (1 << 26, 257), ((1 << 26) + 1, 256), (1 << 24, 2049), (1 << 22, 4097), ((1 << 22) - 1, 4097), ((1 << 23) + 1, 4098),
                          (1 << 22, 16384), (1 << 22, 16385), ((1 << 22) + 7, 16390), (3, B31), (1, B31))],
    "ACT": [("act_bwd", t, r, d, 0) for t in ("f32", "f64") for r, d in ((B31, 1), (1, B31), (70000, 1 << 20), (1 << 20, 70000))],
    "EMBED": [("embed", t, n, v, d) for t in ("f32", "f64") for n, v, d in ((B31, 1, 1), (B31, 5, 29), (B31, 7, 15), (1 << 20, 4, 60001), (3, 2, B31))]
    + [("embed_bwd", t, n, v, d) for t in ("f32", "f64") for n, v, d in ((B31, 1000, 1), (100, (1 << 30) - (1 << 20), 1), (1 << 20, 1 << 20, 50000), (5, 3, 8000000))],
    "SCAN": [(c, t, b, s, d) for t in ("f32", "f64") for c in ("scan", "scan_bwd")
             for b, s, d in ((1, 1, B31), (4000, 1, 1 << 20), (1, (1 << 28) - 100, 1), (2, 1 << 20, 1001), (1 << 20, 1000, 7))],
    "CLIP": [("clip", t, n, e, 0) for t in ("f32", "f64") for n, e in ((1, 1 << 35), (3, B31), (5000, 70), (97, 1 << 26), (1, 1))],
}


@pytest.mark.parametrize("part", PARTS)
def test_sizes_that_one_launch_cannot_hold(binaries, part):
    for case, said in zip(TAKEN[part], run(binaries[part], TAKEN[part])):
        assert said.endswith("launches") and said != "0 launches", (case, said)


def test_sizes_that_are_refused(binaries):
    """With a message, before anything is launched that could not run."""
    cases = {"GEMM": [("linear", "f32", 70000000, 1, 2), ("linear", "f32", 5, B31, 1)],
             "EMBED": [("embed_bwd", "f32", 100, 1 << 30, 1), ("embed_bwd", "f32", 3, 2, 1 << 25), ("embed_bwd", "f64", 3, 2, 1 << 24), ("embed", "f32", 1 << 31, 2, 2)],
             "SCAN": [("scan", "f32", 1, 1 << 30, 1), ("scan_bwd", "f64", 1, 1 << 28, 1), ("scan", "f32", 4, 1, 1 << 30)]}
    for part, list_ in cases.items():
        for case, said in zip(list_, run(binaries[part], list_)):
            assert said.startswith("refused: "), (case, said)
