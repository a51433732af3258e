"""Bounds check on the CPU of the language-model kernels whose addresses do not depend on data (the products' epilogue, RMS norm,
activation backward): the library's own sources compiled as host C++ and every thread of every launch run with each tensor between
inaccessible pages (tests/kernel_walk/walk_lm.cpp)."""
import os
import subprocess
from concurrent.futures import ThreadPoolExecutor

import pytest

from test_patch_kernel_addresses import CLANG, ROOT, WALK_DIR

PARTS = ("GEMM", "NORM", "ACT")


@pytest.fixture(scope="module")
def binaries():
    if not os.path.exists(CLANG):
        pytest.skip("no clang++ to build the host emulation with")
    out = os.path.join(WALK_DIR, "build")
    os.makedirs(out, exist_ok=True)

    def build(part):
        exe = os.path.join(out, "walk_lm_" + part.lower())
        r = subprocess.run([CLANG, "-x", "c++", "-std=c++17", "-O1", "-I", WALK_DIR, "-DFX_HOST_EMULATION=1", "-DWALK_" + part, "-Wno-unknown-attributes",
                            "-Wno-unused-value", "-Wno-psabi", "-fsanitize=signed-integer-overflow,shift,bounds,integer-divide-by-zero",
                            "-fno-sanitize-recover=all", "-o", exe, os.path.join(ROOT, "tests", "kernel_walk", "walk_lm.cpp")],
                           capture_output=True, text=True, cwd=WALK_DIR)
        assert r.returncode == 0, r.stderr[-4000:]
        return exe
    with ThreadPoolExecutor(len(PARTS)) as pool:
        return dict(zip(PARTS, pool.map(build, PARTS)))


def walk(exe, cases, env=None):
    lines = "".join("%s %s %d %d %d %d\n" % ((f"c{i}", dt) + dims) for i, (dt, dims) in enumerate(cases))
    return subprocess.run([exe], input=lines, capture_output=True, text=True, env=dict(os.environ, **(env or {})), timeout=900)


# M, N, K: every kernel of the dispatch (few rows, small tiles of both sizes, split K, slab tiles of 64 and 128 rows with and without a
# remainder of K, thin products, general tiles), edges in both dimensions
GEMM = [(1, 1, 1), (1, 130, 4097), (3, 257, 1001), (4, 64, 512), (5, 7, 3), (33, 65, 31), (100, 100, 64), (256, 64, 784), (10, 300, 300), (130, 260, 192),
        (16, 40, 4096), (300, 129, 100), (8, 8200, 64), (1028, 1028, 132), (1024, 512, 192), (1025, 511, 260), (2052, 1028, 128)]
NORM = [(1, 1), (3, 5), (5, 255), (5, 256), (3, 257), (2, 516), (3, 1001), (1030, 12), (2, 1025), (2, 2052), (1, 4097), (2, 16383), (2, 16385), (3, 20001)]
ACT = [(1, 1), (3, 5), (70, 255), (33, 256), (9, 257), (1030, 12), (5, 1001)]


def test_epilogue_of_the_products(binaries):
    cases = [(dt, dims + (s,)) for dims in GEMM for dt, s in (("f32", 0), ("f32", 2), ("f64", 0))] + [("f32", d + (1,)) for d in GEMM[:10]]
    groups = [cases[k::6] for k in range(6)]
    with ThreadPoolExecutor(6) as pool:
        for r in pool.map(lambda g: walk(binaries["GEMM"], g), groups):
            assert r.returncode == 0 and "every access stayed inside" in r.stdout, r.stderr[-2000:]


@pytest.mark.parametrize("part,sizes", [("NORM", NORM), ("ACT", ACT)])
def test_rows(binaries, part, sizes):
    r = walk(binaries[part], [(dt, d + (0, s)) for d in sizes for dt in ("f32", "f64") for s in (0, 1)])
    assert r.returncode == 0 and "every access stayed inside" in r.stdout, r.stderr[-2000:]


@pytest.mark.parametrize("part,tensor,dims", [("GEMM", "residual", (64, 64, 64)), ("GEMM", "pre", (64, 64, 64)), ("GEMM", "bias", (1, 64, 64)),
                                              ("NORM", "residual", (2, 64, 0)), ("NORM", "w", (2, 64, 0)), ("NORM", "dw", (2, 64, 0)),
                                              ("ACT", "pre", (4, 64, 0)), ("ACT", "db", (4, 64, 0))])
def test_the_walk_notices_a_tensor_that_is_too_short(binaries, part, tensor, dims):
    # one f64 element short: the block then ends 8 bytes in front of the guard, and the kernel's last vector reaches into it
    r = walk(binaries[part], [("f64", dims + (1,))], {"FX_WALK_SHORT": tensor})
    assert r.returncode == 3 and "FAULT" in r.stderr, (r.returncode, r.stderr[-500:])
