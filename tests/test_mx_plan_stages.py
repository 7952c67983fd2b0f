"""CPU check, for 256 CUs, of which products of 128 x 128 FP4 tiles have a CU to each workgroup
(mx_alone in quant_ops_amd/csrc/dispatch_rules.h, compiled as it is): both kernels have GPU cases, whole
and in parts."""
import ctypes
import os
import subprocess

import pytest

from test_gpu_mx_stages import ALONE, SHARED
from test_gpu_mx_tiles import CASES

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CUS = 256
TILES = ("256", "128", "128x64", "64")

SOURCE = r"""
#include "dispatch_rules.h"
extern "C" int plan(int64_t M, int64_t N, int64_t blocks, int fp8, int64_t cus) {
  const qo::MxPlan p = qo::mx_plan(M, N, blocks, fp8 != 0, cus, true);
  return 32 * p.tile + 2 * p.splits + qo::mx_alone(p, M, N, cus);
}
"""


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    d = tmp_path_factory.mktemp("mx_stages")
    src, lib = d / "rules.cpp", d / "libstages.so"
    src.write_text(SOURCE)
    subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", f"-I{ROOT}/quant_ops_amd/csrc", str(src), "-o",
                    str(lib)], check=True)
    rules = ctypes.CDLL(str(lib))
    i64 = ctypes.c_int64
    rules.plan.argtypes = [i64, i64, i64, ctypes.c_int, i64]

    def of(m, n, blocks):
        got = rules.plan(m, n, blocks, 0, CUS)
        return TILES[got // 32], got // 2 % 16, bool(got % 2)

    return of


@pytest.mark.parametrize("m,n,blocks,parts", SHARED)
def test_shared_cases_reach_their_kernel(plan, m, n, blocks, parts):
    assert plan(m, n, blocks) == ("128", parts, False)


@pytest.mark.parametrize("m,n,blocks,parts", ALONE)
def test_alone_cases_reach_their_kernel(plan, m, n, blocks, parts):
    assert plan(m, n, blocks) == ("128", parts, True)


def test_both_kernels_have_cases(plan):
    held = {plan(m, n, blocks) for m, n, blocks, _ in SHARED + ALONE}
    held |= {plan(m, n, blocks) for m, n, blocks, fmt, _, _ in CASES if fmt == "mxfp4"}
    for m in (65, 100, 128, 200, 256, 257, 333, 512, 1000, 1024, 2048, 4096):
        for n in (1024, 2055, 4096, 8201, 11008, 14336, 28672):
            for blocks in (1, 3, 17, 64, 127, 128, 193, 257, 300, 344, 448, 896):
                tile, parts, alone = plan(m, n, blocks)
                if tile == "128":
                    assert (tile, parts, alone) in held, (m, n, blocks, parts, alone)
