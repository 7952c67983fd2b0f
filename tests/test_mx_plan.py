"""CPU check of the rule that gives the microscaled product its tile and the parts of
its sum (mx_plan in quant_ops_amd/csrc/dispatch_rules.h), compiled as it is, for 256 CUs."""
import ctypes
import os
import subprocess

import pytest

from test_gpu_mx_tiles import CASES

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CUS = 256
TILES = ("256", "128", "128x64", "64")

SOURCE = r"""
#include "dispatch_rules.h"
extern "C" int plan(int64_t M, int64_t N, int64_t blocks, int fp8, int64_t cus, int may_split) {
  const qo::MxPlan p = qo::mx_plan(M, N, blocks, fp8 != 0, cus, may_split != 0);
  return 16 * p.tile + p.splits;
}
extern "C" int64_t bytes(int tile, int splits, int64_t M, int64_t N) {
  return qo::mx_plan_bytes({(qo::MxTileKind)tile, splits}, M, N);
}
"""


@pytest.fixture(scope="module")
def rules(tmp_path_factory):
    d = tmp_path_factory.mktemp("mx_rules")
    src, lib = d / "rules.cpp", d / "librules.so"
    src.write_text(SOURCE)
    subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", f"-I{ROOT}/quant_ops_amd/csrc", str(src), "-o",
                    str(lib)], check=True)
    rules = ctypes.CDLL(str(lib))
    i64 = ctypes.c_int64
    rules.plan.argtypes = [i64, i64, i64, ctypes.c_int, i64, ctypes.c_int]
    rules.bytes.argtypes = [ctypes.c_int, ctypes.c_int, i64, i64]
    rules.bytes.restype = i64
    return rules


def _plan(rules, m, n, blocks, fmt, split=True):
    got = rules.plan(m, n, blocks, int(fmt == "mxfp8"), CUS, int(split))
    return TILES[got // 16], got % 16


@pytest.mark.parametrize("m,n,blocks,fmt,tile,parts", CASES)
def test_cases_reach_their_kernel(rules, m, n, blocks, fmt, tile, parts):
    assert _plan(rules, m, n, blocks, fmt) == (tile, parts)
    assert _plan(rules, m, n, blocks, fmt, split=False)[1] == 1


def test_cases_hold_every_plan_of_a_range(rules):
    """Every tile and number of parts that these sizes take has a case."""
    held = {(c[3], c[4], c[5]) for c in CASES}
    for fmt in ("mxfp4", "mxfp8"):
        for m in (17, 18, 33, 64, 65, 100, 128, 200, 256, 257, 333, 512, 1000, 1024, 2048, 4096):
            for n in (32, 41, 300, 1024, 2055, 4096, 8201, 11008, 14336, 28672):
                for blocks in (1, 3, 17, 64, 127, 128, 193, 257, 300, 344, 448, 896):
                    assert (fmt, *_plan(rules, m, n, blocks, fmt)) in held, (m, n, blocks, fmt)


@pytest.mark.parametrize("fmt", ("mxfp4", "mxfp8"))
def test_large_products_take_large_tiles(rules, fmt):
    for m, n, blocks in [(4096, 4096, 448), (8192, 8192, 256), (4096, 14336, 128), (2048, 28672, 128)]:
        assert _plan(rules, m, n, blocks, fmt) == ("256", 1)
    assert _plan(rules, 64, 64, 448, fmt)[1] == 8    # one tile: its sum is divided


def test_parts_have_quads_and_room(rules):
    """No part is empty, and the parts' room is whole tiles of float32."""
    for fmt in ("mxfp4", "mxfp8"):
        for blocks in range(1, 260, 3):
            for m, n in ((17, 41), (65, 4097), (257, 300)):
                assert _plan(rules, m, n, blocks, fmt)[1] <= (blocks + 15) // 16
    assert rules.bytes(TILES.index("64"), 8, 65, 64) == 8 * 2 * 64 * 64 * 4
    assert rules.bytes(TILES.index("128x64"), 2, 128, 65) == 2 * 2 * 128 * 64 * 4
