"""CPU checks of the rule that shares attention over the 4-bit cache out (kv4_plan in quant_ops_amd/csrc/dispatch_rules.h),
compiled as it is, for 256 CUs: the GPU tests' cases reach every kernel, and every row has its workgroup."""
import ctypes
import os
import random
import subprocess

import pytest

from test_gpu_kv4 import EVERY_KERNEL, GPU_CASES
from test_kv4_cpu import CASES

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CUS = 256

SOURCE = r"""
#include "dispatch_rules.h"
extern "C" void plan(int64_t tokens, int64_t q_heads, int64_t kv_heads, int64_t head_dim, int64_t capacity, int64_t sequences,
                     int ragged, int64_t window, int f32, int64_t cus, int64_t* out) {
  const qo::Kv4Plan p = qo::kv4_plan(tokens, q_heads, kv_heads, head_dim, capacity, sequences, ragged != 0, window, f32 != 0, cus);
  out[0] = p.rows, out[1] = p.tiles, out[2] = p.splits;
}
"""


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    d = tmp_path_factory.mktemp("kv4_rules")
    src, lib = d / "rules.cpp", d / "librules.so"
    src.write_text(SOURCE)
    subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", f"-I{ROOT}/quant_ops_amd/csrc", str(src), "-o",
                    str(lib)], check=True)
    call = ctypes.CDLL(str(lib)).plan
    i64, flag = ctypes.c_int64, ctypes.c_int
    call.argtypes = [i64] * 6 + [flag, i64, flag, i64, ctypes.POINTER(i64)]
    call.restype = None

    def run(tokens, q_heads, kv_heads, dim, capacity, sequences, ragged, window, f32):
        out = (i64 * 3)()
        call(tokens, q_heads, kv_heads, dim, capacity, sequences, ragged, window, f32, CUS, out)
        return tuple(out)

    return run


def _case(plan, case, f32):
    lengths, heads, kv, dim, page, queries, window = case
    ragged = not isinstance(queries, int)
    rows = sum(queries) + 2 if ragged else queries * len(lengths)
    width = max([-(-max(n, 0) // page) for n in lengths] + [1])
    return plan(rows, heads, kv, dim, width * page, len(lengths), ragged, window, f32)


def test_cases_reach_every_kernel(plan):
    """Rows of a wave (4, 8, 16; prompts of 16-bit types 32 and 64), head sizes, and one, few or many parts."""
    want = {(r, dim, False) for r in (4, 8, 16, 32, 64) for dim in (64, 96, 128, 192, 256) if r < 64 or dim <= 128}
    want |= {(r, dim, True) for r in (4, 8, 16) for dim in (64, 96, 128, 192, 256)}
    parts = {(kind, f32) for kind in ("one", "few", "many") for f32 in (False, True)}
    for case in CASES + GPU_CASES + EVERY_KERNEL:
        for f32 in (False, True):
            rows, _, splits = _case(plan, case, f32)
            want.discard((rows, case[3], f32))
            parts.discard(("one" if splits == 1 else "few" if splits <= 4 else "many", f32))
    assert not want and not parts


@pytest.mark.parametrize("f32", [False, True])
def test_plans_hold(plan, f32):
    rng = random.Random(1)
    for _ in range(3000):
        group, kv = rng.choice((1, 2, 3, 4, 7, 8, 16, 64)), int(2 ** rng.uniform(0, 5))
        dim = rng.choice((64, 96, 128, 192, 256))
        sequences = int(2 ** rng.uniform(0, 8))
        ragged, window = rng.random() < 0.5, rng.choice((0, 0, 1, 100, 5000))
        counts = [int(2 ** rng.uniform(0, 9)) - 1 if ragged else 0 for _ in range(sequences)]
        each = int(2 ** rng.uniform(0, 9))
        tokens = max(1, sum(counts) + rng.randint(0, 9)) if ragged else each * sequences
        capacity = int(2 ** rng.uniform(0, 20))
        rows, tiles, splits = plan(tokens, group * kv, kv, dim, capacity, sequences, ragged, window, f32)
        assert rows in ((4, 8, 16) if f32 or not tokens else (4, 8, 16, 32, 64)) and (rows < 64 or dim <= 128)
        assert 1 <= splits <= 64 and (splits == 1 or splits * 128 <= capacity)
        tile = 4 * rows
        if not ragged:
            assert tiles == sequences * -(-each * group // tile)
            continue
        # a tile's place is start * group / tile + sequence + its number: none taken twice, none beyond the last
        taken, start = set(), 0
        for b, n in enumerate(counts + [tokens - sum(counts)]):
            for i in range(-(-n * group // tile)):
                at = start * group // tile + b + i
                assert at < tiles and at not in taken
                taken.add(at)
            start += n


def test_a_split_does_not_lengthen_the_work(plan):
    """More tokens never get fewer parts, for one sequence on an empty machine."""
    last = 0
    for tokens in (1, 100, 700, 1500, 4000, 16000, 60000, 131072, 1 << 20):
        splits = plan(1, 64, 8, 128, tokens, 1, False, 0, False)[2]
        assert splits >= last
        last = splits
    assert last == 64
