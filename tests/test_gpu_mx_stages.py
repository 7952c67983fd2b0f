"""FP4 products on 128 x 128 tiles with more workgroups than CUs, whose kernel has fewer stages than
the one of workgroups that have a CU each (mx_alone in dispatch_rules.h), with ragged edges and last
quads, on its own output and in parts. test_mx_plan_stages.py checks that the sizes go there."""
import pytest

import test_gpu_mx_tiles as tiles

pytestmark = pytest.mark.gpu

# M, N, blocks of 32 values; parts
SHARED = [
    (300, 11007, 1, 1),         # one block
    (257, 12300, 16, 1),        # one whole quad of k-steps
    (257, 11007, 33, 1),        # the last of three quads holds one block
    (333, 11007, 45, 1),
    (129, 16391, 40, 1),        # ends between the two stages of its last quad
    (65, 16391, 603, 2),        # parts of nineteen quads, the last of eleven blocks
    (99, 8201, 564, 4),         # parts of nine quads, the last of four blocks
    (65, 4097, 711, 8),
]
# in parts, with a CU each
ALONE = [(65, 4097, 502, 4), (77, 2055, 449, 8)]


@pytest.mark.parametrize("m,n,blocks,parts", SHARED + ALONE)
def test_shared_cu(gpu, m, n, blocks, parts):
    tiles.test_tile(gpu, m, n, blocks, "mxfp4", "128", parts)


def test_nan_blocks(gpu):
    tiles.test_nan_blocks_stay_in_their_rows(gpu, "mxfp4", 257, 11007, 33)
