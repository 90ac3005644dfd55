"""Every kernel that the gated linear unit's products are cut into, against 64 bits.

A kernel is one of a type, a product (y's and dp's, which share their cut; dx's; dw's),
a tile, a way to LDS (pieces of 16 bytes, or element by element) and whole or in splits.
SHAPES reach each that any sizes lead to, with enough k for the loop of whole stages,
tiles inside of the result and tiles past its edges."""

import math
import random

import pytest
import torch

from pytorch_r2d2_dpg_amd.ops import ext_available, hip_ext

BF16, FP32 = torch.bfloat16, torch.float32

SHAPES = [
    (BF16, 242, 248, 118), (BF16, 898, 250, 528), (BF16, 2428, 240, 648), (BF16, 278, 72, 120),
    (BF16, 2713, 344, 1060), (BF16, 2757, 340, 1076), (BF16, 4564, 778, 334), (BF16, 2516, 320, 1972),
    (BF16, 2070, 449, 2096), (BF16, 811, 234, 6348), (BF16, 2095, 464, 2392), (BF16, 10651, 264, 692),
    (BF16, 5313, 411, 1336), (BF16, 792, 5672, 260), (BF16, 776, 4651, 436), (BF16, 1627, 592, 3276),
    (BF16, 1435, 5971, 641), (BF16, 1846, 4448, 904), (BF16, 236, 546, 7062), (BF16, 14000, 527, 144),
    (BF16, 317, 536, 6840), (BF16, 8192, 1040, 124), (BF16, 2013, 1328, 4539), (BF16, 16959, 545, 124),
    (BF16, 252, 840, 6240), (BF16, 13078, 776, 144), (BF16, 8550, 1061, 1224), (BF16, 4133, 584, 4528),
    (BF16, 14742, 320, 1552),
    (FP32, 121, 114, 60), (FP32, 133, 120, 58), (FP32, 1584, 120, 1284), (FP32, 2848, 121, 716),
    (FP32, 746, 4670, 325), (FP32, 890, 3472, 474), (FP32, 2663, 1288, 1999), (FP32, 3988, 808, 2004),
]


def kernels(dtype, M, K, F):
    """The kernels of a forward and backward pass, each with whether it enters the loop
    of whole stages (entered with six, at five of them in LDS) and has tiles inside of
    the result and past both its edges."""
    piece, depth = (8, 32) if dtype == BF16 else (4, 16)
    x = K % piece == 0          # x and w lie in pieces; for dx and dw dp does too
    dp = x and 2 * F % piece == 0
    found = set()
    for (bm, bn, splits), name, m, n, k, direct in zip(
            hip_ext().gated_linear_cuts(dtype == BF16, M, K, F), ("y", "dx", "dw"),
            (M, M, 2 * F), (2 * F, K, K), (K, 2 * F, M), (x, dp, dp)):
        long = math.ceil(k / splits) > 6 * depth
        edges = m > bm and n > bn and m % bm and n % bn
        found.add((dtype, name, bm, bn, direct, splits > 1, bool(long and edges)))
    return found


@pytest.mark.skipif(not ext_available(), reason="the extension is not built")
def test_shapes_reach_every_kernel():
    reached = set().union(*(kernels(*s) for s in SHAPES))
    rng = random.Random(7)
    for _ in range(20000):
        M, K, F = (round(math.exp(rng.uniform(0, math.log(most)))) for most in (65536, 8192, 8192))
        K, F = (max(8, v // 8 * 8) if rng.random() < 0.5 else v for v in (K, F))
        for dtype in (BF16, FP32):
            for kernel in kernels(dtype, M, K, F):
                assert kernel[:-1] + (True,) in reached, (kernel, M, K, F)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype, M, K, F", SHAPES)
def test_kernel(dtype, M, K, F):
    from test_gated_ops_gpu import run_linear
    run_linear(M, K, F, dtype, seed=K, oracle_on="cuda")
