"""Layer norm and gated recurrence where a block walks on: several rows one after the
other, and several passes over time without segments."""

import pytest
import torch

from test_gated_ops_gpu import run_norm, run_recurrence

pytestmark = pytest.mark.gpu
BF16, FP32 = torch.bfloat16, torch.float32


# more rows than a launch has blocks, forward (2048) and backward (512), in each shape of
# threads and runs a row: 64 x 1 and x 2, 128, 256 and 512 x 2, and in fp32 512 x 4
@pytest.mark.parametrize("rows, dim", [(8300, 200), (8300, 400), (8300, 700), (2100, 1300), (2100, 2500), (2100, 4099), (2100, 8190)])
@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("residual", [False, True])
def test_norm_rows_one_after_the_other(rows, dim, dtype, residual):
    run_norm(rows, dim, dtype, residual, seed=dim)


# 4 waves and 4 passes, 5 and 2, 7 and 3; even and odd, ragged and not
@pytest.mark.parametrize("T, B, H", [(100, 1100, 128), (70, 300, 301), (160, 130, 513)])
@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("ragged", [False, True])
def test_recurrence_passes(T, B, H, dtype, ragged):
    lengths = [(37 * b) % (T + 2) for b in range(B)] if ragged else None
    run_recurrence(T, B, H, dtype, lengths=lengths, seed=T)
