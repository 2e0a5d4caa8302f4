"""The output-head operators on the GPU where their kernels' schedules have corners:
short launches, rows and tiles that some warps skip, several pieces of the vocabulary,
targets that repeat, waits that give up in odd places. Formulas and bounds as in
tests/test_head_gpu.py (tests/head_ref.py derives them)."""
import math

import pytest
import torch

import head_ref
from test_head_gpu import BF, HF, check_ce, fp8_operands, gen, operands

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d", [8, 64, 200])
def test_short_launches_back_to_back(mxs, d):
    """Launches of one to four blocks of operands, pairs of CTAs that end within
    microseconds of their last hand-back, each followed at once by the next: the same
    bits every time and nothing reported."""
    h, w, t = operands(300, 640, d, BF, seed=d)
    a = fp8_operands(300, 640, d)
    first = mxs.ce_from_hidden(h, w, t) + (mxs.matmul_fp8(*a),)
    out = [mxs.ce_from_hidden(h, w, t) + (mxs.matmul_fp8(*a),) for _ in range(100)]
    torch.cuda.synchronize()
    assert mxs.get_status(clear=True) == 0
    for o in out:
        assert all(torch.equal(x, y) for x, y in zip(o, first))
