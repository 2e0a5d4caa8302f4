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


def tile_width(m_tiles, n, units, lo=64, step=64):
    """The planner's width of a tile (tile_width in mxs_gemm.cu)."""
    return min(range(256, lo - 1, -step), key=lambda w: (-(-m_tiles * -(-n // w) // units)) * (w + 16))


def skipped_between(rows, kept, vocab, pairs):
    """How often, over all pairs of CTAs and runs of 32 rows, a warp joins a tile, skips an
    odd number of tiles without a row of its own, and joins the next one."""
    n = tile_width(-(-rows // 256), vocab, pairs)
    mt, found = -(-kept // 256), 0
    for pair in range(pairs):
        ms = [i % mt for i in range(pair, mt * -(-vocab // n), pairs)]
        for run in range(8):
            live = [i for i, m in enumerate(ms) if m * 256 + run * 32 < kept]
            found += sum((b - a) % 2 == 0 for a, b in zip(live, live[1:]))
    return found


@pytest.mark.parametrize("rows,left_out,vocab,d", [(520, 0, 33000, 40), (700, 0, 50001, 64), (900, 0, 33000, 200),
                                                   (1500, 211, 40000, 24), (2100, 1, 20001, 72)])
def test_rows_that_skip_tiles(mxs, rows, left_out, vocab, d):
    """Row counts that end inside a tile: warps without rows in a unit's tile skip it and
    join the next one, while short sums leave several accumulators in flight. What four
    warps exchange for a tile is never overwritten by the one after the skipped one."""
    pairs = torch.cuda.get_device_properties(0).multi_processor_count // 2
    assert skipped_between(rows, rows - left_out, vocab, pairs) > 0
    h, w, t = operands(rows, vocab, d, BF, seed=rows)
    if left_out:
        t[torch.randperm(rows, generator=gen(1), device="cuda")[:left_out]] = -100
    l0, e0 = head_ref.ce(h, w, t, 0.9)
    tl, te = head_ref.ce_tol(h, w, t, 0.9, l0, e0)
    first = mxs.ce_from_hidden(h, w, t, temperature=0.9)
    keep = t >= 0
    assert ((first[0].double() - l0).abs() <= tl)[keep].all() and ((first[1].double() - e0).abs() <= te)[keep].all()
    for _ in range(20):
        again = mxs.ce_from_hidden(h, w, t, temperature=0.9)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


@pytest.mark.parametrize("rows,tile", [(9, 0), (100, 0), (300, 0), (300, 1)])
def test_warps_that_meet_give_up(mxs, rows, tile):
    """One of the four warps that meet in the loss's epilogue leaves early (a test
    hook), while its accumulators arrive as ever: the others' wait for it ends after
    about a second, the status word says so, and the next call gives the same bits."""
    h, w, t = operands(rows, 20000, 512, BF, seed=40)
    before = mxs.ce_from_hidden(h, w, t)
    torch.cuda.synchronize()
    mxs.get_status(clear=True)
    mxs.set_test_hooks(drop_tile=-2 - tile)
    try:
        mxs.ce_from_hidden(h, w, t)
        torch.cuda.synchronize()
    finally:
        mxs.set_test_hooks()
    assert mxs.get_status(clear=True) & mxs.ROW_TIMEOUT
    after = mxs.ce_from_hidden(h, w, t)
    torch.cuda.synchronize()
    assert mxs.get_status(clear=True) == 0
    assert torch.equal(before[0], after[0]) and torch.equal(before[1], after[1])
