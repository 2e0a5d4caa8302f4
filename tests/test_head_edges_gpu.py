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


@pytest.mark.parametrize("tile", [0, 1])
def test_warps_that_gather_give_up(mxs, tile):
    """The same for the warps of a CTA that sum a target's rows together in the gradient
    product: the one that leaves does so before a tile whose vocabulary rows have such a
    target."""
    rows, vocab, d = 600, 40000, 64
    h, w, _ = operands(rows, vocab, d, BF, seed=41)
    t = torch.where(torch.arange(rows, device="cuda") % 2 == 0, 5, 74 * 256 + 5)  # CTA 0's first and second tile
    grad = torch.ones(rows, device="cuda")
    _, lse = mxs.ce_from_hidden(h, w, t)
    def call():
        out = mxs.ce_from_hidden_backward(h, w, t, lse, grad, need_hidden=False)[1]
        torch.cuda.synchronize()
        return out
    before = call()
    mxs.get_status(clear=True)
    mxs.set_test_hooks(drop_tile=-2 - tile)
    try:
        call()
    finally:
        mxs.set_test_hooks()
    assert mxs.get_status(clear=True) & mxs.ROW_TIMEOUT
    after = call()
    assert mxs.get_status(clear=True) == 0
    assert torch.equal(before, after)


def repeated(kind, rows, vocab, g):
    """Targets as tokens have them: some far more often than others."""
    t = torch.randint(0, vocab, (rows,), generator=g, device="cuda")
    if kind == "one":
        t[:] = vocab // 2
    elif kind == "most":
        t[torch.rand(rows, generator=g, device="cuda") < 0.6] = vocab - 1
    elif kind == "neighbours":
        t %= 32
    elif kind == "zipf":
        p = 1.0 / torch.arange(1, vocab + 1, device="cuda", dtype=torch.float64)
        t = torch.multinomial(p, rows, replacement=True, generator=g)
    elif kind == "counts":  # groups of 1, 2, ... rows on either side of 16, in any order
        sizes = torch.tensor([1, 2, 3, 15, 16, 17, 18, 33] * (rows // 105 + 1), device="cuda")
        t = (torch.arange(len(sizes), device="cuda") * 5 % vocab).repeat_interleave(sizes)[:rows]
        t = t[torch.randperm(rows, generator=g, device="cuda")]
    elif kind == "large":  # and on either side of 256
        sizes = torch.tensor([256, 1, 257, 2, 300, 5, 255, 40] * (rows // 1116 + 1), device="cuda")
        t = (torch.arange(len(sizes), device="cuda") * 3 % vocab).repeat_interleave(sizes)[:rows]
        t = t[torch.randperm(rows, generator=g, device="cuda")]
    elif kind == "runs":  # each target's rows side by side
        t = torch.arange(rows, device="cuda") * 7 // max(rows, 7) * (vocab // 7)
    return t


@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("kind", ["one", "most", "neighbours", "zipf", "runs", "counts", "large"])
@pytest.mark.parametrize("rows,vocab,d", [(2, 300, 9), (130, 1000, 200), (700, 513, 264), (2500, 4001, 72)])
def test_repeated_targets(mxs, rows, vocab, d, kind, dt):
    g = gen(rows + vocab)
    h, w, _ = operands(rows, vocab, d, dt, seed=rows)
    t = repeated(kind, rows, vocab, g)
    grad = torch.randn(rows, generator=g, device="cuda")
    grad[torch.rand(rows, generator=g, device="cuda") < 0.2] = 0  # rows without weight repeat too
    _, lse, gh, gw = check_ce(mxs, h, w, t, 1.0, grad)
    for _ in range(3):
        again = mxs.ce_from_hidden_backward(h, w, t, lse, grad)
        assert torch.equal(again[0], gh) and torch.equal(again[1], gw)


@pytest.mark.parametrize("dt,vocab", [(BF, 512), (HF, 4096)])
@pytest.mark.parametrize("kind", ["one", "most", "neighbours", "zipf", "runs", "counts", "large", "uniform"])
@pytest.mark.parametrize("rows,d", [(90, 33), (1000, 300), (3000, 100)])
def test_target_entries_keep_32_bits(mxs, rows, d, kind, dt, vocab):
    """A weight of zeros makes every probability 1 / vocab, a power of two, which the
    type holds, and every target entry 1 / vocab - 1, which it does not: the weight's
    gradient is then the formula's, rounded once (fp32 sums are within 2^-16 of it, so
    that two elements in a hundred at most lie next to a midpoint), if and only if
    what the entries' rounding leaves out is added for every row."""
    g = gen(rows + vocab)
    h = (torch.rand((rows, d), generator=g, device="cuda") + 0.5).to(dt)
    w = torch.zeros((vocab, d), dtype=dt, device="cuda")
    t = repeated(kind, rows, vocab, g)
    _, lse = mxs.ce_from_hidden(h, w, t)
    _, gw = mxs.ce_from_hidden_backward(h, w, t, lse, torch.ones(rows, device="cuda"), need_hidden=False)
    def gradient(entry):
        dw = (h.double().sum(0) / vocab).repeat(vocab, 1)
        return dw.index_add_(0, t, h.double() * (entry - 1 / vocab))
    want, hit = gradient(1 / vocab - 1), torch.unique(t)
    rounded = torch.tensor(1 / vocab - 1, dtype=dt, device="cuda").double().item()
    wrong = gradient(rounded)[hit].to(dt) != want[hit].to(dt)
    assert wrong.float().mean() > 0.1  # without the rests
    assert (gw != want.to(dt)).float().mean() <= 0.02
    assert (gw[hit] != want[hit].to(dt)).float().mean() <= 0.02
    u = head_ref.U[dt]
    assert ((gw.double() - want).abs() <= (u + 2.0 ** -16) * want.abs() + 2.0 ** -25).all()


def test_a_million_rows_of_one_target(mxs):
    """Padding that keeps its token id and its weight: no wait runs out, and the time is
    the products'. fp32 sums of so many products of one sign lose up to 2^-23 of
    themselves at every 16 of them."""
    rows, vocab, d = 1200000, 512, 8
    g = gen(1)
    h = (torch.rand((rows, d), generator=g, device="cuda") + 0.5).to(BF)
    w = torch.zeros((vocab, d), dtype=BF, device="cuda")
    t = torch.full((rows,), 77, device="cuda")
    t[::1000] = 78
    mxs.get_status(clear=True)
    _, lse = mxs.ce_from_hidden(h, w, t)
    _, gw = mxs.ce_from_hidden_backward(h, w, t, lse, torch.ones(rows, device="cuda"), need_hidden=False)
    torch.cuda.synchronize()
    assert mxs.get_status(clear=True) == 0
    want = (h.double().sum(0) / vocab).repeat(vocab, 1).index_add_(0, t, -h.double())
    size = (h.double().sum(0) / vocab).repeat(vocab, 1).index_add_(0, t, h.double())
    assert ((gw.double() - want).abs() <= 2.0 ** -8 * want.abs() + rows / 16 * 2.0 ** -23 * size).all()


# ---------------------------------------------------------------------------
# Several pieces of the vocabulary, real heads' widths
# ---------------------------------------------------------------------------

def ceil_div(a, b):
    return -(-a // b)


def piece_of(rows, vocab):
    """Columns of a piece of the gradients (make_plan in mxs_ce.cu: 256 MB of G)."""
    most = max(256, (256 << 20) // (2 * ceil_div(rows, 256) * 256))
    return ceil_div(ceil_div(vocab, ceil_div(vocab, most)), 256) * 256


def in_pieces(mxs, rows, vocab, d, dt, seed, pieces):
    """operands() with targets on both sides of every piece's edge and in the last rows of
    the vocabulary; that G is not held whole shows in the workspace's size."""
    import ctypes
    piece = piece_of(rows, vocab)
    assert ceil_div(vocab, piece) == pieces
    h, w, t = operands(rows, vocab, d, dt, seed=seed)
    need = ctypes.c_size_t()
    assert mxs.load().mxs_ce_workspace_size(ctypes.c_void_p(w.data_ptr()), w.stride(0), rows, d, vocab, 1,
                                            ctypes.byref(need)) == 0
    if rows * d < 1 << 20:  # else the rows' own scratch hides it
        assert need.value < 2 * ceil_div(rows, 256) * 256 * vocab
    at = [0, vocab - 1, vocab - 2, vocab - 31, vocab - 33]
    for p in range(1, pieces):
        at += [p * piece - 33, p * piece - 2, p * piece - 1, p * piece, p * piece + 1, p * piece + 32]
    t[:2 * len(at)] = torch.tensor(at * 2, device="cuda")  # each twice
    t[rows // 2] = -100
    return h, w, t


@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("rows,vocab,d,pieces", [(4000, 40001, 24, 2), (4000, 40001, 264, 2), (4000, 70001, 72, 3),
                                                 (1500, 200003, 40, 3), (300, 600001, 16, 3), (128, 1100001, 8, 3)])
def test_gradients_in_several_pieces(mxs, rows, vocab, d, pieces, dt):
    check_ce(mxs, *in_pieces(mxs, rows, vocab, d, dt, rows + d, pieces), 0.9)


@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("rows,vocab,d", [(4000, 70001, 72), (4000, 40001, 300)])
def test_repeated_targets_at_the_edges_of_pieces(mxs, rows, vocab, d, dt):
    """Groups of every kind (2, 3, 16, 17, 256, 257 rows and more) on both sides of an edge
    and in the vocabulary's last rows; again with the same bits."""
    piece = piece_of(rows, vocab)
    h, w, t = in_pieces(mxs, rows, vocab, d, dt, 7, ceil_div(vocab, piece))
    at = 100
    for target, count in ((piece - 1, 700), (piece, 257), (piece + 1, 17), (piece - 2, 3), (vocab - 1, 256),
                          (vocab - 2, 300), (vocab - 3, 16), (0, 400), (piece - 128, 40), (piece - 129, 5)):
        t[at:at + count] = target
        at += count
    t = t[torch.randperm(rows, generator=gen(2), device="cuda")]
    grad = torch.randn(rows, generator=gen(9), device="cuda")
    _, lse, gh, gw = check_ce(mxs, h, w, t, 0.9, grad)
    again = mxs.ce_from_hidden_backward(h, w, t, lse, grad, temperature=0.9)
    assert torch.equal(again[0], gh) and torch.equal(again[1], gw)


def hidden_splits(rows, nt, width, units):
    """Splits of K for grad_hidden alone (grad_hidden_splits in mxs_ce.cu)."""
    tiles, blocks = ceil_div(rows, 256) * nt, ceil_div(width, 64)
    s = max(1, min(ceil_div(blocks * units, tiles * blocks), ceil_div(blocks, 8), units // tiles))
    return ceil_div(blocks, ceil_div(blocks, s))


@pytest.mark.parametrize("need", ["hidden", "weight"])
@pytest.mark.parametrize("rows,vocab,d", [(130, 533024, 8), (130, 541759, 200), (2000, 140000, 40)])
def test_one_gradient_in_several_pieces(mxs, rows, vocab, d, need):
    """One gradient alone; for 130 rows the last, narrower piece leaves the last split of
    grad_hidden's sum without a column."""
    h, w, t = in_pieces(mxs, rows, vocab, d, BF, 3, ceil_div(vocab, piece_of(rows, vocab)))
    pairs = torch.cuda.get_device_properties(0).multi_processor_count // 2
    if rows == 130 and pairs == 74:
        piece, last = piece_of(rows, vocab), vocab % piece_of(rows, vocab)
        s = hidden_splits(rows, 1, piece, pairs)
        blocks = ceil_div(last, 64)
        assert (s - 1) * ceil_div(blocks, s) >= blocks
    grad = torch.randn(rows, generator=gen(9), device="cuda")
    _, lse = mxs.ce_from_hidden(h, w, t)
    gh, gw = mxs.ce_from_hidden_backward(h, w, t, lse, grad, need_hidden=need == "hidden",
                                         need_weight=need == "weight")
    dh, dw, eh, ew = head_ref.ce_grads(h, w, t, grad, 1.0)
    got, want, tol = (gh, dh, eh) if need == "hidden" else (gw, dw, ew)
    assert (gw if need == "hidden" else gh) is None
    assert ((got.double() - want).abs() <= tol).all()


@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("rows,vocab,d", [(130, 3001, 1100), (300, 2000, 896), (257, 1500, 3584), (520, 5000, 2048),
                                          (700, 1999, 1037), (100, 1999, 3584)])
def test_heads_of_real_widths(mxs, rows, vocab, d, dt):
    """More than 128 rows with a d_model of several joins of the loss's accumulators."""
    check_ce(mxs, *operands(rows, vocab, d, dt, seed=d), 0.9)


@pytest.mark.parametrize("rows,n,k,out", [(65, 3000, 3584, torch.float32), (100, 5001, 1040, BF),
                                          (128, 700, 8192, HF), (260, 3001, 3584, torch.float32),
                                          (1000, 1024, 8192, BF)])
def test_matmul_fp8_real_widths(mxs, rows, n, k, out):
    ops = fp8_operands(rows, n, k, seed=k)
    got = mxs.matmul_fp8(*ops, out_dtype=out)
    want, tol = head_ref.matmul_fp8(*ops, out)
    assert ((got.double() - want).abs() <= tol).all()


@pytest.mark.parametrize("dt", [HF, BF])
@pytest.mark.parametrize("wrt,step", [("hidden", 2.0 ** -5), ("weight", 2.0 ** -8)])
@pytest.mark.parametrize("seed", [0, 1, 2, 3])
def test_gradients_against_differences(mxs, wrt, step, seed, dt):
    """Central differences of the kernel's own losses along a direction of 64 elements,
    in steps that the types hold exactly. The error: the losses' own (their bounds, as a
    random walk over the rows), a third derivative's, at most the cube of a row's
    largest move of a logit, over 6, and the gradients' (their elementwise bounds along
    the direction). The derivative is at least 20 times that, so that a gradient 5 % off
    fails."""
    rows, vocab, d = 60, 300, 32
    g = gen(seed)
    h = (torch.randint(-16, 17, (rows, d), generator=g, device="cuda") / 8).to(dt)
    w = (torch.randint(-16, 17, (vocab, d), generator=g, device="cuda") / 32).to(dt)
    t = torch.randint(0, vocab, (rows,), generator=g, device="cuda")
    if seed == 3:
        t %= 8
    loss, lse = mxs.ce_from_hidden(h, w, t)
    gh, gw = mxs.ce_from_hidden_backward(h, w, t, lse, torch.ones(rows, device="cuda"))
    x, grad = (h, gh) if wrt == "hidden" else (w, gw)
    at = torch.randperm(x.numel(), generator=g, device="cuda")[:64]
    move = torch.zeros_like(x)
    move.view(-1)[at] = step * grad.view(-1)[at].sign()
    assert ((x + move).double() == x.double() + move.double()).all()
    assert ((x - move).double() == x.double() - move.double()).all()
    def total(sign):
        y = x + sign * move
        return mxs.ce_from_hidden(y if wrt == "hidden" else h, w if wrt == "hidden" else y, t)[0].double().sum().item()
    difference = (total(1) - total(-1)) / 2
    derivative = (grad.double() * move.double()).sum().item()
    moved = move.double() @ w.double().t() if wrt == "hidden" else h.double() @ move.double().t()
    cubic = (moved.abs().amax(1) ** 3).sum().item() / 6
    _, _, eh, ew = head_ref.ce_grads(h, w, t, torch.ones(rows, device="cuda"), 1.0)
    own = ((eh if wrt == "hidden" else ew) * move.double().abs()).sum().item()
    tl, _ = head_ref.ce_tol(h, w, t, 1.0, *head_ref.ce(h, w, t, 1.0))
    tol = tl.norm().item() + cubic + own
    assert abs(difference - derivative) <= tol, (difference, derivative, tol)
    assert abs(derivative) >= 20 * tol


@pytest.mark.parametrize("temperature", [1.0, 0.5, 0.7, 3.0])
def test_gradient_weights_near_the_largest_float(mxs, temperature):
    """A row's gradient scales with its own weight, however large another's: zero for a
    weight of zero, finite where the formula's is."""
    h, w, t = operands(6, 400, 64, BF, seed=4)
    w *= 2.0 ** -8
    t[:] = torch.arange(6, device="cuda") * 40
    grad = torch.tensor([0.0, 1e30, -1e20, 3.3e38, -3.3e38, 0.0], device="cuda")
    _, lse = mxs.ce_from_hidden(h, w, t, temperature=temperature)
    gh, gw = mxs.ce_from_hidden_backward(h, w, t, lse, grad, temperature=temperature)
    dh, _, eh, _ = head_ref.ce_grads(h, w, t, grad, temperature)
    assert (gh[[0, 5]] == 0).all()
    assert (dh.abs() < 3.0e38).all() and ((gh.double() - dh).abs() <= eh).all()
    tiny = h * 2.0 ** -8  # the weight's gradient stays in range too
    _, lse = mxs.ce_from_hidden(tiny, w, t, temperature=temperature)
    _, gw = mxs.ce_from_hidden_backward(tiny, w, t, lse, grad, temperature=temperature)
    _, dw, _, ew = head_ref.ce_grads(tiny, w, t, grad, temperature)
    assert (dw.abs() < 3.0e38).all() and ((gw.double() - dw).abs() <= ew).all()


# ---------------------------------------------------------------------------
# 8 bits: layouts, graphs, arguments
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("out", [torch.float32, BF, HF])
@pytest.mark.parametrize("rows", [1, 20, 61, 100, 150, 300])
@pytest.mark.parametrize("pad,offset", [(0, 0), (3, 0), (11, 1), (8, 8)])
def test_matmul_fp8_output_layouts(mxs, rows, pad, offset, out):
    """Every kernel's stores, into rows of any alignment; nothing is written between them."""
    ops = fp8_operands(rows, 301, 200, seed=rows)
    flat = torch.full((rows * (301 + pad) + offset,), -7.0, dtype=out, device="cuda")
    view = flat[offset:].view(rows, 301 + pad)
    mxs.matmul_fp8(*ops, out=view[:, :301])
    want, tol = head_ref.matmul_fp8(*ops, out)
    assert ((view[:, :301].double() - want).abs() <= tol).all()
    assert (view[:, 301:] == -7.0).all() and (flat[:offset] == -7.0).all()


@pytest.mark.parametrize("rows", [1, 40, 140])
@pytest.mark.parametrize("d,pad", [(200, 0), (208, 0), (99, 13)])
def test_sample_from_hidden_fp8_layouts(mxs, rows, d, pad):
    """Weights and logits with rows of any alignment: the same logits and draws."""
    g = gen(rows + d)
    vocab = 3001
    h = torch.randn((rows, d), generator=g, device="cuda").to(BF)
    wq, ws = mxs.quantize_fp8((torch.randn((vocab, d), generator=g, device="cuda") * (3 / d ** 0.5)).to(BF), 128)
    u = torch.rand(rows, generator=g, device="cuda", dtype=torch.float64)
    loose = torch.empty((vocab, d + pad), dtype=torch.uint8, device="cuda")[:, :d].view(torch.float8_e4m3fn)
    loose.copy_(wq)
    want = mxs.matmul_fp8(*mxs.quantize_fp8(h, 1), wq, ws)
    n0, i0, p0 = mxs.sample(want, 0.8, 40, u)
    for extra in (None, 0, 5):
        logits = None if extra is None else torch.empty((rows, vocab + extra), device="cuda")[:, :vocab]
        n, i, p = mxs.sample_from_hidden_fp8(h, loose, ws, 0.8, 40, u, logits_out=logits)
        assert torch.equal(n, n0) and torch.equal(i, i0) and torch.equal(p, p0)
        assert logits is None or torch.equal(logits, want)


@pytest.mark.parametrize("rows", [1, 33, 200])
def test_fp8_calls_in_a_graph(mxs, rows):
    """Quantiser, product and draw captured, and replayed on other hidden states; and on
    a stream of their own."""
    g = gen(rows)
    vocab, d = 5000, 384
    h = torch.randn((rows, d), generator=g, device="cuda").to(HF)
    wq, ws = mxs.quantize_fp8((torch.randn((vocab, d), generator=g, device="cuda") * 0.15).to(HF), 128)
    u = torch.rand(rows, generator=g, device="cuda", dtype=torch.float64)
    def step(stream=None):
        q, s = mxs.quantize_fp8(h, 1, stream=stream)
        return (mxs.matmul_fp8(q, s, wq, ws, out_dtype=BF, stream=stream),) + mxs.sample_from_hidden_fp8(
            h, wq, ws, 1.1, 20, u, stream=stream)
    first = step()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    other = step(side)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(first, other))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    h.copy_(torch.randn((rows, d), generator=g, device="cuda"))
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(out, step()))


def test_fp8_draws_of_no_rows(mxs):
    wq, ws = mxs.quantize_fp8(torch.ones((50, 64), dtype=BF, device="cuda"), 128)
    h = torch.empty((0, 64), dtype=BF, device="cuda")
    n, i, p = mxs.sample_from_hidden_fp8(h, wq, ws, 1.0, 5, torch.empty(0, dtype=torch.float64, device="cuda"))
    assert n.shape == (0,) and i.shape == (0, 5) and p.shape == (0, 5)


@pytest.mark.parametrize("rows", [9, 300])
def test_loss_or_lse_alone(mxs, rows):
    """Either output of the C call may be left out."""
    import ctypes
    P = ctypes.c_void_p
    h, w, t = operands(rows, 700, 96, BF, seed=rows)
    loss, lse = mxs.ce_from_hidden(h, w, t)
    need = ctypes.c_size_t()
    lib = mxs.load()
    assert lib.mxs_ce_workspace_size(P(w.data_ptr()), 96, rows, 96, 700, 0, ctypes.byref(need)) == 0
    ws = torch.empty(need.value, dtype=torch.uint8, device="cuda")
    for which in (0, 1):
        out = torch.full((rows,), -1.0, device="cuda")
        at = [P(out.data_ptr()), None] if which == 0 else [None, P(out.data_ptr())]
        torch.cuda.synchronize()
        assert lib.mxs_ce_from_hidden(P(h.data_ptr()), 96, P(w.data_ptr()), 96, 0, rows, 96, 700, P(t.data_ptr()), 8,
                                      1.0, *at, P(ws.data_ptr()), need.value, None) == 0
        torch.cuda.synchronize()
        assert torch.equal(out, loss if which == 0 else lse)


def test_f16_gradient_weights_of_many_sizes(mxs):
    """f16 holds entries relative to the largest weight: down to 2^-28 of it as exactly as
    ever, below with an absolute error that the bound has."""
    h, w, t = operands(120, 900, 72, HF, seed=14)
    grad = torch.exp2(-torch.arange(120, device="cuda") / 3) * 3e3  # down to 2^-40 of the largest
    grad[::2] *= -1
    check_ce(mxs, h, w, t, 1.0, grad)
    _, lse = mxs.ce_from_hidden(h, w, t)
    for scale in (2.0 ** -12, 2.0 ** 3):  # the division by the largest weight is exact for powers of two
        a = mxs.ce_from_hidden_backward(h, w, t, lse, grad)[0]
        b = mxs.ce_from_hidden_backward(h, w, t, lse, grad * scale)[0]
        ok = (a.abs() >= 2.0 ** -2) & (b.abs() >= 2.0 ** -13)  # both in f16's normal range
        assert ok.any() and torch.equal((a.double() * scale)[ok], b.double()[ok])


@pytest.mark.parametrize("rows,dt,vocab,kind", [(200000, BF, 512, "one"), (200000, HF, 4096, "uniform"),
                                                (1000000, BF, 512, "uniform"), (1000000, HF, 512, "one"),
                                                (33000, HF, 4096, "one"), (65536, HF, 4096, "one")])
def test_weight_gradient_of_many_rows(mxs, rows, dt, vocab, kind):
    """Sums over the rows in which all terms have one sign (a weight of zeros makes every
    probability 1 / vocab). The MMA's own fp32 sum loses up to 2^-23 of itself at every
    16 products, 2^-13 of the whole over 32768 of them; joined after so many, the
    total loses no more than that, and the result's rounding."""
    g = gen(rows + vocab)
    h = (torch.rand((rows, 16), generator=g, device="cuda") + 0.5).to(dt)
    w = torch.zeros((vocab, 16), dtype=dt, device="cuda")
    t = repeated(kind, rows, vocab, g)
    grad = torch.full((rows,), 2.0 ** -10, device="cuda")  # f16 results stay in range
    _, lse = mxs.ce_from_hidden(h, w, t)
    gh, gw = mxs.ce_from_hidden_backward(h, w, t, lse, grad)
    p = h.double().sum(0) / vocab * 2.0 ** -10
    hot = torch.zeros((vocab, 16), dtype=torch.float64, device="cuda").index_add_(0, t, h.double() * 2.0 ** -10)
    want = p - hot
    assert ((gw.double() - want).abs() <= head_ref.U[dt] * want.abs() + 2.0 ** -13 * (p + hot) + 2.0 ** -25).all()
    assert (gh == 0).all()


def test_hidden_gradient_of_a_long_vocabulary(mxs):
    """The same for sums over a piece of 32768 columns and more: 2500 rows whose weight
    rows are all alike, 40000 columns in one piece."""
    rows, vocab, d = 2500, 40000, 16
    assert piece_of(rows, vocab) > 32768
    g = gen(3)
    w = (torch.rand((1, d), generator=g, device="cuda") + 0.5).to(HF).repeat(vocab, 1)
    h = torch.zeros((rows, d), dtype=HF, device="cuda")
    w[7] = 0
    t = torch.full((rows,), 7, device="cuda")
    _, lse = mxs.ce_from_hidden(h, w, t)
    gh, _ = mxs.ce_from_hidden_backward(h, w, t, lse, torch.ones(rows, device="cuda"), need_weight=False)
    want = w.double().sum(0) / vocab  # the target's own row is zero
    # the probabilities' rounding to f16 is common to all columns: 2^-11 of the sum, and the result's
    assert ((gh.double() - want).abs() <= (2 * 2.0 ** -11 + 2.0 ** -13) * want).all()


@pytest.mark.parametrize("d", [896, 3584])
@pytest.mark.parametrize("rows,dt,units", [(64, BF, 2), (64, HF, 12), (200, BF, 8), (200, HF, 56)])
def test_logits_of_one_sign(mxs, rows, dt, units, d):
    """Target logits whose products are all positive, where the tensor core's rounding
    towards zero adds up, read from the lse of rows that are sure of their target: the
    mean error in units of 2^-24 of the logit. An addition of 16 products to a sum loses
    half a unit of it for bf16's products and several for f16's, over runs of 128 (up to
    128 rows) and 512 products: 0.3, 7, 5.5 and 44 units were measured."""
    g = gen(d)
    w = (torch.rand((2000, d), generator=g, device="cuda") * 0.1 + 0.05).to(dt)
    w[64:] *= -1
    h = (torch.rand((64, d), generator=g, device="cuda") + 0.5).to(dt).repeat(4, 1)[:rows]
    t = torch.arange(64, device="cuda").repeat(4)[:rows]
    loss, lse = mxs.ce_from_hidden(h, w, t)
    want = torch.logsumexp(h.double() @ w.double().t(), 1)
    assert ((lse.double() - want) / want).mean().abs().item() <= units * 2.0 ** -24
