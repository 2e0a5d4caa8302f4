"""The output-head operators on the GPU against 64-bit restatements of their
formulas (tests/head_ref.py, which derives the bounds): cross entropy from hidden
states and its gradients, the 8-bit quantiser and block-scaled product, and the
sampler on an 8-bit head."""
import math

import numpy as np
import pytest
import torch

import head_ref
import oracle_lib

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def operands(rows, vocab, d, dt, seed=1, pad=0, offset=0, sharp=2.0):
    """hidden and weight, rows `pad` elements longer than d and starting `offset`
    elements into their buffers, with targets that stand out by up to `sharp`."""
    g = gen(seed)
    def strided(n):
        flat = torch.full((n * (d + pad) + offset + 8,), float("nan"), dtype=dt, device="cuda")
        return flat[offset:offset + n * (d + pad)].view(n, d + pad)[:, :d]
    w, h = strided(vocab), strided(rows)
    w.copy_(torch.randn((vocab, d), generator=g, device="cuda") * (2.5 / math.sqrt(d)))
    t = torch.randint(0, vocab, (rows,), generator=g, device="cuda")
    learnt = torch.rand((rows, 1), generator=g, device="cuda") * sharp
    h.copy_(torch.randn((rows, d), generator=g, device="cuda") + learnt * w[t].float())
    return h, w, t


def check_ce(mxs, h, w, t, temperature, grad=None):
    loss, lse = mxs.ce_from_hidden(h, w, t, temperature=temperature)
    l0, e0 = head_ref.ce(h, w, t, temperature)
    tl, te = head_ref.ce_tol(h, w, t, temperature, l0, e0)
    assert ((loss.double() - l0).abs() <= tl).all(), ((loss.double() - l0).abs() / tl).max()
    left = (t < 0) | (t >= w.shape[0])
    assert ((lse.double() - e0).abs() <= te)[~left].all()
    assert (loss[left] == 0).all() and (lse[left] == 0).all()
    if grad is None:
        grad = torch.randn(h.shape[0], generator=gen(9), device="cuda")
    gh, gw = mxs.ce_from_hidden_backward(h, w, t, lse, grad, temperature=temperature)
    dh, dw, eh, ew = head_ref.ce_grads(h, w, t, grad, temperature)
    assert gh.shape == h.shape and gw.shape == w.shape and gh.dtype == h.dtype and gw.dtype == h.dtype
    assert ((gh.double() - dh).abs() <= eh).all(), ((gh.double() - dh).abs() / eh.clamp_min(1e-300)).max()
    assert ((gw.double() - dw).abs() <= ew).all(), ((gw.double() - dw).abs() / ew.clamp_min(1e-300)).max()
    assert (gh[left] == 0).all()
    return loss, lse, gh, gw


@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("rows,vocab,d,temperature", [
    (1, 1, 1, 1.0), (1, 2, 8, 1.0), (1, 1000, 64, 0.7), (2, 257, 72, 1.3), (5, 63, 15, 1.0), (31, 1001, 130, 1.0),
    (64, 4097, 128, 0.8), (127, 255, 200, 1.0), (128, 256, 64, 1.0), (129, 640, 96, 2.0), (256, 513, 512, 1.0),
    (257, 2000, 264, 1.0), (300, 1999, 333, 0.9), (700, 777, 40, 1.0), (3, 40001, 48, 1.0), (130, 70000, 24, 1.0),
    (520, 33000, 80, 1.0),
])
def test_cross_entropy_and_gradients(mxs, rows, vocab, d, temperature, dt):
    check_ce(mxs, *operands(rows, vocab, d, dt, seed=rows + vocab + d), temperature)


@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("pad,offset", [(8, 0), (5, 0), (0, 8), (0, 1), (3, 7), (64, 16)])
def test_cross_entropy_strides_and_alignment(mxs, pad, offset, dt):
    check_ce(mxs, *operands(70, 500, 104, dt, seed=pad + offset, pad=pad, offset=offset), 0.9)


@pytest.mark.parametrize("rows", [1, 9, 140, 300])
@pytest.mark.parametrize("kind", ["some", "all", "but_one", "first_half"])
def test_rows_left_out(mxs, rows, kind):
    """Targets outside [0, vocab) of every kind; the rows' hidden states hold NaN
    and infinities, their lse and gradient weights NaN, and none of it reaches an output."""
    h, w, t = operands(rows, 900, 64, BF, seed=rows)
    marks = torch.tensor([-100, -1, 900, 2 ** 31 - 1, 2 ** 32 + 5, -2 ** 40, 2 ** 63 - 1], device="cuda")
    r = torch.arange(rows, device="cuda")
    out = {"some": r % 3 == 1, "all": r >= 0, "but_one": r != rows // 2, "first_half": r < rows // 2}[kind]
    t = torch.where(out, marks[r % 7], t)
    clean = h.clone()
    clean[out] = 0
    h[out] = float("nan")
    h[out, ::2] = float("inf")
    grad = torch.randn(rows, generator=gen(3), device="cuda")
    grad[out] = float("nan")
    loss, lse = mxs.ce_from_hidden(h, w, t)
    bad_lse = torch.where(out, torch.full_like(lse, float("nan")), lse)
    gh, gw = mxs.ce_from_hidden_backward(h, w, t, bad_lse, grad)
    l2, e2, gh2, gw2 = check_ce(mxs, clean, w, t, 1.0, torch.where(out, torch.zeros_like(grad), grad))
    for a, b in ((loss, l2), (lse, e2), (gh, gh2), (gw, gw2)):
        assert torch.equal(a, b)
    if kind == "all":
        assert (gw == 0).all() and (loss == 0).all()


def test_int32_targets_equal_int64(mxs):
    h, w, t = operands(50, 300, 64, BF)
    t[3], t[4] = -1, 300
    a, b = mxs.ce_from_hidden(h, w, t), mxs.ce_from_hidden(h, w, t.int())
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_confident_rows_keep_relative_accuracy(mxs):
    """Targets with probability up to 1 - 1e-9: the loss keeps its relative accuracy
    (lse - logit would leave one rounding of lse, 1e-6)."""
    h, w, t = operands(64, 2000, 128, BF, sharp=0.0)
    for i in range(64):
        h[i] = (w[t[i]].float() * (2.0 + i / 16)).to(BF)
    check_ce(mxs, h, w, t, 1.0)
    loss, _ = mxs.ce_from_hidden(h, w, t)
    assert loss.min() < 1e-5 and (loss > 0).all()


@pytest.mark.parametrize("temperature", [0.02, 50.0])
def test_wide_and_flat_logits(mxs, temperature):
    check_ce(mxs, *operands(40, 1500, 64, HF, seed=5), temperature)


def test_nan_and_infinite_rows_stay_their_own(mxs):
    """A kept row with a NaN or infinite hidden state: its own loss and gradient are
    not finite, every other row's are those without it."""
    h, w, t = operands(200, 600, 64, BF, seed=8)
    grad = torch.ones(200, device="cuda")
    l0, e0 = mxs.ce_from_hidden(h, w, t)
    g0, _ = mxs.ce_from_hidden_backward(h, w, t, e0, grad, need_weight=False)
    h[17, 3], h[150, 9] = float("nan"), float("inf")
    loss, lse = mxs.ce_from_hidden(h, w, t)
    gh, none = mxs.ce_from_hidden_backward(h, w, t, lse, grad, need_weight=False)
    assert none is None
    ok = torch.ones(200, dtype=torch.bool, device="cuda")
    ok[[17, 150]] = False
    assert torch.equal(loss[ok], l0[ok]) and torch.equal(lse[ok], e0[ok]) and torch.equal(gh[ok], g0[ok])
    assert torch.isnan(loss[17]) and torch.isnan(gh[17]).all()
    assert not torch.isfinite(lse[150])


def test_gradient_weights_of_any_size(mxs):
    """grad_loss of zero, tiny, huge and infinite rows: a row's own hidden gradient
    scales with it alone."""
    h, w, t = operands(6, 400, 64, BF, seed=4)
    grad = torch.tensor([0.0, 1e-20, -1e-4, 1.0, float("inf"), 3e4], device="cuda")
    _, lse = mxs.ce_from_hidden(h, w, t)
    gh, _ = mxs.ce_from_hidden_backward(h, w, t, lse, grad, need_weight=False)
    fin = [0, 1, 2, 3, 5]
    dh, _, eh, _ = head_ref.ce_grads(h[fin], w, t[fin], grad[fin], 1.0)
    assert ((gh[fin].double() - dh).abs() <= eh).all()
    assert (gh[0] == 0).all() and not torch.isfinite(gh[4]).any()
    _, gw = mxs.ce_from_hidden_backward(h, w, t, lse, torch.zeros(6, device="cuda"), need_hidden=False)
    assert (gw == 0).all()


def test_gradient_against_differences(mxs):
    """Central differences of the kernel's own losses along random directions, in
    steps that the type holds exactly. The error: the losses' rounding over the step
    (2 * 300 rows * 2^-21 / 2 step, as a random walk over rows), the third derivative's
    step^2 / 6 * max |slope|^3, and G's and the gradients' roundings (2^-10 of the sum of magnitudes)."""
    rows, vocab, d, step = 60, 300, 32, 2.0 ** -5
    g = gen(2)
    h = (torch.randint(-16, 17, (rows, d), generator=g, device="cuda") / 8).to(HF)
    w = (torch.randint(-16, 17, (vocab, d), generator=g, device="cuda") / 32).to(HF)
    t = torch.randint(0, vocab, (rows,), generator=g, device="cuda")
    grad = torch.ones(rows, device="cuda")
    _, lse = mxs.ce_from_hidden(h, w, t)
    gh, gw = mxs.ce_from_hidden_backward(h, w, t, lse, grad)
    for k in range(4):
        dh = torch.zeros_like(h)
        dw = torch.zeros_like(w)
        if k < 2:
            at = torch.randperm(h.numel(), generator=g, device="cuda")[:64]
            dh.view(-1)[at] = step * gh.view(-1)[at].sign()
        else:
            at = torch.randperm(w.numel(), generator=g, device="cuda")[:64]
            dw.view(-1)[at] = step * gw.view(-1)[at].sign()
        up = mxs.ce_from_hidden(h + dh, w + dw, t)[0].double().sum().item()
        dn = mxs.ce_from_hidden(h - dh, w - dw, t)[0].double().sum().item()
        num = (up - dn) / 2
        ana = ((gh.double() * dh.double()).sum() + (gw.double() * dw.double()).sum()).item()
        mag = ((gh.double() * dh.double()).abs().sum() + (gw.double() * dw.double()).abs().sum()).item()
        # a row's logits move by at most `slope` along the direction
        slope = (dh.double().norm(dim=1).max() * w.double().norm(dim=1).max()
                 + dw.double().norm(dim=1).max() * h.double().norm(dim=1).max()).item()
        tol = math.sqrt(rows) * 2.0 ** -19 + rows * slope ** 3 / 6 + 2.0 ** -10 * mag
        assert abs(num - ana) <= tol, (num, ana, tol)
        assert abs(ana) > 4 * tol or k >= 2  # the direction says something


def test_autograd_function(mxs):
    h, w, t = operands(90, 700, 64, BF, seed=12)
    t[5] = -100
    hp, wp = h.clone().requires_grad_(), w.clone().requires_grad_()
    loss = mxs.cross_entropy_from_hidden(hp, wp, t, 0.9)
    (loss.sum() / 89).backward()
    l0, lse = mxs.ce_from_hidden(h, w, t, 0.9)
    gh, gw = mxs.ce_from_hidden_backward(h, w, t, lse, torch.full((90,), 1 / 89, device="cuda"), 0.9)
    assert torch.equal(loss, l0) and torch.equal(hp.grad, gh) and torch.equal(wp.grad, gw)
    wp.grad = None
    mxs.cross_entropy_from_hidden(h, wp, t, 0.9).mean().backward()  # hidden needs no gradient
    assert wp.grad is not None


def test_repeats_streams_and_graphs(mxs):
    """The same bits on every call, on another stream, and replayed from a graph
    with other inputs in the buffers."""
    h, w, t = operands(150, 3000, 128, BF, seed=20)
    g1 = torch.ones(150, device="cuda")
    def step(stream=None):
        loss, lse = mxs.ce_from_hidden(h, w, t, stream=stream)
        return (loss, lse) + mxs.ce_from_hidden_backward(h, w, t, lse, g1, stream=stream)
    first, again = step(), step()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    other = step(side)
    side.synchronize()
    for a, b, c in zip(first, again, other):
        assert torch.equal(a, b) and torch.equal(a, c)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    h2, _, t2 = operands(150, 3000, 128, BF, seed=21)
    h.copy_(h2)
    t.copy_(t2)
    graph.replay()
    torch.cuda.synchronize()
    want = step()
    for a, b in zip(out, want):
        assert torch.equal(a, b)


def test_only_one_gradient(mxs):
    h, w, t = operands(40, 500, 64, HF)
    _, lse = mxs.ce_from_hidden(h, w, t)
    g = torch.ones(40, device="cuda")
    gh, gw = mxs.ce_from_hidden_backward(h, w, t, lse, g)
    a, n1 = mxs.ce_from_hidden_backward(h, w, t, lse, g, need_weight=False)
    n2, b = mxs.ce_from_hidden_backward(h, w, t, lse, g, need_hidden=False)
    assert n1 is None and n2 is None and torch.equal(a, gh) and torch.equal(b, gw)


def test_no_rows(mxs):
    w = torch.ones((30, 16), dtype=BF, device="cuda")
    h = torch.empty((0, 16), dtype=BF, device="cuda")
    t = torch.empty(0, dtype=torch.int64, device="cuda")
    loss, lse = mxs.ce_from_hidden(h, w, t)
    gh, gw = mxs.ce_from_hidden_backward(h, w, t, lse, torch.empty(0, device="cuda"))
    assert loss.shape == (0,) and gh.shape == (0, 16) and gw.shape == (30, 16) and (gw == 0).all()


# ---------------------------------------------------------------------------
# 8 bits
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("dt", [BF, HF, torch.float32])
@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("rows,cols,pad", [(1, 1, 0), (1, 128, 0), (3, 129, 0), (127, 100, 4), (128, 256, 0),
                                           (129, 300, 8), (200, 1037, 3), (64, 3584, 0), (1000, 8, 0)])
def test_quantize_bits(mxs, rows, cols, pad, block_rows, dt):
    g = gen(rows + cols)
    x = (torch.randn((rows, cols + pad), generator=g, device="cuda")
         * torch.exp(3 * torch.randn((1, cols + pad), generator=g, device="cuda"))).to(dt)[:, :cols]
    if rows > 2:
        x[rows // 2] = 0
    q, s = mxs.quantize_fp8(x, block_rows)
    q0, s0 = head_ref.quantize(x, block_rows)
    assert q.shape == x.shape and q.stride(0) % 16 == 0 and q.dtype == torch.float8_e4m3fn
    assert torch.equal(s, s0) and torch.equal(q.float().double(), q0)


@pytest.mark.parametrize("block_rows", [1, 128])
def test_quantize_special_values(mxs, block_rows):
    """Infinities saturate and do not set the scale, NaN stays NaN, zeros, values
    near the types' smallest, halves between 8-bit values."""
    x = torch.zeros((130, 256), dtype=torch.float32, device="cuda")
    x[0, :8] = torch.tensor([float("inf"), -float("inf"), float("nan"), 1.0, -2.0, 448.0, 17.0, 19.0], device="cuda")
    x[1, 130] = float("inf")  # alone in its block
    x[2, :3] = torch.tensor([1e-45, -3e-39, 1e-38], device="cuda")
    x[129, 0], x[129, 200] = 3.4e38, -1e-30
    q, s = mxs.quantize_fp8(x, block_rows)
    q0, s0 = head_ref.quantize(x, block_rows)
    assert torch.equal(s, s0)
    same = (q.float().double() == q0) | (torch.isnan(q.float()) & torch.isnan(q0))
    assert same.all()
    assert torch.isnan(q.float()[0, 2]) and q.float()[0, 0] == 448 and q.float()[0, 1] == -448


def fp8_operands(rows, n, k, seed=1, pad=0, offset=0):
    g = gen(seed)
    a = torch.randn((rows, k), generator=g, device="cuda") * torch.exp(torch.randn((1, k), generator=g, device="cuda"))
    b = torch.randn((n, k), generator=g, device="cuda") * torch.exp(torch.randn((n, 1), generator=g, device="cuda"))
    def place(v, br):
        q, s = head_ref.quantize(v, br)
        m = v.shape[0]
        flat = torch.full((m * (k + pad) + offset + 16,), 127, dtype=torch.uint8, device="cuda")  # NaN outside
        view = flat[offset:offset + m * (k + pad)].view(m, k + pad)[:, :k].view(torch.float8_e4m3fn)
        view.copy_(q.float().to(torch.float8_e4m3fn))
        return view, s
    return place(a, 1) + place(b, 128)


def check_matmul(mxs, ops, out_dtype, out=None):
    got = mxs.matmul_fp8(*ops, out_dtype=out_dtype, out=out)
    want, tol = head_ref.matmul_fp8(*ops, out_dtype)
    assert got.dtype == out_dtype and got.shape == want.shape
    err = (got.double() - want).abs()
    assert (err <= tol).all(), (err / tol).max()
    return got


@pytest.mark.parametrize("out_dtype", [torch.float32, BF, HF])
@pytest.mark.parametrize("rows,n,k", [
    (1, 1, 1), (1, 128, 128), (1, 1000, 3584), (2, 129, 130), (17, 500, 256), (64, 2049, 1024), (127, 127, 127),
    (128, 256, 128), (129, 257, 384), (200, 1111, 900), (256, 512, 640), (300, 700, 1040), (513, 3333, 272),
    (1000, 400, 2048), (5, 20000, 96), (40, 151, 8192),
])
def test_matmul_fp8(mxs, rows, n, k, out_dtype):
    check_matmul(mxs, fp8_operands(rows, n, k, seed=rows + n + k), out_dtype)


@pytest.mark.parametrize("pad,offset", [(16, 0), (0, 16), (7, 0), (0, 3), (1, 8)])
def test_matmul_fp8_strides_and_alignment(mxs, pad, offset):
    check_matmul(mxs, fp8_operands(150, 300, 240, pad=pad, offset=offset), torch.float32)


def test_matmul_fp8_strided_output(mxs):
    ops = fp8_operands(40, 301, 256)
    for pad, off in ((0, 0), (3, 0), (11, 1), (4, 4)):
        flat = torch.full((40 * (301 + pad) + off,), -7.0, device="cuda")
        out = flat[off:].view(40, 301 + pad)[:, :301]
        got = check_matmul(mxs, ops, torch.float32, out)
        assert got.data_ptr() == out.data_ptr()
        if pad:
            assert (flat[off:].view(40, 301 + pad)[:, 301:] == -7.0).all()


def test_matmul_fp8_zero_rows_and_nan(mxs):
    a, sa, b, sb = fp8_operands(150, 300, 256)
    a.view(torch.uint8)[7, 5] = 127  # NaN
    clean = a.clone()
    clean.view(torch.uint8)[7, 5] = 0
    x, y = mxs.matmul_fp8(a, sa, b, sb), mxs.matmul_fp8(clean, sa, b, sb)
    assert torch.isnan(x[7]).all()
    x[7], y[7] = 0, 0
    assert torch.equal(x, y)
    assert mxs.matmul_fp8(a[:0], sa[:0], b, sb).shape == (0, 300)


def test_matmul_fp8_scales_of_any_size(mxs):
    a, sa, b, sb = fp8_operands(20, 200, 512)
    sa *= torch.exp(8 * torch.randn(sa.shape, generator=gen(3), device="cuda"))
    sb *= torch.exp(8 * torch.randn(sb.shape, generator=gen(4), device="cuda"))
    check_matmul(mxs, (a, sa, b, sb), torch.float32)


def test_quantized_product_is_near_the_product(mxs):
    """Quantiser and product together: 2^-4 relative per element of each operand at
    most, 3 bits of mantissa; sums of random signs come within 2^-4 of the norm."""
    g = gen(6)
    x = torch.randn((33, 777), generator=g, device="cuda").to(BF)
    w = torch.randn((250, 777), generator=g, device="cuda").to(BF)
    y = mxs.matmul_fp8(*mxs.quantize_fp8(x, 1), *mxs.quantize_fp8(w, 128)).double()
    ref = x.double() @ w.double().t()
    assert (y - ref).norm() <= 2.0 ** -4 * ref.norm()


@pytest.mark.parametrize("rows,d,vocab,k", [(1, 896, 32000, 8), (33, 200, 5001, 40), (130, 512, 4096, 300)])
def test_sample_from_hidden_fp8(mxs, rows, d, vocab, k):
    """The sampled ids, order and probabilities are the oracle's on the call's own
    logits, which are the 8-bit product's."""
    g = gen(rows)
    h = torch.randn((rows, d), generator=g, device="cuda").to(BF)
    wq, ws = mxs.quantize_fp8((torch.randn((vocab, d), generator=g, device="cuda") * (3 / d ** 0.5)).to(BF), 128)
    u = torch.rand(rows, generator=g, device="cuda", dtype=torch.float64)
    logits = torch.empty((rows, vocab), dtype=torch.float32, device="cuda")
    nxt, idx, prob = mxs.sample_from_hidden_fp8(h, wq, ws, 0.8, k, u, logits_out=logits)
    assert torch.equal(logits, mxs.matmul_fp8(*mxs.quantize_fp8(h, 1), wq, ws))
    n0, i0, p0 = oracle_lib.oracle_sample(logits.cpu().numpy(), 0.8, k, u.cpu().numpy())
    np.testing.assert_array_equal(nxt.cpu().numpy(), n0)
    np.testing.assert_array_equal(idx.cpu().numpy(), i0)
    np.testing.assert_allclose(prob.cpu().numpy(), p0, rtol=1e-6, atol=0)
    n2, i2, _ = mxs.sample_from_hidden_fp8(h, wq, ws, 0.8, k, u)
    assert torch.equal(n2, nxt) and torch.equal(i2, idx)


def test_refusals(mxs):
    h, w, t = operands(4, 20, 16, BF)
    g = torch.ones(4, device="cuda")
    _, lse = mxs.ce_from_hidden(h, w, t)
    for bad in (lambda: mxs.ce_from_hidden(h.cpu(), w, t), lambda: mxs.ce_from_hidden(h.float(), w.float(), t),
                lambda: mxs.ce_from_hidden(h, w.to(HF), t), lambda: mxs.ce_from_hidden(h, w[:, :8], t),
                lambda: mxs.ce_from_hidden(h, w, t[:3]), lambda: mxs.ce_from_hidden(h, w, t.float()),
                lambda: mxs.ce_from_hidden(h, w, t, temperature=0.0), lambda: mxs.ce_from_hidden(h.t(), w.t(), t),
                lambda: mxs.ce_from_hidden(h, w, t, temperature=float("nan")),
                lambda: mxs.ce_from_hidden(h, w, t.cpu()), lambda: mxs.ce_from_hidden(h, w, t[::2]),
                lambda: mxs.ce_from_hidden_backward(h, w, t, lse.double(), g),
                lambda: mxs.ce_from_hidden_backward(h, w, t, lse, g[:2]),
                lambda: mxs.quantize_fp8(h, 64), lambda: mxs.quantize_fp8(h.double(), 1),
                lambda: mxs.quantize_fp8(h.t(), 1)):
        with pytest.raises(ValueError):
            bad()
    a, sa, b, sb = fp8_operands(4, 20, 200)
    for bad in (lambda: mxs.matmul_fp8(a, sa[:, :1], b, sb), lambda: mxs.matmul_fp8(a, sa, b[:, :100], sb),
                lambda: mxs.matmul_fp8(h, sa, b, sb), lambda: mxs.matmul_fp8(a, sa, b, sb, out_dtype=torch.int32),
                lambda: mxs.matmul_fp8(a, sa, b, sb, out=torch.empty((4, 19), device="cuda")),
                lambda: mxs.matmul_fp8(a, sa.double(), b, sb),
                lambda: mxs.sample_from_hidden_fp8(h, b, sb, 1.0, 5, torch.zeros(4, device="cuda"))):
        with pytest.raises(ValueError):
            bad()
    # a workspace that is too small or not aligned is refused before anything is launched
    import ctypes
    lib, P = mxs.load(), ctypes.c_void_p
    ws = torch.empty(64, dtype=torch.uint8, device="cuda")
    loss = torch.empty(4, device="cuda")
    rc = lib.mxs_ce_from_hidden(P(h.data_ptr()), 16, P(w.data_ptr()), 16, 0, 4, 16, 20, P(t.data_ptr()), 8, 1.0,
                                P(loss.data_ptr()), None, P(ws.data_ptr()), 64, None)
    assert rc == mxs.MXS_ERR_WORKSPACE


# ---------------------------------------------------------------------------
# Large offsets, give-ups, the example
# ---------------------------------------------------------------------------

def test_offsets_past_32_bits(mxs):
    """A weight of 2.24e9 elements: the last vocabulary rows' logits, targets and
    gradients, against the formula on those rows (lse from pieces in doubles)."""
    rows, vocab, d = 3, 140000, 16000
    g = gen(31)
    w = torch.empty((vocab, d), dtype=BF, device="cuda")
    for i in range(0, vocab, 10000):
        w[i:i + 10000] = torch.randn((10000, d), generator=g, device="cuda") * (2.5 / math.sqrt(d))
    h = torch.randn((rows, d), generator=g, device="cuda").to(BF)
    t = torch.tensor([vocab - 1, 5, vocab - 700], device="cuda")
    loss, lse = mxs.ce_from_hidden(h, w, t)
    x = torch.cat([h.double() @ w[i:i + 10000].double().t() for i in range(0, vocab, 10000)], 1)
    tol = head_ref.logit_tol(h, w[:10000], 1.0)  # rows of one distribution: the largest norm of 10000 stands for all
    want = torch.logsumexp(x, 1)
    assert ((lse.double() - want).abs() <= 2 * tol + 1e-5).all()
    assert ((loss.double() - (want - x.gather(1, t[:, None])[:, 0])).abs() <= 4 * tol + 1e-5).all()
    grad = torch.tensor([1.0, -0.5, 2.0], device="cuda")
    _, gw = mxs.ce_from_hidden_backward(h, w, t, lse, grad, need_hidden=False)
    p = torch.exp(x - want[:, None])
    p.scatter_add_(1, t[:, None], torch.full((rows, 1), -1.0, dtype=torch.float64, device="cuda"))
    p *= grad.double()[:, None]
    for part in (slice(0, 300), slice(vocab - 1000, vocab)):
        dw = p[:, part].t() @ h.double()
        mag = p[:, part].abs().t() @ h.double().abs()
        # G and the result rounded to bf16 (2^-8 each), the probabilities' own error
        assert ((gw[part].double() - dw).abs() <= (2 * 2.0 ** -8 + 4 * tol) * mag + 1e-30).all()


def test_output_offsets_past_32_bits(mxs):
    """An 8-bit product with 2.4e9 outputs: its last rows against those computed alone."""
    a, sa, b, sb = fp8_operands(16000, 300, 128, seed=3)
    b, sb = b.view(torch.uint8).repeat(500, 1).view(torch.float8_e4m3fn), None
    n = b.shape[0]  # 150000
    sb = torch.rand((-(-n // 128), 1), generator=gen(5), device="cuda") + 0.5
    out = mxs.matmul_fp8(a, sa, b, sb, out_dtype=BF)
    check = mxs.matmul_fp8(a[15990:], sa[15990:], b, sb, out_dtype=BF)
    assert torch.equal(out[15990:], check)
    want, tol = head_ref.matmul_fp8(a[15990:], sa[15990:], b, sb, BF)
    assert ((check.double() - want).abs() <= tol).all()


def big_head(mxs):
    h, w, t = operands(300, 20000, 512, BF, seed=40)
    a = fp8_operands(300, 9000, 512)
    few = (a[0][:20], a[1][:20], a[2], a[3])
    mid = (a[0][:100], a[1][:100], a[2], a[3])
    loss, lse = mxs.ce_from_hidden(h, w, t)
    grad = torch.ones(300, device="cuda")
    return {
        "loss": lambda: mxs.ce_from_hidden(h, w, t),
        "loss of few rows": lambda: mxs.ce_from_hidden(h[:9], w, t[:9]),
        "gradients": lambda: mxs.ce_from_hidden_backward(h, w, t, lse, grad),
        "product": lambda: (mxs.matmul_fp8(*a),),
        "product of some rows": lambda: (mxs.matmul_fp8(*mid),),
        "product of few rows": lambda: (mxs.matmul_fp8(*few),),
    }


@pytest.mark.parametrize("name", ["loss", "loss of few rows", "gradients", "product", "product of some rows",
                                  "product of few rows"])
def test_bounded_waits_give_up(mxs, name):
    """A producer that stops before one of its copies (a test hook): the waits give
    up after about a second, the status word says so, nothing hangs, and the next
    call on the same inputs gives the same bits as before."""
    call = big_head(mxs)[name]
    before = call()
    torch.cuda.synchronize()
    mxs.get_status(clear=True)
    mxs.set_test_hooks(drop_tile=1)  # every case has two blocks for its first CTA
    try:
        call()
        torch.cuda.synchronize()
    finally:
        mxs.set_test_hooks()
    assert mxs.get_status(clear=True) & mxs.ROW_TIMEOUT
    after = call()
    torch.cuda.synchronize()
    assert mxs.get_status(clear=True) == 0
    for x, y in zip(before, after):
        assert torch.equal(x, y)


def test_example_learns(mxs):
    """The example's step (8-bit draw, score, gradient, update): the reward rises."""
    import os
    import sys
    sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))
    import head_step
    log = head_step.train(rows=128, d=256, vocab=4000, steps=25)
    first, last = sum(r for r, _ in log[:5]) / 5, sum(r for r, _ in log[-5:]) / 5
    assert all(math.isfinite(l) for _, l in log)
    assert last > first
