"""64-bit restatements of the output-head operators, written from their formulas
(torch doubles on whatever device the inputs are on), with the error bounds the
tests hold the kernels to. Unit roundoffs: U[t] of the stored type, 2^-24 of fp32.
"""
import math

import torch

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}  # 8, 11 and 24 significant bits


def kept_rows(targets, vocab):
    return torch.nonzero((targets >= 0) & (targets < vocab))[:, 0]


def logit_tol(h, w, temperature):
    """Bound on a logit's error: every partial sum of a dot product is at most
    |h||w| (Cauchy-Schwarz), each of the d additions loses at most 2^-23 of it
    when it truncates, and the losses of different additions add up like a random
    walk (sqrt d) with a factor 2 to spare; scaling by 1 / temperature loses two
    more roundings of the logit."""
    d = h.shape[1]
    big = (h.double().norm(dim=1).max() * w.double().norm(dim=1).max()).item() if h.numel() else 0.0
    return 2.0 ** -22 * (math.sqrt(d) + 4) * big / temperature


def ce(h, w, targets, temperature):
    """(loss, lse) in doubles; rows left out read 0."""
    rows, vocab = h.shape[0], w.shape[0]
    loss = torch.zeros(rows, dtype=torch.float64, device=h.device)
    lse = torch.zeros_like(loss)
    keep = kept_rows(targets, vocab)
    if keep.numel() == 0:
        return loss, lse
    x = h[keep].double() @ w.double().t() / temperature
    t = targets[keep].long()[:, None]
    xt = x.gather(1, t)[:, 0]
    others = torch.logsumexp(x.scatter(1, t, -math.inf), dim=1) if vocab > 1 else torch.full_like(xt, -math.inf)
    diff = others - xt
    loss[keep] = diff.clamp_min(0) + torch.log1p(torch.exp(-diff.abs()))
    lse[keep] = torch.logsumexp(x, dim=1)
    return loss, lse


def ce_tol(h, w, targets, temperature, loss, lse):
    """Errors of loss and lse: a logit's error moves others' log-sum and the
    target's logit by at most itself each; the sums of exponentials lose 2^-21
    relative (exp2 and at most 2^10 fp32 additions in a chain, as a random walk), and each result is
    rounded at its own size (4 roundings, of the largest of lse and loss)."""
    keep = kept_rows(targets, w.shape[0])
    tx = logit_tol(h[keep], w, temperature)
    # d loss / d (others - target) = 1 - p_target <= min(1, loss)
    e = 2 * tx + 2.0 ** -20
    size = torch.maximum(lse.abs(), loss.abs())
    return e * loss.clamp_max(1.0) + 2.0 ** -22 * loss + 1e-37, tx + 2.0 ** -20 + 2.0 ** -22 * size


def ce_grads(h, w, targets, grad, temperature):
    """(grad_hidden, grad_weight) in doubles and their elementwise bounds for G
    held in the operands' type: G's rounding u and the probabilities' relative
    error (from the logits' and lse's) multiply the sums' absolute values; fp32
    accumulation adds 2^-22 sqrt(terms) of them; the result is rounded once."""
    rows, vocab, dt = h.shape[0], w.shape[0], h.dtype
    keep = kept_rows(targets, vocab)
    dh = torch.zeros(h.shape, dtype=torch.float64, device=h.device)
    dw = torch.zeros(w.shape, dtype=torch.float64, device=h.device)
    eh, ew = torch.zeros_like(dh), torch.zeros_like(dw)
    if keep.numel() == 0:
        return dh, dw, eh, ew
    hk, wd = h[keep].double(), w.double()
    x = hk @ wd.t() / temperature
    p = torch.softmax(x, dim=1)
    t = targets[keep].long()[:, None]
    hot = torch.zeros_like(p).scatter_(1, t, 1.0)
    g = grad[keep].double()[:, None] / temperature
    dh[keep] = (p - hot) * g @ wd
    dw[:] = ((p - hot) * g).t() @ hk
    u = U[dt]
    rel = 2 * logit_tol(h[keep], w, temperature) + 2.0 ** -20 + 2.0 ** -22 * x.abs().max().item()
    # f16 holds G times 2^14, relative to the largest |grad|: below 2^-28 it loses an absolute 2^-39 of that
    floor = 2.0 ** -39 * g.abs().max().item() if dt == torch.float16 else 0.0
    a = ((p - hot).abs() * u + p * rel) * g.abs() + floor
    terms = max(vocab, keep.numel())
    acc = 2.0 ** -22 * math.sqrt(terms)
    full = (p + hot) * g.abs()
    eh[keep] = (a + acc * full) @ wd.abs()
    ew[:] = (a + acc * full).t() @ hk.abs()
    tiny = 2.0 ** -25 if dt == torch.float16 else 1e-40  # results below the type's normal range
    return dh, dw, eh + u * (dh.abs() + eh) + tiny, ew + u * (dw.abs() + ew) + tiny


def quantize(x, block_rows):
    """(values of q as doubles, scale as float32) bit for bit: the fp32 quotients are
    the doubles' rounded to fp32 (correct, since 53 >= 2 * 24 + 2), then rounded to
    3 mantissa bits, half to even."""
    rows, cols = x.shape
    xd = x.double()
    br, bc = -(-rows // block_rows), -(-cols // 128)
    mag = torch.where(torch.isfinite(xd), xd.abs(), torch.zeros_like(xd))
    mag = torch.nn.functional.pad(mag, (0, bc * 128 - cols, 0, br * block_rows - rows))
    top = mag.view(br, block_rows, bc, 128).amax(dim=(1, 3))
    scale = torch.where(top > 0, (top / 448.0).float().clamp_min(2.0 ** -126), torch.ones_like(top).float())
    s = scale.repeat_interleave(block_rows, 0)[:rows].repeat_interleave(128, 1)[:, :cols].double()
    y = (xd / s).float().double()
    exp = (torch.frexp(y.abs().clamp_min(2.0 ** -6)).exponent.long() - 1).clamp(-6, 9)
    step = ((exp - 3 + 1023) << 52).view(torch.float64)  # 2^(exp - 3), exactly
    q = torch.where(torch.isinf(y), y, torch.round(y / step) * step).clamp(-448, 448)
    return torch.where(torch.isnan(xd), xd, q), scale


def spread(scale, block_rows, rows, cols):
    s = scale.repeat_interleave(block_rows, 0)[:rows] if block_rows > 1 else scale
    return s.repeat_interleave(128, 1)[:, :cols]


def matmul_fp8(a, a_scale, b, b_scale, out_dtype):
    """The product in doubles and its bound: each addition of 32 products loses at
    most 2^-23 of the sum of magnitudes, and there are k / 32 of them, a join of
    two roundings for each block of 128, and the output's rounding."""
    rows, k = a.shape
    n = b.shape[0]
    ad = a.float().double() * spread(a_scale.double(), 1, rows, k)
    bd = b.float().double() * spread(b_scale.double(), 128, n, k)
    out = ad @ bd.t()
    mag = ad.abs() @ bd.abs().t()
    tol = 2.0 ** -23 * (k / 32 + 2 * (k / 128 + 1) + 4) * mag
    tiny = 2.0 ** -25 if out_dtype == torch.float16 else 1e-40
    return out, tol + U[out_dtype] * (out.abs() + tol) + tiny
