"""Cases of the output-head operators: the cross entropy of a softmax over the
vocabulary taken from hidden states (with its gradients), the matrix product of
8-bit floats with a scale for each block of 128, and the quantiser that makes its
operands.

Three kinds of callers stand behind the cases: a sampler that also wants the
log-probability of tokens it was given (scoring, one row to a full batch), a
training step of the output head (loss and both gradients; prompts left out), and
a decode step whose output projection is held in 8 bits.
"""
import math
import os
import sys

import torch

own = False

FP8_MAX = 448.0  # largest finite value of the 8-bit type (4 exponent bits, 3 mantissa bits)
BLOCK = 128
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def _package():
    """The framework's Python side (its folder's name has a dot, so it is reached through the path)."""
    at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "minxfmr.cpp_b200")
    if at not in sys.path:
        sys.path.insert(0, at)
    import mxs_sampler
    return mxs_sampler


# ---------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------

def listed():
    return [
        # the log-probability of one drafted token, a small model's head: latency
        dict(name="score_1", op="score", rows=1, vocab=151936, d=896, dtype="bf16", temperature=1.0, pad=0),
        # a few sequences of odd width, rows padded to a wider stride, f16
        dict(name="score_45_ragged", op="score", rows=45, vocab=50001, d=1000, dtype="f16", temperature=0.8, pad=24),
        # a full batch of rows scored at the sampler's temperature
        dict(name="score_4096", op="score", rows=4096, vocab=151936, d=3584, dtype="bf16", temperature=0.8, pad=0),
        # a short training step of a small head, mean reduction
        dict(name="train_200", op="train", rows=200, vocab=32000, d=512, dtype="f16", temperature=1.0, pad=0,
             ignored=0.0, grad="mean"),
        # policy gradient over sampled tokens: prompts left out, a weight of either sign for each row
        dict(name="train_2048_prompts", op="train", rows=2048, vocab=128256, d=1024, dtype="bf16", temperature=0.7,
             pad=0, ignored=0.4, grad="advantage"),
        # a full training batch
        dict(name="train_4096", op="train", rows=4096, vocab=151936, d=3584, dtype="bf16", temperature=1.0, pad=0,
             ignored=0.0, grad="mean"),
        # decode: logits of one row from an 8-bit head
        dict(name="fp8_decode_1", op="matmul", rows=1, n=151936, k=3584, out="f32"),
        # decode: a batch of rows, odd sizes that end inside blocks of 128
        dict(name="fp8_61_ragged", op="matmul", rows=61, n=50001, k=1040, out="f32"),
        # an inner projection of a prompt in 8 bits
        dict(name="fp8_1000_inner", op="matmul", rows=1000, n=4096, k=8192, out="bf16"),
        # logits of a full batch
        dict(name="fp8_4096", op="matmul", rows=4096, n=151936, k=3584, out="f32"),
        # the rows of a decode batch, a scale for each row's 128 columns
        dict(name="quant_rows_64", op="quant", rows=64, cols=3584, dtype="bf16", block_rows=1),
        # the output head's weight, a scale for each 128 x 128 block
        dict(name="quant_head", op="quant", rows=151936, cols=3584, dtype="bf16", block_rows=128),
    ]


def _log_int(rng, lo, hi):
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    return v + 1 if v == 3072 else v


def _width(rng, lo, hi):
    """A row's length: a multiple of 64 half the time, else any."""
    v = _log_int(rng, lo, hi)
    v = max(64, v // 64 * 64) if rng.random() < 0.5 else v
    return v + 64 if v == 3072 else v


def draw(rng):
    op = rng.choice(["score", "score", "train", "train", "matmul", "matmul", "matmul", "quant"])
    if op in ("score", "train"):
        c = dict(op=op, rows=_log_int(rng, 1, 4096), vocab=_log_int(rng, 1000, 151936), d=_width(rng, 64, 3584),
                 dtype=rng.choice(["bf16", "f16"]), temperature=rng.choice([1.0, 0.7, 1.3]),
                 pad=rng.choice([0, 0, 8, 40]))
        if op == "train":
            c.update(ignored=rng.choice([0.0, 0.25, 0.6]), grad=rng.choice(["mean", "advantage"]))
        return c
    if op == "matmul":
        rows, n = _log_int(rng, 1, 4096), _log_int(rng, 256, 151936)
        k = min(_width(rng, 64, 8192), 4096 * 151936 * 3584 // (rows * n))
        return dict(op=op, rows=rows, n=n, k=k + (k == 3072), out=rng.choice(["f32", "bf16", "f16"]))
    return dict(op=op, rows=_log_int(rng, 1, 151936), cols=_width(rng, 64, 3584),
                dtype=rng.choice(["bf16", "f16", "f32"]), block_rows=rng.choice([1, 128]))


def _left_out(rows, share):
    """Rows that carry no loss: the last part (the next prompt) of each of up to 8 runs of rows."""
    seq = max(4, rows // 8)
    return [r % seq >= seq - share * seq for r in range(rows)]


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------

def _randn(shape, gen, scale=1.0):
    return torch.randn(shape, generator=gen, device="cuda").mul_(scale)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    op = case["op"]
    if op in ("score", "train"):
        rows, vocab, d, dt = case["rows"], case["vocab"], case["d"], DTYPES[case["dtype"]]
        # logits of a spread of 2 to 3, and a target that stands out by what a model has learnt of it
        weight = torch.empty((vocab, d + case["pad"]), dtype=dt, device="cuda")[:, :d]
        weight.copy_(_randn((vocab, d), gen, 2.5 / math.sqrt(d)))
        targets = torch.randint(0, vocab, (rows,), generator=gen, device="cuda")
        learnt = torch.rand((rows, 1), generator=gen, device="cuda") * 2.5
        hidden = (_randn((rows, d), gen) + learnt * weight[targets].float()).to(dt)
        state = dict(case=case, hidden=hidden, weight=weight)
        if op == "train":
            out = torch.tensor(_left_out(rows, case["ignored"]), device="cuda")
            targets = torch.where(out, torch.full_like(targets, -100), targets)
            kept = max(1, rows - int(sum(_left_out(rows, case["ignored"]))))
            if case["grad"] == "mean":
                state["grad"] = torch.full((rows,), 1.0 / kept, device="cuda")
            else:
                state["grad"] = _randn((rows,), gen, 1.0 / kept)
        state["targets"] = targets
        return state
    if op == "matmul":
        rows, n, k = case["rows"], case["n"], case["k"]
        # activations with a few wide channels; weights whose blocks differ in size
        a = _randn((rows, k), gen) * torch.exp(_randn((1, k), gen, 0.5))
        b = _randn((n, k), gen, 1.0 / math.sqrt(k))
        b *= torch.exp(_randn((n, 1), gen, 0.3))
        a, a_scale = _plain_quant(a, 1)
        b, b_scale = _plain_quant(b, BLOCK)
        return dict(case=case, a=a, a_scale=a_scale, b=b, b_scale=b_scale)
    x = _randn((case["rows"], case["cols"]), gen) * torch.exp(_randn((1, case["cols"]), gen, 0.7))
    x = x.to(DTYPES[case["dtype"]])
    if case["rows"] > 4:
        x[case["rows"] // 2] = 0  # a padding row: its blocks may hold nothing but zeros
    return dict(case=case, x=x)


# ---------------------------------------------------------------------------
# Plain forms: 32-bit arithmetic, rounded once at the end
# ---------------------------------------------------------------------------

def _spread(scale, rows_each, rows, cols):
    """A scale for each element of [rows, cols]."""
    s = scale.repeat_interleave(rows_each, 0)[:rows] if rows_each > 1 else scale
    return s.repeat_interleave(BLOCK, 1)[:, :cols]


def _plain_quant(x, block_rows):
    """Every block_rows x 128 block divided by (its largest magnitude / 448), rounded to 8 bits."""
    rows, cols = x.shape
    x = x.float()
    br, bc = -(-rows // block_rows), -(-cols // BLOCK)
    p = torch.nn.functional.pad(x.abs(), (0, bc * BLOCK - cols, 0, br * block_rows - rows))
    top = p.view(br, block_rows, bc, BLOCK).amax(dim=(1, 3))
    scale = torch.where(top > 0, (top / FP8_MAX).clamp_min(2.0 ** -126), torch.ones_like(top))
    q = (x / _spread(scale, block_rows, rows, cols)).clamp(-FP8_MAX, FP8_MAX).to(torch.float8_e4m3fn)
    return q, scale


def _plain_logits(hidden, weight, temperature):
    return (hidden.float() @ weight.float().t()) / temperature


def _plain_lse(logits):
    top = logits.amax(dim=1, keepdim=True)
    return (top + torch.log(torch.exp(logits - top).sum(dim=1, keepdim=True)))[:, 0]


def _plain_ce(state):
    """Cross entropy and, for a training step, its gradients."""
    c = state["case"]
    targets, weight = state["targets"], state["weight"]
    kept = (targets >= 0) & (targets < c["vocab"])
    at = torch.where(kept, targets, torch.zeros_like(targets))[:, None]
    logits = _plain_logits(state["hidden"], weight, c["temperature"])
    picked = logits.gather(1, at)[:, 0]
    # -log p of the target from the others' sum: lse - picked would cancel where p is near 1
    others = _plain_lse(logits.scatter(1, at, -math.inf)) - picked
    zero = torch.zeros_like(others)
    loss = others.clamp_min(0) + torch.log1p(torch.exp(-others.abs()))
    loss, lse = torch.where(kept, loss, zero), torch.where(kept, loss + picked, zero)
    if c["op"] == "score":
        return loss, lse
    p = torch.exp(logits - lse[:, None])
    del logits
    p.scatter_add_(1, at, torch.full_like(picked, -1.0)[:, None])
    p.mul_(torch.where(kept, state["grad"], zero)[:, None] / c["temperature"])
    d_hidden = p @ weight.float()
    d_weight = p.t() @ state["hidden"].float()
    return loss, lse, d_hidden.to(state["hidden"].dtype), d_weight.to(weight.dtype)


def _plain_matmul(state):
    c = state["case"]
    a = state["a"].float() * _spread(state["a_scale"], 1, c["rows"], c["k"])
    b = state["b"].float() * _spread(state["b_scale"], BLOCK, c["n"], c["k"])
    return (a @ b.t()).to(DTYPES[c["out"]])


def run(state):
    c = state["case"]
    if not own:
        if c["op"] == "quant":
            return _plain_quant(state["x"], c["block_rows"])
        return _plain_matmul(state) if c["op"] == "matmul" else _plain_ce(state)
    mxs = _package()
    if c["op"] == "quant":
        return mxs.quantize_fp8(state["x"], c["block_rows"])
    if c["op"] == "matmul":
        return mxs.matmul_fp8(state["a"], state["a_scale"], state["b"], state["b_scale"], out_dtype=DTYPES[c["out"]])
    loss, lse = mxs.ce_from_hidden(state["hidden"], state["weight"], state["targets"], temperature=c["temperature"])
    if c["op"] == "score":
        return loss, lse
    d_hidden, d_weight = mxs.ce_from_hidden_backward(state["hidden"], state["weight"], state["targets"], lse,
                                                     state["grad"], temperature=c["temperature"])
    return loss, lse, d_hidden, d_weight


# ---------------------------------------------------------------------------
# Work and 64-bit values
# ---------------------------------------------------------------------------

def work(case):
    op = case["op"]
    if op in ("score", "train"):
        rows, vocab, d = case["rows"], case["vocab"], case["d"]
        if op == "score":
            return {"bytes": 2 * (rows + vocab) * d + 16 * rows, "flops": 2 * rows * vocab * d}
        # loss: one product; gradients: the logits again (they are not kept), and a product for each operand,
        # for the rows that carry a loss
        kept = rows - int(sum(_left_out(rows, case["ignored"])))
        return {"bytes": 2 * d * (kept + rows + 2 * vocab) + 24 * rows, "flops": 8 * kept * vocab * d}
    if op == "matmul":
        rows, n, k = case["rows"], case["n"], case["k"]
        kb = -(-k // BLOCK)
        return {"bytes": (rows + n) * k + 4 * kb * (rows + -(-n // BLOCK)) + rows * n * (4 if case["out"] == "f32" else 2),
                "flops": 2 * rows * n * k}
    rows, cols = case["rows"], case["cols"]
    blocks = -(-rows // case["block_rows"]) * -(-cols // BLOCK)
    return {"bytes": rows * cols * ((4 if case["dtype"] == "f32" else 2) + 1) + 4 * blocks, "flops": 3 * rows * cols}


def _exact_ce(case, seed):
    st = prepare(case, seed)
    rows, vocab, t = case["rows"], case["vocab"], case["temperature"]
    h = st["hidden"].double()
    step = max(1, min(vocab, (1 << 28) // max(rows, case["d"])))
    pieces = [(v, min(vocab, v + step)) for v in range(0, vocab, step)]
    # log-sum-exp piece by piece
    lse = torch.full((rows,), -math.inf, dtype=torch.float64, device="cuda")
    for a, b in pieces:
        lse = torch.logaddexp(lse, torch.logsumexp(h @ st["weight"][a:b].double().t() / t, dim=1))
    tg = st["targets"]
    live = torch.nonzero((tg >= 0) & (tg < vocab))[:, 0]
    loss, norm = torch.zeros_like(lse), torch.zeros_like(lse)
    norm[live] = lse[live]
    loss[live] = lse[live] - (h[live] * st["weight"][tg[live]].double()).sum(1) / t
    if case["op"] == "score":
        return loss, norm
    g = st["grad"].double()[live] / t
    hl = h[live]
    dh = torch.zeros_like(h)
    dw = torch.empty((vocab, case["d"]), dtype=torch.float64, device="cuda")
    for a, b in pieces:
        w = st["weight"][a:b].double()
        p = torch.exp(hl @ w.t() / t - lse[live][:, None])
        here = torch.nonzero((tg[live] >= a) & (tg[live] < b))[:, 0]
        p[here, tg[live][here] - a] -= 1.0
        p *= g[:, None]
        dh[live] += p @ w
        dw[a:b] = p.t() @ hl
    return loss, norm, dh, dw


def _exact_matmul(case, seed):
    st = prepare(case, seed)
    kb = torch.arange(case["k"], device="cuda") // BLOCK
    a = st["a"].double() * st["a_scale"].double()[:, kb]
    out = torch.empty((case["rows"], case["n"]), dtype=torch.float64, device="cuda")
    step = 64 * BLOCK
    for i in range(0, case["n"], step):
        j = min(case["n"], i + step)
        nb = torch.arange(i, j, device="cuda") // BLOCK
        out[:, i:j] = a @ (st["b"][i:j].double() * st["b_scale"].double()[nb][:, kb]).t()
    return out


def _exact_quant(case, seed):
    x = prepare(case, seed)["x"].double()
    rows, cols = x.shape
    each = case["block_rows"]
    scale = torch.empty((-(-rows // each), -(-cols // BLOCK)), dtype=torch.float64, device="cuda")
    for j in range(scale.shape[1]):
        top = x[:, j * BLOCK:(j + 1) * BLOCK].abs().amax(1)
        if each > 1:
            top = torch.cat([top, top.new_zeros(scale.shape[0] * each - rows)]).view(-1, each).amax(1)
        scale[:, j] = torch.where(top > 0, (top / FP8_MAX).clamp_min(2.0 ** -126), torch.ones_like(top))
    # a value that lies next to the middle of two 8-bit ones may go to either after 32-bit division: the
    # 8-bit values are held to the plain form's alone
    return None, scale


def exact(case, seed):
    if case["op"] == "matmul":
        return _exact_matmul(case, seed)
    return _exact_quant(case, seed) if case["op"] == "quant" else _exact_ce(case, seed)
