"""The output head's operators (include/mxs_head.h): softmax cross entropy from
hidden states with its gradients, the 8-bit quantiser and block-scaled matrix
product, and sampling from an 8-bit head.

As in the rest of the package torch only carries memory and streams. Outputs and
scratch are torch tensors of the call's stream (`stream`, or the current one), so
calls on different streams share none. Inputs are the caller's, as with torch's
operations under torch.cuda.stream: the call does not wait for the stream they were
made on, and a tensor given to another stream than its own is kept (or recorded
there) until that stream has used it.
"""
import contextlib
import ctypes

import torch

from . import _check, k_use, load

BF16, F16, F32 = 0, 1, 2
_CODES = {torch.bfloat16: BF16, torch.float16: F16, torch.float32: F32}
FP8 = torch.float8_e4m3fn
BLOCK = 128


def _ptr(t):
    return None if t is None else t.data_ptr()


def _stream(stream, dev):
    """The stream's handle (the current one's is read without making a Stream: that
    costs 3 us, as much as a small call's launch)."""
    return stream.cuda_stream if stream is not None else torch._C._cuda_getCurrentRawStream(dev)


_HERE = contextlib.nullcontext()


@contextlib.contextmanager
def _elsewhere(dev, stream):
    with torch.cuda.device(dev), torch.cuda.stream(stream):
        yield


def _on(dev, stream):
    """The device and stream of a call made current, where they are not."""
    if stream is None and dev == torch.cuda.current_device():
        return _HERE
    if stream is not None and stream.device_index != dev:
        raise ValueError(f"stream is on cuda:{stream.device_index}, the operands on cuda:{dev}")
    return _elsewhere(dev, stream)


# The checks below read each attribute of a tensor once: a small call's time is
# the host's.


def _matrix(t, name, dtypes, dev=None):
    """(rows, cols, leading dimension) of a [rows, cols] CUDA tensor with unit column stride."""
    d = t.get_device()
    if d < 0:
        raise ValueError(f"{name} must be a CUDA tensor")
    if dev is not None and d != dev:
        raise ValueError(f"{name} must be on cuda:{dev}")
    if t.dtype not in dtypes:
        raise ValueError(f"{name} must be one of {', '.join(str(a) for a in dtypes)}")
    if t.dim() != 2:
        raise ValueError(f"{name} must be [rows, cols]")
    (rows, cols), (ld, one) = t.shape, t.stride()
    if rows <= 1:
        ld = max(ld, cols)
    if (one != 1 and cols > 1) or ld < cols:
        raise ValueError(f"{name} must have unit column stride and rows that do not overlap")
    return rows, cols, ld


def _dense(t, shape, name, dtypes, dev):
    if t.get_device() != dev or t.dtype not in dtypes or t.shape != shape or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous {list(shape)} tensor of "
                         f"{' or '.join(str(d) for d in dtypes)} on cuda:{dev}")


def _scratch(query, *args):
    n = ctypes.c_size_t()
    _check(query, getattr(load(), query)(*args, ctypes.byref(n)))
    return torch.empty(n.value, dtype=torch.uint8, device="cuda") if n.value else None


def _size(ws):
    return ws.numel() if ws is not None else 0


_HALF = (torch.bfloat16, torch.float16)
_FLOATS = (torch.bfloat16, torch.float16, torch.float32)
_F32, _F64, _INTS, _FP8 = (torch.float32,), (torch.float64,), (torch.int32, torch.int64), (FP8,)


def _ce_operands(hidden, weight, targets, temperature):
    rows, d, ldh = _matrix(hidden, "hidden", _HALF)
    dev = hidden.get_device()
    vocab, dw, ldw = _matrix(weight, "weight", (hidden.dtype,), dev)
    if dw != d or d == 0 or vocab == 0:
        raise ValueError("hidden [rows, d] and weight [vocab, d] must share d")
    _dense(targets, (rows,), "targets", _INTS, dev)
    if not temperature > 0:
        raise ValueError("temperature must be positive")
    return dev, _CODES[hidden.dtype], rows, d, vocab, ldh, ldw, targets.element_size()


def ce_from_hidden(hidden, weight, targets, temperature=1.0, stream=None):
    """Softmax cross entropy over the vocabulary (mxs_ce_from_hidden): hidden
    [rows, d] and weight [vocab, d] bf16 or f16 (rows may be strided), targets
    [rows] int32 or int64; the logits <hidden, weight> / temperature are never
    stored. Returns (loss [rows] f32, lse [rows] f32). Rows whose target is
    outside [0, vocab) are left out (loss and lse 0). -loss is the targets'
    log-probability."""
    dev, dt, rows, d, vocab, ldh, ldw, tb = _ce_operands(hidden, weight, targets, temperature)
    with _on(dev, stream):
        loss = torch.empty(rows, dtype=torch.float32, device="cuda")
        lse = torch.empty(rows, dtype=torch.float32, device="cuda")
        ws = _scratch("mxs_ce_workspace_size", _ptr(weight), ldw, rows, d, vocab, 0)
        rc = load().mxs_ce_from_hidden(_ptr(hidden), ldh, _ptr(weight), ldw, dt, rows, d, vocab, _ptr(targets), tb,
                                       float(temperature), _ptr(loss), _ptr(lse), _ptr(ws), _size(ws),
                                       _stream(stream, dev))
    _check("mxs_ce_from_hidden", rc)
    return loss, lse


def ce_from_hidden_backward(hidden, weight, targets, lse, grad_loss, temperature=1.0, need_hidden=True,
                            need_weight=True, stream=None):
    """Gradients of (grad_loss * loss).sum() (mxs_ce_from_hidden_backward) from
    ce_from_hidden's lse: (grad_hidden, grad_weight) in the operands' type; one
    that is not needed is None and is not computed."""
    dev, dt, rows, d, vocab, ldh, ldw, tb = _ce_operands(hidden, weight, targets, temperature)
    _dense(lse, (rows,), "lse", _F32, dev)
    _dense(grad_loss, (rows,), "grad_loss", _F32, dev)
    with _on(dev, stream):
        gh = torch.empty((rows, d), dtype=hidden.dtype, device="cuda") if need_hidden else None
        gw = torch.empty((vocab, d), dtype=hidden.dtype, device="cuda") if need_weight else None
        ws = _scratch("mxs_ce_workspace_size", _ptr(weight), ldw, rows, d, vocab, 1)
        rc = load().mxs_ce_from_hidden_backward(_ptr(hidden), ldh, _ptr(weight), ldw, dt, rows, d, vocab,
                                                _ptr(targets), tb, float(temperature), _ptr(lse), _ptr(grad_loss),
                                                _ptr(gh), d, _ptr(gw), d, _ptr(ws), _size(ws), _stream(stream, dev))
    _check("mxs_ce_from_hidden_backward", rc)
    return gh, gw


class _CrossEntropy(torch.autograd.Function):
    @staticmethod
    def forward(ctx, hidden, weight, targets, temperature):
        loss, lse = ce_from_hidden(hidden, weight, targets, temperature)
        ctx.save_for_backward(hidden, weight, targets, lse)
        ctx.temperature = temperature
        return loss

    @staticmethod
    def backward(ctx, grad_loss):
        hidden, weight, targets, lse = ctx.saved_tensors
        with torch.no_grad():
            gh, gw = ce_from_hidden_backward(hidden, weight, targets, lse, grad_loss.float().contiguous(),
                                             ctx.temperature, ctx.needs_input_grad[0], ctx.needs_input_grad[1])
        if torch.is_grad_enabled():  # create_graph
            gh, gw = _DifferentiatedOnce.apply(gh, gw, hidden, weight, grad_loss)
        return gh, gw, None, None


class _DifferentiatedOnce(torch.autograd.Function):
    """Gradients with a place in the graph of what they were computed from, where
    differentiating them raises. (torch's once_differentiable looks at grad_loss
    alone: a constant one, a plain sum's, would leave the gradients without a graph
    and a second derivative without their part.)"""

    @staticmethod
    def forward(ctx, gh, gw, hidden, weight, grad_loss):
        return gh, gw

    @staticmethod
    def backward(ctx, *grads):
        raise RuntimeError("cross_entropy_from_hidden can be differentiated once only")


def cross_entropy_from_hidden(hidden, weight, targets, temperature=1.0):
    """ce_from_hidden's loss [rows] as a function of hidden and weight that
    torch.autograd can differentiate once (second derivatives raise)."""
    return _CrossEntropy.apply(hidden, weight, targets, float(temperature))


def quantize_fp8(x, block_rows, stream=None):
    """8-bit floats with a scale for each block_rows x 128 block
    (mxs_quantize_fp8): block_rows 1 for activations, 128 for weights. x [rows,
    cols] bf16, f16 or f32. Returns (q [rows, cols] float8_e4m3fn, scale
    [ceil(rows / block_rows), ceil(cols / 128)] f32); q's rows start on 16-byte
    boundaries (its leading dimension is cols rounded up to 16)."""
    rows, cols, ldx = _matrix(x, "x", _FLOATS)
    if block_rows not in (1, BLOCK):
        raise ValueError("block_rows must be 1 or 128")
    if cols == 0:
        raise ValueError("x must have columns")
    dev = x.get_device()
    ldq = -(-cols // 16) * 16
    with _on(dev, stream):
        q = torch.empty((rows, ldq), dtype=FP8, device="cuda")
        if ldq != cols:
            q = q[:, :cols]
        scale = torch.empty((-(-rows // block_rows), -(-cols // BLOCK)), dtype=torch.float32, device="cuda")
        rc = load().mxs_quantize_fp8(_ptr(x), ldx, _CODES[x.dtype], rows, cols, block_rows, _ptr(q), ldq, _ptr(scale),
                                     _stream(stream, dev))
    _check("mxs_quantize_fp8", rc)
    return q, scale


def matmul_fp8(a, a_scale, b, b_scale, out_dtype=torch.float32, out=None, stream=None):
    """a @ b.T for 8-bit a [rows, k] with a scale for each 1 x 128 block and b
    [n, k] with one for each 128 x 128 block (mxs_matmul_fp8), as quantize_fp8
    makes them. Returns [rows, n] of out_dtype (f32, bf16 or f16), or fills `out`."""
    rows, k, lda = _matrix(a, "a", _FP8)
    dev = a.get_device()
    n, kw, ldb = _matrix(b, "b", _FP8, dev)
    if kw != k or k == 0 or n == 0:
        raise ValueError("a [rows, k] and b [n, k] must share k")
    kb = -(-k // BLOCK)
    _dense(a_scale, (rows, kb), "a_scale", _F32, dev)
    _dense(b_scale, (-(-n // BLOCK), kb), "b_scale", _F32, dev)
    with _on(dev, stream):
        if out is None:
            if out_dtype not in _CODES:
                raise ValueError("out_dtype must be float32, bfloat16 or float16")
            out, ldo = torch.empty((rows, n), dtype=out_dtype, device="cuda"), n
        else:
            ro, no, ldo = _matrix(out, "out", _FLOATS, dev)
            if (ro, no) != (rows, n):
                raise ValueError(f"out must be [{rows}, {n}]")
        ws = _scratch("mxs_matmul_fp8_workspace_size", _ptr(a), lda, _ptr(b), ldb, rows, n, k)
        rc = load().mxs_matmul_fp8(_ptr(a), lda, _ptr(a_scale), _ptr(b), ldb, _ptr(b_scale), rows, n, k, _ptr(out),
                                   ldo, _CODES[out.dtype], _ptr(ws), _size(ws), _stream(stream, dev))
    _check("mxs_matmul_fp8", rc)
    return out


def sample_from_hidden_fp8(hidden, weight_q, weight_scale, temperature, top_k, u, top_p=1.0, min_p=0.0,
                           logits_out=None, return_topk=True, stream=None):
    """sample_from_hidden with the head in 8 bits (mxs_sample_from_hidden_fp8):
    hidden [rows, d] bf16 or f16, weight_q [vocab, d] and weight_scale from
    quantize_fp8(weight, 128). Returns (next, topk_idx, topk_prob)."""
    rows, d, ldh = _matrix(hidden, "hidden", _HALF)
    dev = hidden.get_device()
    vocab, dw, ldw = _matrix(weight_q, "weight_q", _FP8, dev)
    if dw != d or d == 0 or vocab == 0:
        raise ValueError("hidden [rows, d] and weight_q [vocab, d] must share d")
    _dense(weight_scale, (-(-vocab // BLOCK), -(-d // BLOCK)), "weight_scale", _F32, dev)
    _dense(u, (rows,), "u", _F64, dev)
    ldl = 0
    if logits_out is not None:
        rl, cl, ldl = _matrix(logits_out, "logits_out", _F32, dev)
        if (rl, cl) != (rows, vocab):
            raise ValueError(f"logits_out must be [{rows}, {vocab}]")
    k = k_use(int(top_k), vocab)
    with _on(dev, stream):
        nxt = torch.empty(rows, dtype=torch.int32, device="cuda")
        idx = torch.empty((rows, k), dtype=torch.int32, device="cuda") if return_topk else None
        prob = torch.empty((rows, k), dtype=torch.float64, device="cuda") if return_topk else None
        ws = _scratch("mxs_sample_from_hidden_fp8_workspace_size", _ptr(weight_q), ldw, rows, d, vocab, int(top_k))
        rc = load().mxs_sample_from_hidden_fp8(_ptr(hidden), ldh, _CODES[hidden.dtype], _ptr(weight_q), ldw,
                                               _ptr(weight_scale), rows, d, vocab, float(temperature), int(top_k),
                                               float(top_p), float(min_p), _ptr(u), _ptr(nxt), _ptr(idx), _ptr(prob),
                                               _ptr(logits_out), ldl, _ptr(ws), _size(ws), _stream(stream, dev))
    _check("mxs_sample_from_hidden_fp8", rc)
    return nxt, idx, prob
