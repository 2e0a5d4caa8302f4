"""The output head's operators (include/mxs_head.h): softmax cross entropy from
hidden states with its gradients, the 8-bit quantiser and block-scaled matrix
product, and sampling from an 8-bit head.

As in the rest of the package torch only carries memory and streams. Outputs and
scratch are torch tensors of the call's stream (`stream`, or the current one), so
calls on different streams share none.
"""
import contextlib
import ctypes

import torch

from . import _check, _need_cuda, k_use, load

BF16, F16, F32 = 0, 1, 2
_CODES = {torch.bfloat16: BF16, torch.float16: F16, torch.float32: F32}
FP8 = torch.float8_e4m3fn
BLOCK = 128


def _ptr(t):
    return None if t is None else t.data_ptr()


def _stream(stream, dev):
    """The stream's handle (the current one's is read without making a Stream: that
    costs 3 us, as much as a small call's launch)."""
    return stream.cuda_stream if stream is not None else torch._C._cuda_getCurrentRawStream(dev.index)


_HERE = contextlib.nullcontext()


@contextlib.contextmanager
def _elsewhere(dev, stream):
    with torch.cuda.device(dev), torch.cuda.stream(stream):
        yield


def _on(dev, stream):
    """The device and stream of a call made current, where they are not."""
    if stream is None and dev.index == torch.cuda.current_device():
        return _HERE
    return _elsewhere(dev, stream)


def _code(t, name, allowed):
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor")
    if t.dtype not in allowed:
        raise ValueError(f"{name} must be one of {', '.join(str(a) for a in allowed)}")
    return _CODES.get(t.dtype)


def _matrix(t, name):
    """Leading dimension of a [rows, cols] tensor with unit column stride."""
    if t.dim() != 2 or (t.stride(1) != 1 and t.shape[1] > 1) or (t.shape[0] > 1 and t.stride(0) < t.shape[1]):
        raise ValueError(f"{name} must be [rows, cols] with unit column stride and rows that do not overlap")
    return t.stride(0) if t.shape[0] > 1 else max(t.stride(0), t.shape[1])


def _vector(t, n, name, dtypes):
    if not t.is_cuda or t.dtype not in dtypes or t.dim() != 1 or t.numel() != n or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous [{n}] CUDA tensor of {' or '.join(str(d) for d in dtypes)}")


def _scratch(query, args, dev):
    n = ctypes.c_size_t()
    _check(query, getattr(load(), query)(*args, ctypes.byref(n)))
    return torch.empty(n.value, dtype=torch.uint8, device=dev) if n.value else None


def _same_device(dev, **tensors):
    for name, t in tensors.items():
        if t is not None and t.device != dev:
            raise ValueError(f"{name} must be on {dev}")


def _ce_operands(hidden, weight, targets, temperature):
    dt = _code(hidden, "hidden", (torch.bfloat16, torch.float16))
    if weight.dtype != hidden.dtype:
        raise ValueError("hidden and weight must have the same type")
    _same_device(hidden.device, weight=weight, targets=targets)
    ldh, ldw = _matrix(hidden, "hidden"), _matrix(weight, "weight")
    rows, d = hidden.shape
    if weight.shape[1] != d or d == 0 or weight.shape[0] == 0:
        raise ValueError("hidden [rows, d] and weight [vocab, d] must share d")
    _vector(targets, rows, "targets", (torch.int32, torch.int64))
    if not temperature > 0:
        raise ValueError("temperature must be positive")
    return dt, rows, d, weight.shape[0], ldh, ldw, targets.element_size()


def ce_from_hidden(hidden, weight, targets, temperature=1.0, stream=None):
    """Softmax cross entropy over the vocabulary (mxs_ce_from_hidden): hidden
    [rows, d] and weight [vocab, d] bf16 or f16 (rows may be strided), targets
    [rows] int32 or int64; the logits <hidden, weight> / temperature are never
    stored. Returns (loss [rows] f32, lse [rows] f32). Rows whose target is
    outside [0, vocab) are left out (loss and lse 0). -loss is the targets'
    log-probability."""
    dt, rows, d, vocab, ldh, ldw, tb = _ce_operands(hidden, weight, targets, temperature)
    dev = hidden.device
    with _on(dev, stream):
        loss = torch.empty(rows, dtype=torch.float32, device=dev)
        lse = torch.empty(rows, dtype=torch.float32, device=dev)
        ws = _scratch("mxs_ce_workspace_size", (_ptr(weight), ldw, rows, d, vocab, 0), dev)
        rc = load().mxs_ce_from_hidden(_ptr(hidden), ldh, _ptr(weight), ldw, dt, rows, d, vocab, _ptr(targets), tb,
                                       float(temperature), _ptr(loss), _ptr(lse), _ptr(ws), ws.numel() if ws is not None else 0,
                                       _stream(stream, dev))
    _check("mxs_ce_from_hidden", rc)
    return loss, lse


def ce_from_hidden_backward(hidden, weight, targets, lse, grad_loss, temperature=1.0, need_hidden=True,
                            need_weight=True, stream=None):
    """Gradients of (grad_loss * loss).sum() (mxs_ce_from_hidden_backward) from
    ce_from_hidden's lse: (grad_hidden, grad_weight) in the operands' type; one
    that is not needed is None and is not computed."""
    dt, rows, d, vocab, ldh, ldw, tb = _ce_operands(hidden, weight, targets, temperature)
    dev = hidden.device
    _same_device(dev, lse=lse, grad_loss=grad_loss)
    _vector(lse, rows, "lse", (torch.float32,))
    _vector(grad_loss, rows, "grad_loss", (torch.float32,))
    with _on(dev, stream):
        gh = torch.empty((rows, d), dtype=hidden.dtype, device=dev) if need_hidden else None
        gw = torch.empty((vocab, d), dtype=hidden.dtype, device=dev) if need_weight else None
        ws = _scratch("mxs_ce_workspace_size", (_ptr(weight), ldw, rows, d, vocab, 1), dev)
        rc = load().mxs_ce_from_hidden_backward(_ptr(hidden), ldh, _ptr(weight), ldw, dt, rows, d, vocab,
                                                _ptr(targets), tb, float(temperature), _ptr(lse), _ptr(grad_loss),
                                                _ptr(gh), d, _ptr(gw), d, _ptr(ws), ws.numel() if ws is not None else 0, _stream(stream, dev))
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
        gh, gw = ce_from_hidden_backward(hidden, weight, targets, lse, grad_loss.float().contiguous(),
                                         ctx.temperature, ctx.needs_input_grad[0], ctx.needs_input_grad[1])
        return gh, gw, None, None


def cross_entropy_from_hidden(hidden, weight, targets, temperature=1.0):
    """ce_from_hidden's loss [rows] as a differentiable function of hidden and
    weight, for torch.autograd."""
    return _CrossEntropy.apply(hidden, weight, targets, float(temperature))


def quantize_fp8(x, block_rows, stream=None):
    """8-bit floats with a scale for each block_rows x 128 block
    (mxs_quantize_fp8): block_rows 1 for activations, 128 for weights. x [rows,
    cols] bf16, f16 or f32. Returns (q [rows, cols] float8_e4m3fn, scale
    [ceil(rows / block_rows), ceil(cols / 128)] f32); q's rows start on 16-byte
    boundaries (its leading dimension is cols rounded up to 16)."""
    dt = _code(x, "x", (torch.bfloat16, torch.float16, torch.float32))
    ldx = _matrix(x, "x")
    if block_rows not in (1, BLOCK):
        raise ValueError("block_rows must be 1 or 128")
    rows, cols = x.shape
    if cols == 0:
        raise ValueError("x must have columns")
    dev = x.device
    ldq = -(-cols // 16) * 16
    with _on(dev, stream):
        q = torch.empty((rows, ldq), dtype=FP8, device=dev)[:, :cols]
        scale = torch.empty((-(-rows // block_rows), -(-cols // BLOCK)), dtype=torch.float32, device=dev)
        rc = load().mxs_quantize_fp8(_ptr(x), ldx, dt, rows, cols, block_rows, _ptr(q), ldq, _ptr(scale),
                                     _stream(stream, dev))
    _check("mxs_quantize_fp8", rc)
    return q, scale


def _scale(t, shape, name):
    if not t.is_cuda or t.dtype != torch.float32 or tuple(t.shape) != shape or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous {list(shape)} float32 CUDA tensor")


def matmul_fp8(a, a_scale, b, b_scale, out_dtype=torch.float32, out=None, stream=None):
    """a @ b.T for 8-bit a [rows, k] with a scale for each 1 x 128 block and b
    [n, k] with one for each 128 x 128 block (mxs_matmul_fp8), as quantize_fp8
    makes them. Returns [rows, n] of out_dtype (f32, bf16 or f16), or fills `out`."""
    _code(a, "a", (FP8,))
    _code(b, "b", (FP8,))
    lda, ldb = _matrix(a, "a"), _matrix(b, "b")
    (rows, k), n = a.shape, b.shape[0]
    if b.shape[1] != k or k == 0 or n == 0:
        raise ValueError("a [rows, k] and b [n, k] must share k")
    kb = -(-k // BLOCK)
    _scale(a_scale, (rows, kb), "a_scale")
    _scale(b_scale, (-(-n // BLOCK), kb), "b_scale")
    dev = a.device
    _same_device(dev, a_scale=a_scale, b=b, b_scale=b_scale, out=out)
    with _on(dev, stream):
        if out is None:
            if out_dtype not in _CODES:
                raise ValueError("out_dtype must be float32, bfloat16 or float16")
            out = torch.empty((rows, n), dtype=out_dtype, device=dev)
        elif out.dtype not in _CODES or tuple(out.shape) != (rows, n):
            raise ValueError(f"out must be [{rows}, {n}] float32, bfloat16 or float16")
        ldo = _matrix(out, "out")
        ws = _scratch("mxs_matmul_fp8_workspace_size", (_ptr(a), lda, _ptr(b), ldb, rows, n, k), dev)
        rc = load().mxs_matmul_fp8(_ptr(a), lda, _ptr(a_scale), _ptr(b), ldb, _ptr(b_scale), rows, n, k, _ptr(out),
                                   ldo, _CODES[out.dtype], _ptr(ws), ws.numel() if ws is not None else 0, _stream(stream, dev))
    _check("mxs_matmul_fp8", rc)
    return out


def sample_from_hidden_fp8(hidden, weight_q, weight_scale, temperature, top_k, u, top_p=1.0, min_p=0.0,
                           logits_out=None, return_topk=True, stream=None):
    """sample_from_hidden with the head in 8 bits (mxs_sample_from_hidden_fp8):
    hidden [rows, d] bf16 or f16, weight_q [vocab, d] and weight_scale from
    quantize_fp8(weight, 128). Returns (next, topk_idx, topk_prob)."""
    dt = _code(hidden, "hidden", (torch.bfloat16, torch.float16))
    _code(weight_q, "weight_q", (FP8,))
    _need_cuda(u, "u", torch.float64)
    ldh, ldw = _matrix(hidden, "hidden"), _matrix(weight_q, "weight_q")
    (rows, d), vocab = hidden.shape, weight_q.shape[0]
    if weight_q.shape[1] != d or d == 0 or vocab == 0:
        raise ValueError("hidden [rows, d] and weight_q [vocab, d] must share d")
    _scale(weight_scale, (-(-vocab // BLOCK), -(-d // BLOCK)), "weight_scale")
    dev = hidden.device
    _same_device(dev, weight_q=weight_q, weight_scale=weight_scale, u=u, logits_out=logits_out)
    _vector(u, rows, "u", (torch.float64,))
    if logits_out is not None and (logits_out.dtype != torch.float32 or tuple(logits_out.shape) != (rows, vocab)):
        raise ValueError(f"logits_out must be [{rows}, {vocab}] float32")
    ldl = 0 if logits_out is None else _matrix(logits_out, "logits_out")
    k = k_use(int(top_k), vocab)
    with _on(dev, stream):
        nxt = torch.empty(rows, dtype=torch.int32, device=dev)
        idx = torch.empty((rows, k), dtype=torch.int32, device=dev) if return_topk else None
        prob = torch.empty((rows, k), dtype=torch.float64, device=dev) if return_topk else None
        ws = _scratch("mxs_sample_from_hidden_fp8_workspace_size", (_ptr(weight_q), ldw, rows, d, vocab, int(top_k)),
                      dev)
        rc = load().mxs_sample_from_hidden_fp8(_ptr(hidden), ldh, dt, _ptr(weight_q), ldw, _ptr(weight_scale), rows, d,
                                               vocab, float(temperature), int(top_k), float(top_p), float(min_p),
                                               _ptr(u), _ptr(nxt), _ptr(idx), _ptr(prob), _ptr(logits_out), ldl,
                                               _ptr(ws), ws.numel() if ws is not None else 0, _stream(stream, dev))
    _check("mxs_sample_from_hidden_fp8", rc)
    return nxt, idx, prob
