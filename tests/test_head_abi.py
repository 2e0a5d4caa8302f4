"""CPU tests of the output-head entry points: bad arguments are refused before a
device is touched, empty calls succeed, and workspace sizes follow the shape."""
import ctypes

import pytest

import mxs_sampler
from mxs_sampler import MXS_ERR_INVALID, MXS_OK

P = ctypes.c_void_p
A = P(4096)


@pytest.fixture(scope="module")
def lib():
    import mxs_build
    mxs_build.build()
    return mxs_sampler.load()


def ce(lib, h=A, ldh=64, w=A, ldw=64, dt=0, rows=4, d=64, vocab=100, t=A, tb=8, temp=1.0, loss=A, lse=A, ws=A,
       n=1 << 40):
    return lib.mxs_ce_from_hidden(h, ldh, w, ldw, dt, rows, d, vocab, t, tb, temp, loss, lse, ws, n, None)


@pytest.mark.parametrize("bad", [
    dict(rows=-1), dict(d=0), dict(vocab=0), dict(ldh=63), dict(ldw=63), dict(dt=2), dict(dt=-1), dict(tb=2),
    dict(temp=0.0), dict(temp=-1.0), dict(temp=float("nan")), dict(temp=float("inf")), dict(h=None), dict(w=None),
    dict(t=None), dict(rows=2 ** 31), dict(vocab=2 ** 31), dict(d=2 ** 31, ldh=2 ** 31, ldw=2 ** 31),
])
def test_ce_refuses(lib, bad):
    assert ce(lib, **bad) == MXS_ERR_INVALID


def bwd(lib, rows=4, lse=A, g=A, gh=A, ldgh=64, gw=A, ldgw=64, **k):
    return lib.mxs_ce_from_hidden_backward(k.get("h", A), 64, A, 64, 0, rows, 64, 100, A, 8, 1.0, lse, g, gh, ldgh, gw,
                                           ldgw, A, 1 << 40, None)


def test_backward_refuses(lib):
    assert bwd(lib, lse=None) == MXS_ERR_INVALID
    assert bwd(lib, g=None) == MXS_ERR_INVALID
    assert bwd(lib, ldgh=63) == MXS_ERR_INVALID
    assert bwd(lib, ldgw=10) == MXS_ERR_INVALID
    assert bwd(lib, h=None) == MXS_ERR_INVALID
    assert bwd(lib, gh=None, gw=None) == MXS_OK  # nothing asked for
    assert bwd(lib, rows=0, gw=None) == MXS_OK


def test_empty_calls(lib):
    assert ce(lib, rows=0, h=None, t=None) == MXS_OK
    assert lib.mxs_quantize_fp8(None, 10, 0, 0, 10, 1, None, 10, None, None) == MXS_OK
    assert lib.mxs_matmul_fp8(None, 10, None, A, 10, A, 0, 5, 10, None, 5, 2, None, 0, None) == MXS_OK


def test_fp8_refuses(lib):
    q = lambda ldx=64, dt=0, rows=4, cols=64, br=1, ldq=64, x=A: lib.mxs_quantize_fp8(x, ldx, dt, rows, cols, br, A,
                                                                                     ldq, A, None)
    for bad in (dict(ldx=63), dict(ldq=63), dict(dt=3), dict(rows=-1), dict(cols=0), dict(br=2), dict(x=None)):
        assert q(**bad) == MXS_ERR_INVALID
    m = lambda lda=64, ldb=64, rows=4, n=32, k=64, ldo=32, dt=2, a=A, o=A: lib.mxs_matmul_fp8(
        a, lda, A, A, ldb, A, rows, n, k, o, ldo, dt, A, 1 << 40, None)
    for bad in (dict(lda=63), dict(ldb=63), dict(rows=-1), dict(n=0), dict(k=0), dict(ldo=31), dict(dt=7),
                dict(a=None), dict(o=None)):
        assert m(**bad) == MXS_ERR_INVALID
    s = lambda **k: lib.mxs_sample_from_hidden_fp8(
        k.get("h", A), k.get("ldh", 64), k.get("dt", 0), A, 64, A, k.get("rows", 4), 64, 100, 1.0, 5, 1.0, 0.0,
        k.get("u", A), A, None, None, A, k.get("ldl", 100), A, 1 << 40, None)
    for bad in (dict(h=None), dict(ldh=1), dict(dt=2), dict(rows=-1), dict(u=None), dict(ldl=99)):
        assert s(**bad) == MXS_ERR_INVALID


def test_workspace_queries_refuse(lib):
    n = ctypes.c_size_t()
    r = ctypes.byref(n)
    assert lib.mxs_ce_workspace_size(A, 64, 4, 64, 100, 0, None) == MXS_ERR_INVALID
    assert lib.mxs_ce_workspace_size(A, 63, 4, 64, 100, 0, r) == MXS_ERR_INVALID
    assert lib.mxs_ce_workspace_size(A, 64, -1, 64, 100, 0, r) == MXS_ERR_INVALID
    assert lib.mxs_matmul_fp8_workspace_size(A, 64, A, 10, 4, 4, 64, r) == MXS_ERR_INVALID


def test_python_refuses_cpu_tensors():
    import torch
    h = torch.zeros((2, 16), dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        mxs_sampler.ce_from_hidden(h, h, torch.zeros(2, dtype=torch.int64))
    with pytest.raises(ValueError):
        mxs_sampler.quantize_fp8(h, 1)
