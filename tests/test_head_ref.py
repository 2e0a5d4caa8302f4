"""CPU tests of the 64-bit restatements that the GPU tests compare with: the loss
and its gradients against torch's own cross entropy and autograd in doubles, the
quantiser against torch's 8-bit conversion."""
import pytest
import torch

import head_ref


@pytest.mark.parametrize("temperature", [1.0, 0.6])
def test_cross_entropy_restatement(temperature):
    g = torch.Generator().manual_seed(1)
    h = torch.randn((9, 12), generator=g).to(torch.bfloat16)
    w = torch.randn((31, 12), generator=g).to(torch.bfloat16)
    t = torch.randint(0, 31, (9,), generator=g)
    t[4] = -100
    grad = torch.randn(9, generator=g)
    hd, wd = h.double().requires_grad_(), w.double().requires_grad_()
    x = hd @ wd.t() / temperature
    want = torch.nn.functional.cross_entropy(x, t, reduction="none")
    (want * grad.double()).sum().backward()
    loss, lse = head_ref.ce(h, w, t, temperature)
    torch.testing.assert_close(loss, want.detach(), rtol=1e-12, atol=1e-12)
    keep = t >= 0
    torch.testing.assert_close(lse[keep], torch.logsumexp(x.detach(), 1)[keep], rtol=1e-12, atol=1e-12)
    dh, dw, _, _ = head_ref.ce_grads(h, w, t, grad, temperature)
    torch.testing.assert_close(dh, hd.grad, rtol=1e-11, atol=1e-13)
    torch.testing.assert_close(dw, wd.grad, rtol=1e-11, atol=1e-13)


@pytest.mark.parametrize("block_rows", [1, 128])
def test_quantize_restatement(block_rows):
    g = torch.Generator().manual_seed(2)
    x = torch.randn((150, 300), generator=g) * torch.exp(3 * torch.randn((1, 300), generator=g))
    x[70] = 0
    q, s = head_ref.quantize(x, block_rows)
    y = x / head_ref.spread(s, block_rows, 150, 300)
    assert torch.equal(q, y.clamp(-448, 448).to(torch.float8_e4m3fn).double())
    assert q.abs().max() == 448
    planted = x.clone()
    planted[3, 5] *= 1.5  # more than an 8-bit step
    assert not torch.equal(head_ref.quantize(planted, block_rows)[0], q)
