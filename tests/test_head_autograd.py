"""CPU tests of cross_entropy_from_hidden's place in torch.autograd, with the two
device calls replaced by their formulas on the CPU: first derivatives reach both
operands, second derivatives are refused and not dropped."""
import pytest
import torch

import mxs_sampler
from mxs_sampler import head


@pytest.fixture
def stand_ins(monkeypatch):
    def probabilities(h, w, temperature):
        return torch.softmax(h @ w.t() / temperature, 1)

    def forward(h, w, t, temperature=1.0, stream=None):
        with torch.no_grad():
            x = h @ w.t() / temperature
            lse = torch.logsumexp(x, 1)
            return lse - x.gather(1, t[:, None])[:, 0], lse

    def backward(h, w, t, lse, grad, temperature=1.0, need_hidden=True, need_weight=True, stream=None):
        with torch.no_grad():
            g = probabilities(h, w, temperature)
            g[torch.arange(len(t)), t] -= 1
            g *= grad[:, None].to(g.dtype) / temperature
            return g @ w if need_hidden else None, g.t() @ h if need_weight else None

    monkeypatch.setattr(head, "ce_from_hidden", forward)
    monkeypatch.setattr(head, "ce_from_hidden_backward", backward)


def operands():
    g = torch.Generator().manual_seed(3)
    h = torch.randn((6, 5), generator=g).requires_grad_()
    w = torch.randn((9, 5), generator=g).requires_grad_()
    return h, w, torch.randint(0, 9, (6,), generator=g)


def test_first_derivatives(stand_ins):
    h, w, t = operands()
    got = torch.autograd.grad(mxs_sampler.cross_entropy_from_hidden(h, w, t, 0.8).sum(), (h, w))
    want = torch.autograd.grad(torch.nn.functional.cross_entropy(h @ w.t() / 0.8, t, reduction="sum"), (h, w))
    for a, b in zip(got, want):
        torch.testing.assert_close(a, b, rtol=1e-5, atol=1e-6)


@pytest.mark.parametrize("wanted", ["hidden", "weight", "both"])
def test_second_derivatives_are_refused(stand_ins, wanted):
    """A penalty on the gradients has a derivative of its own, which the operator
    does not compute: an error, not a gradient without it."""
    h, w, t = operands()
    inputs = {"hidden": (h,), "weight": (w,), "both": (h, w)}[wanted]
    loss = mxs_sampler.cross_entropy_from_hidden(h, w, t).sum()
    grads = torch.autograd.grad(loss, inputs, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiated once"):
        (loss + sum((g * g).sum() for g in grads)).backward()


def test_create_graph_alone_changes_nothing(stand_ins):
    h, w, t = operands()
    loss = mxs_sampler.cross_entropy_from_hidden(h, w, t).sum()
    plain = torch.autograd.grad(loss, (h, w), retain_graph=True)
    kept = torch.autograd.grad(loss, (h, w), create_graph=True)
    for a, b in zip(plain, kept):
        assert torch.equal(a, b) and not a.requires_grad and b.requires_grad


def test_second_derivatives_through_the_loss_weights_are_refused(stand_ins):
    """Only grad_loss needs a gradient of its own: the same error."""
    h, w, t = operands()
    scale = torch.ones(6, requires_grad=True)
    loss = (mxs_sampler.cross_entropy_from_hidden(h, w.detach(), t) * scale).sum()
    (gh,) = torch.autograd.grad(loss, (h,), create_graph=True)
    with pytest.raises(RuntimeError, match="differentiated once"):
        (gh * gh).sum().backward()
