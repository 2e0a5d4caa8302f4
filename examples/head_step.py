"""One policy-gradient step of an output head, with the head served in 8 bits.

Tokens are drawn from the 8-bit head (quantise the hidden states, multiply, sample),
scored under the 16-bit head that is trained (their log-probability is minus the
cross entropy), and the head is moved along the gradient of the advantage-weighted
log-probability; the 8-bit copy is then made again from the new weight. No step
stores the logits of the 16-bit head.

    python examples/head_step.py [--rows 256] [--d 896] [--vocab 32000] [--steps 20]

The reward of a token is 1 when it is one of a row's `good` tokens; its average
rises from chance towards 1 within the steps.
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "minxfmr.cpp_b200"))
import mxs_sampler  # noqa: E402


def train(rows=256, d=896, vocab=32000, steps=20, temperature=1.0, lr=400.0, seed=0):
    """Returns (mean reward, mean loss of the drawn tokens) of each step."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    hidden = torch.randn((rows, d), generator=gen, device="cuda").to(torch.bfloat16)
    master = torch.randn((vocab, d), generator=gen, device="cuda") * (2.0 / d ** 0.5)
    good = torch.randint(0, vocab, (rows, 64), generator=gen, device="cuda")
    # a head that already leans towards the good tokens, so that some are drawn
    master.index_add_(0, good.view(-1), (hidden.float() * (5.0 / d)).repeat_interleave(64, 0))
    log = []
    for _ in range(steps):
        weight = master.to(torch.bfloat16)
        weight_q, weight_scale = mxs_sampler.quantize_fp8(weight, 128)
        u = torch.rand(rows, generator=gen, device="cuda", dtype=torch.float64)
        token, _, _ = mxs_sampler.sample_from_hidden_fp8(hidden, weight_q, weight_scale, temperature, 128, u,
                                                         return_topk=False)
        reward = (good == token[:, None]).any(1).float()
        advantage = (reward - reward.mean()) / rows
        loss, lse = mxs_sampler.ce_from_hidden(hidden, weight, token, temperature)
        _, grad = mxs_sampler.ce_from_hidden_backward(hidden, weight, token, lse, advantage, temperature,
                                                      need_hidden=False)
        master.add_(grad.float(), alpha=-lr / d)
        log.append((reward.mean(), loss.mean()))
    return [(r.item(), l.item()) for r, l in log]


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--rows", type=int, default=256)
    ap.add_argument("--d", type=int, default=896)
    ap.add_argument("--vocab", type=int, default=32000)
    ap.add_argument("--steps", type=int, default=20)
    a = ap.parse_args()
    for i, (reward, loss) in enumerate(train(a.rows, a.d, a.vocab, a.steps)):
        print(f"step {i:3d}  reward {reward:.3f}  loss of the drawn tokens {loss:.3f}")
