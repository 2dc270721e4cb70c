"""The example's path (examples/learn_from_samples.py): the 4-bit head, the exact candidates, the sampler, the log probabilities and
the two losses, each against the others and the gradients against the formulas in 64 bits."""
import importlib.util
from pathlib import Path

import pytest
import torch

import qwen_warp_amd as q

pytestmark = pytest.mark.gpu
B, STEPS, N, K, T = 6, 5, 8000, 256, 0.8


def example():
    spec = importlib.util.spec_from_file_location("example_learn", Path(__file__).resolve().parents[1] / "examples" / "learn_from_samples.py")
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


@pytest.fixture(scope="module")
def world():
    torch.manual_seed(2)
    w = torch.randn(N, K, device="cuda").mul_(0.1).to(torch.bfloat16)
    x = torch.randn(STEPS, B, K, device="cuda").to(torch.bfloat16)
    ex = example()
    tokens, old = ex.rollout(q.Int4Head(w), w, q.HeadSelect("cuda"), q.Sampler("cuda"), q.LogProbs("cuda"), x, T, seed=3)
    return ex, w, x, tokens, old


def bf16_logits(w, x):
    return example().logits_of(w, x).double()


def test_rollout(world):
    """A token's log probability is that of the logits it was drawn from: those of the 4-bit head, the 64 best made exact."""
    ex, w, x, tokens, old = world
    assert tokens.shape == (B, STEPS) and (tokens >= 0).all() and (old <= 0).all()
    head, select = q.Int4Head(w), q.HeadSelect("cuda")
    for s in range(STEPS):
        logits = head(x[s])
        select(logits, w, x[s], 64)
        lp = torch.log_softmax(logits.double() / T, 1).gather(1, tokens[:, s].long().view(-1, 1))[:, 0]
        assert torch.allclose(old[:, s].double(), lp, atol=1e-4)


def test_policy_update(world):
    """dw = sum over rows of dlogits x: the gradient at the logits is the formula's, rounded to bf16 (half a step, 2^-8), and the product
    that takes it to w sums bf16 values in fp32 and rounds once more."""
    ex, w, x, tokens, old = world
    advantages = torch.linspace(-1, 1, B, device="cuda")
    leaf = w.clone().requires_grad_()
    out = ex.policy_update(q.PolicyLoss("cuda", clip=(0.2, 0.2), kl=0.1), leaf, x, tokens, old, advantages, T, ref=old)
    z = (bf16_logits(w, x) / T).requires_grad_()
    lp = torch.log_softmax(z, 2).gather(2, tokens.long().unsqueeze(2))[..., 0]
    r, a = torch.exp(lp - old.double()), advantages.double().view(-1, 1)
    d = old.double() - lp
    loss = (0.1 * (torch.exp(d) - 1 - d) - torch.minimum(r * a, r.clamp(0.8, 1.2) * a)).mean()
    assert abs(float(out.loss.detach()) - float(loss.detach())) < 1e-5 and torch.allclose(out.ratio.double(), r, rtol=1e-4)
    (gz,) = torch.autograd.grad(loss, z)
    g = (gz / T).reshape(-1, N)
    states = x.transpose(0, 1).reshape(-1, K).double()
    want, size = g.t() @ states, g.abs().t() @ states.abs()
    off = (leaf.grad.double() - want).abs()
    assert (off <= size * (2.0 ** -8 + 2.0 ** -10) + want.abs() * 2.0 ** -8 + 1e-12).all()


def test_preference_update(world):
    ex, w, x, tokens, old = world
    order = torch.tensor([4, 1, 0, 5, 2, 3], device="cuda")
    leaf = w.clone().requires_grad_()
    out = ex.preference_update(q.PreferenceLoss("cuda", beta=0.2), leaf, x, tokens, order)
    z = bf16_logits(w, x)[order].requires_grad_()
    s = torch.log_softmax(z, 2).gather(2, tokens[order].long().unsqueeze(2))[..., 0].sum(1)
    u = 0.2 * (s[0::2] - s[1::2])
    loss = -torch.nn.functional.logsigmoid(u).mean()
    assert abs(float(out.loss.detach()) - float(loss.detach())) < 1e-5 and torch.allclose(out.margins.double(), u, atol=1e-5) and torch.allclose(out.logprobs.double(), s, atol=1e-4)
    (gz,) = torch.autograd.grad(loss, z)
    g, states = gz.reshape(-1, N), x.transpose(0, 1)[order].reshape(-1, K).double()
    want, size = g.t() @ states, g.abs().t() @ states.abs()
    off = (leaf.grad.double() - want).abs()
    assert (off <= size * (2.0 ** -8 + 2.0 ** -10) + want.abs() * 2.0 ** -8 + 1e-12).all()


def test_example_runs(monkeypatch, capsys):
    monkeypatch.setattr("sys.argv", ["learn_from_samples.py", "--vocab", "4000", "--hidden", "128", "--batch", "4", "--steps", "3"])
    example().main()
    printed = capsys.readouterr().out
    assert "policy: loss" in printed and "preference: loss" in printed and "nan" not in printed
