"""Tokens drawn behind a head held in 4 bits, and two updates of the head from them: a clipped policy loss on the drawn tokens, and
a preference loss on pairs of the drawn texts.

    python examples/learn_from_samples.py [--vocab 32000 --hidden 1024 --batch 8 --steps 16]

Weights and hidden states are random; the "model" is the head alone (hidden states do not depend on the drawn tokens)."""
import argparse
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))
import qwen_warp_amd as qws  # noqa: E402


def rollout(head, w, select, sampler, logprobs, x, temperature, seed):
    """Texts for hidden states x [steps, B, K]: (tokens int32 [B, steps], their log probabilities at the temperature).  Each step's logits come
    from the 4-bit head, the best candidates' are made exact from the bf16 weights, a token a row is drawn, and its log
    probability is read from the same logits."""
    tokens, old = [], []
    for step, states in enumerate(x):
        logits = head(states)
        select(logits, w, states, 64)
        rows = [qws.RowSpec(temperature=temperature, seed=seed, position=step, row_key=b) for b in range(len(states))]
        t = sampler.sample(logits, rows)
        at = torch.full((len(states),), temperature, device=states.device)
        tokens.append(t)
        old.append(logprobs(logits, t, temperature=at).logprobs)
    return torch.stack(tokens, 1).contiguous(), torch.stack(old, 1).contiguous()


def logits_of(w, x):
    """[B, steps, N] logits of hidden states x [steps, B, K] (one product of two matrices)."""
    return (x.transpose(0, 1).reshape(-1, x.shape[2]) @ w.t()).view(x.shape[1], x.shape[0], -1)


def policy_update(loss_fn, w, x, tokens, old, advantages, temperature, ref=None):
    """The policy loss of texts under the head w (a leaf that requires a gradient); the gradient goes to w.grad."""
    logits = logits_of(w, x)
    at = torch.full(tokens.shape, temperature, device=x.device)
    out = loss_fn(logits, tokens, old, advantages.view(-1, 1).expand_as(old).contiguous(), ref_logprobs=ref, temperature=at)
    out.loss.backward()
    return out


def preference_update(loss_fn, w, x, tokens, order, ref=None):
    """The preference loss of pairs of texts, rows order[0], order[1] of tokens the first pair (the better text first), and so on."""
    logits = logits_of(w, x)[order]
    out = loss_fn(logits, tokens[order].contiguous(), ref=ref)
    out.loss.backward()
    return out


def main():
    p = argparse.ArgumentParser()
    p.add_argument("--vocab", type=int, default=32000)
    p.add_argument("--hidden", type=int, default=1024)
    p.add_argument("--batch", type=int, default=8)
    p.add_argument("--steps", type=int, default=16)
    a = p.parse_args()
    torch.manual_seed(0)
    w = torch.randn(a.vocab, a.hidden, device="cuda", dtype=torch.bfloat16).mul_(0.05)
    x = torch.randn(a.steps, a.batch, a.hidden, device="cuda", dtype=torch.bfloat16)
    tokens, old = rollout(qws.Int4Head(w), w, qws.HeadSelect("cuda"), qws.Sampler("cuda"), qws.LogProbs("cuda"), x, 0.8, seed=7)
    reward = -(tokens.float() / a.vocab).mean(1)  # any score of a text: here low ids
    advantages = (reward - reward.mean()) / (reward.std() + 1e-6)
    w.requires_grad_()
    out = policy_update(qws.PolicyLoss("cuda", clip=(0.2, 0.28), kl=0.02), w, x, tokens, old, advantages, 0.8, ref=old)
    print(f"policy: loss {float(out.loss.detach()):.4f}, mean ratio {float(out.ratio.mean()):.3f}, mean KL term {float(out.kl.mean()):.4f}, |dw| {float(w.grad.float().norm()):.4f}")
    w.grad = None
    order = reward.argsort(descending=True)[:a.batch // 2 * 2].view(2, -1).t().reshape(-1)  # a better text with a worse one
    out = preference_update(qws.PreferenceLoss("cuda", beta=0.1), w, x, tokens, order)
    print(f"preference: loss {float(out.loss.detach()):.4f}, margins {[round(m, 3) for m in out.margins.tolist()]}, |dw| {float(w.grad.float().norm()):.4f}")


if __name__ == "__main__":
    main()
