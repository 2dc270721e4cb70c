"""A decode step whose requests ask for log probabilities, behind a head held in 8 bits, and the scoring of a text.

    python examples/logprobs.py [--vocab 248320 --hidden 5120 --batch 8 --text 512]

Weights and hidden states are random (hidden states lean to the token that follows, as a trained model's do)."""
import argparse
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))
import qwen_warp_amd as qws  # noqa: E402


def decode_step(head, w, select, sampler, logprobs, x, rows, top):
    """One step of a batch: hidden states x [B, K] -> (tokens, LogProbsResult, logits).  The 8-bit head gives the logits, the
    best candidates' are made exact from the bf16 weights, a token is drawn, and its log probability, rank and the row's
    entropy and `top` alternatives are read from the same logits."""
    logits = head(x)
    select(logits, w, x, 64)
    tokens = sampler.sample(logits, rows)
    return tokens, logprobs(logits, tokens, top=top), logits


def score_text(head, x, ids):
    """Hidden states x [n, K] of a text's positions and its ids [n] -> (log p of each id behind the first, entropies)."""
    return head.score(x[:-1], ids[1:])


def states_before(w, ids, gain=8.0):
    """Random hidden states [n, K] whose next token, ids [n], is likely."""
    rows = w[ids.long()].float()
    return (torch.randn(rows.shape, device=w.device) + gain * rows / rows.square().sum(1, keepdim=True)).to(torch.bfloat16)


def main():
    p = argparse.ArgumentParser()
    p.add_argument("--vocab", type=int, default=248320)
    p.add_argument("--hidden", type=int, default=5120)
    p.add_argument("--batch", type=int, default=8)
    p.add_argument("--text", type=int, default=512)
    a = p.parse_args()
    torch.manual_seed(0)
    w = torch.randn(a.vocab, a.hidden, device="cuda", dtype=torch.bfloat16).mul_(0.02)
    head, select, sampler, logprobs = qws.Fp8Head(w), qws.HeadSelect("cuda"), qws.Sampler("cuda"), qws.LogProbs("cuda")
    rows = [qws.RowSpec(temperature=0.8, top_p=0.95, seed=7, position=0, row_key=b) for b in range(a.batch)]
    likely = torch.randint(0, a.vocab, (a.batch,), device="cuda")
    tokens, out, _ = decode_step(head, w, select, sampler, logprobs, states_before(w, likely, 16.0), rows, top=5)
    for b in range(a.batch):
        best = ", ".join(f"{i}: {lp:.3f}" for i, lp in zip(out.top_ids[b].tolist(), out.top_logprobs[b].tolist()))
        print(f"row {b}: token {int(tokens[b])} log p {float(out.logprobs[b]):.3f} rank {int(out.ranks[b])} entropy {float(out.entropy[b]):.3f} | {best}")
    ids = torch.randint(0, a.vocab, (a.text,), device="cuda", dtype=torch.int32)
    x = states_before(w, torch.cat([ids[1:], ids[:1]]), 16.0)
    lp, h = score_text(head, x, ids)
    print(f"text of {a.text} tokens: mean log p {float(lp.mean()):.3f}, perplexity {float(torch.exp(-lp.mean())):.2f}, mean entropy {float(h.mean()):.3f}")


if __name__ == "__main__":
    main()
