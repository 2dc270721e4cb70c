"""The example's path (examples/logprobs.py): the 8-bit head, the exact candidates, the sampler, the log probabilities, and the
scoring of a text, each against the others and against torch on the same logits."""
import importlib.util
from pathlib import Path

import pytest
import torch

import qwen_warp_amd as q

pytestmark = pytest.mark.gpu


def example():
    spec = importlib.util.spec_from_file_location("example_logprobs", Path(__file__).resolve().parents[1] / "examples" / "logprobs.py")
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


@pytest.fixture(scope="module")
def world():
    torch.manual_seed(1)
    w = torch.randn(32000, 512, device="cuda").mul_(0.05).to(torch.bfloat16)
    return example(), w, q.Fp8Head(w)


@pytest.mark.parametrize("B", [1, 5, 16])
def test_decode_step(world, B):
    ex, w, head = world
    likely = torch.randint(0, 32000, (B,), device="cuda")
    rows = [q.RowSpec(temperature=0.0 if b % 2 else 0.7, top_p=0.9, seed=3, position=5, row_key=b) for b in range(B)]
    tokens, out, logits = ex.decode_step(head, w, q.HeadSelect("cuda"), q.Sampler("cuda"), q.LogProbs("cuda"), ex.states_before(w, likely, 20.0), rows, 5)
    lp = torch.log_softmax(logits.double(), 1)
    assert torch.allclose(out.logprobs.double(), lp.gather(1, tokens.long().view(-1, 1))[:, 0], atol=1e-4)
    assert torch.allclose(out.entropy.double(), -(lp.exp() * lp).sum(1), atol=1e-3)
    assert torch.equal(out.top_ids[:, 0].long(), logits.argmax(1))
    greedy = torch.arange(B, device="cuda") % 2 == 1
    assert (out.ranks[greedy] == 0).all() and (out.ranks >= 0).all()
    for b in range(B):
        if int(out.ranks[b]) < 5:
            assert int(out.top_ids[b, int(out.ranks[b])]) == int(tokens[b]) and float(out.top_logprobs[b, int(out.ranks[b])]) == float(out.logprobs[b])


@pytest.mark.parametrize("n", [2, 20, 70, 300])
def test_score_text(world, n):
    ex, w, head = world
    ids = torch.randint(0, 32000, (n,), device="cuda", dtype=torch.int32)
    x = ex.states_before(w, torch.cat([ids[1:], ids[:1]]), 20.0)
    lp, h = ex.score_text(head, x, ids)
    want = torch.log_softmax(head(x[:-1]).double(), 1)
    assert lp.shape == (n - 1,)
    assert torch.allclose(lp.double(), want.gather(1, ids[1:].long().view(-1, 1))[:, 0], atol=1e-4)
    assert torch.allclose(h.double(), -(want.exp() * want).sum(1), atol=1e-3)


def test_verify_rows(world):
    """A verify call's tokens (-1 behind the accepted ones) with the target logits it verified."""
    _, w, head = world
    B, K, V = 3, 4, 32000
    target = head(torch.randn(B * (K + 1), 512, device="cuda").mul_(3).to(torch.bfloat16)).view(B, K + 1, V)
    idmap = torch.arange(V, dtype=torch.int32, device="cuda")
    sampler = q.Sampler("cuda")
    drafts = target[:, :K].argmax(2).to(torch.int32)
    drafts[1, 2] = int(target[1, 2].argmin())
    probs = torch.zeros(B, K, V, device="cuda").scatter_(2, drafts.long().unsqueeze(2), 1.0)
    seqs = [q.RowSpec(temperature=0.0, seed=1, position=0, row_key=b) for b in range(B)]
    tokens, n = sampler.verify(target, probs, sampler.verify_map(idmap, V), drafts, seqs)
    out = q.LogProbs("cuda")(target, tokens, top=2)
    assert n.tolist() == [5, 3, 5]
    taken = tokens >= 0
    assert (out.ranks[taken] == 0).all() and (out.ranks[~taken] == -1).all() and (out.logprobs[~taken] == 0).all()
    assert torch.equal(out.logprobs[taken], out.top_logprobs[..., 0][taken])
