"""The log-probability operators and the 8-bit head for timing and comparison: single calls over the ranges that `draw` spans.

Kinds of case:
  logprobs  LogProbs: per row of logits the log probabilities and ranks of given tokens, the entropy and the best
            alternatives.  M given tokens a row (M = 0: one, without an axis of its own); pad: the rows lie in a buffer of
            V + pad columns; masks: rows with few allowed tokens (-inf and the type's lowest value elsewhere), one with none.
  head      Fp8Head: logits of T hidden states from the head's weights in 8 bits (a power-of-two scale per 128 weights).
  score     Fp8Head.score: the log probabilities of the tokens that followed T hidden states, and the entropies, without
            the logits in memory.

The plain forms are elementary torch operations in 32 bits; `exact` is the definition in 64 bits."""
import math

import torch

own = False

DEV = "cuda"
V = 248320  # the vocabulary
K = 5120    # the hidden size of the full head
BLOCK = 128


def listed():
    return [
        # one user's step: a token's log probability and five alternatives
        dict(name="lp_1", kind="logprobs", R=1, V=V, dtype="bfloat16", M=0, top=5, temperature=False, pad=0, masks=False, tail=False),
        # the nine verify rows of four speculating sequences at their temperatures; -1 behind the accepted tokens
        dict(name="lp_verify_36", kind="logprobs", R=36, V=V, dtype="float32", M=0, top=20, temperature=True, pad=0, masks=False, tail=True),
        # a choice among sixteen labels in an odd vocabulary, under masks that leave some rows little or nothing
        dict(name="lp_labels_24", kind="logprobs", R=24, V=32001, dtype="bfloat16", M=16, top=8, temperature=False, pad=7, masks=True, tail=False),
        # a server's full batch with twenty alternatives
        dict(name="lp_256", kind="logprobs", R=256, V=V, dtype="float32", M=0, top=20, temperature=False, pad=0, masks=False, tail=False),
        # the positions of a long prompt
        dict(name="lp_prompt_2048", kind="logprobs", R=2048, V=V, dtype="bfloat16", M=0, top=5, temperature=False, pad=0, masks=False, tail=False),
        # a small drafter's head, ragged both ways: the smallest product
        dict(name="head_ragged_3", kind="head", T=3, N=8191, K=1000, out="float32", pad=0),
        # a drafter's reduced vocabulary for five sequences
        dict(name="head_draft_5", kind="head", T=5, N=64000, K=K, out="float32", pad=0),
        # one user's step: bound by the weights' bytes
        dict(name="head_1", kind="head", T=1, N=V, K=K, out="float32", pad=0),
        # the verify rows of a few sequences
        dict(name="head_16", kind="head", T=16, N=V, K=K, out="float32", pad=0),
        # a server's batch of verify rows, the logits in bf16
        dict(name="head_300", kind="head", T=300, N=V, K=K, out="bfloat16", pad=0),
        # a short text scored by a small model
        dict(name="score_77", kind="score", T=77, N=32001, K=1280, temperature=True, pad=8),
        # a long prompt scored at the full head: the largest call
        dict(name="score_2048", kind="score", T=2048, N=V, K=K, temperature=False, pad=0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("logprobs", "logprobs", "head", "head", "score"))
    if kind == "logprobs":
        vocab = rng.choice((V, _log(rng, 500, V)))
        M = rng.choice((0, 0, 1, rng.randint(2, 16)))
        dtype = rng.choice(("float32", "bfloat16"))
        most = min(2048, 2048 * V // (vocab * max(M, 1) * (2 if dtype == "float32" else 1)))
        return dict(kind=kind, R=_log(rng, 1, most), V=vocab, dtype=dtype, M=M, top=rng.choice((0, 1, 5, 20, rng.randint(1, 64))), temperature=rng.random() < 0.4,
                    pad=rng.choice((0, 0, 8, rng.randint(1, 40))), masks=rng.random() < 0.25, tail=M == 0 and rng.random() < 0.3)
    N, hidden = rng.choice((V, _log(rng, 1000, V))), rng.choice((K, _log(rng, 200, K), 128 * (2 * rng.randint(1, 19) + 1)))
    T = rng.choice((rng.randint(1, 16), _log(rng, 1, 2048)))
    if kind == "head":
        return dict(kind=kind, T=min(T, 1024), N=N, K=hidden, out=rng.choice(("float32", "float32", "bfloat16")), pad=rng.choice((0, 0, 8, 3)))
    return dict(kind=kind, T=T, N=N, K=hidden, temperature=rng.random() < 0.4, pad=rng.choice((0, 0, 8, 3)))


# ------------------------------------------------------------------------------------------ inputs
def _logits(g, c):
    """[R, V] logits of a model that knows a few continuations: N(0, 2.5) with 32 ids a row 8 higher; masked rows last."""
    R, n, dtype = c["R"], c["V"], getattr(torch, c["dtype"])
    x = torch.empty(R, n + c["pad"], device=DEV, dtype=dtype)[:, :n]
    x.copy_(torch.randn(R, n, device=DEV, generator=g, dtype=torch.float32).mul_(2.5))
    ids = torch.randint(0, n, (R, 32), device=DEV, generator=g)
    x.scatter_add_(1, ids, torch.full(ids.shape, 8.0, device=DEV, dtype=dtype))
    if c["masks"]:
        few = torch.rand(R, n, device=DEV, generator=g) * n < 12  # about twelve allowed tokens a row
        row = torch.arange(R, device=DEV).view(R, 1)
        x.masked_fill_(~few & (row % 3 == 1), -math.inf)
        x.masked_fill_(~few & (row % 3 == 2), torch.finfo(dtype).min)
        x.masked_fill_(row == R - 1, -math.inf)  # the mask leaves nothing
    return x


def _weights(g, c):
    """[N, K] weights whose rows differ in size, a few columns larger than the rest, as a trained head's."""
    N, k = c["N"], c["K"]
    w = torch.randn(N, k, device=DEV, generator=g, dtype=torch.bfloat16)
    w *= (0.01 + 0.02 * torch.rand(N, 1, device=DEV, generator=g)).to(torch.bfloat16)
    w[:, ::97] *= 3.0
    return w


def _scales(x):
    """The exponent e of each row's blocks of 128 (the last one shorter): the least whole number with max|x| <= 448 * 2^e, >= -127."""
    rows, k = x.shape
    a = torch.nn.functional.pad(x.abs(), (0, -k % BLOCK)).view(rows, -1, BLOCK).amax(2).float()
    m, p = torch.frexp(a)  # a = m * 2^p with m in [0.5, 1); 448 = 0.875 * 2^9
    return torch.where(a > 0, p - 9 + (m > 0.875), -127).clamp_(min=-127)


def _scaled(x, e):
    """x * 2^e in 32 bits, e one exponent in [-127, 127] for each block of 128 (-127 stands for 0: blocks of zeros)."""
    return x.float() * ((e.int() + 127) << 23).view(torch.float32).repeat_interleave(BLOCK, 1)[:, :x.shape[1]]


def _eight_bits(x, e):
    """x / 2^e of its block, rounded to the nearest e4m3 value (ties to even)."""
    return _scaled(x, -e).to(torch.float8_e4m3fn)


def prepare(case, seed):
    c = case
    g = torch.Generator(device=DEV).manual_seed(seed)
    if c["kind"] == "logprobs":
        R, n = c["R"], c["V"]
        s = dict(case=c, logits=_logits(g, c))
        # half of the given tokens are likely ones, as a sampler's, the others anything
        pick = (s["logits"].float() / 2 + torch.empty(R, n, device=DEV).exponential_(generator=g).log_().neg_()).argmax(1)
        tokens = torch.randint(0, n, (R, max(c["M"], 1)), device=DEV, generator=g)
        tokens[::2, 0] = pick[::2]
        if c["tail"]:
            tokens[torch.arange(R, device=DEV) % 9 >= 1 + torch.randint(0, 9, (R,), device=DEV, generator=g)] = -1
        s["tokens"] = tokens.to(torch.int32) if c["M"] else tokens[:, 0].to(torch.int32)
        if own:
            import qwen_warp_amd as q
            s["op"] = q.LogProbs(DEV)
    else:
        T, N, k = c["T"], c["N"], c["K"]
        w = _weights(g, c)
        s = dict(case=c, x=torch.empty(T, k + c["pad"], device=DEV, dtype=torch.bfloat16)[:, :k])
        tokens = torch.randint(0, N, (T,), device=DEV, generator=g)
        x = torch.randn(T, k, device=DEV, generator=g)
        x[:, ::61] *= 4.0
        if c["kind"] == "score":  # hidden states that lean to the token that follows, as a trained model's
            x[::2] += 8.0 * w[tokens[::2]].float() / w[tokens[::2]].float().square().sum(1, keepdim=True)
            s["tokens"] = tokens.to(torch.int32)
        s["x"].copy_(x)
        if own:
            import qwen_warp_amd as q
            s["op"] = q.Fp8Head(w)
        else:
            e = _scales(w)
            s["w8"], s["we"] = _eight_bits(w, e), e.to(torch.int16)
    n = c["R"] if c["kind"] == "logprobs" else c["T"]
    s["temperature"] = 0.5 + torch.rand(n, device=DEV, generator=g) if c.get("temperature") else None
    return s


# ------------------------------------------------------------------------------------------ one pass
def _log_softmax_parts(x, temperature):
    """(z, max, sum) of x / temperature in 32 bits, NaN as -inf, a row without a finite value summed to 0."""
    z = x.float() if temperature is None else x.float() / temperature.view(-1, 1)
    z = torch.where(z.isnan(), -math.inf, z)
    m = z.amax(1, keepdim=True)
    m = torch.where(m == -math.inf, 0.0, m)
    z = z - m
    return z, m, torch.exp(z).sum(1, keepdim=True)


def _entropy(z, total):
    e = torch.exp(z)
    h = torch.log(total) - torch.where(e > 0, e * z, 0.0).sum(1, keepdim=True) / total
    return torch.where(total > 0, h, 0.0)[:, 0]


def _plain_logprobs(x, tokens, top, temperature):
    R, n = x.shape
    given = tokens.view(R, -1).long()
    skipped = (given < 0) | (given >= n)
    given = given.clamp(0, n - 1)
    z, _, total = _log_softmax_parts(x, temperature)
    lse = torch.log(total)
    logprobs = torch.where(skipped, 0.0, torch.where(total > 0, z.gather(1, given) - lse, -math.inf))
    clean = torch.where(x.isnan(), -math.inf, x.float())
    mine, at = clean.gather(1, given).unsqueeze(2), torch.arange(n, device=x.device)
    before = ((clean.unsqueeze(1) > mine) | ((clean.unsqueeze(1) == mine) & (at < given.unsqueeze(2)))).sum(2)
    ranks = torch.where(skipped, -1, before).to(torch.int32)
    # the order of (value, lowest index first) as whole numbers: the bits of a float, those of negative ones turned over
    bits = (clean + 0.0).view(torch.int32).long()
    keys = torch.where(bits < 0, -(bits & 0x7FFFFFFF), bits) * 2**32 + (2**31 - at)
    ids = torch.topk(keys, min(top, n), 1).indices if top else keys[:, :0].long()
    alive = clean.gather(1, ids) > -math.inf
    top_logprobs = torch.where(alive, z.gather(1, ids) - lse, -math.inf)
    ids = torch.where(alive, ids, -1).to(torch.int32)
    return logprobs.view(tokens.shape), ranks.view(tokens.shape), _entropy(z, total), ids, top_logprobs


def _plain_head(s):
    x = s["x"]
    e = _scales(x)
    return _scaled(_eight_bits(x, e), e) @ _scaled(s["w8"], s["we"]).t()


def run(state):
    s, c = state, state["case"]
    if c["kind"] == "logprobs":
        if own:
            o = s["op"](s["logits"], s["tokens"], top=c["top"], temperature=s["temperature"])
            return o.logprobs, o.ranks, o.entropy, o.top_ids, o.top_logprobs
        return _plain_logprobs(s["logits"], s["tokens"], c["top"], s["temperature"])
    if c["kind"] == "head":
        dtype = getattr(torch, c["out"])
        return s["op"](s["x"], dtype=dtype) if own else _plain_head(s).to(dtype)
    if own:
        return s["op"].score(s["x"], s["tokens"], temperature=s["temperature"])
    z, _, total = _log_softmax_parts(_plain_head(s), s["temperature"])
    return z.gather(1, s["tokens"].long().view(-1, 1))[:, 0] - torch.log(total)[:, 0], _entropy(z, total)


def work(case):
    c = case
    if c["kind"] == "logprobs":
        R, n, M = c["R"], c["V"], max(c["M"], 1)
        size = 4 if c["dtype"] == "float32" else 2
        # an element: difference, scale, exponential, two sums; a comparison for each given token and one for the alternatives
        return dict(bytes=R * (n * size + 12 * M + 4 + 8 * c["top"] + (4 if c["temperature"] else 0)), flops=R * n * (6 + M + (1 if c["top"] else 0)))
    T, N, k = c["T"], c["N"], c["K"]
    read = N * k + N * -(-k // BLOCK) + 2 * T * k
    if c["kind"] == "head":
        return dict(bytes=read + T * N * (4 if c["out"] == "float32" else 2), flops=2 * T * N * k)
    return dict(bytes=read + 12 * T + (4 * T if c["temperature"] else 0), flops=T * N * (2 * k + 6))


# ------------------------------------------------------------------------------------------ in 64 bits
def _exact_rows(x, temperature):
    """log p of every token of rows x (float64) and the rows' entropies."""
    if temperature is not None:
        x = x / temperature.double().view(-1, 1)
    x = x.nan_to_num(nan=-math.inf, posinf=math.inf, neginf=-math.inf)
    lp = x - x.logsumexp(1, keepdim=True)
    lp = lp.nan_to_num(nan=-math.inf, posinf=math.inf, neginf=-math.inf)  # a row of nothing: -inf - -inf
    return lp, -(lp.exp() * lp.clamp(min=-1e30)).sum(1)


def _power(e):
    """2^e in 64 bits, without a rounding (pow's would move ties)."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _exact_values(x):
    """The values that x stands for in 8 bits, from its definition: blocks of 128 divided by a power of two, three bits after the leading one."""
    rows, k = x.shape
    b = torch.nn.functional.pad(x.double(), (0, -k % BLOCK)).view(rows, -1, BLOCK)
    most = b.abs().amax(2, keepdim=True)
    e = torch.where(most > 0, torch.ceil(torch.log2(most.clamp(min=1e-300) / 448)), 0.0)
    e = torch.where(448 * _power(e - 1) >= most, e - 1, e)
    e = torch.where(448 * _power(e) < most, e + 1, e)
    b = b * _power(-e)
    step = _power(torch.floor(torch.log2(b.abs().clamp(min=2.0 ** -6))) - 3)
    return (torch.round(b / step) * step * _power(e)).view(rows, -1)[:, :k]


def exact(case, seed):
    c = case
    if c["kind"] == "logprobs":
        s = prepare(c, seed)
        x, given = s["logits"], s["tokens"].view(c["R"], -1).long()
        lp, h = _exact_rows(x.double(), s["temperature"])
        of_given = torch.where(given < 0, 0.0, lp.gather(1, given.clamp(min=0)))
        best = torch.topk(lp, min(c["top"], c["V"]), 1).values if c["top"] else lp[:, :0]
        return of_given.view(s["tokens"].shape), None, h, None, best
    g = torch.Generator(device=DEV).manual_seed(seed)
    w = _weights(g, c)
    s = prepare(c, seed)
    x, parts = _exact_values(s["x"]), 8
    n = -(-c["N"] // parts)
    y = torch.cat([x @ _exact_values(w[i * n:(i + 1) * n]).t().contiguous() for i in range(parts) if i * n < c["N"]], 1)
    if c["kind"] == "head":
        return y
    lp, h = _exact_rows(y, s["temperature"])
    return lp.gather(1, s["tokens"].long().view(-1, 1))[:, 0], h
