"""The 4-bit head and the losses over sampled tokens for timing and comparison: single calls over the ranges that `draw` spans.

Kinds of case:
  int4        Int4Head: logits of T hidden states from a head's weights in 4 bits, a scale and a zero point for each `group` of
              them.  codes: the weights come as codes with scales (and zeros), as a quantised checkpoint holds them.
  policy      PolicyLoss: the clipped policy loss of R drawn tokens with a KL term.  grad: with the gradient at the logits,
              through autograd or (one_call) as one call.  pad: the rows lie in a buffer of V + pad columns.
  preference  PreferenceLoss: the paired log ratios of P chosen and P rejected texts of `length` tokens on average, packed.

The plain forms are elementary torch operations in 32 bits, with the sums over a row and what follows from them (a few numbers a
row) in 64; `exact` is the definition in 64 bits."""
import math

import torch

own = False

DEV = "cuda"
V = 248320  # the vocabulary
K = 5120    # the hidden size of the full head


def listed():
    return [
        # a small drafter's head, ragged both ways, from a checkpoint's symmetric codes
        dict(name="int4_ragged_3", kind="int4", T=3, N=8191, K=1000, group=32, codes=True, zeros=False, out="float32", pad=0),
        # a drafter's reduced vocabulary for five sequences
        dict(name="int4_draft_5", kind="int4", T=5, N=64000, K=K, group=64, codes=True, zeros=True, out="float32", pad=0),
        # one user's step
        dict(name="int4_1", kind="int4", T=1, N=V, K=K, group=128, codes=False, zeros=True, out="float32", pad=0),
        # the nine verify rows of four speculating sequences
        dict(name="int4_36", kind="int4", T=36, N=V, K=K, group=128, codes=False, zeros=True, out="float32", pad=0),
        # a server's batch of verify rows, the logits in bf16
        dict(name="int4_200", kind="int4", T=200, N=V, K=K, group=128, codes=False, zeros=True, out="bfloat16", pad=0),
        # a few tokens of a small vocabulary, odd sizes, masks: latency
        dict(name="policy_24", kind="policy", R=24, V=32001, dtype="bfloat16", kl=True, temperature=False, weights=True, masks=True, pad=7, grad=True, one_call=True),
        # an evaluation without a gradient, at the tokens' temperatures
        dict(name="policy_eval_256", kind="policy", R=256, V=V, dtype="float32", kl=True, temperature=True, weights=False, masks=False, pad=0, grad=False, one_call=False),
        # a micro-batch in fp32
        dict(name="policy_512_fp32", kind="policy", R=512, V=V, dtype="float32", kl=True, temperature=True, weights=False, masks=False, pad=0, grad=True, one_call=False),
        # a step's tokens at the full vocabulary: the largest
        dict(name="policy_2048", kind="policy", R=2048, V=V, dtype="bfloat16", kl=False, temperature=False, weights=True, masks=False, pad=0, grad=True, one_call=False),
        # a pair of short answers, length-normalised
        dict(name="pref_1", kind="preference", P=1, length=20, V=32001, dtype="float32", ref=False, average=True, smoothing=0.1, weights=False, pad=0, grad=True, one_call=True),
        # eight pairs scored without a gradient
        dict(name="pref_eval_8", kind="preference", P=8, length=40, V=V, dtype="bfloat16", ref=True, average=False, smoothing=0.0, weights=True, pad=0, grad=False, one_call=False),
        # pairs of answers of some hundred tokens
        dict(name="pref_6", kind="preference", P=6, length=100, V=V, dtype="bfloat16", ref=True, average=False, smoothing=0.0, weights=False, pad=0, grad=True, one_call=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("int4", "int4", "policy", "policy", "preference"))
    if kind == "int4":
        n, k = rng.choice((V, _log(rng, 1000, V))), rng.choice((K, _log(rng, 200, K), 32 * (2 * rng.randint(3, 79) + 1)))
        codes = rng.random() < 0.5
        return dict(kind=kind, T=rng.choice((1, rng.randint(1, 16), _log(rng, 1, 200))), N=n, K=k, group=rng.choice((32, 64, 128, 128)), codes=codes,
                    zeros=not codes or rng.random() < 0.5, out=rng.choice(("float32", "float32", "bfloat16")), pad=rng.choice((0, 0, 8, 3)))
    vocab, dtype = rng.choice((V, _log(rng, 500, V))), rng.choice(("float32", "bfloat16"))
    common = dict(V=vocab, dtype=dtype, weights=rng.random() < 0.5, pad=rng.choice((0, 0, 8, rng.randint(1, 40))), grad=rng.random() < 0.75, one_call=rng.random() < 0.3)
    rows = min(4096, 2048 * V // (vocab * (2 if dtype == "float32" else 1)))
    if kind == "policy":
        return dict(kind=kind, R=_log(rng, 1, rows), kl=rng.random() < 0.5, temperature=rng.random() < 0.4, masks=rng.random() < 0.25, **common)
    pairs = _log(rng, 1, 32)
    return dict(kind=kind, P=pairs, length=_log(rng, 2, max(4, rows // (3 * pairs))), ref=rng.random() < 0.7, average=rng.random() < 0.3,
                smoothing=rng.choice((0.0, 0.0, 0.1)), **common)


# ------------------------------------------------------------------------------------------ inputs
CLIP_LOW, CLIP_HIGH, KL = 0.2, 0.28, 0.05
BETA, MARGIN = 0.1, 0.25


def _logits(g, c, R):
    """[R, V] logits of a model that knows a few continuations, N(0, 2.5) with 32 ids a row 8 higher, and a token drawn from each
    (one in sixteen rows has none: a prompt's or padding).  masks: rows of few allowed tokens, one without any."""
    n, dtype = c["V"], getattr(torch, c["dtype"])
    x = torch.empty(R, n + c["pad"], device=DEV, dtype=dtype)[:, :n]
    x.copy_(torch.randn(R, n, device=DEV, generator=g, dtype=torch.float32).mul_(2.5))
    ids = torch.randint(0, n, (R, 32), device=DEV, generator=g)
    x.scatter_add_(1, ids, torch.full(ids.shape, 8.0, device=DEV, dtype=dtype))
    if c.get("masks"):
        few = torch.rand(R, n, device=DEV, generator=g) * n < 12  # about twelve allowed tokens a row
        row = torch.arange(R, device=DEV).view(R, 1)
        x.masked_fill_(~few & (row % 3 == 1), -math.inf)
        x.masked_fill_(~few & (row % 3 == 2), torch.finfo(dtype).min)
        x.masked_fill_(row == R - 1, -math.inf)  # the mask leaves nothing
    tokens = (x.float() / 1.25 + torch.empty(R, n, device=DEV).exponential_(generator=g).log_().neg_()).argmax(1)
    return x, torch.where(torch.rand(R, device=DEV, generator=g) < 1 / 16, -1, tokens).to(torch.int32)


def _logprobs_about(x, tokens, temperature):
    """log p of the tokens to some 1e-5, as a rollout recorded them."""
    z = x.float() if temperature is None else x.float() / temperature.view(-1, 1)
    lp = z.log_softmax(1).gather(1, tokens.clamp(min=0).long().view(-1, 1))[:, 0]
    return torch.where(lp.isfinite(), lp, -20.0)


def _weights(g, c):
    """[N, K] weights whose rows differ in size, a few columns larger than the rest, as a trained head's."""
    w = torch.randn(c["N"], c["K"], device=DEV, generator=g, dtype=torch.bfloat16)
    w *= (0.01 + 0.02 * torch.rand(c["N"], 1, device=DEV, generator=g)).to(torch.bfloat16)
    w[:, ::97] *= 3.0
    return w


def _quantised(g, c):
    """Codes [N, K], scales and zero points [N, groups] of a checkpoint."""
    groups = -(-c["K"] // c["group"])
    codes = torch.randn(c["N"], c["K"], device=DEV, generator=g, dtype=torch.bfloat16).mul_(2.7).add_(8).clamp_(0, 15).to(torch.uint8)
    scales = (0.002 + 0.004 * torch.rand(c["N"], groups, device=DEV, generator=g)).to(torch.float16 if c["zeros"] else torch.bfloat16)
    return codes, scales, torch.randint(6, 11, (c["N"], groups), device=DEV, generator=g, dtype=torch.uint8) if c["zeros"] else None


def _groups(x, group):
    return torch.nn.functional.pad(x, (0, -x.shape[1] % group)).view(x.shape[0], -1, group)


def _quantise(w, group):
    """Weights as codes 0 .. 15 with a scale in bf16 and a zero point for each group of a row: the range [lo, hi] of the group's
    values and 0 in fifteen steps."""
    parts = []
    for p in w.split(1 << 15):
        b = _groups(p, group).float()
        lo, hi = b.amin(2).clamp(max=0), b.amax(2).clamp(min=0)
        s = ((hi - lo) / 15).to(torch.bfloat16)
        d = torch.where(s > 0, s, 1.0).float()
        z = torch.round(-lo / d).clamp(0, 15)
        q = (torch.round(b / d.unsqueeze(2)) + z.unsqueeze(2)).clamp(0, 15)
        parts.append((q.flatten(1)[:, :p.shape[1]].to(torch.uint8), s, z.to(torch.uint8)))
    return tuple(torch.cat(p) for p in zip(*parts))


def prepare(case, seed):
    c = case
    g = torch.Generator(device=DEV).manual_seed(seed)
    s = dict(case=c)
    if c["kind"] == "int4":
        if c["codes"]:
            codes, scales, zeros = _quantised(g, c)
        else:
            w = _weights(g, c)
        s["x"] = torch.empty(c["T"], c["K"] + c["pad"], device=DEV, dtype=torch.bfloat16)[:, :c["K"]]
        s["x"].copy_(torch.randn(c["T"], c["K"], device=DEV, generator=g))
        s["x"][:, ::61] *= 4.0
        if own:
            import qwen_warp_amd as q
            s["op"] = q.Int4Head.from_codes(codes, scales, zeros, group=c["group"]) if c["codes"] else q.Int4Head(w, group=c["group"])
        else:
            s["codes"], s["scales"], s["zeros"] = (codes, scales, zeros) if c["codes"] else _quantise(w, c["group"])
        return s
    if c["kind"] == "policy":
        R = c["R"]
        s["logits"], s["tokens"] = _logits(g, c, R)
        s["temperature"] = 0.5 + torch.rand(R, device=DEV, generator=g) if c["temperature"] else None
        lp = _logprobs_about(s["logits"], s["tokens"], s["temperature"])
        # the policy has moved since the rollout; log ratios keep some distance from the two borders of the clip, where a rounding decides
        drift = 0.2 * torch.randn(R, device=DEV, generator=g)
        for border in (math.log(1 - CLIP_LOW), math.log(1 + CLIP_HIGH)):
            drift = torch.where((drift - border).abs() < 2e-3, border - 4e-3, drift)
        s["old"] = lp - drift
        s["ref"] = lp + 0.3 * torch.randn(R, device=DEV, generator=g) if c["kl"] else None
        s["advantages"] = torch.randn(R, device=DEV, generator=g) + 0.5
        s["weights"] = (0.5 + torch.rand(R, device=DEV, generator=g)) / R if c["weights"] else None
    else:
        P = c["P"]
        shares = (0.5 + torch.rand(2 * P, device=DEV, generator=g)).cumsum(0)
        starts = torch.zeros(2 * P + 1, device=DEV, dtype=torch.int64)
        starts[1:] = (shares / shares[-1] * (2 * P * c["length"])).round()
        lengths = starts.diff()
        s["logits"], s["tokens"] = _logits(g, c, 2 * P * c["length"])
        s["starts"] = starts.to(torch.int32)
        total = torch.zeros(2 * P, device=DEV).index_add_(0, torch.repeat_interleave(torch.arange(2 * P, device=DEV), lengths),
                                                          torch.where(s["tokens"] >= 0, _logprobs_about(s["logits"], s["tokens"], None), 0.0))
        s["ref"] = (total / lengths.clamp(min=1) if c["average"] else total) + 2.0 * torch.randn(2 * P, device=DEV, generator=g) if c["ref"] else None
        s["weights"] = (0.5 + torch.rand(P, device=DEV, generator=g)) / P if c["weights"] else None
    s["logits"].requires_grad_(c["grad"] and not c["one_call"])
    if own:
        import qwen_warp_amd as q
        s["op"] = (q.PolicyLoss(DEV, clip=(CLIP_LOW, CLIP_HIGH), kl=KL if c["kl"] else 0.0) if c["kind"] == "policy" else
                   q.PreferenceLoss(DEV, beta=BETA, margin=MARGIN, smoothing=c["smoothing"], average=c["average"]))
    return s


# ------------------------------------------------------------------------------------------ one pass
def _plain_head(s):
    c = s["case"]
    zeros = 8.0 if s["zeros"] is None else s["zeros"].float().unsqueeze(2)
    w = (_groups(s["codes"].float(), c["group"]) - zeros) * s["scales"].float().unsqueeze(2)
    return (s["x"].float() @ w.flatten(1)[:, :c["K"]].t()).to(getattr(torch, c["out"]))


def _token_logprobs(x, tokens, temperature):
    """(log p of the tokens in 64 bits, whether each row has a token that its mask allows, e^(z - max), its sum): NaN as -inf."""
    z = x.float() if temperature is None else x.float() / temperature.view(-1, 1)
    z = torch.where(z.isnan(), -math.inf, z)
    m = z.amax(1, keepdim=True)
    z = z - torch.where(m == -math.inf, 0.0, m)
    e = torch.exp(z)
    total = e.sum(1, dtype=torch.float64)
    lp = z.gather(1, tokens.clamp(min=0).long().view(-1, 1))[:, 0].double() - torch.log(total)
    lp = torch.where(total > 0, lp, -math.inf)
    return lp, (tokens >= 0) & (lp > -math.inf), e, total


def _gradient(x, tokens, temperature, coef, e, total):
    """coef ([j = token] - p_j) / temperature in the logits' type."""
    coef = torch.where(coef == 0, 0.0, coef if temperature is None else coef / temperature)
    g = e * (-coef / torch.where(total > 0, total, 1.0)).float().view(-1, 1)
    return g.scatter_add_(1, tokens.clamp(min=0).long().view(-1, 1), coef.float().view(-1, 1)).to(x.dtype)


def _plain_policy(s):
    c, tokens = s["case"], s["tokens"]
    x = s["logits"].detach()
    lp, used, e, total = _token_logprobs(x, tokens, s["temperature"])
    w = s["weights"].double() if c["weights"] else 1.0 / (tokens >= 0).sum().clamp(min=1)
    a = s["advantages"].double()
    ratio = torch.exp(torch.where(used, lp - s["old"], 0.0))
    straight, clipped = ratio * a, ratio.clamp(1 - CLIP_LOW, 1 + CLIP_HIGH) * a
    d = torch.where(used, s["ref"] - lp, 0.0) if c["kl"] else torch.zeros_like(lp)
    kl = torch.expm1(d) - d
    loss = torch.where(used, w * (KL * kl - torch.minimum(straight, clipped)), 0.0).sum()
    out = [loss.float(), torch.where(tokens >= 0, lp, 0.0).float(), ratio.float(), kl.float() if c["kl"] else None]
    if c["grad"]:
        coef = torch.where(used, w * (torch.where(straight <= clipped, -straight, 0.0) - KL * torch.expm1(d)), 0.0)
        out.append(_gradient(x, tokens, s["temperature"], coef, e, total))
    return out


def _plain_preference(s):
    c, tokens = s["case"], s["tokens"]
    x = s["logits"].detach()
    lp, used, e, total = _token_logprobs(x, tokens, None)
    of = torch.bucketize(torch.arange(len(tokens), device=DEV, dtype=torch.int32), s["starts"], right=True) - 1  # each row's sequence
    sums = torch.zeros(2 * c["P"], device=DEV, dtype=torch.float64).index_add_(0, of, torch.where(used, lp, 0.0))
    count = torch.zeros_like(sums).index_add_(0, of, (tokens >= 0).double()).clamp(min=1) if c["average"] else torch.ones_like(sums)
    sums = sums / count
    above = sums - s["ref"] if c["ref"] else sums
    u = BETA * (above[0::2] - above[1::2]) - MARGIN
    w = s["weights"].double() if c["weights"] else 1.0 / c["P"]
    eps = c["smoothing"]
    softplus = torch.clamp(-u, min=0) + torch.log1p(torch.exp(-u.abs()))  # -log sigmoid(u)
    loss = (w * (softplus + eps * u)).sum()
    out = [loss.float(), sums.float(), u.float(), torch.where(tokens >= 0, lp, 0.0).float()]
    if c["grad"]:
        slope = BETA * w * (eps - 1 / (1 + torch.exp(u)))
        coef = torch.where(used, (torch.stack((slope, -slope), 1).view(-1) / count)[of], 0.0)
        out.append(_gradient(x, tokens, None, coef, e, total))
    return out


def run(state):
    s, c = state, state["case"]
    if c["kind"] == "int4":
        return s["op"](s["x"], dtype=getattr(torch, c["out"])) if own else _plain_head(s)
    if not own:
        return _plain_policy(s) if c["kind"] == "policy" else _plain_preference(s)
    if c["kind"] == "policy":
        args, more = (s["logits"], s["tokens"], s["old"], s["advantages"]), dict(ref_logprobs=s["ref"], weights=s["weights"], temperature=s["temperature"])
    else:
        args, more = (s["logits"], s["tokens"], s["starts"]), dict(ref=s["ref"], weights=s["weights"])
    grad = []
    if c["grad"] and c["one_call"]:
        o, g = s["op"].value_and_grad(*args, **more)
        grad = [g]
    else:
        o = s["op"](*args, **more)
        if c["grad"]:
            grad = list(torch.autograd.grad(o.loss, s["logits"]))
    if c["kind"] == "policy":
        return [o.loss.detach(), o.logprobs, o.ratio, o.kl] + grad
    return [o.loss.detach(), o.logprobs, o.margins, o.token_logprobs] + grad


def _mean_rows(c):
    return c["R"] if c["kind"] == "policy" else 2 * c["P"] * c["length"]


def work(case):
    c = case
    if c["kind"] == "int4":
        T, N, k = c["T"], c["N"], c["K"]
        scale = 3 if c["zeros"] else 2  # bytes of a group's scale and, rounded up, its zero point
        return dict(bytes=N * k // 2 + N * -(-k // c["group"]) * scale + 2 * T * k + T * N * (4 if c["out"] == "float32" else 2), flops=2 * T * N * k)
    R, n, size = _mean_rows(c), c["V"], 4 if c["dtype"] == "float32" else 2
    # an element: difference, scale, exponential, sum; for the gradient an exponential again, a product, a difference
    return dict(bytes=R * (n * size * (2 if c["grad"] else 1) + 24), flops=R * n * (9 if c["grad"] else 5))


# ------------------------------------------------------------------------------------------ in 64 bits
def _exact_weights(c, g):
    """The values that the weights stand for, float64, in parts of rows."""
    group = c["group"]
    if c["codes"]:
        codes, scales, zeros = _quantised(g, c)
        for i in range(0, c["N"], 1 << 15):
            part = slice(i, i + (1 << 15))
            z = zeros[part].double() if c["zeros"] else torch.full(scales[part].shape, 8.0, device=DEV, dtype=torch.float64)
            spread = lambda t: t.repeat_interleave(group, 1)[:, :c["K"]]  # noqa: E731
            yield spread(scales[part].double()) * (codes[part].double() - spread(z))
        return
    for p in _weights(g, c).split(1 << 15):
        b = _groups(p.double(), group)
        hi, lo = b.amax(2, keepdim=True).clamp(min=0), b.amin(2, keepdim=True).clamp(max=0)
        step = ((hi - lo) / 15).to(torch.float32).to(torch.bfloat16).double()
        q = torch.round(torch.where(step > 0, b / step, 0.0))
        low = -torch.round(torch.where(step > 0, -lo / step, 0.0)).clamp(0, 15)  # the least code stands for this many steps
        yield (torch.minimum(torch.maximum(q, low), low + 15) * step).flatten(1)[:, :c["K"]]


def _exact_rows(x, T):
    """log p of rows x in 64 bits."""
    x = x.double().nan_to_num(nan=-math.inf, posinf=math.inf, neginf=-math.inf)
    lp = torch.log_softmax(x if T is None else x / T.double().view(-1, 1), 1)
    return torch.where(lp.isnan(), -math.inf, lp)


def exact(case, seed):
    c = case
    s = prepare(c, seed)
    if c["kind"] == "int4":
        x = s["x"].double()
        s.clear()
        return torch.cat([x @ w.t().contiguous() for w in _exact_weights(c, torch.Generator(device=DEV).manual_seed(seed))], 1)
    x, tokens = s["logits"].detach(), s["tokens"].long()
    R, T = len(tokens), s.get("temperature")
    rows = max(1, (1 << 27) // c["V"])  # a part of 1 GB in 64 bits
    parts = [slice(i, i + rows) for i in range(0, R, rows)]
    at = tokens.clamp(min=0).view(-1, 1)
    lp = torch.cat([_exact_rows(x[p], None if T is None else T[p]).gather(1, at[p])[:, 0] for p in parts])
    has = tokens >= 0
    used = has & (lp > -math.inf)
    safe = torch.where(used, lp, 0.0).requires_grad_()
    if c["kind"] == "policy":
        w = s["weights"].double() if c["weights"] else torch.full_like(lp, 1 / max(1, int(has.sum())))
        ratio = torch.where(used, (safe - s["old"].double()).exp(), 1.0)
        a = s["advantages"].double()
        inside = torch.where(a >= 0, ratio <= 1 + CLIP_HIGH, ratio >= 1 - CLIP_LOW)
        gain = torch.where(inside, ratio, torch.where(a >= 0, 1 + CLIP_HIGH, 1 - CLIP_LOW)) * a
        d = torch.where(used, s["ref"].double() - safe, 0.0) if c["kl"] else torch.zeros_like(lp)
        kl = d.exp() - 1 - d
        loss = (used * w * (KL * kl - gain)).sum()
        out = [loss, torch.where(has, lp, 0.0), ratio, kl if c["kl"] else None]
    else:
        ends = s["starts"].tolist()
        sums = torch.stack([(safe[i:j] * used[i:j]).sum() / (max(1, int(has[i:j].sum())) if c["average"] else 1) for i, j in zip(ends, ends[1:])])
        above = (sums - (s["ref"].double() if c["ref"] else 0.0)).view(-1, 2)
        u = BETA * (above[:, 0] - above[:, 1]) - MARGIN
        w = s["weights"].double() if c["weights"] else torch.full_like(u, 1 / c["P"])
        log_sigma = torch.nn.functional.logsigmoid
        loss = -(w * ((1 - c["smoothing"]) * log_sigma(u) + c["smoothing"] * log_sigma(-u))).sum()
        out = [loss, sums, u, torch.where(has, lp, 0.0)]
    if c["grad"]:
        (slope,) = torch.autograd.grad(loss, safe, retain_graph=True)
        grad = torch.empty(R, c["V"], device=DEV, dtype=torch.float32 if c["dtype"] == "bfloat16" else torch.float64)
        for p in parts:
            k = torch.where(used[p], slope[p], 0.0).view(-1, 1)
            row = _exact_rows(x[p], None if T is None else T[p]).exp().mul_(-k).scatter_add_(1, at[p], k)
            grad[p] = row if T is None else row / T[p].double().view(-1, 1)
        out.append(grad)
    return [v if v is None else v.detach() for v in out]
