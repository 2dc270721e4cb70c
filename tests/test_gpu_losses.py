"""PolicyLoss and PreferenceLoss (qws_policy_loss, qws_preference_loss, qws_loss_grad through the Python wrappers) against the 64-bit
definitions (oracle/losses.py).

Bounds.  U = 2^-24, a rounding to fp32.  A term of a row's sum is 2^d with d = c (x - m): c's rounding, the multiply-add's and the
exponential's put it off by (2 |d| + 4) U of itself at most (with those of the reference it is relative to), the additions by one U
each: a lane adds V / 256 terms, then some twenty joins.  Over the row the |d| weigh as its probabilities do: sum p |d| <=
log2 V + 1.  So ln s, and with it log p, is within delta = (V / 256 + 2 log2 V + 40) U; log p itself is then rounded once.
A ratio, a KL term, a slope move by their derivatives times delta.  A gradient's element is slope / T ([j = token] - p_j): p_j is off by
(2 |d_j| + 8) U of itself and delta, products and the sum at the token by a few U of the slope; then it is rounded to
the logits' type.  What lies below 2^-126 may be 0."""
import numpy as np
import pytest
import torch
import torch.utils.checkpoint

import qwen_warp_amd as q
from oracle import losses as O

pytestmark = pytest.mark.gpu
INF, NAN = float("inf"), float("nan")
U = 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}


def delta(V):
    return (V / 256 + 2 * np.log2(V) + 40) * U


def close(got, want, tol, what):
    got, want = got.detach().double().cpu().numpy(), np.asarray(want, np.float64)
    tol = np.broadcast_to(tol, want.shape)
    fine = np.isfinite(want)
    assert got.shape == want.shape and (np.isnan(got) == np.isnan(want)).all() and (got[~fine & ~np.isnan(want)] == want[~fine & ~np.isnan(want)]).all(), what
    off = np.abs(got[fine] - want[fine])
    assert (off <= tol[fine]).all(), f"{what}: off by {off.max()}, {(off / np.maximum(tol[fine], 1e-300)).max()} of the bound"


def check_gradient(grad, want, slope_tol, dtype, V, T=None):
    """want: the oracle's answer; slope_tol [R]: how far the slopes may be off."""
    R = len(want["slope"])
    T = np.ones(R) if T is None else np.where(np.asarray(T) > 0, T, 1.0)
    g = grad.double().cpu().numpy()
    for r in range(R):
        slope, lp = abs(want["slope"][r]) / T[r], want["table"][r]
        d = np.minimum(np.abs(lp) * 1.4427 + 20, 200)  # |d_j|: below its log p's size in log2 units and the row's ln s
        p = np.exp(lp)
        tol = slope * p * ((2 * d + 12) * U + delta(V)) + 8 * U * slope * p + slope_tol[r] / T[r] * p
        at = np.zeros(V)
        at[want["tokens"][r]] = 1 if slope else 0
        tol = tol + at * (8 * U * slope + slope_tol[r] / T[r])
        tol = tol * (1 + HALF[dtype]) + HALF[dtype] * np.abs(want["grad"][r]) + 2.0 ** -126 * (1 + slope)
        off = np.abs(g[r] - want["grad"][r])
        assert (off <= tol).all(), f"row {r}: {off.max()} at {int(np.argmax(off - tol))}, bound {tol[int(np.argmax(off - tol))]}"


def logits_of(R, V, dtype, seed, pad=0, masks=False):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(R, V, generator=g) * 2.5
    x.scatter_add_(1, torch.randint(0, V, (R, 3), generator=g), torch.full((R, 3), 6.0))
    if masks:
        few = torch.rand(R, V, generator=g) * V < 5
        row = torch.arange(R).view(R, 1)
        x = torch.where(~few & (row % 4 == 1), torch.tensor(-INF), x)
        x = torch.where(~few & (row % 4 == 2), torch.tensor(torch.finfo(dtype).min), x)
        x = torch.where(row % 8 == 7, torch.tensor(-INF), x)
    buf = torch.full((R, V + pad), NAN, dtype=dtype, device="cuda")[:, pad // 2:pad // 2 + V]
    buf.copy_(x)
    x = buf.float().cpu()
    tokens = torch.randint(0, V, (R,), generator=g)
    tokens[::2] = (x / 1.5 - torch.log(-torch.log(torch.rand(R, V, generator=g).clamp(1e-9, 1 - 1e-7)))).nan_to_num(nan=-INF).argmax(1)[::2]
    return buf, x, tokens.to(torch.int32)


def policy_inputs(x, tokens, seed, temperature, clip=(0.2, 0.28)):
    rng = np.random.default_rng(seed)
    R, V = x.shape
    T = rng.uniform(0.5, 2.0, R).astype(np.float32) if temperature else None
    lp = np.array([O.log_softmax(r, 1.0 if T is None else T[i])[int(t) if 0 <= t < V else 0] for i, (r, t) in enumerate(zip(x.numpy(), tokens))])
    lp = np.where(np.isfinite(lp), lp, -20.0)
    drift = rng.normal(size=R) * 0.25
    for border in (np.log(1 - clip[0]), np.log(1 + clip[1])):  # away from the borders, where a rounding decides
        drift = np.where(np.abs(drift - border) < 0.01, border + 0.02, drift)
    old = (lp - drift).astype(np.float32)
    return T, old, (rng.normal(size=R) + 0.3).astype(np.float32), (lp + rng.normal(size=R) * 0.4).astype(np.float32), rng.uniform(0, 2, R).astype(np.float32)


def dev(a):
    return None if a is None else torch.from_numpy(np.ascontiguousarray(a)).cuda()


def policy_tolerances(want, adv, kl, ref, w, V):
    dl = delta(V) + 2 * U  # with the rounding of what came in 64 bits
    r, k = want["ratio"], want["kl"]
    ed = np.abs(np.expm1(np.minimum(np.asarray(ref, np.float64) - np.where(np.isfinite(want["logprobs"]), want["logprobs"], 0), 80))) if ref is not None else 0 * r
    slope = w * (r * np.abs(adv) + kl * (ed + 1)) * (dl + 4 * U)
    return dl, ed, slope


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("R,V,pad,temperature,kl,weights,masks", [
    (1, 1, 0, False, 0.0, False, False), (1, 2, 1, True, 0.1, True, False), (3, 7, 0, False, 0.05, False, False), (5, 255, 3, True, 0.0, True, False),
    (17, 1000, 8, False, 0.1, True, True), (64, 4096, 0, True, 0.05, False, False), (9, 32001, 7, False, 0.05, True, True), (70, 3001, 1, True, 0.1, False, True),
    (3, 248320, 0, False, 0.05, True, False), (2, 100003, 5, True, 0.1, False, True), (700, 513, 2, False, 0.05, True, True), (2100, 64, 0, False, 0.0, False, False),
    (130, 100003, 5, True, 0.1, False, True), (20, 100003, 1, False, 0.05, False, True), (6, 65432, 0, False, 0.05, True, False), (600, 9001, 3, False, 0.0, True, False)])
def test_policy(dtype, R, V, pad, temperature, kl, weights, masks):
    logits, x, tokens = logits_of(R, V, dtype, R + V, pad, masks)
    T, old, adv, ref, w = policy_inputs(x, tokens, R, temperature)
    if R > 4:
        tokens[1], tokens[4] = -1, V
        old[1] = adv[4] = NAN  # rows left out
    ref, w = ref if kl else None, w if weights else None
    clip, kl32 = (float(np.float32(0.2)), float(np.float32(0.28))), float(np.float32(kl))
    want = O.policy(x.numpy(), tokens.tolist(), old, adv, clip, kl32, ref, w, T)
    want["tokens"] = np.clip(tokens.numpy(), 0, V - 1)
    has = (tokens >= 0).numpy() & (tokens < V).numpy()
    wt = np.full(R, 1.0 / max(1, has.sum())) if w is None else w.astype(np.float64)
    adv_used = np.where(has, adv, 0.0)
    dl, ed, slope_tol = policy_tolerances(want, adv_used, kl32, ref, wt, V)
    fn = q.PolicyLoss("cuda", clip=(0.2, 0.28), kl=kl)
    args = (tokens.cuda(), dev(old), dev(adv))
    more = dict(ref_logprobs=dev(ref), weights=dev(w), temperature=dev(T))
    out, grad = fn.value_and_grad(logits, *args, **more)
    lpw = np.where(np.isfinite(want["logprobs"]), want["logprobs"], 0)
    close(out.logprobs, want["logprobs"], dl + U * np.abs(lpw), "log p")
    close(out.ratio, want["ratio"], want["ratio"] * (dl + 2 * U), "ratio")
    if kl:
        close(out.kl, want["kl"], ed * dl + dl * dl + 2 * U * want["kl"] + 1e-15, "kl")
    else:
        assert out.kl is None
    terms = wt * (want["ratio"] * np.abs(adv_used) + kl32 * (ed + want["kl"]))
    close(out.loss, want["loss"], terms.sum() * dl + 2 * U * abs(want["loss"]) + 1e-30, "loss")
    assert grad.dtype == dtype and grad.shape == logits.shape and grad.is_contiguous()
    check_gradient(grad, want, slope_tol, dtype, V, T)
    zero = want["slope"] == 0
    assert (grad[torch.from_numpy(zero).cuda()] == 0).all()
    # through autograd: the same numbers
    leaf = logits.detach().requires_grad_()
    again = fn(leaf, *args, **more)
    again.loss.backward()
    assert torch.equal(again.loss, out.loss) and torch.equal(leaf.grad, grad)
    for a, b in zip(again[1:], out[1:]):
        assert (a is None and b is None) or (torch.equal(a, b) and not a.requires_grad)
    # without a gradient the sums may be taken in another order: the same bounds
    plain = fn(logits, *args, **more)
    assert not plain.loss.requires_grad
    close(plain.logprobs, want["logprobs"], dl + U * np.abs(lpw), "log p")
    close(plain.ratio, want["ratio"], want["ratio"] * (dl + 2 * U), "ratio")
    close(plain.loss, want["loss"], terms.sum() * dl + 2 * U * abs(want["loss"]) + 1e-30, "loss")


def pairs(seed, P, most):
    """Ascending starts with empty sequences among them, rows before the first and behind the last."""
    rng = np.random.default_rng(seed)
    n = rng.integers(0, most + 1, 2 * P)
    if P > 1:
        n[1] = 0
    starts = np.concatenate([[0], n.cumsum()]) + (2 if P > 1 else 0)
    return rng, starts.astype(np.int32), int(starts[-1]) + (3 if P > 1 else 0)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("P,most,V,pad,average,smoothing,ref,weights,masks", [
    (1, 3, 5, 0, False, 0.0, True, False, False), (1, 40, 32001, 7, True, 0.1, False, False, True), (3, 9, 1000, 1, False, 0.0, True, True, True),
    (8, 20, 3001, 3, True, 0.0, True, False, False), (2, 3, 248320, 0, False, 0.2, True, True, False), (70, 4, 255, 2, False, 0.1, False, True, True),
    (400, 5, 33, 0, True, 0.0, True, False, False)])
def test_preference(dtype, P, most, V, pad, average, smoothing, ref, weights, masks):
    rng, starts, R = pairs(P + V, P, most)
    R = max(R, 1)
    logits, x, tokens = logits_of(R, V, dtype, R + V, pad, masks)
    tokens[::5] = -1
    if R > 6:
        tokens[6] = V + 3
    w = rng.uniform(0, 2, P).astype(np.float32) if weights else None
    base = O.preference(x.numpy(), tokens.tolist(), starts, average=average)["logprobs"]
    rf = (base + rng.normal(size=2 * P) * 4).astype(np.float32) if ref else None
    f32 = lambda v: float(np.float32(v))  # noqa: E731
    want = O.preference(x.numpy(), tokens.tolist(), starts, f32(0.1), f32(0.25), f32(smoothing), average, rf, w)
    want["tokens"] = np.clip(tokens.numpy(), 0, V - 1)
    fn = q.PreferenceLoss("cuda", beta=0.1, margin=0.25, smoothing=smoothing, average=average)
    args, more = (tokens.cuda(), dev(starts)), dict(ref=dev(rf), weights=dev(w))
    out, grad = fn.value_and_grad(logits, *args, **more)
    dl = delta(V) + 2 * U
    n = np.diff(starts)
    lpw = np.where(np.isfinite(want["token_logprobs"]), want["token_logprobs"], 0)
    close(out.token_logprobs, want["token_logprobs"], dl + U * np.abs(lpw), "token log p")
    seq_tol = dl * (1 if average else n)
    close(out.logprobs, want["logprobs"], seq_tol + 2 * U * np.abs(want["logprobs"]), "sums")
    pair_tol = 0.1 * (np.broadcast_to(seq_tol, 2 * P)[0::2] + np.broadcast_to(seq_tol, 2 * P)[1::2])
    close(out.margins, want["margins"], pair_tol + 2 * U * np.abs(want["margins"]), "margins")
    wt = np.full(P, 1.0 / P) if w is None else w.astype(np.float64)
    close(out.loss, want["loss"], (wt * pair_tol).sum() + 2 * U * abs(want["loss"]), "loss")
    of = np.searchsorted(starts, np.arange(R), side="right") - 1
    inside = (of >= 0) & (of < 2 * P)
    # a slope is beta w (eps - sigma(-u)) / count: sigma moves by a quarter of u's error
    slope_tol = np.where(inside, 0.1 * (wt * (pair_tol / 4 + 4 * U))[np.clip(of, 0, 2 * P - 1) // 2], 0.0)
    check_gradient(grad, want, slope_tol, dtype, V)
    assert (grad[torch.from_numpy(want["slope"] == 0).cuda()] == 0).all()
    leaf = logits.detach().requires_grad_()
    again = fn(leaf, *args, **more)
    again.loss.backward()
    assert torch.equal(again.loss, out.loss) and torch.equal(leaf.grad, grad)
    assert all(torch.equal(a, b) and not a.requires_grad for a, b in zip(again[1:], out[1:]))
    plain = fn(logits, *args, **more)
    assert torch.equal(plain.loss, out.loss) and torch.equal(plain.margins, out.margins)


def test_sequences_of_a_batch():
    """Without starts, [2 P, L, V] logits are a sequence for each leading index."""
    P, L, V = 3, 7, 500
    logits, _, tokens = logits_of(2 * P * L, V, torch.float32, 1)
    fn = q.PreferenceLoss("cuda", beta=0.2)
    a, ga = fn.value_and_grad(logits, tokens.cuda(), torch.arange(0, 2 * P * L + 1, L, dtype=torch.int32, device="cuda"))
    b, gb = fn.value_and_grad(logits.view(2 * P, L, V), tokens.cuda().view(2 * P, L))
    assert torch.equal(a.loss, b.loss) and torch.equal(ga.view(2 * P, L, V), gb) and torch.equal(a.margins, b.margins)
    assert b.token_logprobs.shape == (2 * P, L)
    # the positions that predict, a slice at two strides
    x = logits.view(2 * P, L, V)
    cut, keep = x[:, :-1], x[:, :-1].contiguous()
    t = tokens.cuda().view(2 * P, L)[:, :-1].contiguous()
    a, ga = fn.value_and_grad(cut, t)
    b, gb = fn.value_and_grad(keep, t)
    assert torch.equal(a.loss, b.loss) and torch.equal(ga, gb)
    leaf = x.detach().requires_grad_()
    fn(leaf[:, :-1], t).loss.backward()
    assert torch.equal(leaf.grad[:, :-1], ga) and (leaf.grad[:, -1] == 0).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_special_logits(dtype):
    """Infinities, NaN in masked places, extreme values and temperatures: the definition's answers, in each row alone."""
    R, V = 12, 3000
    logits, x, tokens = logits_of(R, V, dtype, 3)
    low = torch.finfo(dtype).min
    t = tokens.tolist()
    other = [(k + 1) % V for k in t]
    logits[0] = -INF
    logits[1, t[1]] = -INF
    logits[2, other[2]], logits[2, (t[2] + 7) % V] = NAN, NAN
    logits[3, t[3]] = INF
    logits[4, t[4]], logits[4, other[4]] = INF, INF
    logits[5] = low
    logits[6] = -INF
    logits[6, t[6]] = low
    logits[7] += 30000
    logits[8] = NAN
    logits[9] = logits[9] * 1e30
    logits[10, t[10]] = NAN
    logits[11] = -1e9
    logits[11, t[11]] = -1e9
    T = np.ones(R, np.float32)
    T[7], T[9], T[2] = 0.5, NAN, 0.0
    x = logits.float().cpu().numpy()
    lp = np.array([O.log_softmax(r, T[i])[k] for i, (r, k) in enumerate(zip(x, t))])
    old = np.where(np.isfinite(lp), lp, -5.0).astype(np.float32) - 0.1
    adv = np.ones(R, np.float32)
    want = O.policy(x, t, old, adv, (float(np.float32(0.2)),) * 2, 0.0, None, None, T)
    want["tokens"] = tokens.numpy()
    out, grad = q.PolicyLoss("cuda").value_and_grad(logits, tokens.cuda(), dev(old), dev(adv), temperature=dev(T))
    dl, _, slope_tol = policy_tolerances(want, adv, 0.0, None, np.full(R, 1 / R), V)
    close(out.logprobs, want["logprobs"], dl + U * np.abs(np.where(np.isfinite(want["logprobs"]), want["logprobs"], 0)), "log p")
    close(out.loss, want["loss"], (want["ratio"] / R).sum() * dl + 2 * U * abs(want["loss"]), "loss")
    assert torch.isfinite(grad).all()
    check_gradient(grad, want, slope_tol, dtype, V, T)
    assert (grad[[0, 1, 8, 10]] == 0).all()


def test_not_a_number_stays():
    """NaN among what a used row brings: the loss is NaN, and that row's gradient; the other rows' are as without it."""
    logits, x, tokens = logits_of(6, 900, torch.float32, 5)
    _, old, adv, ref, w = policy_inputs(x, tokens, 5, False)
    fn = q.PolicyLoss("cuda", kl=0.1)
    _, good = fn.value_and_grad(logits, tokens.cuda(), dev(old), dev(adv), dev(ref), dev(w))
    for k in range(4):
        v = [a.copy() for a in (old, adv, ref, w)]
        v[k][2] = NAN
        out, grad = fn.value_and_grad(logits, tokens.cuda(), *(dev(a) for a in v))
        assert torch.isnan(out.loss) and torch.isnan(grad[2]).all()
        rest = [0, 1, 3, 4, 5]
        assert torch.equal(grad[rest], good[rest])
    starts = dev(np.array([0, 1, 2, 4, 6], np.int32))
    pl = q.PreferenceLoss("cuda")
    _, good = pl.value_and_grad(logits, tokens.cuda(), starts, weights=dev(np.ones(2, np.float32)))
    for kw in (dict(ref=dev(np.array([0, 0, NAN, 0], np.float32)), weights=dev(np.ones(2, np.float32))), dict(weights=dev(np.array([1, NAN], np.float32)))):
        out, grad = pl.value_and_grad(logits, tokens.cuda(), starts, **kw)
        assert torch.isnan(out.loss) and torch.isnan(grad[2:]).all() and torch.equal(grad[:2], good[:2])


def test_far_ratios():
    """Log ratios past e^80 count as 80; a clipped one has no gradient; old log probabilities of -inf or far off stay finite."""
    logits, x, tokens = logits_of(4, 100, torch.float32, 6)
    old = np.array([-500.0, -500.0, 500.0, -INF], np.float32)
    adv = np.array([1.0, -1.0, 1.0, 1.0], np.float32)
    want = O.policy(x.numpy(), tokens.tolist(), old, adv, (float(np.float32(0.2)),) * 2)
    out, grad = q.PolicyLoss("cuda").value_and_grad(logits, tokens.cuda(), dev(old), dev(adv))
    close(out.ratio, want["ratio"], 4 * U * want["ratio"] + 1e-30, "ratio")
    close(out.loss, want["loss"], 4 * U * abs(want["loss"]), "loss")
    assert (grad[0] == 0).all() and (grad[3] == 0).all() and torch.isfinite(grad).all() and grad[1].abs().max() > 1e30


@pytest.mark.parametrize("loss", ["policy", "preference"])
def test_upstream_gradients(loss):
    """A scaled loss, a loss used twice, logits that came from a product, rows shared by a broadcast."""
    R, V = 10, 1003
    logits, x, tokens = logits_of(R, V, torch.float32, 7)
    _, old, adv, _, _ = policy_inputs(x, tokens, 7, False)
    if loss == "policy":
        fn, args = q.PolicyLoss("cuda"), (tokens.cuda(), dev(old), dev(adv))
    else:
        fn, args = q.PreferenceLoss("cuda"), (tokens.cuda(), dev(np.array([0, 2, 5, 6, 10], np.int32)))
    _, g = fn.value_and_grad(logits, *args)
    leaf = logits.detach().requires_grad_()
    (4 * fn(leaf, *args).loss).backward()  # a power of two: exact
    assert torch.equal(leaf.grad, 4 * g)
    leaf.grad = None
    l = fn(leaf, *args).loss
    l.backward(retain_graph=True)
    l.backward()
    assert torch.equal(leaf.grad, 2 * g)
    first = torch.autograd.grad(fn(leaf, *args).loss, leaf)[0]
    l = fn(leaf, *args).loss
    a = torch.autograd.grad(l, leaf, retain_graph=True)[0]
    b = torch.autograd.grad(l * 0.5, leaf)[0]
    assert torch.equal(a, first) and torch.equal(a, g) and torch.equal(b, 0.5 * g)
    if loss == "policy":  # an upstream gradient that was named beforehand, met and missed (powers of two: exact)
        fn.upstream = 0.25
        l = fn(leaf, *args).loss
        assert torch.equal(torch.autograd.grad(l * 0.25, leaf, retain_graph=True)[0], 0.25 * g) and torch.equal(torch.autograd.grad(l, leaf)[0], g)
        assert torch.equal(torch.autograd.grad(fn(leaf, *args).loss, leaf)[0], g) and torch.equal(fn.value_and_grad(logits, *args)[1], g)
        fn.upstream = 0.0
        assert (torch.autograd.grad(fn(leaf, *args).loss * 0.0, leaf)[0] == 0).all() and torch.equal(torch.autograd.grad(fn(leaf, *args).loss, leaf)[0], g)
        fn.upstream = 1.0
    h = torch.randn(R, 32, device="cuda", requires_grad=True)
    w = torch.randn(V, 32, device="cuda", requires_grad=True)
    y = h @ w.t()
    (gh, gw, gy) = torch.autograd.grad(fn(y, *args).loss, (h, w, y))
    assert torch.allclose(gh, gy @ w, rtol=1e-4, atol=1e-6) and torch.allclose(gw, gy.t() @ h, rtol=1e-4, atol=1e-6)
    one = logits[:1].detach().clone().requires_grad_()
    _, gs = fn.value_and_grad(one.detach().expand(R, V), *args)
    fn(one.expand(R, V), *args).loss.backward()
    assert torch.allclose(one.grad[0], gs.sum(0), rtol=1e-5, atol=1e-7)
    with torch.no_grad():
        assert not fn(leaf, *args).loss.requires_grad
    changed = logits.detach().clone().requires_grad_()
    y = changed * 1.0
    l = fn(y, *args).loss
    y.mul_(2)
    with pytest.raises(RuntimeError):  # the logits were changed in place since
        l.backward()


def test_directional_differences():
    """The loss along a direction moves as the gradient says: fp32 logits, a step whose cubed term and the loss's rounding
    are bounded.  |l(x + h v) - l(x - h v) - 2 h g v| <= h^3 max|l'''| / 3 + 2 err(l), with |v| = 1 per row and l''' of a few units."""
    logits, x, tokens = logits_of(8, 400, torch.float32, 8)
    _, old, adv, ref, w = policy_inputs(x, tokens, 8, False)
    ratio = np.exp(np.array([O.log_softmax(r)[t] for r, t in zip(x.numpy(), tokens)]) - old)
    old = np.where(np.abs(np.log(ratio) - np.log(0.8)) + np.abs(np.log(ratio) - np.log(1.2)) > 0.43, old + np.log(ratio), old).astype(np.float32)  # inside the clip or at r = 1
    fn = q.PolicyLoss("cuda", kl=0.1)
    args = (tokens.cuda(), dev(old), dev(adv), dev(ref), dev(w))
    _, g = fn.value_and_grad(logits, *args)
    v = torch.randn(8, 400, device="cuda", generator=torch.Generator("cuda").manual_seed(1))
    v /= v.norm(dim=1, keepdim=True)
    h = 2.0 ** -7
    up, down = fn(logits + h * v, *args).loss.double(), fn(logits - h * v, *args).loss.double()
    size = float((dev(w) * (dev(adv).abs() * 2 + 1)).sum())
    assert abs(float(up - down) - 2 * h * float((g.double() * v.double()).sum())) <= h ** 3 * 8 * size + 4 * delta(400) * size


def test_no_rows_and_refusals():
    fn, pl = q.PolicyLoss("cuda"), q.PreferenceLoss("cuda")
    none = torch.empty(0, 50, device="cuda", requires_grad=True)
    i, f = torch.empty(0, dtype=torch.int32, device="cuda"), torch.empty(0, device="cuda")
    out = fn(none, i, f, f)
    out.loss.backward()
    assert float(out.loss.detach()) == 0 and none.grad.shape == (0, 50) and out.ratio.shape == (0,)
    out = pl(torch.randn(3, 50, device="cuda"), torch.zeros(3, dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda"))
    assert float(out.loss) == 0 and out.logprobs.shape == (0,) and out.margins.shape == (0,)
    out, g = pl.value_and_grad(torch.randn(3, 50, device="cuda"), torch.zeros(3, dtype=torch.int32, device="cuda"), torch.zeros(3, dtype=torch.int32, device="cuda"))
    assert abs(float(out.loss) - np.log(2)) < 1e-6 and (g == 0).all()  # a pair of empty texts
    x = torch.randn(4, 50, device="cuda")
    t, v = torch.zeros(4, dtype=torch.int32, device="cuda"), torch.zeros(4, device="cuda")
    out, g = fn.value_and_grad(x, t - 1, v, v)
    assert float(out.loss) == 0 and (g == 0).all() and (out.ratio == 1).all()  # no row with a token
    for bad in ((x.half(), t, v, v), (x.cpu(), t, v, v), (x[0], t, v, v), (x, t.long(), v, v), (x, t[:3], v, v), (x, t, v.double(), v), (x, t, v, v[:2]), (x, t, v.cpu(), v),
                (x.t().contiguous().t(), t, v, v), (x, t, v.clone().requires_grad_(), v), (x[:, :0], t, v, v), (x, t, None, v)):
        with pytest.raises(q.ValidationError):
            fn(*bad)
    for kw in (dict(ref_logprobs=v[:1]), dict(weights=v.double()), dict(temperature=t)):
        with pytest.raises(q.ValidationError):
            fn(x, t, v, v, **kw)
    s = torch.tensor([0, 2, 4], dtype=torch.int32, device="cuda")
    for bad in ((x, t, s.long()), (x, t, s[:2]), (x, t, s.cpu()), (x, t, None), (x.view(1, 4, 50), t.view(1, 4), None)):
        with pytest.raises(q.ValidationError):
            pl(*bad)
    for kw in (dict(ref=v[:1]), dict(weights=v)):
        with pytest.raises(q.ValidationError):
            pl(x, t, s, **kw)


def test_starts_out_of_order_or_range():
    """Nothing outside is read or written; rows of no sequence have no gradient."""
    logits, _, tokens = logits_of(10, 300, torch.float32, 9)
    for s in ([0, 7, 3, 9, 4], [-5, 2, 4, 1000, 2000], [100, 200, 300, 400, 500]):
        out, g = q.PreferenceLoss("cuda").value_and_grad(logits, tokens.cuda(), torch.tensor(s, dtype=torch.int32, device="cuda"))
        assert torch.isfinite(out.loss) and torch.isfinite(g).all()
    assert (g == 0).all()


def test_offsets_past_32_bits():
    """Logits and a gradient of more than 2^31 elements: the last rows as those of a call of their own."""
    R, V = 9000, 248320
    x = torch.zeros(R, V, dtype=torch.bfloat16, device="cuda")
    tail = torch.randn(20, V, device="cuda").to(torch.bfloat16)
    x[-20:] = tail
    tokens = torch.full((R,), -1, dtype=torch.int32, device="cuda")
    tokens[-20:] = torch.arange(20, device="cuda") * 1000
    zero, one = torch.full((R,), -12.0, device="cuda"), torch.ones(R, device="cuda")
    fn = q.PolicyLoss("cuda", clip=(1.0, 1e6))
    out, g = fn.value_and_grad(x, tokens, zero, one, weights=one)
    want, gw = fn.value_and_grad(tail, tokens[-20:], zero[-20:], one[-20:], weights=one[-20:])
    assert torch.allclose(out.logprobs[-20:], want.logprobs, atol=2 * delta(V)) and (g[:-20] == 0).all()
    assert torch.allclose(g[-20:].float(), gw.float(), rtol=2.0 ** -7, atol=1e-9)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("R", [2, 140])
def test_longest_rows(dtype, R):
    """V at its limit, and a value past it refused; the log probabilities against torch's in 64 bits."""
    V = 1 << 24 if R == 2 else 1 << 21
    x = torch.randn(R, V, device="cuda", generator=torch.Generator("cuda").manual_seed(R)).mul_(2).to(dtype)
    tokens = torch.arange(R, device="cuda", dtype=torch.int32) * 7 + V - 2000
    old, adv = torch.full((R,), -14.0, device="cuda"), torch.ones(R, device="cuda")
    fn = q.PolicyLoss("cuda", clip=(1.0, 1e6))
    out, g = fn.value_and_grad(x, tokens, old, adv)
    for r in (0, 1, R - 1):
        lp = torch.log_softmax(x[r].double(), 0)
        assert abs(float(out.logprobs[r]) - float(lp[int(tokens[r])])) <= delta(V) + U * 20
        p, slope = lp.exp(), -float(out.ratio[r]) / R
        want = -slope * p
        want[int(tokens[r])] += slope
        off = (g[r].double() - want).abs()
        # |d| of any logit here: below 40 log2 units
        assert (off <= (abs(slope) * p * (92 * U + 2 * delta(V)) + 8 * U * abs(slope) * (want.abs() == want.abs().max())) * (1 + HALF[dtype]) + HALF[dtype] * want.abs() + 1e-37).all()
    with pytest.raises(q.ValidationError):
        fn(torch.empty(1, 1, device="cuda").expand(1, (1 << 24) + 1).contiguous(), tokens[:1], old[:1], adv[:1])


def test_calls_repeat_and_streams():
    logits, x, tokens = logits_of(40, 9001, torch.bfloat16, 10, pad=3)
    _, old, adv, ref, w = policy_inputs(x, tokens, 10, False)
    fn = q.PolicyLoss("cuda", kl=0.1)
    args = (tokens.cuda(), dev(old), dev(adv), dev(ref), dev(w))
    out, grad = fn.value_and_grad(logits, *args)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    leaf = logits.detach().requires_grad_()
    with torch.cuda.stream(side):
        again = fn(leaf, *args)
        (g,) = torch.autograd.grad(again.loss, leaf)
    here, h = fn.value_and_grad(logits, *args)
    torch.cuda.synchronize()
    assert torch.equal(again.loss, out.loss) and torch.equal(g, grad) and torch.equal(h, grad) and torch.equal(here.ratio, out.ratio)


def test_graphs():
    """Captured calls replay on new inputs, two graphs between each other and eager calls; autograd is refused in one."""
    R, V = 12, 5000
    logits, x, tokens = logits_of(R, V, torch.float32, 11)
    _, old, adv, _, _ = policy_inputs(x, tokens, 11, False)
    args = (tokens.cuda(), dev(old), dev(adv))
    starts = dev(np.array([0, 3, 6, 8, 12], np.int32))
    fn, pl = q.PolicyLoss("cuda"), q.PreferenceLoss("cuda")
    eager_leaf = logits.detach().clone().requires_grad_()
    eager = fn(eager_leaf, *args).loss  # an eager graph of a leaf lives meanwhile
    fn.value_and_grad(logits, *args), pl.value_and_grad(logits, args[0], starts)
    torch.cuda.synchronize()
    a, b = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(a):
        oa, ga = fn.value_and_grad(logits, *args)
    with torch.cuda.graph(b):
        ob, gb = pl.value_and_grad(logits, args[0], starts)
    for refused in (lambda: fn(eager_leaf, *args), lambda: pl(eager_leaf * 1.0, args[0], starts)):
        with pytest.raises(q.ValidationError):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                refused()
    for seed in range(20, 24):
        logits.copy_(logits_of(R, V, torch.float32, seed)[0])
        a.replay()
        b.replay()
        wa, wga = fn.value_and_grad(logits, *args)
        wb, wgb = pl.value_and_grad(logits, args[0], starts)
        torch.cuda.synchronize()
        assert torch.equal(oa.loss, wa.loss) and torch.equal(ga, wga) and torch.equal(ob.loss, wb.loss) and torch.equal(gb, wgb)
    eager.backward()
    assert torch.isfinite(eager_leaf.grad).all()


@pytest.mark.parametrize("loss,R,V", [("policy", 6, 100003), ("policy", 20, 5000), ("policy", 130, 33003), ("preference", 6, 100003), ("preference", 60, 700)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_saved_tensor_hooks_and_checkpoints(loss, R, V, dtype):
    """The backward pass reads the logits that autograd hands it: copies in other strides whose original was overwritten, copies
    brought back from the host, logits that a checkpoint made anew.  Each equals the plain one, with and without a gradient
    that the forward pass wrote, at another upstream gradient (a power of two: exact) and in a second pass."""
    logits, x, tokens = logits_of(R, V, dtype, R + 1)
    _, old, adv, _, _ = policy_inputs(x, tokens, 13, False)
    if loss == "policy":
        fn, args = q.PolicyLoss("cuda"), (tokens.cuda(), dev(old), dev(adv))
    else:
        fn, args = q.PreferenceLoss("cuda"), (tokens.cuda(), dev(np.array([0, 2, R // 2, R - 1, R], np.int32)))
    _, g = fn.value_and_grad(logits, *args)
    _, g2 = fn.value_and_grad(logits * 2, *args)  # of the logits that the model below makes

    def padded(t):
        buf = torch.full((R, V + 3), NAN, dtype=dtype, device="cuda")[:, 1:V + 1]
        return buf.copy_(t)

    leaf = logits.detach().requires_grad_()
    for pack, unpack in ((torch.clone, lambda t: t), (torch.clone, padded), (torch.clone, lambda t: t.t().contiguous().t())):
        with torch.autograd.graph.saved_tensors_hooks(pack, unpack):
            y = leaf * 1.0
            l = fn(y, *args).loss
        y.detach().fill_(NAN)
        (a,) = torch.autograd.grad(4 * l, leaf, retain_graph=True)
        (b,) = torch.autograd.grad(l, leaf)
        assert torch.equal(a, 4 * g) and torch.equal(b, g)
    with torch.autograd.graph.save_on_cpu():
        l = fn(leaf * 1.0, *args).loss
    junk = [torch.full_like(logits, NAN) for _ in range(3)]  # what was freed is used again
    (a,) = torch.autograd.grad(4 * l, leaf, retain_graph=True)
    (b,) = torch.autograd.grad(l, leaf)
    assert torch.equal(a, 4 * g) and torch.equal(b, g)
    del junk
    for factor in (1.0, 4.0):
        l = torch.utils.checkpoint.checkpoint(lambda t: fn(t * 2, *args).loss, leaf, use_reentrant=False)
        junk = [torch.full_like(logits, NAN) for _ in range(3)]
        (a,) = torch.autograd.grad(factor * l, leaf)
        assert torch.equal(a, 2 * factor * g2)
        del junk


@pytest.mark.parametrize("R,V", [(6, 100003), (6, 300), (140, 50001)])
@pytest.mark.parametrize("temperature", [2.0 ** -100, 1e-39, 2.0 ** -149])
def test_no_slope_at_the_smallest_temperatures(R, V, temperature):
    """A row without a slope (clipped, no advantage, no weight) has a gradient of zeros at every temperature, where 1 / T
    is past fp32 as well; the others' stay finite.  At such a temperature the best token's p is 1, and its gradient 0."""
    logits, x, _ = logits_of(R, V, torch.float32, 21)
    tokens = logits.argmax(1).to(torch.int32)
    old, adv, w = torch.zeros(R, device="cuda"), torch.ones(R, device="cuda"), torch.ones(R, device="cuda")
    old[0] = -1.0  # r = e: clipped
    adv[1], w[2] = 0.0, 0.0
    T = torch.full((R,), temperature, device="cuda")
    fn = q.PolicyLoss("cuda")
    for weights in (None, w):
        out, g = fn.value_and_grad(logits, tokens, old, adv, weights=weights, temperature=T)
        assert torch.isfinite(out.loss) and (out.logprobs == 0).all() and (g[:2] == 0).all() and torch.isfinite(g).all()
        leaf = logits.detach().requires_grad_()
        l = fn(leaf, tokens, old, adv, weights=weights, temperature=T).loss
        (a,) = torch.autograd.grad(l, leaf, retain_graph=True)
        (b,) = torch.autograd.grad(l * 0.0, leaf)
        assert (a[:2] == 0).all() and torch.isfinite(a).all() and (b == 0).all()
    assert (g[2] == 0).all()


@pytest.mark.parametrize("loss", ["policy", "preference"])
@pytest.mark.parametrize("upstream", [INF, -INF, NAN])
def test_upstream_gradients_that_are_not_finite(loss, upstream):
    """They reach the gradient of every row that has a slope (a loss scaler looks for them there); the others stay 0."""
    R, V = 8, 1003
    logits, x, tokens = logits_of(R, V, torch.float32, 7)
    tokens[3] = -1
    old = np.array([O.log_softmax(r)[max(int(t), 0)] for r, t in zip(x.numpy(), tokens)], np.float32)
    if loss == "policy":
        fn, args = q.PolicyLoss("cuda"), (tokens.cuda(), dev(old), torch.ones(R, device="cuda"))
    else:
        fn, args = q.PreferenceLoss("cuda"), (tokens.cuda(), dev(np.array([0, 2, 5, 6, 8], np.int32)))
    leaf = logits.detach().requires_grad_()
    (g,) = torch.autograd.grad(fn(leaf, *args).loss, leaf, grad_outputs=torch.tensor(upstream, device="cuda"))
    has = [0, 1, 2, 4, 5, 6, 7]
    assert not torch.isfinite(g[has]).any() and (g[3] == 0).all()
