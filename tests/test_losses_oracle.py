"""The losses' definitions (oracle/losses.py): gradients against differences in 64 bits, torch's autograd and the cases left out;
the entry points' refusals and sizes, without a GPU."""
import ctypes as C

import numpy as np
import pytest
import torch

import qwen_warp_amd as q
from oracle import losses as O
from qwen_warp_amd import _lib


def world(seed, R=7, V=11):
    rng = np.random.default_rng(seed)
    x = rng.normal(size=(R, V)) * 2
    tokens = rng.integers(0, V, R)
    lp = np.array([O.log_softmax(r)[t] for r, t in zip(x, tokens)])
    return rng, x, tokens, lp


def differences(f, x, h=1e-6):
    g = np.zeros_like(x)
    for i in np.ndindex(*x.shape):
        y = x.copy()
        y[i] += h
        up = f(y)
        y[i] -= 2 * h
        g[i] = (up - f(y)) / (2 * h)
    return g


@pytest.mark.parametrize("kl,weights,temperature", [(0.0, False, False), (0.3, True, False), (0.1, False, True)])
def test_policy_gradient_against_differences(kl, weights, temperature):
    rng, x, tokens, lp = world(1)
    T = rng.uniform(0.5, 2, 7) if temperature else None
    lp = np.array([O.log_softmax(r, 1 if T is None else t)[k] for r, k, t in zip(x, tokens, np.ones(7) if T is None else T)])
    old = lp - np.array([0.3, -0.3, 0.1, -0.1, 0.5, -0.5, 0.0])  # inside and outside the clip, both ways
    args = dict(old=old, adv=np.array([1.0, 1.0, -1.0, 2.0, -2.0, -1.0, 0.5]), clip=(0.2, 0.28), kl=kl, ref=lp + rng.normal(size=7) * 0.3,
                weights=rng.uniform(0.1, 1, 7) if weights else None, temperature=T)
    tokens[3] = -1
    got = O.policy(x, tokens, **args)
    want = differences(lambda y: O.policy(y, tokens, **args)["loss"], x)
    assert np.abs(got["grad"] - want).max() < 1e-8 and (got["grad"][3] == 0).all()
    if kl == 0.0:
        assert (got["grad"][0] == 0).all() and np.abs(got["grad"][1]).max() > 0  # r = 1.35, A > 0: clipped; r = 0.74, A > 0: not


@pytest.mark.parametrize("average,smoothing,weights,ref", [(False, 0.0, False, True), (True, 0.1, True, False)])
def test_preference_gradient_against_differences(average, smoothing, weights, ref):
    rng, x, tokens, _ = world(2, R=12)
    tokens[[0, 6]] = -1
    starts = [1, 4, 6, 6, 10]  # rows 0, 10 and 11 outside, the third sequence empty
    args = dict(starts=starts, beta=0.3, margin=0.2, smoothing=smoothing, average=average, ref=rng.normal(size=4) * 3 if ref else None,
                weights=rng.uniform(0.1, 1, 2) if weights else None)
    got = O.preference(x, tokens, **args)
    want = differences(lambda y: O.preference(y, tokens, **args)["loss"], x)
    assert np.abs(got["grad"] - want).max() < 1e-8 and (got["grad"][[0, 6, 10, 11]] == 0).all() and got["logprobs"][2] == 0


def test_against_autograd():
    rng, x, tokens, lp = world(3)
    old, adv = lp + rng.normal(size=7) * 0.1, rng.normal(size=7)
    t = torch.tensor(x, requires_grad=True)
    l = torch.log_softmax(t, 1).gather(1, torch.tensor(tokens).view(-1, 1))[:, 0]
    r = torch.exp(l - torch.tensor(old))
    a = torch.tensor(adv)
    loss = -torch.minimum(r * a, r.clamp(0.8, 1.2) * a).mean()
    loss.backward()
    got = O.policy(x, tokens, old, adv)
    assert abs(got["loss"] - float(loss.detach())) < 1e-12 and np.abs(got["grad"] - t.grad.numpy()).max() < 1e-12
    t.grad = None
    s = torch.log_softmax(t, 1).gather(1, torch.tensor(tokens).view(-1, 1))[:, 0]
    loss = -torch.nn.functional.logsigmoid(0.1 * (s[:3].sum() - s[3:].sum()))
    loss.backward()
    got = O.preference(x, tokens, [0, 3, 7])
    assert abs(got["loss"] - float(loss.detach())) < 1e-12 and np.abs(got["grad"] - t.grad.numpy()).max() < 1e-12


def test_rows_left_out():
    rng, x, tokens, lp = world(4)
    x[1] = -np.inf                    # the mask leaves nothing
    x[2, tokens[2]] = -np.inf         # the token is forbidden
    x[3, (tokens[3] + 1) % 11] = np.nan  # a masked place
    tokens[4], tokens[5] = -1, 11
    adv = rng.normal(size=7)
    old = lp.copy()
    old[4] = adv[5] = np.nan          # not used
    got = O.policy(x, tokens, old, adv)
    assert np.isfinite(got["loss"]) and np.isfinite(got["grad"]).all()
    assert (got["grad"][[1, 2, 4, 5]] == 0).all() and got["grad"][3, (tokens[3] + 1) % 11] == 0
    assert got["logprobs"][1] == got["logprobs"][2] == -np.inf and got["logprobs"][4] == got["logprobs"][5] == 0
    assert abs(got["grad"][6].sum()) < 1e-15


def test_sizes_and_refusals():
    lib = _lib.load()
    assert C.sizeof(_lib.LossRows) == 56 and C.sizeof(_lib.PolicyBatch) == 136 and C.sizeof(_lib.PreferenceBatch) == 136
    assert lib.qws_policy_state_bytes(0, 0, 10) > 0 and lib.qws_preference_state_bytes(1, 5, 10, 0) > 0
    for bad in ((2, 5, 10), (0, -1, 10), (0, 5, 0), (0, 1 << 24, 10), (0, 5, (1 << 24) + 1)):
        assert lib.qws_policy_state_bytes(*bad) == 0
        assert lib.qws_preference_state_bytes(*bad, 2) == 0
    assert lib.qws_preference_state_bytes(0, 5, 10, -1) == 0
    n = 1 << 20

    def rows(**kw):
        r = _lib.LossRows(256, 0, 4, 10, 0, 10, 0, 256, None)
        for k, v in kw.items():
            setattr(r, k, v)
        return r

    def policy(state=256, size=n, grad=None, stride=10, r=None, scale=1.0, **kw):
        b = _lib.PolicyBatch(r or rows(), 256, 256, None, None, 0.2, 0.2, 0.0, 256, None, None, None)
        for k, v in kw.items():
            setattr(b, k, v)
        return lib.qws_policy_loss(C.byref(b), state, size, grad, stride, scale, None)

    def preference(state=256, size=n, grad=None, stride=10, r=None, scale=1.0, **kw):
        b = _lib.PreferenceBatch(r or rows(), 256, 2, 0, None, None, 0.1, 0.0, 0.0, 256, None, None, None)
        for k, v in kw.items():
            setattr(b, k, v)
        return lib.qws_preference_loss(C.byref(b), state, size, grad, stride, scale, None)

    nan, inf = float("nan"), float("inf")
    for f in (policy, preference):
        for kw in (dict(state=None), dict(state=257), dict(size=100), dict(grad=258), dict(grad=256, stride=9), dict(out_loss=None), dict(scale=nan), dict(scale=inf), dict(r=rows(logits=None)),
                   dict(r=rows(logits=258)), dict(r=rows(dtype=5)), dict(r=rows(tokens=None)), dict(r=rows(R=-1)), dict(r=rows(V=0)), dict(r=rows(block=-1)),
                   dict(r=rows(row_stride=-1)), dict(r=rows(block_stride=-1))):
            assert f(**kw) == _lib.ERR_INVALID, kw
        assert f(r=rows(V=(1 << 24) + 1, row_stride=1 << 25)) == _lib.ERR_NOT_SUPPORTED
        assert f(r=rows(R=1 << 24)) == _lib.ERR_NOT_SUPPORTED
    for kw in (dict(old_logprobs=None), dict(advantages=None), dict(clip_low=-0.1), dict(clip_low=1.1), dict(clip_low=nan), dict(clip_high=-0.1), dict(clip_high=inf),
               dict(clip_high=nan), dict(kl=nan), dict(kl=inf)):
        assert policy(**kw) == _lib.ERR_INVALID, kw
    for kw in (dict(starts=None), dict(P=-1), dict(beta=nan), dict(margin=inf), dict(smoothing=-0.1), dict(smoothing=1.1), dict(smoothing=nan)):
        assert preference(**kw) == _lib.ERR_INVALID, kw
    r = rows()
    assert lib.qws_loss_grad(None, 256, None, 256, 10, 0, None) == _lib.ERR_INVALID
    assert lib.qws_loss_grad(C.byref(r), None, None, 256, 10, 0, None) == _lib.ERR_INVALID
    assert lib.qws_loss_grad(C.byref(r), 256, None, None, 10, 0, None) == _lib.ERR_INVALID
    assert lib.qws_loss_grad(C.byref(r), 256, None, 256, 9, 0, None) == _lib.ERR_INVALID
    assert lib.qws_loss_grad(C.byref(r), 256, None, 256, 10, nan, None) == _lib.ERR_INVALID
    r = rows(R=0)
    assert lib.qws_loss_grad(C.byref(r), 256, None, None, 0, 0, None) == _lib.OK


def test_python_refusals():
    for bad in (dict(clip=(-0.1, 0.2)), dict(clip=(0.2, float("nan"))), dict(kl=float("inf")), dict(upstream=float("nan"))):
        with pytest.raises(q.ValidationError):
            q.PolicyLoss("cuda", **bad)
    for bad in (dict(beta=float("nan")), dict(margin=float("inf")), dict(smoothing=1.5)):
        with pytest.raises(q.ValidationError):
            q.PreferenceLoss("cuda", **bad)
    with pytest.raises(q.ValidationError):
        q.PolicyLoss("cuda")(torch.zeros(2, 3), torch.zeros(2, dtype=torch.int32), torch.zeros(2), torch.zeros(2))  # not on a GPU


def test_blocks_of():
    from qwen_warp_amd.losses import blocks_of
    x = torch.zeros(4, 6, 10)
    assert blocks_of(x, "x") == (24, 0, 10, 0)
    assert blocks_of(x[:, :-1], "x") == (20, 5, 10, 60)
    assert blocks_of(x[:, 1:2], "x") == (4, 0, 60, 0)
    assert blocks_of(x.transpose(0, 1), "x") == (24, 4, 60, 10)
    assert blocks_of(x[0], "x") == (6, 0, 10, 0)
    assert blocks_of(x[:1, :1], "x") == (1, 0, 0, 0)
    assert blocks_of(x[:0], "x") == (0, 0, 0, 0)
    assert blocks_of(torch.zeros(1, 10).expand(5, 10), "x") == (5, 0, 0, 0)
    with pytest.raises(q.ValidationError):
        blocks_of(x[0, 0], "x")
    with pytest.raises(q.ValidationError):
        blocks_of(x.transpose(1, 2), "x")
    with pytest.raises(q.ValidationError):
        blocks_of(torch.zeros(3, 4, 5, 10)[:, :-1, :-1], "x")
