"""The 4-bit head's definition (oracle/int4.py), its refusals and its size queries, without a GPU."""
import ctypes as C

import numpy as np
import pytest
import torch

import qwen_warp_amd as q
from oracle import int4 as I
from qwen_warp_amd import _lib


@pytest.mark.parametrize("K,group", [(1, 32), (31, 32), (33, 32), (128, 128), (129, 128), (300, 64)])
def test_values_lie_within_half_a_step(K, group):
    """A value is off by at most half a step and what the scale's and the zero point's rounding take at the range's ends."""
    rng = np.random.default_rng(K)
    w = rng.normal(size=(40, K)).astype(np.float32)
    w[3] = np.abs(w[3])
    w[4] = 0
    codes, s, z = I.quantise(w, group)
    assert codes.max() <= 15 and z.max() <= 15 and s.shape == (40, -(-K // group))
    v = I.values(codes, s, z, group)
    step = np.repeat(s, group, 1)[:, :K]
    # the range's ends: 15 steps of s cover hi - lo but for its rounding (2^-8 of it, 15 steps), the zero point moves them by half a step
    assert (np.abs(v - w) <= step * (0.5 + 0.5 + 15 * 2.0 ** -8)).all()
    assert (v[4] == 0).all()


def test_exact_grid_is_kept():
    """Weights that are whole steps of a power of two, with both ends in a group, come back as they were."""
    rng = np.random.default_rng(0)
    k = rng.integers(-8, 8, size=(20, 64))
    k[:, 0], k[:, 1] = -8, 7
    w = (k * 0.25).astype(np.float32)
    codes, s, z = I.quantise(w, 64)
    assert (I.values(codes, s, z, 64) == w).all() and (s == 0.25).all() and (z == 8).all()


def test_not_finite_and_overflow():
    w = np.zeros((4, 32), np.float32)
    w[0, 3], w[1, 4] = np.nan, np.inf
    w[2, 0], w[2, 1] = 3e38, -3e38
    w[3, 0] = 1.0
    v = I.values(*I.quantise(w, 32), 32)
    assert np.isnan(v[:3]).all() and v[3, 0] == float(I.round_bf16(np.float32(1 / 15))) * 15


def test_sizes_and_refusals():
    lib = _lib.load()
    # 64 rows x 128 values in 4 KB, a word per row and group
    assert lib.qws_int4_pack_bytes(65, 129, 128) == 2 * 2 * 4096 + 2 * 2 * 256
    assert lib.qws_int4_pack_bytes(64, 128, 32) == 4096 + 4 * 256
    for bad in ((0, 5, 32), (5, 0, 32), (5, 5, 16), (5, 5, 0), ((1 << 24) + 1, 5, 32), (5, (1 << 20) + 1, 32)):
        assert lib.qws_int4_pack_bytes(*bad) == 0
    assert lib.qws_int4_head_ws_bytes(3, 10, 100, 32) == 768 and lib.qws_int4_head_ws_bytes(0, 10, 100, 32) == 0
    p, odd = C.c_void_p(256), C.c_void_p(257)
    head = lambda packed=p, N=64, K=128, group=32, x=p, xs=128, T=2, out=p, dt=0, os=64, ws=p, n=512: lib.qws_int4_head(  # noqa: E731
        packed, N, K, group, x, xs, T, out, dt, os, ws, n, None)
    assert head(T=0) == _lib.OK
    for kw in (dict(packed=None), dict(packed=odd), dict(N=0), dict(group=48), dict(x=None), dict(x=odd), dict(xs=-1), dict(T=-1), dict(out=None), dict(out=C.c_void_p(258)),
               dict(dt=2), dict(os=63), dict(ws=odd), dict(ws=None), dict(n=511)):
        assert head(**kw) == _lib.ERR_INVALID, kw
    assert head(T=(1 << 22) + 1, n=1 << 40) == _lib.ERR_NOT_SUPPORTED
    pack = lambda w=p, dt=0, N=4, K=4, stride=4, group=64, to=p: lib.qws_int4_pack(w, dt, N, K, stride, group, to, None)  # noqa: E731
    for kw in (dict(w=None), dict(w=odd), dict(dt=3), dict(N=0), dict(K=0), dict(stride=-1), dict(group=100), dict(to=odd)):
        assert pack(**kw) == _lib.ERR_INVALID, kw
    assert pack(N=(1 << 24) + 1) == _lib.ERR_NOT_SUPPORTED
    codes = lambda c=p, cs=4, s=p, ss=1, z=None, zs=0, group=64, to=p: lib.qws_int4_pack_codes(c, cs, s, 0, ss, z, zs, 4, 4, group, to, None)  # noqa: E731
    for kw in (dict(c=None), dict(s=None), dict(s=odd), dict(cs=-1), dict(ss=-1), dict(zs=-1), dict(group=1), dict(to=None)):
        assert codes(**kw) == _lib.ERR_INVALID, kw


def test_python_refusals():
    with pytest.raises(q.ValidationError):
        q.Int4Head(torch.zeros(4, 4))  # not on a GPU
    with pytest.raises(q.ValidationError):
        q.Int4Head.from_codes(torch.zeros(4, 4, dtype=torch.uint8), torch.ones(4, 1, dtype=torch.bfloat16))


def test_hidden_states_that_want_a_derivative_are_refused():
    """The head gives none: its logits would come back as constants.  Under no_grad, and detached, they go in."""
    head = q.Int4Head.__new__(q.Int4Head)
    head.K, head.device = 4, torch.device("cpu")
    x = torch.zeros(2, 4, dtype=torch.bfloat16, requires_grad=True)
    with pytest.raises(q.ValidationError, match="gradient"):
        head(x)
    with torch.autograd.forward_ad.dual_level():
        with pytest.raises(q.ValidationError, match="tangent"):
            head(torch.autograd.forward_ad.make_dual(x.detach(), torch.ones(2, 4, dtype=torch.bfloat16)))


def test_products_of_too_many_workgroups():
    """Refused before anything is launched; N / 64 times T / 16 says which."""
    lib = _lib.load()
    p = C.c_void_p(256)
    for N, T in ((1 << 24, 1 << 22), (1 << 24, 1 << 14), (1 << 20, 1 << 21)):
        n = lib.qws_int4_head_ws_bytes(T, N, 128, 128)
        assert n > 0 and lib.qws_int4_head(p, N, 128, 128, p, 128, T, p, 0, N, p, n, None) == _lib.ERR_NOT_SUPPORTED
