"""The CPU definitions of the log probabilities and of the 8-bit head against independent calculations, and the argument
checks of their entry points and Python wrappers, without a GPU."""
import ctypes as C
import math

import numpy as np
import pytest
import torch

import qwen_warp_amd as q
from oracle import fp8 as F
from oracle import logprobs as L
from qwen_warp_amd import _lib
from qwen_warp_amd.logprobs import rows_of


# ------------------------------------------------------------------------------------------ definitions
def test_row_against_torch():
    g = torch.Generator().manual_seed(0)
    x = torch.randn(1000, generator=g, dtype=torch.float64) * 3
    lp, rank, h, ids, top = L.row(x.numpy(), [5, 999, -1, 1000], 7, 0.5)
    want = torch.log_softmax(x / 0.5, 0)
    assert np.allclose(lp, [want[5], want[999], 0, 0], atol=1e-12)
    assert rank[2] == rank[3] == -1 and rank[0] == int((x > x[5]).sum())
    assert abs(h + float((want.exp() * want).sum())) < 1e-12
    best = torch.topk(want, 7)
    assert ids.tolist() == best.indices.tolist() and np.allclose(top, best.values.numpy(), atol=1e-12)


def test_row_edges():
    inf, nan = math.inf, math.nan
    lp, rank, h, ids, top = L.row([-inf, nan, -inf], [0, 1], 2)
    assert (lp == -inf).all() and rank.tolist() == [0, 1] and h == 0 and ids.tolist() == [-1, -1] and (top == -inf).all()
    lp, rank, h, ids, top = L.row([0.0, inf, 3.0, inf], [1, 3, 2], 3)
    assert np.allclose(lp[:2], -math.log(2)) and lp[2] < -1e37 and rank.tolist() == [0, 1, 2] and abs(h - math.log(2)) < 1e-12
    lp, rank, _, ids, _ = L.row([0.0, -0.0, 1.0, 1.0], [0, 1, 2, 3], 4)  # zeros of both signs tie
    assert rank.tolist() == [2, 3, 0, 1] and ids.tolist() == [2, 3, 0, 1]
    assert L.row([1.0, 2.0], [0], 0, 0.0)[0] == L.row([1.0, 2.0], [0], 0, 1.0)[0]


def test_e4m3_against_torch():
    t = F.e4m3_values()
    assert (t == torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy()).all()
    v = np.concatenate([t, (t[1:] + t[:-1]) / 2, np.random.default_rng(0).uniform(-448, 448, 5000)]).astype(np.float32)
    assert (F.round_e4m3(v.astype(np.float64)) == torch.from_numpy(v).to(torch.float8_e4m3fn).double().numpy()).all()


def test_block_exponents():
    x = np.zeros((6, 200))
    x[0, 3], x[1, 150], x[2, 0], x[3, 0] = 448.0, 449.0, 1.0, 2.0 ** -140
    e = F.block_exponents(x)
    assert e[0].tolist() == [0, -127] and e[1].tolist() == [-127, 1] and e[2, 0] == -8 and e[3, 0] == -127
    y = np.random.default_rng(1).standard_normal((4, 300))
    a = np.abs(np.pad(y, ((0, 0), (0, 84)))).reshape(4, 3, 128).max(2)
    e = F.block_exponents(y)
    assert (a <= 448 * 2.0 ** e).all() and (a > 448 * 2.0 ** (e - 1)).all()
    assert np.abs(F.values(y) - y).max() <= np.abs(y).max() / 16
    assert np.isnan(F.values(np.array([[1.0, math.inf, math.nan]])))[0].tolist() == [False, True, True]


# ------------------------------------------------------------------------------------------ refusals
@pytest.fixture(scope="module")
def lib():
    return _lib.load()


P = 4096  # a device address that no call may reach


def _batch(**kw):
    b = _lib.LogprobsBatch(logits=P, dtype=0, R=2, V=100, row_stride=100, tokens=P, M=1, top=3, out_logprobs=P, out_ranks=P, out_entropy=P, out_top_ids=P,
                           out_top_logprobs=P)
    for k, v in kw.items():
        setattr(b, k, v)
    return b


@pytest.mark.parametrize("kw", [dict(dtype=2), dict(V=0), dict(R=-1), dict(M=-1), dict(top=-1), dict(logits=None), dict(logits=P + 2), dict(row_stride=-1),
                                dict(tokens=None), dict(out_logprobs=None), dict(out_top_ids=None), dict(out_top_logprobs=None),
                                dict(M=0, tokens=None)])
def test_logprobs_refuses(lib, kw):
    assert lib.qws_logprobs(C.byref(_batch(**kw)), P, 1 << 30, None) == _lib.ERR_INVALID


def test_logprobs_struct_layout():
    """The library's own layout is asserted where it is built (qws_logprobs.hip)."""
    assert C.sizeof(_lib.LogprobsBatch) == 96 and _lib.LogprobsBatch.tokens.offset == 32 and _lib.LogprobsBatch.out_top_logprobs.offset == 88


def test_logprobs_limits(lib):
    for kw in (dict(V=(1 << 19) + 1), dict(M=65), dict(top=65)):
        assert lib.qws_logprobs(C.byref(_batch(**kw)), P, 1 << 30, None) == _lib.ERR_NOT_SUPPORTED
    n = lib.qws_logprobs_ws_bytes(0, 2, 100, 1, 3)
    assert n > 0 and lib.qws_logprobs(C.byref(_batch()), P, n - 1, None) == _lib.ERR_INVALID
    assert lib.qws_logprobs(C.byref(_batch()), P + 16, n, None) == _lib.ERR_INVALID and lib.qws_logprobs(C.byref(_batch()), None, n, None) == _lib.ERR_INVALID
    assert lib.qws_logprobs(None, P, n, None) == _lib.ERR_INVALID
    assert lib.qws_logprobs(C.byref(_batch(R=0)), None, 0, None) == _lib.OK
    for args in ((2, 1, 100, 1, 1), (0, 0, 100, 1, 1), (0, 1, (1 << 19) + 1, 1, 1), (0, 1, 100, 65, 1), (0, 1, 100, 1, 65)):
        assert lib.qws_logprobs_ws_bytes(*args) == 0


def test_fp8_refuses(lib):
    n = lib.qws_fp8_head_ws_bytes(4, 1000, 256)
    s = lib.qws_fp8_score_ws_bytes(4, 1000, 256)
    assert lib.qws_fp8_pack_bytes(1000, 256) >= 1000 * 256 and n > 0 and s > n
    assert lib.qws_fp8_pack_bytes(0, 256) == 0 and lib.qws_fp8_pack_bytes((1 << 24) + 1, 1) == 0 and lib.qws_fp8_pack_bytes(1, (1 << 20) + 1) == 0
    assert lib.qws_fp8_head_ws_bytes(0, 1, 1) == 0 and lib.qws_fp8_score_ws_bytes(1, 1, 0) == 0
    assert lib.qws_fp8_pack(P, 2, 1000, 256, 256, P, None) == _lib.ERR_INVALID
    assert lib.qws_fp8_pack(P + 1, 1, 1000, 256, 256, P, None) == _lib.ERR_INVALID
    assert lib.qws_fp8_pack(P, 1, 1000, 256, 256, P + 16, None) == _lib.ERR_INVALID
    assert lib.qws_fp8_pack(None, 1, 1000, 256, 256, P, None) == _lib.ERR_INVALID

    def head(packed=P, N=1000, K=256, x=P, xs=256, T=4, out=P, dt=0, os=1000, ws=P, nb=n):
        return lib.qws_fp8_head(packed, N, K, x, xs, T, out, dt, os, ws, nb, None)

    assert head(T=0) == _lib.OK
    for kw in (dict(packed=None), dict(packed=P + 8), dict(x=None), dict(x=P + 1), dict(T=-1), dict(out=None), dict(out=P + 2), dict(dt=5), dict(os=999), dict(xs=-1),
               dict(ws=None), dict(ws=P + 4), dict(nb=n - 1), dict(N=0), dict(K=0)):
        assert head(**kw) == _lib.ERR_INVALID, kw
    assert head(T=(1 << 22) + 1) == _lib.ERR_NOT_SUPPORTED

    def score(tok=P, lp=P, nb=s, T=4):
        return lib.qws_fp8_score(P, 1000, 256, P, 256, T, tok, None, lp, None, P, nb, None)

    assert score(T=0) == _lib.OK
    for kw in (dict(tok=None), dict(lp=None), dict(nb=s - 1)):
        assert score(**kw) == _lib.ERR_INVALID, kw


def test_wrappers_refuse():
    op = q.LogProbs("cpu")
    with pytest.raises(q.ValidationError):
        op(torch.zeros(2, 8))
    with pytest.raises(q.ValidationError):
        q.Fp8Head(torch.zeros(8, 8))


def test_rows_of():
    x = torch.zeros(4, 5, 10)
    assert rows_of(x, "x") == (20, 10) and rows_of(x[:, :, :7], "x") == (20, 10) and rows_of(x[:, 2], "x") == (4, 50) and rows_of(x[1:2, 1:2], "x") == (1, 0)
    assert rows_of(torch.zeros(1, 10).expand(6, 10), "x") == (6, 0) and rows_of(torch.zeros(0, 10), "x")[0] == 0
    for bad in (x[:, :3], x.transpose(1, 2), torch.zeros(10), torch.zeros(1, 10).expand(6, 10).view(2, 3, 10).transpose(0, 1)[..., ::2]):
        with pytest.raises(q.ValidationError):
            rows_of(bad, "x")


def test_row_counts_past_the_ranges(lib):
    """More workgroups than a launch has threads for, and counts that do not fit the entry points' int."""
    most = (1 << 24) - 1  # workgroups of 256 threads below 2^32 threads
    for dtype, V in ((0, 1), (0, 1000), (1, 2000), (1, 1)):
        over = most + 1
        assert lib.qws_logprobs(C.byref(_batch(R=over, V=V, dtype=dtype)), P, 1 << 62, None) == _lib.ERR_NOT_SUPPORTED
        assert lib.qws_logprobs_ws_bytes(dtype, over, V, 1, 3) == 0 and lib.qws_logprobs_ws_bytes(dtype, most, V, 1, 3) > 0
    one = torch.zeros(1, 1)
    for bad in (one.expand(1 << 31, 1), one.expand((1 << 32) + 2, 1), one.view(1, 1, 1).expand(1 << 16, 1 << 16, 1), torch.empty(2, 1 << 31, device="meta")):
        with pytest.raises(q.ValidationError):
            rows_of(bad, "x")
    assert rows_of(one.expand((1 << 31) - 1, 1), "x") == ((1 << 31) - 1, 0)
