"""Fp8Head (qws_fp8_* through the Python wrapper) against the 64-bit definition (oracle/fp8.py, oracle/logprobs.py).

The packed weights are read back exactly (products with unit vectors).  A logit is a sum of K exact products in fp32, in
blocks of 128: it is within (128 + K / 128) 2^-23 of sum |qx qw| (a rounding, or a truncation, of each partial sum).  A
logit's error moves ln sum e^z by as much at most, and a log probability or an entropy by the bounds of
tests/test_gpu_logprobs.py beside it."""
import numpy as np
import pytest
import torch

import qwen_warp_amd as q
from oracle import fp8 as F
from oracle import logprobs as L

pytestmark = pytest.mark.gpu
INF = float("inf")


def data(T, N, K, seed, wdtype=torch.bfloat16):
    g = torch.Generator().manual_seed(seed)
    w = torch.randn(N, K, generator=g) * (0.01 + 0.05 * torch.rand(N, 1, generator=g))
    x = torch.randn(T, K, generator=g) * (0.1 + 3 * torch.rand(T, 1, generator=g))
    w[:, ::61] *= 5
    x[:, ::37] *= 8
    return w.to(wdtype), x.to(torch.bfloat16)


def product(w, x):
    """(logits, their bound) in 64 bits"""
    a, b = F.values(x.double().numpy()), F.values(w.double().numpy())
    return a @ b.T, (128 + x.shape[1] / 128) * 2.0 ** -23 * (np.abs(a) @ np.abs(b).T)


@pytest.mark.parametrize("wdtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("N,K", [(1, 1), (5, 127), (16, 128), (300, 129), (257, 300), (64, 640)])
def test_weights_read_back(N, K, wdtype):
    w, _ = data(1, N, K, N + K, wdtype)
    w[0] = 0.0
    w[-1, 0] = 2.0 ** -100
    eye = torch.eye(K, dtype=torch.bfloat16, device="cuda")
    for pad in (0, 1):
        v = torch.zeros(N, K + pad, dtype=wdtype, device="cuda")[:, :K]
        v.copy_(w)
        got = q.Fp8Head(v)(eye).t().double().cpu().numpy()
        assert (got == F.values(w.double().numpy())).all()


def test_scales_at_their_ends():
    """Blocks whose largest value is just at, below and above a scale's range; powers over the whole exponent range."""
    K = 128
    p = 2.0 ** torch.arange(-60, 60, dtype=torch.float64)
    w = torch.zeros(360, K, dtype=torch.float64)
    w[:120, 5], w[120:240, 5], w[240:, 5] = 1.75 * p, 1.75 * p * (1 + 2.0 ** -20), p
    w[:, 6] = w[:, 5] / 3
    w = w.float()
    eye = torch.eye(K, dtype=torch.bfloat16, device="cuda")
    got = q.Fp8Head(w.cuda())(eye).t().double().cpu().numpy()
    assert (got == F.values(w.double().numpy())).all()


@pytest.mark.parametrize("T,N,K", [(1, 1, 1), (1, 1000, 100), (2, 15, 128), (3, 8191, 1000), (7, 129, 5120), (16, 4096, 640), (17, 1000, 257), (33, 700, 512),
                                   (64, 513, 385), (65, 300, 1024), (100, 2001, 130), (128, 256, 128), (129, 255, 2000), (200, 1300, 768), (257, 257, 384), (600, 900, 640)])
def test_logits(T, N, K):
    w, x = data(T, N, K, T + N + K)
    want, tol = product(w, x)
    head = q.Fp8Head(w.cuda())
    for pad in (0, 3):
        y = torch.full((T, K + pad), float("nan"), dtype=torch.bfloat16, device="cuda")[:, :K]
        y.copy_(x)
        got = head(y)
        assert got.shape == (T, N) and got.dtype == torch.float32
        err = np.abs(got.double().cpu().numpy() - want)
        assert (err <= tol).all(), f"off by {(err / tol).max()} of the bound"
        half = head(y, dtype=torch.bfloat16)
        assert torch.equal(half.view(torch.int16), got.to(torch.bfloat16).view(torch.int16))
        # into a wider buffer, at any alignment; nothing around it is touched
        for dtype in (torch.float32, torch.bfloat16):
            buf = torch.full((T, N + 9), 7.0, dtype=dtype, device="cuda")
            head(y, out=buf[:, 5:5 + N])
            assert torch.equal(buf[:, 5:5 + N], got.to(dtype)) and (buf[:, :5] == 7).all() and (buf[:, 5 + N:] == 7).all()


def test_rows_do_not_depend_on_the_batch():
    """A hidden state's logits in batches of other sizes stay within the bound; the same call gives the same bits."""
    w, x = data(300, 3000, 1280, 5)
    head = q.Fp8Head(w.cuda())
    want, tol = product(w, x)
    x = x.cuda()
    for T in (1, 15, 31, 64, 96, 150, 300):
        got = head(x[:T])
        assert (np.abs(got.double().cpu().numpy() - want[:T]) <= tol[:T]).all(), T
        assert torch.equal(got, head(x[:T]))


def test_special_values():
    """Zeros give zeros; a row with NaN or an infinity is NaN, the others are not touched by it."""
    w, x = data(20, 500, 300, 6)
    want, tol = product(w, x)
    x[3] = 0
    x[5, 17], x[6, 299], x[7, 0] = float("nan"), INF, -INF
    wn = w.clone()
    wn[11, 4], wn[12, 299] = INF, float("nan")
    got = q.Fp8Head(wn.cuda())(x.cuda()).double().cpu().numpy()
    nan = np.zeros((20, 500), bool)
    nan[5:8] = True
    nan[:, 11:13] = True
    want[3] = 0
    assert (np.isnan(got) == nan).all()
    assert (np.abs(got - want)[~nan] <= tol[~nan]).all()
    lp, h = q.Fp8Head(wn.cuda()).score(x.cuda(), torch.full((20,), 12, dtype=torch.int32, device="cuda"))
    assert (lp == -INF).all() and (h[5:8] == 0).all() and torch.isfinite(h).all()  # NaN logits count as -inf


@pytest.mark.parametrize("T,N,K", [(1, 1, 1), (1, 5000, 256), (5, 129, 128), (16, 8191, 640), (17, 500, 130), (77, 3001, 384), (130, 1000, 512), (300, 257, 100), (520, 1025, 256)])
@pytest.mark.parametrize("temperature", [False, True])
def test_score(T, N, K, temperature):
    w, x = data(T, N, K, T * N + K)
    y, tol = product(w, x)
    g = torch.Generator().manual_seed(T)
    tokens = torch.randint(0, N, (T,), generator=g).to(torch.int32)
    t = 0.3 + 2 * torch.rand(T, generator=g) if temperature else None
    if T > 4:
        tokens[2], tokens[3] = -1, N
        if temperature:
            t[1] = 0.0
    head = q.Fp8Head(w.cuda())
    lp, h = head.score(x.cuda(), tokens.cuda(), temperature=t.cuda() if temperature else None)
    lp, h = lp.double().cpu().numpy(), h.double().cpu().numpy()
    for r in range(T):
        temp = 1.0 if t is None or t[r] == 0 else float(t[r])
        want, _, wh, _, _ = L.row(y[r], [int(tokens[r])], 0, temp)
        off = tol[r].max() / temp
        sums = (256 + 30) * 2.0 ** -24
        assert abs(lp[r] - want[0]) <= 2 * off + sums + 8 * abs(want[0]) * 2.0 ** -24, f"row {r}: {lp[r]} {want[0]}"
        # dH = -cov(z, log p): a change of off in z moves H by at most off * sd(log p), sd <= ln N + 1 + |mean|
        assert abs(h[r] - wh) <= off * (2 * np.log(N) + 2) + sums * (1 + 2 * wh), f"row {r}: entropy {h[r]} {wh}"
    again = head.score(x.cuda(), tokens.cuda(), temperature=t.cuda() if temperature else None)
    assert (again[0].double().cpu().numpy() == lp).all() and (again[1].double().cpu().numpy() == h).all()


@pytest.mark.parametrize("T,N,K", [(9, 33001, 130), (16, 40000, 257), (17, 140003, 100), (32, 33025, 384), (33, 32769, 129), (50, 140003, 130), (64, 36000, 640)])
def test_few_states_of_a_large_head(T, N, K):
    """More weight rows than 128 tiles of 256, the last one partly filled; more tiles than two a CU among them."""
    w, x = data(T, N, K, T + N + K)
    y, tol = product(w, x)
    head = q.Fp8Head(w.cuda())
    buf = torch.full((T, N + 9), 7.0, device="cuda")
    got = head(x.cuda(), out=buf[:, 5:5 + N])
    err = np.abs(got.double().cpu().numpy() - y)
    assert (err <= tol).all(), f"off by {(err / tol).max()} of the bound"
    assert (buf[:, :5] == 7).all() and (buf[:, 5 + N:] == 7).all()
    assert torch.equal(head(x.cuda(), dtype=torch.bfloat16), got.to(torch.bfloat16))
    tokens = torch.randint(0, N, (T,), generator=torch.Generator().manual_seed(T)).to(torch.int32)
    tokens[1], tokens[2], tokens[3] = -1, N, N - 1
    lp, h = (v.double().cpu().numpy() for v in head.score(x.cuda(), tokens.cuda()))
    for r in range(T):  # the bounds of test_score
        want, _, wh, _, _ = L.row(y[r], [int(tokens[r])], 0, 1.0)
        off, sums = tol[r].max(), (256 + 30) * 2.0 ** -24
        assert abs(lp[r] - want[0]) <= 2 * off + sums + 8 * abs(want[0]) * 2.0 ** -24, f"row {r}: {lp[r]} {want[0]}"
        assert abs(h[r] - wh) <= off * (2 * np.log(N) + 2) + sums * (1 + 2 * wh), f"row {r}: entropy {h[r]} {wh}"


def test_score_agrees_with_the_logits():
    """score() against LogProbs over the same head's logits, through the package."""
    w, x = data(90, 6000, 512, 9)
    head = q.Fp8Head(w.cuda())
    tokens = torch.randint(0, 6000, (90,), generator=torch.Generator().manual_seed(1)).to(torch.int32).cuda()
    lp, h = head.score(x.cuda(), tokens)
    want = q.LogProbs("cuda")(head(x.cuda()), tokens)
    assert torch.allclose(lp, want.logprobs, atol=5e-5, rtol=1e-5) and torch.allclose(h, want.entropy, atol=5e-5, rtol=1e-5)


def test_no_rows_streams_and_graph():
    w, x = data(40, 2000, 256, 10)
    head = q.Fp8Head(w.cuda())
    x = x.cuda()
    assert head(x[:0]).shape == (0, 2000) and head.score(x[:0], torch.empty(0, dtype=torch.int32, device="cuda"))[0].shape == (0,)
    first = head(x)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        head(x[:7])
        with torch.cuda.stream(side):
            other = head(x)
        side.synchronize()
        assert torch.equal(first, other)
    buf, tokens = x.clone(), torch.arange(40, dtype=torch.int32, device="cuda")
    for n in (1, 40):
        head(buf[:n]), head.score(buf[:n], tokens[:n])
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y, (lp, h) = head(buf[:n]), head.score(buf[:n], tokens[:n])
        for i in range(4):
            buf.copy_(data(40, 1, 256, 50 + i)[1])
            want = [head(buf[:n]).clone(), *(t.clone() for t in head.score(buf[:n], tokens[:n]))]
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip((y, lp, h), want)), f"replay {i}"


def test_offsets_past_32_bits():
    """Hidden states and logits whose rows lie 2^31 + 8 elements apart."""
    w, x = data(2, 700, 200, 11)
    stride = (1 << 31) + 8
    xs = torch.zeros(stride + 700, dtype=torch.bfloat16, device="cuda")
    far = xs.as_strided((2, 200), (stride, 1))
    far.copy_(x)
    head = q.Fp8Head(w.cuda())
    want = head(x.cuda(), dtype=torch.bfloat16)
    assert torch.equal(head(far, dtype=torch.bfloat16), want)
    out = xs.as_strided((2, 700), (stride, 1))
    xin = x.cuda()
    head(xin, out=out)
    assert torch.equal(out, want)


def test_behind_the_candidate_select():
    """The head's logits refined by HeadSelect: the argmax is the bf16 head's."""
    w, x = data(8, 4096, 512, 12)
    x[:] = (x.float() + 60 * w[torch.arange(8) * 500].float()).to(torch.bfloat16)
    head, select = q.Fp8Head(w.cuda()), q.HeadSelect("cuda")
    tok, val, _, _ = select(head(x.cuda()), w.cuda(), x.cuda(), 32)
    exact = x.double() @ w.double().t()
    assert tok.tolist() == exact.argmax(1).tolist()


def test_refusals():
    w, x = data(4, 100, 64, 13)
    w, x = w.cuda(), x.cuda()
    head = q.Fp8Head(w)
    i32 = torch.zeros(4, dtype=torch.int32, device="cuda")
    for call in (lambda: q.Fp8Head(w.half()), lambda: q.Fp8Head(w.t()), lambda: q.Fp8Head(w[0]), lambda: q.Fp8Head(w[:0]), lambda: head(x.float()), lambda: head(x[:, :63]),
                 lambda: head(x.cpu()), lambda: head(x[0]), lambda: head(x, dtype=torch.float16), lambda: head(x, out=torch.zeros(4, 99, device="cuda")),
                 lambda: head(x, out=torch.zeros(1, 100, device="cuda").expand(4, 100)), lambda: head.score(x, i32[:3]), lambda: head.score(x, i32.long()),
                 lambda: head.score(x, i32, temperature=torch.ones(4))):
        with pytest.raises(q.ValidationError):
            call()


@pytest.mark.parametrize("T,N,K", [(1, 8191, 130), (7, 1000, 256), (12, 33001, 130), (24, 4000, 300), (40, 33001, 64), (40, 5000, 64), (80, 3001, 384)])
def test_score_small_temperatures(T, N, K):
    """Temperatures down to 1e-30 and large logits, against the definition over the head's own logits (the same products in
    the same order)."""
    w, x = data(T, N, K, T + N)
    temps = torch.tensor([1e-5, 1e-6, 1e-7, 1e-8, 5e-9, 3e-9, 1e-9, 1e-10, 1e-12, 1e-17, 1e-18, 1e-30])
    head = q.Fp8Head(w.cuda())
    y = head(x.cuda()).double().cpu().numpy()
    tokens = torch.randint(0, N, (T,), generator=torch.Generator().manual_seed(T)).to(torch.int32)
    tokens[::2] = torch.from_numpy(y.argmax(1)[::2])
    for i in range(14):  # each temperature alone (a wave takes one form for all its states), then mixed ones, then large logits
        t = torch.ones(T) if i == 13 else temps.repeat(T)[:T] if i == 12 else temps[i].repeat(T)
        if i == 13:
            x = (x.float() * 2.0 ** 36).to(torch.bfloat16)
            y = head(x.cuda()).double().cpu().numpy()
        lp, h = (v.double().cpu().numpy() for v in head.score(x.cuda(), tokens.cuda(), temperature=t.cuda()))
        for r in range(T):
            want, _, wh, _, _ = L.row(y[r], [int(tokens[r])], 0, float(t[r]))
            sums = (256 + 30) * 2.0 ** -24
            assert abs(lp[r] - want[0]) <= sums + 8 * abs(want[0]) * 2.0 ** -24, f"row {r} at {float(t[r])}: {lp[r]} {want[0]}"
            assert abs(h[r] - wh) <= sums * (1 + 2 * wh), f"row {r} at {float(t[r])}: entropy {h[r]} {wh}"


@pytest.mark.parametrize("T,N", [(1, 9000), (8, 4000), (16, 33001), (32, 4000), (64, 33001), (64, 4000), (200, 4000)])
def test_score_signs(T, N):
    """No log probability above 0 and no entropy below 0 where a token is sure, at many temperatures."""
    w, x = data(T, N, 256, T)
    likely = torch.arange(T) * 7 % N
    x = (x.float() + 600 * w[likely].float()).to(torch.bfloat16)
    head = q.Fp8Head(w.cuda())
    for t in (None, torch.full((T,), 0.37), 0.05 + torch.rand(T, generator=torch.Generator().manual_seed(T))):
        lp, h = head.score(x.cuda(), likely.to(torch.int32).cuda(), temperature=t.cuda() if t is not None else None)
        assert (lp <= 0).all() and (h >= 0).all()
        assert T == 1 or (lp > -0.1).float().mean() > 0.5  # mostly sure ones


@pytest.mark.parametrize("wdtype", [torch.float32, torch.bfloat16])
def test_smallest_scales(wdtype):
    """Blocks whose largest value is 2^-95 down to the type's least, ties among them, as weights and as hidden states, by every
    kernel that widens them: read back exactly."""
    K = 128
    g = torch.Generator().manual_seed(14)
    least = -149 if wdtype == torch.float32 else -133
    rows = range(-95, least - 1, -1)
    v = torch.randn(len(rows), K, generator=g, dtype=torch.float64)
    v[:, 0], v[:, 1:40], v[:, 40:60], v[:, 60:90] = 1.0, v[:, 1:40] * 2.0 ** -6, torch.arange(1, 21) * 2.0 ** -10, torch.arange(1, 31) * 2.0 ** -5
    v = (v.clamp(-1, 1) * 2.0 ** torch.tensor(list(rows), dtype=torch.float64).view(-1, 1)).to(wdtype)
    want = F.values(v.double().numpy())
    eye = torch.eye(K, dtype=torch.bfloat16, device="cuda")
    wide = torch.zeros(33000, K, dtype=wdtype, device="cuda")
    wide[:len(rows)] = v.cuda()
    odd = torch.zeros(K, K + 1, dtype=torch.bfloat16, device="cuda")[:, :K]  # rows that k_f8_few does not take as they are
    odd.copy_(eye)
    for w, T in ((v.cuda(), (1, 8, 16, 32, 64, 128)), (wide, (16, 64, 128))):
        head = q.Fp8Head(w)
        for x in (eye, odd):
            for t in T:
                got = torch.cat([head(x[i:i + t]) for i in range(0, K, t)]).t()[:len(rows)].double().cpu().numpy()
                assert (got == want).all(), f"{t} states of {w.shape[0]} rows: {np.abs(got - want).max(1)}"
    if wdtype == torch.bfloat16:  # hidden states of that size
        x = torch.zeros(128, K, dtype=wdtype, device="cuda")
        x[:len(rows)] = v.cuda()
        unit = torch.zeros(33000, K, dtype=wdtype, device="cuda")
        unit[:K] = eye
        for w in (eye, unit):
            head = q.Fp8Head(w)
            for t in (1, 8, 16, 32, 64, 128):
                got = torch.cat([head(x[i:i + t])[:, :K] for i in range(0, 128, t)])[:len(rows)].double().cpu().numpy()
                assert (got == want).all(), f"hidden states, {t} at {w.shape[0]} rows"


# Each instance of the kernel for many hidden states (waves of 16 FN weight rows x 16 FT states, two by two), by sizes that
# f8_plan gives to it: in one round of workgroups, and with more than 256 tiles, so that workgroups take a second one, whose
# copies start under the first one's end.  No size is a multiple of a tile's.
TILES = {(4, 3): ((90, 16449, 257), (70, 65601, 130)), (4, 4): ((100, 16449, 257), (100, 65601, 100)), (4, 5): ((131, 16449, 130), (131, 65601, 130)),
         (4, 6): ((170, 16449, 384), (170, 65601, 130)), (4, 7): ((200, 22081, 130), (200, 65601, 100)), (4, 8): ((230, 22081, 257), (230, 65601, 130)),
         (8, 3): ((70, 32833, 130), (70, 100001, 100)), (8, 4): ((100, 32833, 257), (290, 32833, 130)), (8, 5): ((140, 32833, 130), (390, 32833, 100)),
         (8, 6): ((165, 32833, 384), (485, 32833, 130)), (8, 7): ((200, 32833, 130), (390, 49217, 100)), (8, 8): ((240, 43585, 130), (680, 32833, 257))}


@pytest.mark.parametrize("FN,FT,T,N,K", [(*k, *s) for k, v in TILES.items() for s in v])
def test_many_states(FN, FT, T, N, K):
    w, x = data(T, N, K, T + N + K)
    y, tol = product(w, x)
    head = q.Fp8Head(w.cuda())
    buf = torch.full((T, N + 9), 7.0, device="cuda")
    got = head(x.cuda(), out=buf[:, 5:5 + N])
    err = np.abs(got.double().cpu().numpy() - y)
    assert (err <= tol).all(), f"off by {(err / tol).max()} of the bound"
    assert (buf[:, :5] == 7).all() and (buf[:, 5 + N:] == 7).all()
    wide = torch.full((T, N + 9), 7.0, dtype=torch.bfloat16, device="cuda")
    half = head(x.cuda(), out=wide[:, 3:3 + N])
    assert torch.equal(half, got.to(torch.bfloat16)) and (wide[:, :3] == 7).all() and (wide[:, 3 + N:] == 7).all()
    assert torch.equal(head(x.cuda(), dtype=torch.bfloat16), half)
    g = torch.Generator().manual_seed(T)
    tokens = torch.randint(0, N, (T,), generator=g).to(torch.int32)
    tokens[1], tokens[2], tokens[3], tokens[-1] = -1, N, N - 1, 0
    t = 0.3 + 2 * torch.rand(T, generator=g)
    for temperature in (None, t):
        lp, h = (v.double().cpu().numpy() for v in head.score(x.cuda(), tokens.cuda(), temperature=temperature.cuda() if temperature is not None else None))
        assert np.isfinite(lp).all() and np.isfinite(h).all()
        for r in sorted({*range(5), *range(5, T, 13), *range(T - 5, T)}):  # the bounds of test_score
            temp = 1.0 if temperature is None else float(t[r])
            want, _, wh, _, _ = L.row(y[r], [int(tokens[r])], 0, temp)
            off, sums = tol[r].max() / temp, (256 + 30) * 2.0 ** -24
            assert abs(lp[r] - want[0]) <= 2 * off + sums + 8 * abs(want[0]) * 2.0 ** -24, f"row {r}: {lp[r]} {want[0]}"
            assert abs(h[r] - wh) <= off * (2 * np.log(N) + 2) + sums * (1 + 2 * wh), f"row {r}: entropy {h[r]} {wh}"
        # every row against the log probabilities of the same logits
        same = q.LogProbs("cuda")(got, tokens.cuda(), temperature=temperature.cuda() if temperature is not None else None)
        assert torch.allclose(torch.from_numpy(lp).float(), same.logprobs.cpu(), atol=5e-5, rtol=1e-5)
        assert torch.allclose(torch.from_numpy(h).float(), same.entropy.cpu(), atol=5e-5, rtol=1e-5)
