"""LogProbs (qws_logprobs through the Python wrapper) against the 64-bit definition (oracle/logprobs.py): ranks and
alternatives bit-exact, log probabilities and entropies within the bound of their fp32 sums.

The bound, in units of u = 2^-24.  A lane adds a chain of elements, parts are joined over 6 lane levels, the waves and the
row's workgroups (at most 9 levels of ours, 3 roundings each), every weight 2^d has the error of its exponential (2 u) and of
d (2 u |d| ln 2, and 2^d |d| ln 2 < 1 / e): under (chain + 64) u relative in s, and as much again in t.  So ln s is off by
(chain + 66) u + u ln s, a log probability by that and 4 u |log p|, the entropy by (chain + 66) (1 + 2 H) u + 4 u H."""
import numpy as np
import pytest
import torch

import qwen_warp_amd as q
from oracle import logprobs as L

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
INF = float("inf")


def chain(R, V):
    return 64 + (R * V) // (2048 * 256) * 2


def layout(x, pad=0, offset=0):
    """x [R, V] on the GPU in rows of V + pad elements that start `offset` elements behind an aligned address; NaN around."""
    R, V = x.shape
    buf = torch.full((R * (V + pad) + offset + 16,), float("nan"), dtype=x.dtype, device="cuda")
    y = buf[offset:offset + R * (V + pad)].view(R, V + pad)[:, :V]
    y.copy_(x)
    return y


def compare(x, tokens, top, temperature, out, label):
    """x [R, V] as the kernel reads it, tokens [R, M]; out: a result with those shapes."""
    R, V = x.shape
    xs = x.double().cpu().numpy()
    n = chain(R, V) + 66
    for r in range(R):
        lp, rank, h, ids, tlp = L.row(xs[r], tokens[r].tolist(), top, 1.0 if temperature is None else float(temperature[r]))
        at = f"{label} row {r}"
        assert out.ranks[r].tolist() == rank.tolist(), at
        assert out.top_ids[r].tolist() == ids.tolist(), at
        ln_s = 30.0
        for got, want, what in ((out.logprobs[r], lp, "log p"), (out.top_logprobs[r], tlp, "alternatives")):
            got = got.double().cpu().numpy()
            with np.errstate(over="ignore"):
                want = want.astype(np.float32).astype(np.float64)
            fine = np.isfinite(want)
            assert (got[~fine] == want[~fine]).all(), f"{at}: {what}"
            assert (np.abs(got - want)[fine] <= (n + ln_s + 6 * np.abs(want[fine])) * U).all(), f"{at}: {what} off by {np.abs(got - want)[fine].max()}"
        assert abs(float(out.entropy[r]) - h) <= (n * (1 + 2 * h) + 6 * h) * U, f"{at}: entropy {float(out.entropy[r])} {h}"


def check(x, tokens, top=0, temperature=None, label="", pad=0, offset=0):
    y = layout(x.cuda(), pad, offset)
    out = q.LogProbs("cuda")(y, tokens.cuda(), top=top, temperature=temperature.cuda() if temperature is not None else None)
    torch.cuda.synchronize()
    compare(x, tokens.view(x.shape[0], -1), top, temperature, out._replace(logprobs=out.logprobs.view(x.shape[0], -1), ranks=out.ranks.view(x.shape[0], -1)), label)
    return out


def rows(R, V, dtype, seed, scale=3.0):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(R, V, generator=g) * scale).to(dtype)
    return x, g


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("R,V,pad,offset", [(1, 1, 0, 0), (3, 2, 0, 1), (2, 63, 1, 0), (2, 64, 0, 3), (5, 65, 6, 5), (1, 1023, 0, 7), (3, 2049, 2, 1), (2, 8192, 0, 0),
                                            (4, 12345, 3, 2), (1, 70001, 0, 1)])
def test_shapes(dtype, R, V, pad, offset):
    x, g = rows(R, V, dtype, R * V + pad)
    for M, top in ((1, 0), (1, 1), (3, 5), (64, 64)):
        tokens = torch.randint(0, V, (R, M), generator=g).to(torch.int32)
        check(x, tokens, top, None, f"M={M} top={top}", pad, offset)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_full_vocabulary(dtype):
    x, g = rows(3, 248320, dtype, 7)
    x[0, 1000:1032] += 12
    tokens = torch.tensor([1005, 77, 248319], dtype=torch.int32)
    check(x, tokens, 20, torch.tensor([0.3, 1.0, 2.5]), "full", 0, 0)
    check(x, tokens, 64, None, "full, misaligned", 5, 3)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_many_rows(dtype):
    """Rows enough that a workgroup takes several stripes of one (the parts of a row are then fewer and longer)."""
    x, g = rows(700, 30011, dtype, 8)
    tokens = torch.randint(-1, 30011, (700, 2), generator=g).to(torch.int32)
    check(x, tokens, 6, None, "many rows", 1, 0)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_orders(dtype):
    """Ascending, descending, flat and blockwise rows: the alternatives are exact whatever the order in memory."""
    V = 9001
    up = torch.arange(V, dtype=torch.float32) / 16
    block = torch.zeros(V)
    block[64 * 5:64 * 6] = 3.0  # one group holds every alternative
    stride = torch.zeros(V)
    stride[::64] = 5.0  # every group has the same maximum
    x = torch.stack([up, up.flip(0), torch.zeros(V), block, stride, torch.full((V,), -7.5)]).to(dtype)
    tokens = torch.tensor([[0, V - 1, 320, 4000]] * 6, dtype=torch.int32)
    for top in (1, 20, 64):
        check(x, tokens, top, None, f"orders top={top}", 3, 1)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_ties_in_few_places(dtype):
    """Many groups of 64 logits tie, their ties in fewer places than alternatives are asked for: the selections then list as
    many keys as they ever can."""
    V = 9001
    x = torch.zeros(8, V)
    places = torch.arange(V) % 64
    for r, (groups, lanes) in enumerate(((40, 19), (64, 19), (64, 4), (140, 1), (21, 20), (30, 64), (63, 7), (140, 19))):
        x[r, (torch.arange(V) // 64 < groups) & (places < lanes)] = 5.0
    x[1] -= 3.0
    tokens = torch.tensor([[0, 18, 19, 64, 9000]] * 8, dtype=torch.int32)
    for top in (5, 8, 9, 20, 45, 63, 64):
        for pad, offset in ((0, 0), (3, 1)):
            check(x.to(dtype), tokens, top, None, f"ties top={top}", pad, offset)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("temperature", [None, 0.4, 1.7])
def test_masks(dtype, temperature):
    """Rows of nothing, of one token, with NaN, infinities and the type's lowest value, alone and mixed."""
    V = 5003
    low, nan = torch.finfo(dtype).min, float("nan")
    x, g = rows(14, V, dtype, 9)
    x[0] = -INF
    x[1] = nan
    x[2] = -INF
    x[2, 4321] = -3.0
    x[3] = low
    x[4] = low
    x[4, [7, 4000]] = 2.0
    x[5, :] = -INF
    x[5, ::1000] = low
    x[6, ::2] = nan
    x[7, 1::3] = -INF
    x[8, 17] = INF
    x[9, [3, 5000]] = INF
    x[10] = -INF
    x[10, :3] = torch.tensor([1.0, 3.0, 2.0])
    x[11] = torch.finfo(dtype).max
    x[12] = -INF
    x[12, 9] = INF
    x[13, 0], x[13, 1], x[13, 2:] = 0.0, -0.0, -1.0
    tokens = torch.tensor([[0, 4321, 17, 3, 5000, 7, 1, -1, V, 2 ** 31 - 1]] * 14, dtype=torch.int32)
    t = torch.full((14,), temperature) if temperature else None
    for pad, offset in ((0, 0), (1, 3)):
        check(x, tokens, 5, t, f"masks {pad}", pad, offset)
        check(x, tokens[:, 0].contiguous(), 0, t, f"masks, one token {pad}", pad, offset)


def test_temperatures():
    """0 and NaN read as 1; tiny, huge and infinite ones give the limits (a point mass, a uniform row)."""
    V = 3000
    x, _ = rows(6, V, torch.float32, 10)
    x[:, 11] = 40.0
    t = torch.tensor([0.0, float("nan"), 1e-40, 1e-6, 1e30, INF])
    tokens = torch.full((6,), 11, dtype=torch.int32)
    out = q.LogProbs("cuda")(x.cuda(), tokens.cuda(), top=2, temperature=t.cuda())
    one = q.LogProbs("cuda")(x.cuda(), tokens.cuda(), top=2)
    assert torch.equal(out.logprobs[:2], one.logprobs[:2]) and torch.equal(out.entropy[:2], one.entropy[:2])
    assert (out.logprobs[2:4] == 0).all() and (out.entropy[2:4] == 0).all()
    assert torch.allclose(out.logprobs[4:].cpu(), torch.full((2,), -np.log(V), dtype=torch.float32), atol=1e-4)
    assert torch.allclose(out.entropy[4:].cpu(), torch.full((2,), np.log(V), dtype=torch.float32), atol=1e-4)
    assert torch.equal(out.top_ids, one.top_ids) and torch.equal(out.ranks, one.ranks)


def test_large_logits_and_values():
    """Logits of 1e4 and 1e30: differences to the maximum are taken first."""
    for scale in (1e4, 1e30):
        x, g = rows(3, 4097, torch.float32, 11)
        x = x * scale
        x[1, 5] = x[1].max()
        check(x, torch.tensor([[5, 9], [5, 9], [5, 9]], dtype=torch.int32), 4, None, f"scale {scale}")


def test_leading_dimensions_strides_and_outputs():
    """[B, K + 1, V] logits with a verify call's tokens; rows shared by a stride of 0; nothing but the entropy."""
    x, g = rows(12, 777, torch.float32, 12)
    tokens = torch.randint(0, 777, (4, 3), generator=g).to(torch.int32)
    tokens[1, 2] = -1
    op = q.LogProbs("cuda")
    out = op(x.view(4, 3, 777).cuda(), tokens.cuda(), top=3)
    assert out.logprobs.shape == (4, 3) and out.ranks.shape == (4, 3) and out.entropy.shape == (4, 3) and out.top_ids.shape == (4, 3, 3)
    flat = op(x.cuda(), tokens.view(12).cuda(), top=3)
    assert all(torch.equal(a.flatten(), b.flatten()) for a, b in zip(out, flat))
    assert out.logprobs[1, 2] == 0 and out.ranks[1, 2] == -1
    labels = op(x.view(4, 3, 777).cuda(), tokens.view(4, 3, 1).expand(4, 3, 5).contiguous().cuda())
    assert labels.logprobs.shape == (4, 3, 5) and torch.equal(labels.logprobs[..., 4], out.logprobs) and torch.equal(labels.ranks[..., 2], out.ranks)
    shared = op(x[:1].cuda().expand(6, 777), torch.arange(6, dtype=torch.int32, device="cuda"), top=2)
    assert (shared.entropy == shared.entropy[0]).all() and shared.ranks.unique().numel() == 6
    bare = op(x.cuda())
    assert bare.logprobs is None and bare.ranks is None and torch.equal(bare.entropy.view(4, 3), out.entropy) and bare.top_ids.shape == (12, 0)
    no_ranks = op(x.cuda(), tokens.view(12).cuda(), ranks=False)
    assert no_ranks.ranks is None and torch.equal(no_ranks.logprobs.view(4, 3), out.logprobs)
    empty = op(torch.empty(0, 777, device="cuda"), torch.empty(0, dtype=torch.int32, device="cuda"), top=3)
    assert empty.logprobs.shape == (0,) and empty.top_ids.shape == (0, 3)


def test_widest_vocabulary():
    V = 1 << 19
    for dtype in (torch.float32, torch.bfloat16):
        x, g = rows(2, V, dtype, 13)
        check(x, torch.tensor([[V - 1], [0]], dtype=torch.int32), 64, None, "widest", 1, 1)
    with pytest.raises(RuntimeError):
        q.LogProbs("cuda")(torch.zeros(1, V + 1, device="cuda"))


def test_offsets_past_32_bits():
    """Rows 2^31 + 8 elements apart."""
    stride, V = (1 << 31) + 8, 5000
    buf = torch.zeros(stride + V, dtype=torch.bfloat16, device="cuda")
    x, _ = rows(2, V, torch.bfloat16, 14)
    y = buf.as_strided((2, V), (stride, 1))
    y.copy_(x)
    tokens = torch.tensor([[3], [4999]], dtype=torch.int32)
    out = q.LogProbs("cuda")(y, tokens.cuda(), top=8)
    compare(x, tokens, 8, None, out, "far rows")


def test_streams_and_repeats():
    """The same bits on every run and on another stream, also with calls of other shapes in between."""
    x, g = rows(40, 20000, torch.float32, 15)
    x, tokens = x.cuda(), torch.randint(0, 20000, (40,), generator=g).to(torch.int32).cuda()
    op = q.LogProbs("cuda")
    first = op(x, tokens, top=20)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for i in range(5):
        op(x[: 1 + i], tokens[: 1 + i], top=1)
        with torch.cuda.stream(side):
            other = op(x, tokens, top=20)
        side.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(first, other))
        assert all(torch.equal(a, b) for a, b in zip(first, op(x, tokens, top=20)))


def test_graph():
    """A captured call, replayed with new logits in place and eager work in between."""
    x, g = rows(8, 30000, torch.bfloat16, 16)
    buf, tokens = x.cuda(), torch.randint(0, 30000, (8,), generator=g).to(torch.int32).cuda()
    op = q.LogProbs("cuda")
    op(buf, tokens, top=5)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = op(buf, tokens, top=5)
    for i in range(4):
        buf.copy_(rows(8, 30000, torch.bfloat16, 100 + i)[0])
        want = [t.clone() for t in op(buf, tokens, top=5)]
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want)), f"replay {i}"


def test_refusals():
    op = q.LogProbs("cuda")
    x = torch.zeros(4, 100, device="cuda")
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")  # noqa: E731
    for call in (lambda: op(x.half()), lambda: op(x.t()), lambda: op(x[0]), lambda: op(x, i32(3)), lambda: op(x, i32(4).long()), lambda: op(x, i32(4).cpu()),
                 lambda: op(x, i32(4, 65)), lambda: op(x, i32(4, 0)), lambda: op(x, i32(8)[::2]), lambda: op(x, top=65), lambda: op(x, top=-1),
                 lambda: op(x, temperature=torch.ones(3, device="cuda")), lambda: op(x, temperature=torch.ones(4)), lambda: op(x.double())):
        with pytest.raises(q.ValidationError):
            call()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("R", [12, 84])
def test_small_temperatures(dtype, R):
    """Ordinary logits at temperatures that a near-greedy request may have, down to 1e-30: a sure row, two equal best logits
    and two neighbours, in both forms of the pass (one and several vectors of a thread)."""
    V = 32000
    x, g = rows(R, V, dtype, 17)
    x[:, 77] = 20.0
    x[1::3, 31999] = 20.0
    x[2::3, 5] = float(np.nextafter(np.float32(20), np.float32(0))) if dtype == torch.float32 else 19.875
    t = torch.tensor([1e-5, 1e-6, 1e-7, 1e-8, 5e-9, 3e-9, 1e-9, 1e-10, 1e-12, 1e-17, 1e-18, 1e-30]).repeat_interleave(R // 12)
    tokens = torch.randint(0, V, (R,), generator=g).to(torch.int32)
    tokens[::2] = 77
    check(x, tokens, 3, t[torch.randperm(R, generator=g)], "small temperatures")
    check(x, tokens.view(R, 1).expand(R, 3).contiguous(), 0, t, "small temperatures, several tokens")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("R", [12, 84])
@pytest.mark.parametrize("temperature", [None, 0.7])
def test_finite_masks(dtype, R, temperature):
    """All but a dozen tokens masked with a finite value, rows of nothing but that value, and logits as large."""
    V = 32000
    x, g = rows(R, V, dtype, 18)
    values = [-1e4, -1e7, -1e9, -1e10, -5e10, -1e11, -1e12, -1e13, -1e14, -1e15, -1e20, -1e30]
    few = torch.rand(R, V, generator=g) * V < 12
    for r in range(R):
        value = values[r % 12]
        if r < 60:
            x[r, ~few[r]] = value
        elif r < 72:
            x[r] = value
        else:
            x[r] *= -value
    tokens = torch.randint(0, V, (R,), generator=g).to(torch.int32)
    tokens[::2] = torch.where(few, x.float(), -INF).argmax(1)[::2].to(torch.int32)
    t = torch.full((R,), temperature) if temperature else None
    check(x, tokens, 5, t, "finite masks", 1, 3)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("temperature", [None, 0.37])
def test_signs(dtype, temperature):
    """No log probability above 0 and no entropy below 0: rows with one sure token, whose best logits differ, and rows of one token."""
    for R, V in ((400, 1500), (300, 30011), (64, 1)):
        x, g = rows(R, V, dtype, 19)
        x[:, V // 2] = (60.0 + 10 * torch.rand(R, generator=g)).to(dtype)
        tokens = torch.full((R,), V // 2, dtype=torch.int32)
        t = torch.full((R,), temperature) if temperature else None
        out = check(x, tokens, 2, t, "signs")
        assert (out.logprobs <= 0).all() and (out.top_logprobs <= 0).all() and (out.entropy >= 0).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("R", [6, 180])
def test_signalling_nan(dtype, R):
    """NaN of both kinds and signs counts as -inf: as a given token, among the best, in a row of nothing else, in both forms of the pass."""
    V = 16001
    ints, codes = (torch.int32, (0x7F800001, -0x7FFFFF, 0x7FBFFFFF, 0x7FC00000, -1)) if dtype == torch.float32 else (torch.int16, (0x7F81, -0x7F, 0x7FBF, 0x7FC0, -1))
    x, g = rows(R, V, dtype, 20)
    for r in range(R):
        bits = x[r].view(ints)
        if r % 6 == 5:
            bits[:] = codes[r // 6 % 5]
            if r % 12 == 11:
                x[r, 9000] = -2.0
        else:
            bits[[0, 63, 64, 777, 1023, 9000, 16000]] = codes[r % 5]
    assert x.isnan().sum() > 7 * R // 2
    tokens = torch.tensor([[0, 777, 5, 16000]], dtype=torch.int32).repeat(R, 1)
    check(x, tokens, 3, None, "signalling NaN", 1, 1)
    check(x, tokens[:, 1].contiguous(), 3, torch.full((R,), 0.6), "signalling NaN, one token")


def test_device():
    """The operator's device is the logits': another one's are refused; without an index, any GPU's are taken."""
    x = torch.zeros(2, 50, device="cuda:0")
    want = q.LogProbs("cuda")(x)
    assert torch.equal(q.LogProbs("cuda:0")(x).entropy, want.entropy) and torch.equal(q.LogProbs(torch.device("cuda", 0))(x).entropy, want.entropy)
    for other in ("cpu", "cuda:1"):
        with pytest.raises(q.ValidationError):
            q.LogProbs(other)(x)


# Rows and vocabularies by the stripes that a workgroup then takes (lp_plan): one, a block of them, two, more, and as many as a
# short row has.  The last workgroup of a row is partly filled in most.
@pytest.mark.parametrize("dtype,R,V,stripes", [(torch.float32, 20, 62465, 1), (torch.float32, 70, 62465, 4), (torch.float32, 400, 62465, 8), (torch.float32, 2200, 62465, 12),
                                               (torch.float32, 1024, 248321, 16), (torch.float32, 3000, 3000, 4), (torch.float32, 3000, 1000, 1),
                                               (torch.bfloat16, 20, 62465, 1), (torch.bfloat16, 100, 62465, 4), (torch.bfloat16, 400, 62465, 8),
                                               (torch.bfloat16, 2700, 62465, 12), (torch.bfloat16, 2048, 248321, 28), (torch.bfloat16, 3000, 3000, 4), (torch.bfloat16, 3000, 1000, 1)])
def test_plans(dtype, R, V, stripes):
    """Every form of the pass (no tokens, one, several; ranks or not; alternatives or not) over ordinary, masked and NaN rows.  A
    lane's chain is its share of the workgroup's stripes; the other roundings are those of the bound above."""
    pad, offset = 3, 5
    g = torch.Generator(device="cuda").manual_seed(R + V)
    buf = torch.full((R * (V + pad) + offset + 16,), float("nan"), dtype=dtype, device="cuda")
    y = buf[offset:offset + R * (V + pad)].view(R, V + pad)[:, :V]
    y.normal_(0, 3, generator=g)
    few = torch.rand(V, device="cuda", generator=g) * V < 12
    y[5::11, ~few] = -INF
    y[7::11, ~few] = torch.finfo(dtype).min
    y[9::11, ~few] = -1e9
    y[3::11, ::7] = float("nan")
    y[2] = -INF
    tokens = torch.randint(0, V, (R, 3), device="cuda", generator=g).to(torch.int32)
    for r in range(0, R, 2):
        tokens[r, 0] = y[r].nan_to_num(nan=-INF).argmax()
    tokens[::5, 2] = -1
    tokens[1::5, 2] = V - 1
    t = 0.4 + 2 * torch.rand(R, device="cuda", generator=g)
    rows_ = sorted({*range(14), R // 2, *range(R - 6, R)})
    n = stripes * 16 // dtype.itemsize + 64 + 66
    op = q.LogProbs("cuda")
    for temperature in (None, t):
        want = {r: L.row(y[r].double().cpu().numpy(), tokens[r].tolist(), 6, 1.0 if temperature is None else float(t[r])) for r in rows_}

        def near(got, of, r, what):
            got = np.atleast_1d(got.double().cpu().numpy())
            of = np.atleast_1d(of).astype(np.float32).astype(np.float64)
            fine = np.isfinite(of)
            assert (got[~fine] == of[~fine]).all(), f"row {r}: {what}"
            assert (np.abs(got[fine] - of[fine]) <= (n + 30 + 6 * np.abs(of[fine])) * U).all(), f"row {r}: {what} {got} {of}"

        for M in (0, 1, 3):
            for ranks in (True, False):
                if not M and not ranks:
                    continue
                for top in (0, 6):
                    given = None if not M else tokens[:, 0].contiguous() if M == 1 else tokens
                    out = op(y, given, top=top, temperature=temperature, ranks=ranks)
                    at = f"M={M} ranks={ranks} top={top}"
                    assert (out.logprobs is None) == (M == 0) and (out.ranks is None) == (not ranks or not M) and out.top_ids.shape == (R, top)
                    assert torch.isfinite(out.entropy).all() and (out.entropy >= 0).all()
                    for r in rows_:
                        lp, rank, h, ids, tlp = want[r]
                        assert abs(float(out.entropy[r]) - h) <= (n * (1 + 2 * h) + 6 * h) * U, f"{at} row {r}: entropy {float(out.entropy[r])} {h}"
                        if M:
                            near(out.logprobs[r], lp[:M], r, at)
                            if ranks:
                                assert out.ranks[r].view(-1).tolist() == rank[:M].tolist(), f"{at} row {r}"
                        if top:
                            assert out.top_ids[r].tolist() == ids.tolist(), f"{at} row {r}"
                            near(out.top_logprobs[r], tlp, r, at)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_largest_differences(dtype):
    """+inf (or the type's largest value) and the lowest value in one row: their difference is past fp32, over the temperature it
    is not."""
    V = 3000
    t = torch.tensor([1.0, 2.0, 4.0, 1e3, 1e30, 1e37, 1e38, 3e38, INF])
    x, _ = rows(18, V, dtype, 21)
    x[:, 5], x[:9, 100], x[9:, 100], x[3:, 2000] = torch.finfo(dtype).min, INF, torch.finfo(dtype).max, torch.finfo(dtype).min
    x[6:9, ::2] = torch.finfo(dtype).min
    tokens = torch.tensor([[5, 100, 7, 2000]], dtype=torch.int32).repeat(18, 1)
    check(x, tokens, 3, t.repeat(2), "differences")
    low = x[:, 5:6].expand(18, 64).contiguous()
    low[:, 7] = INF
    check(low, torch.full((18, 1), 3, dtype=torch.int32), 64, t.repeat(2), "nothing between")


def test_temperatures_that_are_none():
    """0, NaN and negative ones (infinity's among them) read as 1, in LogProbs and in score."""
    x, g = rows(6, 1000, torch.float32, 22)
    t = torch.tensor([0.0, -0.0, float("nan"), -1.0, -1e-30, -INF], device="cuda")
    tokens = torch.randint(0, 1000, (6,), generator=g).to(torch.int32).cuda()
    op = q.LogProbs("cuda")
    assert all(torch.equal(a, b) for a, b in zip(op(x.cuda(), tokens, top=3, temperature=t), op(x.cuda(), tokens, top=3)))
    head = q.Fp8Head(x.t().contiguous().cuda())
    states = torch.randn(6, 6, generator=g).to(torch.bfloat16).cuda()
    assert all(torch.equal(a, b) for a, b in zip(head.score(states, tokens, temperature=t), head.score(states, tokens)))
