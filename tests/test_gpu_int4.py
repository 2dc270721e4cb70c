"""Int4Head (qws_int4_* through the Python wrapper) against the 64-bit definition (oracle/int4.py).

The packed weights are read back exactly (products with unit vectors).  A logit is a sum over groups of s (D - (16 + z) X): D and X
are sums of at most `group` exact products in fp32, off by at most group 2^-23 of their terms' magnitudes (a rounding, or a
truncation, of each partial sum), and the K / group scaled ones are summed with a rounding each, in four parts: within
(group + K / group + 8) 2^-23 of sum s ((16 + q) + (16 + z)) |x|."""
import numpy as np
import pytest
import torch

import qwen_warp_amd as q
from oracle import int4 as I
from qwen_warp_amd import _lib

pytestmark = pytest.mark.gpu
INF = float("inf")


def weights(N, K, seed, wdtype=torch.bfloat16):
    g = torch.Generator().manual_seed(seed)
    w = torch.randn(N, K, generator=g) * (0.01 + 0.05 * torch.rand(N, 1, generator=g))
    w[:, ::61] *= 5
    return w.to(wdtype)


def states(T, K, seed):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(T, K, generator=g) * (0.1 + 3 * torch.rand(T, 1, generator=g))
    x[:, ::37] *= 8
    return x.to(torch.bfloat16)


def codes_of(N, K, group, seed, zeros, dtype=torch.float16):
    g = torch.Generator().manual_seed(seed)
    codes = torch.randint(0, 16, (N, K), generator=g, dtype=torch.uint8)
    shape = (N, -(-K // group))
    scales = (0.001 + 0.01 * torch.rand(shape, generator=g)).to(dtype)
    return codes, scales, torch.randint(0, 16, shape, generator=g, dtype=torch.uint8) if zeros else None


def product(x, codes, scales, zeros, group):
    """(logits, their bound) in 64 bits"""
    x = x.double().numpy()
    k = codes.shape[1]
    w = I.values(codes, scales, zeros, group)
    z = np.full(scales.shape, 8.0) if zeros is None else zeros & 15
    size = np.repeat(np.abs(scales), group, 1)[:, :k] * (32.0 + (codes & 15) + np.repeat(z, group, 1)[:, :k])
    return x @ w.T, (group + k / group + 8) * 2.0 ** -23 * (np.abs(x) @ size.T)


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("wdtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("N,K", [(1, 1), (5, 127), (16, 128), (300, 129), (257, 300), (64, 640)])
def test_weights_read_back(N, K, wdtype, group):
    w = weights(N, K, N + K, wdtype)
    w[0] = 0.0
    w[-1, 0] = 2.0 ** -100
    want = I.values(*I.quantise(w.float().numpy(), group), group)
    eye = torch.eye(K, dtype=torch.bfloat16, device="cuda")
    for pad in (0, 1):
        v = torch.zeros(N, K + pad, dtype=wdtype, device="cuda")[:, :K]
        v.copy_(w)
        got = q.Int4Head(v, group=group)(eye).t().double().cpu().numpy()
        assert (got == want).all()


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_codes_read_back(group, zeros, dtype):
    """Codes, scales (subnormal fp16 ones too, negative ones, zero) and zero points at any stride; high bits of a byte do not count."""
    N, K = 70, 333
    codes, scales, z = codes_of(N, K, group, group, zeros, dtype)
    scales[0, 0], scales[1, 0], scales[2, 0] = 0.0, 2.0 ** -24, -0.5
    want = I.values(codes.numpy(), scales.double().numpy(), None if z is None else z.numpy(), group)
    eye = torch.eye(K, dtype=torch.bfloat16, device="cuda")
    wide = lambda t, k: torch.nn.functional.pad(t, (0, k)).cuda()[:, :t.shape[1]]  # noqa: E731
    for pad in (0, 3):
        high = torch.randint(0, 16, codes.shape, dtype=torch.uint8) * 16 if pad else 0
        head = q.Int4Head.from_codes(wide(codes + high, pad), wide(scales, pad), wide(z, pad) if zeros else None, group=group)
        assert (head(eye).t().double().cpu().numpy() == want).all()


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("T,N,K", [(1, 1, 1), (1, 1000, 100), (2, 15, 128), (3, 8191, 1000), (7, 129, 5120), (16, 4096, 640), (17, 1000, 257), (33, 700, 512), (48, 65, 96),
                                   (64, 513, 385), (65, 300, 1024), (100, 2001, 136), (129, 255, 2000), (200, 1300, 768)])
def test_logits(T, N, K, group):
    w, x = weights(N, K, T + N + K), states(T, K, T)
    want, tol = product(x, *I.quantise(w.float().numpy(), group), group)
    head = q.Int4Head(w.cuda(), group=group)
    for pad in (0, 3, 8):
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


@pytest.mark.parametrize("T", [1, 5, 40])
def test_large_head(T):
    """More tiles than the card holds at once; a given checkpoint's codes."""
    N, K, group = 70001, 768, 64
    codes, scales, z = codes_of(N, K, group, T, True)
    x = states(T, K, T)
    want, tol = product(x, codes.numpy(), scales.double().numpy(), z.numpy(), group)
    got = q.Int4Head.from_codes(codes.cuda(), scales.cuda(), z.cuda(), group=group)(x.cuda()).double().cpu().numpy()
    assert (np.abs(got - want) <= tol).all()


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("T,frags", [(5, 0), (12, 1), (16, 1), (25, 2), (41, 3), (64, 4), (100, 4), (70, 3)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_tiles(T, frags, group, dtype):
    """Heads of many rows, 16 frags states a tile (0: the rows' own kernel): an odd number of blocks of K, the last tile partly
    past N; the reference by torch in 64 bits on the GPU.  bf16 logits are the fp32 ones rounded."""
    N, K, kb = 50001, 2600, 21
    head_bytes = _lib.load().qws_int4_head_ws_bytes(T, N, K, group)
    assert head_bytes == (-(-T // (16 * frags)) * (kb + 1) * (4 * frags + 1) * 1024 if frags else (T * kb * 256 + 255) // 256 * 256)
    g = torch.Generator("cuda").manual_seed(T)
    codes = torch.randint(0, 16, (N, K), generator=g, dtype=torch.uint8, device="cuda")
    shape = (N, -(-K // group))
    scales = (0.001 + 0.01 * torch.rand(shape, generator=g, device="cuda")).to(torch.bfloat16)
    z = torch.randint(0, 16, shape, generator=g, dtype=torch.uint8, device="cuda")
    x = states(T, K, T).cuda()
    head = q.Int4Head.from_codes(codes, scales, z, group=group)
    got = head(x)
    spread = lambda t: t.double().repeat_interleave(group, 1)[:, :K]  # noqa: E731
    want = x.double() @ (spread(scales) * (codes.double() - spread(z))).t()
    size = x.double().abs() @ (spread(scales) * (32 + codes.double() + spread(z))).t()
    assert ((got.double() - want).abs() <= (group + K / group + 8) * 2.0 ** -23 * size).all()
    if dtype == torch.bfloat16:
        assert torch.equal(head(x, dtype=dtype).view(torch.int16), got.to(dtype).view(torch.int16))
        buf = torch.full((T, N + 9), 7.0, dtype=dtype, device="cuda")
        head(x, out=buf[:, 5:5 + N])
        assert torch.equal(buf[:, 5:5 + N], got.to(dtype)) and (buf[:, :5] == 7).all() and (buf[:, 5 + N:] == 7).all()


def test_rows_do_not_depend_on_the_batch():
    w, x = weights(3000, 1280, 5), states(300, 1280, 6)
    head = q.Int4Head(w.cuda())
    want, tol = product(x, *I.quantise(w.float().numpy(), 128), 128)
    x = x.cuda()
    for T in (1, 15, 31, 64, 96, 150, 300):
        got = head(x[:T])
        assert (np.abs(got.double().cpu().numpy() - want[:T]) <= tol[:T]).all(), T
        assert torch.equal(got, head(x[:T]))


@pytest.mark.parametrize("T,N,K,group", [(1, 1 << 24, 32, 32), (2, 70, 1 << 20, 128), (3000, 200, 96, 64), (40, 300, 70001, 32)])
def test_largest_sizes(T, N, K, group):
    """The limits of N and K, many hidden states of a small head, a long K for tiles; the reference by torch in 64 bits on the GPU."""
    g = torch.Generator("cuda").manual_seed(T)
    codes = torch.randint(0, 16, (N, K), generator=g, dtype=torch.uint8, device="cuda")
    scales = (0.001 + 0.01 * torch.rand((N, -(-K // group)), generator=g, device="cuda")).to(torch.bfloat16)
    x = states(T, K, 3).cuda()
    got = q.Int4Head.from_codes(codes, scales, group=group)(x)
    for rows in (slice(0, 1 << 13), slice(max(0, N - (1 << 13)), N)):
        s = scales[rows].double().repeat_interleave(group, 1)[:, :K]
        want = x.double() @ (s * (codes[rows].double() - 8)).t()
        size = x.double().abs() @ (s * (40 + codes[rows].double())).t()
        assert ((got[:, rows].double() - want).abs() <= (group + K / group + 8) * 2.0 ** -23 * size).all()
    with pytest.raises(q.ValidationError):
        q.Int4Head(torch.empty(1, 1, device="cuda").expand(1, (1 << 20) + 1))


def test_special_values():
    """Zeros give zeros; a row with NaN or an infinity is NaN, the others are not touched by it."""
    w, x = weights(500, 300, 6), states(20, 300, 7)
    want, tol = product(x, *I.quantise(w.float().numpy(), 32), 32)
    x[3] = 0
    x[5, 17], x[6, 299], x[7, 0] = float("nan"), INF, -INF
    wn = w.clone()
    wn[11, 4], wn[12, 299] = INF, float("nan")
    got = q.Int4Head(wn.cuda(), group=32)(x.cuda()).double().cpu().numpy()
    nan = np.zeros((20, 500), bool)
    nan[5:8] = True
    nan[:, 11:13] = True
    want[3] = 0
    assert (np.isnan(got) == nan).all()
    assert (np.abs(got - want)[~nan] <= tol[~nan]).all()


def test_no_states_and_refusals():
    head = q.Int4Head(weights(70, 40, 1).cuda(), group=32)
    assert head(torch.empty(0, 40, dtype=torch.bfloat16, device="cuda")).shape == (0, 70)
    x = states(2, 40, 1).cuda()
    for bad in (x.float(), x[0], x[:, :39], x.cpu(), x.t().contiguous().t()):
        with pytest.raises(q.ValidationError):
            head(bad)
    for kw in (dict(dtype=torch.float16), dict(out=torch.empty(2, 69, device="cuda")), dict(out=torch.empty(2, 70, dtype=torch.int32, device="cuda")),
               dict(out=torch.empty(2, 70)), dict(out=torch.empty(1, 70, device="cuda").expand(2, 70))):
        with pytest.raises(q.ValidationError):
            head(x, **kw)
    w = weights(8, 64, 1).cuda()
    for bad in (dict(w=w, group=16), dict(w=w.half()), dict(w=w[0]), dict(w=w[:0])):
        with pytest.raises(q.ValidationError):
            q.Int4Head(**bad)
    codes, scales, z = (t.cuda() for t in codes_of(8, 64, 32, 1, True))
    for bad in ((codes.int(), scales, z), (codes, scales.float(), z), (codes, scales[:, :1], z), (codes, scales, z.int()), (codes, scales, z[:4]), (codes, scales.cpu(), z)):
        with pytest.raises(q.ValidationError):
            q.Int4Head.from_codes(*bad, group=32)
    with pytest.raises(q.ValidationError):
        q.Int4Head.from_codes(codes, scales, z, group=48)


def test_streams_and_graph():
    """A captured call replays into its own buffers, with new hidden states and with work between the replays."""
    w, x = weights(2000, 520, 3).cuda(), states(9, 520, 4).cuda()
    head = q.Int4Head(w, group=64)
    other = [states(9, 520, s).cuda() for s in range(5, 9)]
    want = [head(o).clone() for o in other]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        first = head(other[0])
    side.synchronize()
    assert torch.equal(first, want[0])
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = head(x)
    for o, y in zip(other, want):
        x.copy_(o)
        g.replay()
        assert torch.equal(head(o), y)
        torch.cuda.synchronize()
        assert torch.equal(got, y)


def test_hidden_states_of_a_trained_model():
    """Hidden states that require a gradient: taken under no_grad, and weights that do are packed as they are."""
    w, x = weights(300, 64, 1).cuda().requires_grad_(), states(3, 64, 2).cuda()
    head = q.Int4Head(w, group=32)
    leaf = x.clone().requires_grad_()
    with pytest.raises(q.ValidationError):
        head(leaf)
    with torch.no_grad():
        got = head(leaf)
    assert torch.equal(got, head(x)) and torch.equal(head(leaf.detach()), got) and not got.requires_grad


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("T,N,K,frags", [(1, 8191, 5120, 0), (5, 50001, 5120, 0), (30, 8191, 5120, 0), (30, 32001, 5120, 0), (50, 16001, 5120, 0), (100, 39589, 256, 0), (3, 8191, 1000, 0),
                                         (16, 50001, 5120, 1), (30, 50001, 5120, 2), (48, 50001, 5120, 3), (64, 50001, 5120, 4), (129, 32001, 5120, 3), (100, 32001, 5120, 4), (48, 50001, 2600, 3)])
def test_sums_are_fp32(T, N, K, frags, group):
    """The logits' error as a whole, at the sizes where the bound of each (above) is a percent of a logit.  With codes and zero points
    uniform over 0 .. 15 and independent hidden states of size 1, a sum of i terms (16 + q) x or (16 + z) x is about 24 sqrt(i).  Were
    each of a group's g additions rounded, independently and by at most 2^-24 of the sum, a group's two sums would be off by
    24 sqrt(2 g^2 / 2) 2^-24, and its result is about 6.5 sqrt(g) (q - z has variance 2 (16^2 - 1) / 12): 3.7 sqrt(g) 2^-24 of it.  The
    K / g scaled ones add less than sqrt(K / g) 2^-24, the last steps a few.  Group sums in fp16 put the logits off by 1e-3, in 16 bits by 3e-5."""
    if frags:
        kb = -(-K // 128)
        assert _lib.load().qws_int4_head_ws_bytes(T, N, K, group) == -(-T // (16 * frags)) * (kb + kb % 2) * (4 * frags + 1) * 1024
    g = torch.Generator("cuda").manual_seed(T + N)
    codes = torch.randint(0, 16, (N, K), generator=g, dtype=torch.uint8, device="cuda")
    shape = (N, -(-K // group))
    z = torch.randint(0, 16, shape, generator=g, dtype=torch.uint8, device="cuda")
    scales = (0.004 + 0.004 * torch.rand(shape, generator=g, device="cuda")).to(torch.bfloat16)
    x = torch.randn(T, K, generator=g, device="cuda").to(torch.bfloat16)
    got = q.Int4Head.from_codes(codes, scales, z, group=group)(x)
    spread = lambda t: t.double().repeat_interleave(group, 1)[:, :K]  # noqa: E731
    want = x.double() @ (spread(scales) * (codes.double() - spread(z))).t()
    off = float((got.double() - want).norm() / want.norm())
    assert off <= (4 * group ** 0.5 + (K / group) ** 0.5 + 4) * 2.0 ** -24
