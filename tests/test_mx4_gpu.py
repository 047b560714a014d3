"""4-bit matrices (linearcorex_amd.mx4, include/lcx.h lcx_mx4_*) against their definition in float64.

Tolerance of a product: every product of the definition is exact in the kernels, so what is left is (a) the float32 sum - one rounding or
truncation, at most 2^-23 of S = sum |x w|, per accumulation step; an output sees K / 32 steps per bf16 term of x (3 for float32, 2 for
float16, 1) plus 32 inside one instruction and 64 to join partial sums - and (b) one rounding to the output type, finfo.eps / 2."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
from tests import mx4_reference as R                                     # noqa: E402

pytestmark = pytest.mark.gpu
TERMS = {torch.float32: 3, torch.float16: 2, torch.bfloat16: 1}
PRODUCT = [torch.float32, torch.bfloat16, torch.float16]
ids = lambda d: str(d).replace("torch.", "")                            # noqa: E731


@pytest.fixture(scope="module")
def mx4():
    from linearcorex_amd import mx4 as m
    return m


def f64(t):
    return t.detach().cpu().double().numpy()


def tol(xa, wa, dt, terms, want):
    """bound of the module docstring; xa (T, K), wa (N, K) magnitudes"""
    s = xa @ wa.T
    steps = -(-xa.shape[1] // 32) * terms + 32 + 64
    return steps * 2.0 ** -23 * s + torch.finfo(dt).eps / 2 * np.abs(want) * 1.001 + 1e-30 + (2.0 ** -25 if dt == torch.float16 else 0)


def gen(seed):
    return torch.Generator().manual_seed(seed)


def ints(shape, seed, dt, hi=4):
    return torch.randint(-hi, hi + 1, shape, generator=gen(seed)).to(dt).cuda()


# ---- quantisation: to the bit ------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dt", [torch.float32, torch.float64, torch.bfloat16, torch.float16], ids=ids)
@pytest.mark.parametrize("shape", [(1, 1), (1, 33), (5, 31), (7, 513), (3, 256), (65, 100), (130, 2050), (2, 4096), (600, 64)])
@pytest.mark.parametrize("axis", [0, 1])
def test_quantize_to_the_bit(mx4, dt, shape, axis):
    x = torch.randn(shape, generator=gen(shape[0] * 7 + shape[1]), dtype=torch.float64)
    x *= torch.exp2(torch.randint(-12, 12, (shape[0], 1), generator=gen(3)).double())
    x = x.to(dt).cuda()
    q = mx4.quantize(x, axis=axis)
    want = f64(x) if axis == 1 else f64(x).T
    code, byte = R.quantize(want)
    got_code, got_byte = R.unpack(q.codes.cpu().numpy(), q.scales.cpu().numpy(), *want.shape)
    r, c = want.shape
    assert np.array_equal(got_byte[:r, :byte.shape[1]], byte)
    assert np.array_equal(got_code[:r, :c], code)
    # what lies behind the last row and column is defined: zeros and the scale byte 2
    assert not got_code[r:].any() and not got_code[:, c:].any()
    assert (got_byte[r:] == 2).all() and (got_byte[:, byte.shape[1]:] == 2).all()
    val = R.values(code, byte)
    for out in (torch.float32, torch.float64, torch.bfloat16):
        v = mx4.dequantize(q, out)
        assert v.shape == x.shape and v.dtype == out
        assert np.array_equal(f64(v), val if axis == 1 else val.T)
    # float16: one rounding (the bytes of this data reach below its normal range)
    assert np.array_equal(f64(mx4.dequantize(q, torch.float16)), (val if axis == 1 else val.T).astype(np.float16).astype(np.float64))


def edge_values(dt):
    fi = torch.finfo(dt)
    v = [0.0, -0.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 7.0, 7.99, 8.0, -0.25, -5.0, fi.tiny, fi.max, -fi.max, fi.eps, 1.0 - fi.eps]
    m = torch.tensor(v, dtype=torch.float64)
    rows = [torch.cat([m, torch.full((12,), 4.0 * 2.0 ** s, dtype=torch.float64)]) for s in (-3, 0, 1, 5)]
    rows += [torch.full((32,), s, dtype=torch.float64) for s in (0.0, fi.tiny, fi.max, 2.0 ** -14)]
    small = torch.linspace(0, 8, 32, dtype=torch.float64)
    rows += [small * 2.0 ** e for e in (-149, -140, -130, -128, -127, -126, -125, -124, -3, 13, 125)]
    return torch.stack(rows).clamp(-fi.max, fi.max).to(dt)


@pytest.mark.parametrize("dt", [torch.float32, torch.float64, torch.bfloat16, torch.float16], ids=ids)
def test_quantize_ties_extremes_and_non_finite(mx4, dt):
    x = edge_values(dt)
    for bad in (float("inf"), -float("inf"), float("nan")):
        row = torch.ones(1, 32, dtype=dt)
        row[0, 17] = bad
        x = torch.cat([x, row])
    if dt == torch.float64:
        x = torch.cat([x, torch.full((1, 32), 1e300, dtype=dt), torch.full((1, 32), 1e-300, dtype=dt)])
        # a hair beside every tie: must not be rounded to float32 first
        t = torch.tensor([m * s for m in R.MIDS for s in (1 - 2.0 ** -50, 1 + 2.0 ** -50)] + [4.0] * 18, dtype=dt)
        x = torch.cat([x, t[None]])
    x = torch.cat([x, torch.ones_like(x)], dim=1)                       # a clean block beside each
    q = mx4.quantize(x.cuda())
    code, byte = R.quantize(f64(x))
    got_code, got_byte = R.unpack(q.codes.cpu().numpy(), q.scales.cpu().numpy(), *x.shape)
    got_code, got_byte = got_code[:code.shape[0], :code.shape[1]], got_byte[:byte.shape[0], :byte.shape[1]]
    assert np.array_equal(got_byte, byte)
    ok = np.repeat(byte != 255, 32, axis=1)
    assert np.array_equal(got_code[ok], code[ok])
    v = f64(mx4.dequantize(q, torch.float64))
    assert np.isnan(v[~ok]).all() and np.array_equal(v[ok], R.values(code, byte)[ok])


def test_quantize_reads_any_strides(mx4):
    base = torch.randn(260, 1100, generator=gen(5)).cuda()
    views = [base[3:, 5:], base[::2, ::3], base.t(), base.t()[7:300, 1:], base[:, 1:129], base[:1].expand(40, 1100), base[:, :1].expand(260, 77)]
    for x in views + [v.bfloat16() for v in views[:2]] + [base.bfloat16()[1:, 3:]]:
        for axis in (0, 1):
            a, b = mx4.quantize(x, axis=axis), mx4.quantize(x.contiguous(), axis=axis)
            assert torch.equal(a.codes, b.codes) and torch.equal(a.scales, b.scales)


# ---- products ----------------------------------------------------------------------------------------------------------------
# small integers: every partial sum is an integer below 2^24, so any order of summation gives the exact result
SIZES = [(1, 1, 1), (1, 64, 256), (2, 17, 33), (3, 100, 511), (16, 128, 512), (17, 129, 1025), (33, 250, 130), (64, 512, 2048), (100, 333, 777),
         (128, 256, 640), (129, 4100, 96), (200, 70, 3000), (300, 520, 260), (1, 3, 9000), (5, 9000, 40), (40, 31, 5000)]


@pytest.mark.parametrize("dt", PRODUCT, ids=ids)
@pytest.mark.parametrize("m,n,k", SIZES)
def test_products_of_integers_are_exact(mx4, dt, m, n, k):
    x, w, dy = ints((m, k), 1, dt), ints((n, k), 2, torch.float32, hi=2), ints((m, n), 3, dt)
    q = mx4.quantize(w)
    wq = R.round4(f64(w))
    big = 2048.0 if dt == torch.float16 else 256.0 if dt == torch.bfloat16 else 2.0 ** 24
    for got, want in ((mx4.linear(x, q), f64(x) @ wq.T), (mx4.linear_grad(dy, q), f64(dy) @ wq),
                      (mx4.matmul(mx4.quantize(x), q, dt), R.round4(f64(x)) @ wq.T)):
        assert got.dtype == dt and np.abs(want).max() < 2 ** 22
        want = torch.from_numpy(want).to(dt).double().numpy()           # one rounding (exact below 2^8 / 2^11 / 2^24)
        assert np.array_equal(f64(got), want), (np.abs(want).max(), big)


@pytest.mark.parametrize("dt", PRODUCT, ids=ids)
@pytest.mark.parametrize("m,n,k", [(1, 512, 4096), (7, 1000, 2000), (16, 64, 20000), (50, 400, 1500), (256, 300, 700)])
def test_products_of_random_values(mx4, dt, m, n, k):
    x = (torch.randn(m, k, generator=gen(1)) * torch.exp2(torch.randint(-6, 6, (1, k), generator=gen(9)).float())).to(dt).cuda()
    w = torch.randn(n, k, generator=gen(2)) * 0.05
    dy = torch.randn(m, n, generator=gen(3)).to(dt).cuda()
    q = mx4.quantize(w.cuda())
    wq, xf, df = R.round4(w.double().numpy()), f64(x), f64(dy)
    xq = R.round4(xf)
    for got, a, b, terms in ((mx4.linear(x, q), xf, wq, TERMS[dt]), (mx4.linear_grad(dy, q), df, wq.T, TERMS[dt]),
                             (mx4.matmul(mx4.quantize(x), q, dt), xq, wq, 1)):
        want = a @ b.T
        err = np.abs(f64(got) - want)
        assert (err <= tol(np.abs(a), np.abs(b), dt, terms, want)).all(), (err / tol(np.abs(a), np.abs(b), dt, terms, want)).max()


@pytest.mark.parametrize("dt", PRODUCT, ids=ids)
def test_every_bit_of_x_takes_part(mx4, dt):
    """one value per row of W: y is x times a power of two, bit for bit - no term of the split is dropped, no column is mixed up"""
    k, m = 700, 37
    x = torch.randn(m, k, generator=gen(4)).to(dt).cuda()
    w = torch.zeros(k, k)
    perm = torch.randperm(k, generator=gen(5))
    w[torch.arange(k), perm] = 4.0
    q = mx4.quantize(w.cuda())
    assert torch.equal(mx4.linear(x, q), x[:, perm.cuda()] * 4)
    assert torch.equal(mx4.linear_grad(x, q)[:, perm.cuda()], x * 4)
    # tiny and huge values of the type
    fi = torch.finfo(dt)
    for v in (fi.tiny, fi.tiny * 8, fi.max / 8, -fi.max / 8, 1 + fi.eps):
        x[:] = v
        assert torch.equal(mx4.linear(x, q), x[:, perm.cuda()] * 4), v


@pytest.mark.parametrize("dt", PRODUCT, ids=ids)
@pytest.mark.parametrize("m", [1, 5, 40, 200])
def test_blocks_along_the_other_axis(mx4, dt, m):
    w = ints((90, 333), 7, torch.float32, hi=2)
    q = mx4.quantize(w, axis=0)
    wq = R.round4(f64(w).T).T
    x, dy = ints((m, 333), 8, dt), ints((m, 90), 9, dt)
    assert np.array_equal(f64(mx4.linear(x, q)), torch.from_numpy(f64(x) @ wq.T).to(dt).double().numpy())
    assert np.array_equal(f64(mx4.linear_grad(dy, q)), torch.from_numpy(f64(dy) @ wq).to(dt).double().numpy())
    assert torch.equal(mx4.linear(dy, q.t()), mx4.linear_grad(dy, q))
    assert torch.equal(mx4.dequantize(q.t()), mx4.dequantize(q).t())


@pytest.mark.parametrize("dt", PRODUCT, ids=ids)
@pytest.mark.parametrize("m", [1, 4, 70, 140])
def test_activations_of_any_strides(mx4, dt, m):
    q = mx4.quantize(ints((200, 300), 7, torch.float32, hi=2))
    base = ints((2 * m + 3, 901), 8, dt)
    big = ints((901, 2 * m + 3), 8, dt)
    for x in (base[3:3 + m, 1:301], base[:m, :600:2], base[1:1 + 2 * m:2, 601:901], big[:300, :m].t(), big[1:301, 3:3 + m].t(), base[:1, :300].expand(m, 300),
              base[:m, :1].expand(m, 300), base[:1, :1].expand(m, 300)):
        assert torch.equal(mx4.linear(x, q), mx4.linear(x.contiguous(), q))
        assert torch.equal(mx4.linear_grad(x[:, :200], q), mx4.linear_grad(x[:, :200].contiguous(), q))
    x3 = base[:m, :300].reshape(m, 300).expand(2, 3, m, 300)
    y = mx4.linear(x3, q)
    assert y.shape == (2, 3, m, 200) and torch.equal(y[1, 2], mx4.linear(base[:m, :300], q))
    assert torch.equal(mx4.linear(base[0, :300], q), mx4.linear(base[:1, :300], q)[0])


@pytest.mark.parametrize("m", [3, 17, 40, 100, 129, 300])
@pytest.mark.parametrize("n,k", [(64, 128), (192, 384), (640, 1280), (20032, 4096)])
def test_whole_lines_of_bfloat16_take_the_short_way(mx4, m, n, k):
    """rows of whole lines are read in place, others are laid out first: the same sums in the same order, to the bit"""
    q = mx4.quantize(torch.randn(n, k, generator=gen(1)).cuda())
    base, top = torch.randn(2 * m, k + 8, generator=gen(2)).bfloat16().cuda(), torch.randn(2 * m, n + 8, generator=gen(3)).bfloat16().cuda()
    for rows in (slice(0, m), slice(m - 1, 2 * m - 1), slice(0, 2 * m, 2)):
        for f, b, c in ((mx4.linear, base, k), (mx4.linear_grad, top, n)):
            x = b[rows, :c]
            want = f(x, q)
            odd = torch.empty(m, c + 1, dtype=x.dtype, device="cuda")[:, :c].copy_(x)
            col = torch.empty(c, m, dtype=x.dtype, device="cuda").t().copy_(x)
            behind = b[rows, 8:c + 8].clone()[:, :c]
            assert torch.equal(f(odd, q), want) and torch.equal(f(col, q), want) and torch.equal(f(b[rows, 8:], q), f(behind, q))
    one = base[:1, :k].expand(m, k)
    assert torch.equal(mx4.linear(one, q), mx4.linear(one.contiguous(), q))
    # rows and columns behind a matrix are not read into the result
    x = torch.full((2 * m, k + 8), float("nan"), dtype=torch.bfloat16, device="cuda")
    x[:m, :k] = base[:m, :k]
    assert torch.equal(mx4.linear(x[:m, :k], q), mx4.linear(base[:m, :k], q))


@pytest.mark.parametrize("dt", PRODUCT, ids=ids)
@pytest.mark.parametrize("m", [1, 20, 150])
def test_non_finite_values_stay_in_their_rows(mx4, dt, m):
    n, k = 150, 420
    w = ints((n, k), 1, torch.float32, hi=2)
    w[20, 40] = float("nan")
    w[21, k - 1] = float("inf")
    q = mx4.quantize(w)
    wq = R.round4(f64(w))
    assert np.isnan(wq[20, 32:64]).all() and np.isnan(wq).sum() == 32 + (k - 416)
    x, dy = ints((m, k), 2, dt), ints((m, n), 3, dt)
    x[m - 1, 7], dy[0, 9] = float("inf"), float("nan")
    with np.errstate(invalid="ignore"):
        # only the rows / columns that the definition makes NaN or infinite are
        for got, want in ((mx4.linear(x, q), f64(x) @ wq.T), (mx4.linear_grad(dy, q), f64(dy) @ wq)):
            got = f64(got)
            assert np.array_equal(np.isnan(got), np.isnan(want))
            ok = ~np.isnan(want)
            assert np.array_equal(got[ok], torch.from_numpy(want).to(dt).double().numpy()[ok])
        y = f64(mx4.matmul(mx4.quantize(x[: m - 1] if m > 1 else dy[:, :1].expand(1, k).nan_to_num()), q, dt))
    assert np.isnan(y[:, 20:22]).all() and np.isfinite(np.delete(y, (20, 21), axis=1)).all()


def test_empty_sizes(mx4):
    for shape in ((0, 5), (5, 0), (0, 0)):
        for axis in (0, 1):
            q = mx4.quantize(torch.empty(shape, device="cuda"), axis=axis)
            assert q.shape == shape and mx4.dequantize(q).shape == shape
    q0, q = mx4.quantize(torch.ones(4, 0, device="cuda")), mx4.quantize(torch.ones(4, 6, device="cuda"))
    for dt in PRODUCT:
        assert torch.equal(mx4.linear(torch.empty(3, 0, device="cuda", dtype=dt), q0), torch.zeros(3, 4, device="cuda", dtype=dt))
        assert mx4.linear(torch.empty(0, 6, device="cuda", dtype=dt), q).shape == (0, 4)
        assert mx4.linear(torch.empty(2, 0, 6, device="cuda", dtype=dt), q).shape == (2, 0, 4)
        assert mx4.linear_grad(torch.empty(3, 4, device="cuda", dtype=dt), q0).shape == (3, 0)
        e = mx4.quantize(torch.empty(0, 6, device="cuda"))
        assert torch.equal(mx4.linear_grad(torch.empty(3, 0, device="cuda", dtype=dt), e), torch.zeros(3, 6, device="cuda", dtype=dt))
        assert mx4.matmul(e, q, dt).shape == (0, 4)
        assert torch.equal(mx4.matmul(q0, q0, dt), torch.zeros(4, 4, device="cuda", dtype=dt))


# ---- gradients ---------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dt", PRODUCT, ids=ids)
@pytest.mark.parametrize("axis", [0, 1])
@pytest.mark.parametrize("m", [1, 6, 130])
def test_gradient_is_the_formulas(mx4, dt, axis, m):
    w = ints((45, 70), 1, torch.float32, hi=2)
    q = mx4.quantize(w, axis=axis)
    wq = R.round4(f64(w)) if axis == 1 else R.round4(f64(w).T).T
    x = ints((2, m, 70), 2, dt).requires_grad_(True)
    dy = ints((2, m, 45), 3, dt)
    y = mx4.linear(x, q)
    dx, = torch.autograd.grad(y, x, dy, create_graph=False)
    assert dx.shape == x.shape and np.array_equal(f64(dx), torch.from_numpy(f64(dy) @ wq).to(dt).double().numpy())
    # a broadcast gradient (what .sum() hands back has no strides)
    dx, = torch.autograd.grad(mx4.linear(x, q).sum(), x)
    assert np.array_equal(f64(dx[0, 0]), torch.from_numpy(wq.sum(axis=0)).to(dt).double().numpy())
    # the same leaf twice, and through a shared (broadcast) input
    row = ints((70,), 4, dt).requires_grad_(True)
    (mx4.linear(row.expand(m, 70), q) * dy[0]).sum().backward()
    assert row.grad.shape == (70,)
    want = (f64(dy[0]) @ wq)
    tolr = torch.finfo(dt).eps * (m + 1) * np.abs(want).sum(axis=0) + 1e-6
    assert (np.abs(f64(row.grad) - want.sum(axis=0)) <= tolr).all()


def test_gradient_against_differences(mx4):
    """the product is linear in x, so a difference of any step is its derivative up to float32 rounding; the second derivative: the
    gradient of the gradient with respect to dy is the forward product"""
    q = mx4.quantize(torch.randn(33, 64, generator=gen(1)).cuda())
    x = torch.randn(3, 64, generator=gen(2)).cuda().requires_grad_(True)
    dy = torch.randn(3, 33, generator=gen(3)).cuda().requires_grad_(True)
    dx, = torch.autograd.grad(mx4.linear(x, q), x, dy, create_graph=True)
    d = torch.randn(3, 64, generator=gen(4)).cuda()
    ddy, = torch.autograd.grad(dx, dy, d)
    assert torch.allclose(ddy, mx4.linear(d, q), rtol=0, atol=0)
    h = 0.5
    num = ((mx4.linear(x + h * d, q) - mx4.linear(x - h * d, q)) / (2 * h) * dy).sum()
    ana = (dx * d).sum()
    assert abs(float((num - ana).detach())) <= 64 * 33 * 3 * 2.0 ** -23 * float(((x.abs().max() + d.abs().max()) * 6 * dy.abs().max()).detach())


# ---- streams, graphs, one after the other ------------------------------------------------------------------------------------
def _pipeline(mx4, x, q, dy):
    return mx4.matmul(mx4.quantize(x), q, torch.bfloat16), mx4.linear(x, q), mx4.linear_grad(dy, q)


@pytest.mark.parametrize("m", [1, 24, 300])
def test_side_stream_and_captured_graphs(mx4, m):
    n, k = 400, 2100
    q = mx4.quantize(ints((n, k), 1, torch.float32, hi=2))
    xs = [ints((m, k), 10 + i, torch.bfloat16) for i in range(3)]
    dys = [ints((m, n), 20 + i, torch.bfloat16) for i in range(3)]
    want = [_pipeline(mx4, x, q, d) for x, d in zip(xs, dys)]
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = [_pipeline(mx4, x, q, d) for x, d in zip(xs, dys)]
    # two streams at once
    again = [_pipeline(mx4, x, q, d) for x, d in zip(xs, dys)]
    torch.cuda.synchronize()
    for a, b, c in zip(want, got, again):
        assert all(torch.equal(u, v) and torch.equal(u, w) for u, v, w in zip(a, b, c))
    # two graphs of the same calls, replayed in turn with eager work between
    graphs = []
    for _ in range(2):
        x, d = torch.empty_like(xs[0]), torch.empty_like(dys[0])
        g = torch.cuda.CUDAGraph()
        x.copy_(xs[0]); d.copy_(dys[0])
        torch.cuda.synchronize()
        with torch.cuda.graph(g):
            out = _pipeline(mx4, x, q, d)
        graphs.append((g, x, d, out))
    for i in range(3):
        for j, (g, x, d, out) in enumerate(graphs):
            x.copy_(xs[(i + j) % 3]); d.copy_(dys[(i + j) % 3])
            g.replay()
        mid = _pipeline(mx4, xs[0], q, dys[0])
        torch.cuda.synchronize()
        for j, (g, x, d, out) in enumerate(graphs):
            assert all(torch.equal(u, v) for u, v in zip(out, want[(i + j) % 3]))
        assert all(torch.equal(u, v) for u, v in zip(mid, want[0]))


def test_results_do_not_change_from_call_to_call(mx4):
    x = torch.randn(70, 3001, generator=gen(1)).cuda()
    q = mx4.quantize(torch.randn(1111, 3001, generator=gen(2)).cuda())
    dy = torch.randn(70, 1111, generator=gen(3)).cuda()
    first = (mx4.linear(x, q), mx4.linear_grad(dy, q), mx4.matmul(mx4.quantize(x), q), mx4.linear(x[:1], q), mx4.linear_grad(dy[:1], q))
    for _ in range(3):
        again = (mx4.linear(x, q), mx4.linear_grad(dy, q), mx4.matmul(mx4.quantize(x), q), mx4.linear(x[:1], q), mx4.linear_grad(dy[:1], q))
        assert all(torch.equal(a, b) for a, b in zip(first, again))


def test_offsets_beyond_32_bits(mx4):
    """more than 2^32 values: the last rows are right"""
    n, k = 70000, 65536
    w = torch.zeros(64, k, device="cuda")
    w[torch.arange(64), torch.arange(64) * 1000] = 4.0
    q = mx4.quantize(w)
    z = torch.zeros(n // 16 * (k // 128) * 1024, dtype=torch.uint8, device="cuda")
    big = mx4.Mx4((n, k), 1, z, torch.full((z.numel() // 16,), 2, dtype=torch.uint8, device="cuda"))
    big.codes[-q.codes.numel():], big.scales[-q.scales.numel():] = q.codes, q.scales       # (whole tiles of 16 rows)
    for m in (1, 33):
        x = ints((m, k), 1, torch.bfloat16)
        y = mx4.linear(x, big)
        assert not y[:, :-64].any() and torch.equal(y[:, -64:], mx4.linear(x, q))
        dy = ints((m, n), 2, torch.bfloat16)
        assert torch.equal(mx4.linear_grad(dy, big), mx4.linear_grad(dy[:, -64:], q))
        assert torch.equal(mx4.matmul(mx4.quantize(x), big)[:, -64:], mx4.matmul(mx4.quantize(x), q))
    x = torch.randn(16, k, device="cuda", dtype=torch.bfloat16).expand(n // 16, 16, k).reshape(-1, k)
    z = mx4.quantize(x)
    one = k // 128 * 1024
    assert torch.equal(z.codes[-one:], z.codes[:one]) and torch.equal(z.scales[-one // 16:], z.scales[:one // 16])


def test_copies_of_a_matrix_hold_their_own_buffers(mx4):
    import copy
    import pickle
    for axis in (0, 1):
        w, x = ints((70, 300), 1, torch.float32, hi=2), ints((5, 300), 2, torch.bfloat16)
        q = mx4.quantize(w, axis=axis)
        want = mx4.linear(x, q)
        copies = [copy.deepcopy(q), pickle.loads(pickle.dumps(q)), copy.deepcopy(q.t()).t()]
        q.codes.zero_()
        for c in copies:
            assert c.codes.data_ptr() == c._cp != q._cp and c.scales.data_ptr() == c._sp
            assert torch.equal(mx4.linear(x, c), want) and torch.equal(mx4.dequantize(c), w)
        assert not mx4.linear(x, q).any()


def test_views_that_negate_lazily(mx4):
    """the imaginary part of a conjugated view is stored with the other sign"""
    z = torch.complex(ints((40, 96), 1, torch.float32), ints((40, 96), 2, torch.float32))
    x = z.conj().imag
    assert x.is_neg()
    q = mx4.quantize(ints((24, 96), 3, torch.float32, hi=2))
    assert torch.equal(mx4.dequantize(mx4.quantize(x)), mx4.dequantize(mx4.quantize(-z.imag)))
    assert torch.equal(mx4.linear(x, q), -mx4.linear(z.imag, q)) and torch.equal(mx4.linear_grad(x[:, :24], q), -mx4.linear_grad(z.imag[:, :24], q))


@pytest.mark.parametrize("dt", PRODUCT, ids=ids)
def test_captured_gradient(mx4, dt):
    """forward and backward of a leaf in one graph, replayed with new values"""
    q = mx4.quantize(ints((90, 333), 1, torch.float32, hi=2))
    xs, dys = [ints((2, 37, 333), 5 + i, dt) for i in range(3)], [ints((2, 37, 90), 9 + i, dt) for i in range(3)]
    want = [(mx4.linear(a, q), mx4.linear_grad(b, q)) for a, b in zip(xs, dys)]
    x, dy = xs[0].clone().requires_grad_(True), dys[0].clone()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = mx4.linear(x, q)
        dx, = torch.autograd.grad(y, x, dy)
    for i in (0, 1, 2, 0):
        with torch.no_grad():
            x.copy_(xs[i])
        dy.copy_(dys[i])
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(y.detach(), want[i][0]) and torch.equal(dx, want[i][1])
        again = mx4.linear(xs[i], q)
        assert torch.equal(again, want[i][0])


@pytest.mark.parametrize("dt,low", [(torch.float32, -133), (torch.bfloat16, -133), (torch.float16, -24)], ids=["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("m", [1, 40])
def test_subnormal_activations_count(mx4, dt, low, m):
    """down to bfloat16's last place (all of float16): one product by 4 an output, so nothing is rounded"""
    w = torch.zeros(64, 64)
    w[torch.arange(64), torch.arange(64)] = 4.0
    q = mx4.quantize(w.cuda())
    x = torch.exp2(torch.arange(low, low + 64, dtype=torch.float64).clamp(max=8)).expand(m, 64).to(dt).cuda()
    assert (x != 0).all()
    assert torch.equal(f64_t(mx4.linear(x, q)), 4 * f64_t(x)) and torch.equal(f64_t(mx4.linear_grad(x, q)), 4 * f64_t(x))


def f64_t(t):
    return t.detach().cpu().double()
