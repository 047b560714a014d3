"""Every kernel that a 4-bit product can be made of: tile heights, split and whole contractions, one and two row tiles a wave - each at a size of odd
edges that takes it, which the test first makes sure of (the choice follows a model of the times, mx_choose).  Integers: every partial sum is
exact, so results are compared to the bit, whatever the layout of x and of the output; what lies around both stays as it was."""
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu
OPS = ("matmul", "linear", "linear_grad")
F32, BF16, F16 = 0, 2, 3
TORCH = {F32: torch.float32, BF16: torch.bfloat16, F16: torch.float16}
ids = lambda c: "-".join(str(v) for v in c) if isinstance(c, tuple) else str(c)       # noqa: E731

# (op, type, M, N, K), what it takes: a row kernel of so many row tiles, or tiles of 16 ct rows of x, in parts
CASES = [
    ((0, F32, 7, 180, 150), ("row", 1)), ((0, BF16, 13, 8713, 153), ("row", 2)), ((0, F16, 16, 9870, 150), ("row", 2)),
    ((0, F32, 26, 192, 150), (2, 1)), ((0, BF16, 34, 153, 1709), (2, 4)), ((0, F16, 2851, 788, 170), (4, 1)), ((0, F32, 3782, 610, 165), (4, 1)),
    ((0, BF16, 988, 619, 7372), (4, 5)), ((0, F32, 937, 647, 6801), (4, 5)), ((0, BF16, 6589, 1091, 191), (8, 1)), ((0, F32, 2986, 2611, 157), (8, 1)),
    ((0, F16, 1727, 1452, 10374), (8, 3)), ((0, F32, 1366, 1693, 10663), (8, 3)), ((0, BF16, 6802, 364, 10827), (8, 2)),
    ((1, F32, 1, 163, 170), ("row", 1)), ((1, F32, 10, 9105, 160), ("row", 2)), ((1, F32, 12, 153, 11602), (1, 23)), ((1, F32, 31, 182, 154), (2, 1)),
    ((1, F32, 20, 169, 478), (2, 4)), ((1, F32, 8315, 555, 182), (4, 1)), ((1, F32, 774, 2676, 3752), (4, 3)),
    ((1, BF16, 6, 156, 128), ("row", 1)), ((1, BF16, 1, 8436, 128), ("row", 2)), ((1, BF16, 15, 19, 26880), (1, 30)), ((1, BF16, 17, 182, 128), (2, 1)),
    ((1, BF16, 25, 151, 1024), (2, 8)), ((1, BF16, 6429, 571, 128), (4, 1)), ((1, BF16, 936, 1351, 8448), (4, 4)), ((1, BF16, 2721, 2949, 640), (8, 1)),
    ((1, BF16, 2140, 1933, 8219), (8, 3)), ((1, BF16, 2747, 1361, 7680), (8, 3)),
    ((1, F16, 1, 184, 158), ("row", 1)), ((1, F16, 1, 8744, 180), ("row", 2)), ((1, F16, 10, 7942, 8833), (1, 14)), ((1, F16, 17, 174, 176), (2, 1)),
    ((1, F16, 23, 179, 623), (2, 5)), ((1, F16, 5465, 1123, 179), (4, 1)), ((1, F16, 1399, 1441, 4054), (4, 3)),
    ((2, F32, 7, 153, 152), (1, 1)), ((2, F32, 8, 269, 150), (1, 3)), ((2, F32, 24, 155, 177), (2, 1)), ((2, F32, 38, 272, 156), (2, 3)),
    ((2, F32, 7070, 160, 520), (4, 1)), ((2, F32, 2949, 584, 161), (4, 5)),
    ((2, BF16, 2, 128, 158), (1, 1)), ((2, BF16, 8, 403, 169), (1, 4)), ((2, BF16, 24, 128, 186), (2, 1)), ((2, BF16, 24, 320, 178), (2, 3)),
    ((2, BF16, 4445, 152, 1067), (4, 1)), ((2, BF16, 1573, 1559, 536), (4, 5)), ((2, BF16, 1573, 1600, 536), (4, 5)),
    ((2, F16, 3, 157, 150), (1, 1)), ((2, F16, 3, 264, 152), (1, 3)), ((2, F16, 34, 155, 179), (2, 1)), ((2, F16, 44, 347, 174), (2, 3)),
    ((2, F16, 7837, 260, 586), (4, 1)), ((2, F16, 2739, 515, 186), (4, 5)),
]


def taken(case):
    from tests import probe
    row, ct, rt, split = probe.mx4_plan(*case)
    return ("row", rt) if row else (ct, split)


def ints(shape, seed, hi):
    return torch.randint(-hi, hi + 1, shape, generator=torch.Generator().manual_seed(seed)).float().cuda()


def embedded(x, ld, first=0):
    """x inside a buffer of NaN, rows ld apart"""
    b = torch.full((x.shape[0] + 2, ld), float("nan"), dtype=x.dtype, device="cuda")
    v = b[1:-1, first:first + x.shape[1]]
    return v.copy_(x)


def transposed(x):
    b = torch.full((x.shape[1] + 1, x.shape[0] + 3), float("nan"), dtype=x.dtype, device="cuda")
    return b[:x.shape[1], 3:].t().copy_(x)


@pytest.mark.parametrize("case,what", CASES, ids=ids)
def test_every_variant(case, what):
    from linearcorex_amd import mx4
    op, dt, m, n, k = case
    assert taken(case) == what
    t = TORCH[dt]
    w = ints((n, k), 1, 2)
    w *= torch.exp2(torch.randint(-1, 2, (n, -(-k // 32)), generator=torch.Generator().manual_seed(2)).float().cuda()).repeat_interleave(32, dim=1)[:, :k]
    q = mx4.quantize(w)
    assert torch.equal(mx4.dequantize(q), w)
    x = ints((m, n if op == 2 else k), 3, 4).to(t)
    b = w.double() if op == 2 else w.double().t().contiguous()
    want = (x.double() @ b).to(t)
    c, o = x.shape[1], b.shape[1]
    if op == 0:
        layouts, f = [mx4.quantize(x), mx4.quantize(transposed(x))], lambda a: mx4.matmul(a, q, t)         # noqa: E731
    else:
        # rows a multiple of 16 bytes apart (bfloat16 of whole stages is read in place), others, transposed
        layouts = [x, embedded(x, -(-c // 8) * 8 + 8), embedded(x, c + 1 + c % 2, 1), transposed(x)]
        f = lambda a: (mx4.linear if op == 1 else mx4.linear_grad)(a, q)                                   # noqa: E731
    for a in layouts:
        assert torch.equal(f(a), want)
    # outputs of other strides: the C entry points
    a = layouts[0]
    wb = mx4._workspace_bytes(op, dt, m, n, k)
    work = torch.empty(wb, dtype=torch.uint8, device="cuda") if wb else None
    tail = (work.data_ptr() if wb else None, wb)
    for rs, cs, shape in ((o + 3, 1, (m + 2, o + 3)), (1, m + 5, (o + 2, m + 5)), (2 * o + 1, 2, (m + 2, 2 * o + 1))):
        out = torch.full(shape, 77.0, dtype=t, device="cuda")
        at = out.data_ptr() + out[1].storage_offset() * out.element_size()
        if op == 0:
            mx4._call(0, "lcx_mx4_matmul", a._cp, a._sp, m, q._cp, q._sp, n, k, at, dt, rs, cs, *tail)
        else:
            mx4._call(0, "lcx_mx4_" + OPS[op], a.data_ptr(), dt, m, *a.stride(), q._cp, q._sp, n, k, at, rs, cs, *tail)
        got = out.view(-1)[shape[1]:].as_strided((m, o), (rs, cs))
        assert torch.equal(got, want)
        got.fill_(77.0)
        assert (out == 77.0).all()


@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16], ids=str)
def test_large_matrices_are_quantised_as_small_ones(t):
    """128 MB and more are read past the caches, along rows and across: the same codes as pieces of whole tiles that are not"""
    from linearcorex_amd import mx4
    rows, cols = (8208, 4104) if t == torch.float32 else (8208, 8200)
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(rows, cols, generator=g, device="cuda").to(t)
    assert x.numel() * x.element_size() >= 128 << 20
    xt = torch.empty(cols, rows, dtype=t, device="cuda").t().copy_(x)       # rows are neighbours in memory
    half = 4096                                                             # (whole tiles of 16 rows)
    a, b = mx4.quantize(x[:half]), mx4.quantize(x[half:].contiguous())
    codes, scales = torch.cat([a.codes, b.codes]), torch.cat([a.scales, b.scales])
    for v in (x, xt):
        for q in (mx4.quantize(v), mx4.quantize(v.t(), axis=0)):
            assert torch.equal(q.codes, codes) and torch.equal(q.scales, scales)


@pytest.mark.parametrize("m,n,k", [(2000, 4096, 8192), (40, 512, 8960)])
def test_bfloat16_read_in_place_takes_no_copy(m, n, k):
    from linearcorex_amd import mx4
    q = mx4.quantize(ints((n, k), 1, 2))
    for f, c, o in ((mx4.linear, k, n), (mx4.linear_grad, n, k)):
        x = ints((m, c), 3, 4).bfloat16()
        want = f(x, q)
        torch.cuda.synchronize()
        parts = taken((1 if f is mx4.linear else 2, BF16, m, n, k))[1]
        torch.cuda.reset_peak_memory_stats()
        before = torch.cuda.memory_allocated()
        assert torch.equal(f(x, q), want)
        # the result, its comparison, the partial sums (blocks of 2 MB at most beside them)
        assert torch.cuda.max_memory_allocated() - before <= m * o * (2 + 1) + (parts * m * o * 4 if parts > 1 else 0) + 4 * (2 << 20)
        # the space that the C entry asks for does, to the byte
        wb = mx4._workspace_bytes(3 if f is mx4.linear else 4, BF16, m, n, k)
        space = torch.full((wb + 64,), 77, dtype=torch.uint8, device="cuda")
        out = torch.empty(m, o, dtype=torch.bfloat16, device="cuda")
        mx4._call(0, "lcx_mx4_linear" if f is mx4.linear else "lcx_mx4_linear_grad", x.data_ptr(), BF16, m, c, 1, q._cp, q._sp, n, k, out.data_ptr(), o, 1,
                  space.data_ptr(), wb)
        assert torch.equal(out, want) and (space[wb:] == 77).all()
