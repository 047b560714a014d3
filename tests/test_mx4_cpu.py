"""Refusals of the 4-bit operators: wrong arguments are turned down before anything reaches a GPU (none is needed here)."""
import ctypes as C

import numpy as np
import pytest

torch = pytest.importorskip("torch")
from linearcorex_amd import _abi, mx4                                   # noqa: E402
from tests import mx4_reference as R                                     # noqa: E402


@pytest.fixture(scope="module")
def lib():
    import __graft_entry__ as ge
    ge.build()
    return _abi.load()


def fake(shape, axis=1):
    """a matrix on the meta device: what the checks see"""
    r, c = shape if axis == 1 else shape[::-1]
    cb, sb = mx4._sizes(r, c)
    return mx4.Mx4(shape, axis, torch.empty(cb, dtype=torch.uint8, device="meta"), torch.empty(sb, dtype=torch.uint8, device="meta"))


def test_python_refuses_host_tensors_and_wrong_types():
    q = fake((4, 64))
    for call in (lambda: mx4.quantize(torch.zeros(2, 2)), lambda: mx4.linear(torch.zeros(2, 64), q), lambda: mx4.linear_grad(torch.zeros(2, 4), q)):
        with pytest.raises(ValueError, match="must be on the GPU"):
            call()
    for call in (lambda: mx4.quantize(np.zeros((2, 2))), lambda: mx4.linear([1.0], q), lambda: mx4.dequantize(torch.zeros(2, 2)),
                 lambda: mx4.matmul(q, torch.zeros(2, 2)), lambda: mx4.matmul(q, q, torch.float64), lambda: mx4.dequantize(q, torch.int8)):
        with pytest.raises(TypeError):
            call()


def test_python_refuses_shapes_that_do_not_fit():
    with pytest.raises(ValueError, match="columns"):
        mx4.matmul(fake((4, 64)), fake((4, 65)))
    with pytest.raises(ValueError, match="along the blocks"):
        mx4.matmul(fake((4, 64)), fake((4, 64), axis=0))
    q = fake((4, 64))
    assert q.t().shape == (64, 4) and q.t().axis == 0 and q.t().t().axis == 1 and q.t()._stored() == (4, 64)
    assert "Mx4(shape=(4, 64), axis=1" in repr(q)


def _call(lib, name, *args):
    rc = getattr(lib, name)(*args)
    return rc, (lib.lcx_last_error() or b"").decode()


def test_c_entry_points_refuse_bad_arguments(lib):
    p, odd = 4096, 4097                       # never dereferenced: every call below is refused before a launch
    bad = [("lcx_mx4_quantize", (p, 9, 4, 64, 64, 1, p, p, None)), ("lcx_mx4_quantize", (p, 0, -1, 64, 64, 1, p, p, None)),
           ("lcx_mx4_quantize", (p, 0, 4, 1 << 31, 64, 1, p, p, None)), ("lcx_mx4_quantize", (None, 0, 4, 64, 64, 1, p, p, None)),
           ("lcx_mx4_quantize", (p, 0, 4, 64, 64, 1, odd, p, None)), ("lcx_mx4_quantize", (p, 0, 4, 64, 64, 1, p, odd, None)),
           ("lcx_mx4_dequantize", (p, p, 4, 64, None, 0, 64, 1, None)), ("lcx_mx4_dequantize", (p, p, 4, 64, p, 4, 64, 1, None)),
           ("lcx_mx4_dequantize", (odd, p, 4, 64, p, 0, 64, 1, None)),
           ("lcx_mx4_matmul", (p, p, 4, p, p, 4, 64, p, 1, 4, 1, None, 0, None)), ("lcx_mx4_matmul", (p, p, 4, p, None, 4, 64, p, 0, 4, 1, None, 0, None)),
           ("lcx_mx4_matmul", (p, p, -4, p, p, 4, 64, p, 0, 4, 1, None, 0, None)), ("lcx_mx4_matmul", (p, p, 4, odd, p, 4, 64, p, 0, 4, 1, None, 0, None)),
           ("lcx_mx4_linear", (p, 1, 4, 64, 1, p, p, 4, 64, p, 4, 1, None, 0, None)), ("lcx_mx4_linear", (None, 0, 4, 64, 1, p, p, 4, 64, p, 4, 1, None, 0, None)),
           ("lcx_mx4_linear", (p, 0, 4, 64, 1, p, odd, 4, 64, p, 4, 1, None, 0, None)), ("lcx_mx4_linear", (p, 0, 4, 64, 1, p, p, 4, -1, p, 4, 1, None, 0, None)),
           ("lcx_mx4_linear_grad", (p, 1, 4, 4, 1, p, p, 4, 64, p, 64, 1, None, 0, None)), ("lcx_mx4_linear_grad", (p, 0, 4, 4, 1, p, p, 4, 64, None, 64, 1, None, 0, None)),
           ("lcx_mx4_linear_grad", (p, 0, 4, 4, 1, odd, p, 4, 64, p, 64, 1, None, 0, None))]
    for name, args in bad:
        rc, msg = _call(lib, name, *args)
        assert rc == 1 and msg.startswith(name), (name, args, rc, msg)
    b, n = C.c_int64(), C.c_int64()
    for args in ((3, 0, 1, 1, 1), (0, 1, 1, 1, 1), (1, 0, -1, 1, 1)):
        assert _call(lib, "lcx_mx4_workspace", *args, C.byref(b))[0] == 1
    assert _call(lib, "lcx_mx4_workspace", 1, 0, 1, 1, 1, None)[0] == 1 and _call(lib, "lcx_mx4_layout", 4, -1, None, None)[0] == 1
    for rows in (0, 1, 16, 17, 5000):
        for cols in (0, 1, 31, 256, 257, 512, 513, 5000):
            assert lib.lcx_mx4_layout(rows, cols, C.byref(b), C.byref(n)) == 0
            assert (b.value, n.value) == mx4._sizes(rows, cols)
    # nothing to do: no device is needed either
    assert lib.lcx_mx4_quantize(None, 0, 0, 64, 64, 1, None, None, None) == 0
    assert lib.lcx_mx4_linear(None, 0, 0, 64, 1, None, None, 4, 64, None, 4, 1, None, 0, None) == 0


def test_reference_format():
    """the restatement the GPU tests compare with, on values worked out by hand"""
    x = np.zeros((1, 64))
    x[0, :9] = [4.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, -7.9]
    x[0, 32:35] = [1.0, 2.0 ** -4, -2.0 ** -3]
    code, byte = R.quantize(x)
    assert byte.tolist() == [[127, 125]]
    assert code[0, :9].tolist() == [6, 0, 2, 2, 4, 4, 6, 6, 15] and code[0, 32:35].tolist() == [6, 0, 9]
    assert R.values(code, byte)[0, [0, 8, 32, 34]].tolist() == [4.0, -6.0, 1.0, -0.125]


def test_a_fit_refuses_4_bit_data_where_they_do_not_exist(lib):
    from linearcorex_amd import Corex
    for kw in (dict(x_storage="int8"), dict(x_storage="mx4", dtype=np.float64), dict(x_storage="mx4", n_hidden=129)):
        with pytest.raises(ValueError, match="x_storage"):
            Corex(**{"n_hidden": 4, **kw})
    assert Corex(n_hidden=4).x_storage == "dense" and Corex(n_hidden=4, x_storage="mx4").x_storage == "mx4"
    h = C.c_void_p()
    for args in ((100, 20, 4, 1, 0, 1), (100, 20, 129, 0, 0, 1), (100, 20, 4, 0, 0, 2)):
        assert lib.lcx_create_stored(C.byref(h), *args) == 1 and not h.value
        assert b"lcx_create_stored" in lib.lcx_last_error()


def test_a_matrix_of_buffers_that_do_not_fit_is_refused():
    import copy
    cb, sb = mx4._sizes(20, 300)
    c, s = torch.zeros(cb, dtype=torch.uint8), torch.zeros(sb, dtype=torch.uint8)
    for shape, axis, codes, scales in (((20, 300), 1, c[1:], s), ((20, 300), 1, c, s[1:]), ((20, 300), 0, c, s), ((20, 300), 1, c.int(), s),
                                       ((20, 300), 1, c, torch.zeros(2 * sb, dtype=torch.uint8)[::2]), ((20, 300), 2, c, s), ((20,), 1, c, s)):
        with pytest.raises(ValueError):
            mx4.Mx4(shape, axis, codes, scales)
    # on the host: copies hold their own buffers, no operator takes them
    q = mx4.Mx4((20, 300), 1, c, s)
    d, e = copy.deepcopy(q), copy.copy(q)
    assert d._cp == d.codes.data_ptr() != q._cp and d._sp == d.scales.data_ptr() != q._sp and e._cp == q._cp and e.shape == q.shape
    for call in (lambda: mx4.dequantize(q), lambda: mx4.matmul(q, q)):
        with pytest.raises(ValueError, match="must be on the GPU"):
            call()


def test_sizes_beyond_one_launch_are_refused(lib):
    """a launch counts its threads in 32 bits; what needs more is turned down (before a launch: the pointers are not real)"""
    p, big = 4096, (1 << 31) - 1
    for name, args in (("lcx_mx4_quantize", (p, 0, big, 1, 1, 1, p, p, None)), ("lcx_mx4_quantize", (p, 2, big, 1024, 1, big, p, p, None)),
                       ("lcx_mx4_quantize", (p, 3, (1 << 28) + 1, 16, 16, 1, p, p, None)), ("lcx_mx4_dequantize", (p, p, big, 1, p, 0, 1, 1, None)),
                       ("lcx_mx4_dequantize", (p, p, big, 1024, p, 0, 1, big, None)), ("lcx_mx4_linear", (p, 0, 1, 8, 1, p, p, big, 8, p, big, 1, None, 0, None)),
                       ("lcx_mx4_matmul", (p, p, 1, p, p, big, 8, p, 0, big, 1, None, 0, None))):
        rc, msg = _call(lib, name, *args)
        assert rc == 1 and "too large" in msg, (name, args, rc, msg)


def test_work_space_that_does_not_do_is_refused(lib):
    p, b = 4096, C.c_int64()
    for op, name, args in ((0, "lcx_mx4_matmul", (p, p, 40, p, p, 500, 9000, p, 0, 500, 1)),
                           (1, "lcx_mx4_linear", (p, 0, 40, 9000, 1, p, p, 500, 9000, p, 500, 1)),
                           (2, "lcx_mx4_linear_grad", (p, 0, 40, 500, 1, p, p, 500, 9000, p, 9000, 1))):
        assert lib.lcx_mx4_workspace(op, 0, 40, 500, 9000, C.byref(b)) == 0 and b.value > 0
        for space, size in ((None, b.value), (None, 0), (p, b.value - 1), (p + 8, b.value)):
            rc, msg = _call(lib, name, *args, space, size, None)
            assert rc == 1 and msg.startswith(name) and "work space" in msg, (name, space, size, rc, msg)
