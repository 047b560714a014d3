"""What the 4-bit operators ask for as work space, and the sizes that they refuse, from the host's side (nothing is launched)."""
import ctypes as C

import pytest

pytest.importorskip("torch")
from linearcorex_amd import _abi                                         # noqa: E402

F32, BF16, F16 = 0, 2, 3
BIG = (1 << 31) - 1


@pytest.fixture(scope="module")
def lib():
    import __graft_entry__ as ge
    ge.build()
    return _abi.load()


def workspace(lib, *args):
    b = C.c_int64(-7)
    rc = lib.lcx_mx4_workspace(*args, C.byref(b))
    return b.value if rc == 0 else (lib.lcx_last_error() or b"").decode()


@pytest.mark.parametrize("m,n,k", [(4096, 8192, 4096), (40, 512, 8960), (2048, 8192, 4096), (17, 128, 128), (200, 20032, 20096)])
def test_what_is_read_in_place_needs_no_copy(lib, m, n, k):
    for op, c, o in ((1, k, n), (2, n, k)):
        whole, place = workspace(lib, op, BF16, m, n, k), workspace(lib, op + 2, BF16, m, n, k)
        assert place % (m * o * 4) == 0                                  # partial sums, or nothing
        assert whole >= place + m * c * 2
    assert "in place" in workspace(lib, 3, F32, m, n, k) and "in place" in workspace(lib, 4, F16, m, n, k)
    assert "bad argument" in workspace(lib, 5, BF16, m, n, k)


def test_sizes_that_overflow_are_refused(lib):
    """pieces of 16 rows x 128 of the contraction are counted by a launch; sizes whose space would not fit 64 bits used to wrap around"""
    for dt in (F32, BF16, F16):
        for op, m, n, k in ((1, BIG, BIG, BIG), (2, BIG, BIG, BIG), (1, 16 << 12, 100, 128 * ((1 << 12) + 1)), (2, 16 << 12, 128 * ((1 << 12) + 1), 100)):
            assert "too large" in workspace(lib, op, dt, m, n, k), (op, dt, m, n, k)
        assert workspace(lib, 1, dt, 128 << 8, 100, 128 << 12) > 0       # well below
    # read in place there is no such limit, the tiles of the output are what counts
    assert workspace(lib, 3, BF16, 16 << 12, 100, 128 * ((1 << 12) + 1)) >= 0
    # the calls say so as well, whatever space they are given (the pointers are not real: nothing is launched)
    p, m, c = 4096, 16 << 12, 128 * ((1 << 12) + 1)
    for name, args in (("lcx_mx4_linear", (p, F32, m, c, 1, p, p, 100, c, p, 100, 1)), ("lcx_mx4_linear_grad", (p, F32, m, c, 1, p, p, c, 100, p, 100, 1)),
                       ("lcx_mx4_linear", (p + 2, BF16, m, c + 1, 1, p, p, 100, c, p, 100, 1))):
        assert getattr(lib, name)(*args, p, 1 << 62, None) == 1 and "too large" in (lib.lcx_last_error() or b"").decode()
    # sizes whose bytes do not fit 64 bits: refused before they are counted
    assert lib.lcx_mx4_quantize(p, 1, BIG, BIG, BIG, 1, p, p, None) == 1 and "too large" in (lib.lcx_last_error() or b"").decode()
    assert lib.lcx_mx4_quantize(p, 1, BIG, BIG, 1, BIG, p, p, None) == 1 and "too large" in (lib.lcx_last_error() or b"").decode()
