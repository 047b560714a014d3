"""The sizes of tests/test_mx4_variants_gpu.py take the kernels that they are there for, and every kernel has one."""
import itertools

import pytest

pytest.importorskip("torch")
from tests import test_mx4_variants_gpu as V                             # noqa: E402


@pytest.fixture(scope="module", autouse=True)
def lib():
    import __graft_entry__ as ge
    ge.build()


@pytest.mark.parametrize("case,what", V.CASES, ids=V.ids)
def test_the_case_takes_its_variant(case, what):
    assert V.taken(case) == what


def test_every_variant_has_a_case():
    have = {(op, dt, w[0], w[1] if w[0] == "row" else w[1] > 1) for (op, dt, *_), w in V.CASES}
    for dt in (V.F32, V.BF16, V.F16):
        want = {(1, dt, "row", 1), (1, dt, "row", 2), (1, dt, 1, True)} | {(1, dt, ct, s) for ct, s in itertools.product((2, 4), (False, True))}
        want |= {(2, dt, ct, s) for ct, s in itertools.product((1, 2, 4), (False, True))}
        if dt == V.BF16:
            want |= {(1, dt, 8, False), (1, dt, 8, True)}
        assert want <= have, want - have
    mat = {(w, s) for op, _, w, s in have if op == 0}
    assert mat >= {("row", 1), ("row", 2)} | set(itertools.product((2, 4, 8), (False, True)))
    # read in place and laid out, where both exist
    for op, edge in ((1, 128), (2, 64)):
        for ct in ((2, 4, 8) if op == 1 else (1, 2, 4)):
            assert any(c[:2] == (op, V.BF16) and w[0] == ct and (c[4] if op == 1 else c[3]) % edge == 0 for c, w in V.CASES), (op, ct)


def test_two_row_tiles_where_one_would_leave_more_blocks_than_cus():
    from tests import probe
    for dt, m in ((V.BF16, 8), (V.F32, 16), (V.F16, 1)):
        for n, rt in ((1, 1), (4096, 1), (4097, 2), (8191, 2), (8192, 2), (16384, 2), (100000, 2)):
            assert probe.mx4_plan(0, dt, m, n, 4096)[:3] == (True, 1, rt), (dt, m, n)
