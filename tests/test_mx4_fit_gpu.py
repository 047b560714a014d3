"""A fit whose data are resident in 4 bits per value (Corex(x_storage="mx4"), include/lcx.h lcx_create_stored).

What is fitted is the rounded matrix X~ that lcx_download_x returns, and the two passes over it are exact up to float32 sums: so the moments
and the whole fit are compared with a dense float32 handle / fit OF THAT MATRIX, at the bars float32 has against itself elsewhere in this
suite (2e-4 of an array's scale for a step; final TC 5e-5, iterations 6 %)."""
import pickle

import numpy as np
import pytest

from linearcorex_amd import Corex
from linearcorex_amd.backend import HipBackend
from oracle import corex_oracle as O
from tests import mx4_reference as R

pytestmark = pytest.mark.gpu


def planted(n, v, k, seed):
    x, grp = O.gen_planted(n, v, k, seed=seed)
    return np.asarray(x, np.float32), grp


def standardised(n, v, seed):
    r = np.random.RandomState(seed)
    x = r.randn(n, v) + r.randn(n, 1) * np.linspace(0, 1, v)
    x[:, v // 2] = 0.0                                       # a constant variable
    s = x.std(axis=0)
    return ((x - x.mean(axis=0)) / np.where(s > 0, s, 1)).astype(np.float32)


def rounded(x):
    """X~: the 4-bit values (blocks along the variables), every variable brought back to mean square 1"""
    v = R.round4(x.astype(np.float64))
    q = (v ** 2).mean(axis=0)
    unit = np.where(q > 0, 1 / np.sqrt(np.where(q > 0, q, 1)), 1.0).astype(np.float32)
    return (v.astype(np.float32) * unit), unit


@pytest.mark.parametrize("n,v,m", [(1, 1, 1), (70, 33, 3), (130, 600, 16), (1000, 1300, 20), (700, 2000, 64), (2100, 900, 100), (65, 5000, 128)])
def test_moments_are_those_of_the_rounded_matrix(n, v, m, monkeypatch):
    if v == 1300:
        monkeypatch.setenv("LCX_PANEL_BLOCK_COLS", "512")    # several staging blocks
    x = standardised(n, v, seed=n) if n > 1 else np.ones((1, 1), np.float32)
    be = HipBackend(n, v, m, np.float32, x_storage="mx4")
    be.upload_x(x)
    xq = be.download_x()
    want, unit = rounded(x)
    assert np.abs(xq - want).max() <= 4 * 2.0 ** -24 * np.abs(want).max()        # one float32 factor, one product
    info = be.bytes_resident()
    assert info["x_layout"] == "4 bits per value"
    dense = HipBackend(n, v, m, np.float32)
    dense.upload_x(xq)
    w = (np.random.RandomState(1).randn(m, v) / np.sqrt(v)).astype(np.float32)
    for b in (be, dense):
        b.set_ws(w * 0.3)
        b.moments_a(0)
        b.moments_b(0, 0.3, False)
        b.moments_c(0)
        b.moments_detail(0)
    # a pass: exact products (every float32 in three bf16 numbers), float32 sums; the small operand is rounded once where it takes the factor in
    y, wd = be.get_moment(0, "Y"), w * 0.3
    s = np.abs(xq.astype(np.float64)) @ np.abs(wd.T.astype(np.float64))
    steps = 3 * -(-v // 32) + 96
    err = np.abs(y - xq.astype(np.float64) @ wd.T.astype(np.float64))
    assert (err <= (steps + 2) * 2.0 ** -23 * s + 1e-30).all()
    for key in ("Y", "uj", "rho", "ry", "invrho", "rhoinvrho", "Qij", "Si", "Qi-Si^2", "MI", "X_i Z_j", "X_i^2 | Y"):
        a, b = be.get_moment(0, key, 0.3), dense.get_moment(0, key, 0.3)
        assert np.abs(a - b).max() <= 2e-4 * max(1e-3, np.abs(b).max()), key
    # an update (the direction, a trial)
    for b in (be, dense):
        b.update_a()
        b.update_b(0.3)
        b.update_c(0.3)
        b.update_d()
        b.make_trial(0.5)
        b.moments_a(1)
        b.moments_b(1, 0.3, True)
        b.moments_c(1)
    for key in ("grad", "update", "sig_grad"):
        a, b = be.get_moment(0, key), dense.get_moment(0, key)
        assert np.abs(a - b).max() <= 5e-4 * max(1e-3, np.abs(b).max()), key
    a, b = be.read_state(1), dense.read_state(1)             # (a random start's trial may be invalid: then it is on both)
    assert a[2] == b[2] and np.isnan(a[0]) == np.isnan(b[0])
    assert np.isnan(b[0]) or abs(a[0] - b[0]) <= 2e-4 * max(1.0, abs(b[0]))
    be.close(); dense.close()


def test_resident_bytes():
    be = HipBackend(4096, 20000, 64, np.float32, x_storage="mx4")
    dense = HipBackend(4096, 20000, 64, np.float32)
    a, b = be.bytes_resident(), dense.bytes_resident()
    assert a["x"] < b["x"] / 7 and a["total"] < b["total"]
    be.close(); dense.close()


@pytest.mark.parametrize("n,v,m", [(400, 300, 4), (1500, 1000, 20)])
def test_fit_is_the_fit_of_the_rounded_matrix(n, v, m):
    x, grp = planted(n, v, m, seed=5)
    a = Corex(n_hidden=m, seed=0, x_storage="mx4").fit(x)
    assert a.x_storage == "mx4" and "mx_" in a._backend.kernel_name(0)
    xq = a._backend.download_x()
    b = Corex(n_hidden=m, seed=0, gaussianize="none").fit(xq)
    assert abs(a.tc - b.tc) <= 5e-5 * abs(b.tc)
    na, nb = len(a.history["TC"]), len(b.history["TC"])
    assert abs(na - nb) <= 0.06 * nb + 2
    # the groups that were planted, as a dense fit finds them
    c = Corex(n_hidden=m, seed=0).fit(x)
    assert np.array_equal(a.clusters(), b.clusters())
    assert (a.clusters() == c.clusters()).mean() == 1.0
    assert abs(a.tc - c.tc) < 0.15 * abs(c.tc)               # rounding noise weakens every correlation a little
    # transform of new data, and of the fitted data: dense, as always
    y = a.transform(x)
    assert np.array_equal(a.fit_transform(x) * 0 + y, y)
    cov = a.get_covariance()
    assert cov.shape == (v, v) and np.isfinite(cov).all()
    back = pickle.loads(pickle.dumps(a))
    assert np.abs(back.transform(x) - a.transform(x)).max() <= 1e-4 * np.abs(y).max() and back.x_storage == "mx4"
    yd, mo = a.transform(x[:50], details=True)
    assert yd.shape == (50, m) and np.isfinite(mo["TC"])


@pytest.mark.parametrize("gz,missing", [("standard", -999.0), ("outliers", None), ("empirical", None), ("none", None)])
def test_preprocessing_comes_before_the_rounding(gz, missing):
    x, _ = planted(300, 200, 3, seed=8)
    if missing is not None:
        x[np.random.RandomState(2).rand(*x.shape) < 0.03] = missing
    kw = dict(n_hidden=3, seed=0, max_iter=3, gaussianize=gz, missing_values=missing)
    a, b = Corex(x_storage="mx4", **kw).fit(x), Corex(**kw).fit(x)
    want, _ = rounded(b._backend.download_x())
    assert np.abs(a._backend.download_x() - want).max() <= 4 * 2.0 ** -24 * np.abs(want).max()


def test_other_paths_run_on_it():
    x, _ = planted(300, 260, 3, seed=9)
    for kw in (dict(line_search="linear"), dict(line_search="exact-y"), dict(discourage_overlap=False, max_iter=20), dict(f32_gemm="split")):
        a = Corex(n_hidden=3, seed=0, x_storage="mx4", max_iter=kw.pop("max_iter", 30), **kw).fit(x)
        xq = a._backend.download_x()
        b = Corex(n_hidden=3, seed=0, gaussianize="none", max_iter=a.max_iter, **{k: v for k, v in kw.items() if k != "f32_gemm"}).fit(xq)
        assert a.f32_gemm == "mfma" and np.isfinite(a.tc) and abs(a.tc - b.tc) <= 2e-3 * max(1.0, abs(b.tc)), kw
    g = Corex(n_hidden=4, seed=0, x_storage="mx4", max_iter=5).fit_generated(500, 700, seed=3, kind=1, n_groups=4)
    assert np.isfinite(g.tc)


@pytest.mark.parametrize("n,v,m", [(300, 200, 3), (4000, 3000, 30), (2000, 9000, 64), (700, 2000, 128)])
def test_kernel_names_are_those_that_run(n, v, m):
    """what a profiler shows of the passes, templates included"""
    import re
    be = HipBackend(n, v, m, np.float32, 0, x_storage="mx4")
    try:
        a, b = re.fullmatch(r"lcx::mx_linear_tile_kernel<float, ([124]), 4, ([24]), false>", be.kernel_name(0)), \
            re.fullmatch(r"lcx::mx_grad_tile_kernel<float, ([124]), 1, false>", be.kernel_name(1))
        assert a and b and be.kernel_name(2) == "" and int(a[2]) == (2 if a[1] == "4" else 4)
        rows = max(16, 1 << (m - 1).bit_length())                        # factors, padded
        assert int(a[1]) * 16 <= rows and int(b[1]) * 16 <= rows
    finally:
        be.close()
