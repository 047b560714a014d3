"""The shard of a fit with Corex(x_storage="mx4") where preprocessed variables do not have mean square 1: missing cells (the standard deviation is
that of the observed ones, the others are 0), squashed outliers, ranks, no scaling at all.  X~ is the 4-bit rounding times one float32 factor
per variable, sqrt(sum x^2 / sum rounded^2): every variable keeps the mean square it had."""
import os
import subprocess
import sys
import threading

import numpy as np
import pytest

torch = pytest.importorskip("torch")          # before the library, which must resolve against the HIP runtime of torch's wheel
from linearcorex_amd import Corex                                       # noqa: E402
from linearcorex_amd.backend import HipBackend                          # noqa: E402
from linearcorex_amd.comm import Comm                                   # noqa: E402
from oracle import corex_oracle as O                                    # noqa: E402
from tests import mx4_reference as R                                    # noqa: E402
from tests.test_thread_ranks_gpu import TIMEOUT, ThreadComm, _run_loop, _Shared       # noqa: E402

pytestmark = pytest.mark.gpu


def kept(x):
    """X~ of preprocessed data, in float64"""
    x = x.astype(np.float64)
    v = R.round4(x)
    a, b = (x ** 2).sum(axis=0), (v ** 2).sum(axis=0)
    return v * np.sqrt(np.where((a > 0) & (b > 0), a, 1) / np.where((a > 0) & (b > 0), b, 1))


def data(kind, n, v, k):
    """data whose preprocessed variables have a mean square of their own"""
    x, _ = O.gen_planted(n, v, k, seed=5)
    r = np.random.RandomState(2)
    kw = dict(gaussianize="standard", missing_values=None)
    if kind == "missing":
        x[r.rand(*x.shape) < 0.3] = -999.0
        kw["missing_values"] = -999.0
    elif kind == "none":
        x *= np.linspace(0.3, 0.7, v)
        kw["gaussianize"] = "none"
    elif kind == "outliers":
        x *= np.exp(0.8 * r.randn(n, 1))
        kw["gaussianize"] = "outliers"
    elif kind == "empirical":
        kw["gaussianize"] = "empirical"
    return np.asarray(x, np.float32), kw


KINDS = ["standard", "missing", "none", "outliers", "empirical"]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("n,v", [(400, 60), (130, 1200)])
def test_every_variable_keeps_its_mean_square(kind, n, v, monkeypatch):
    if v > 1000:
        monkeypatch.setenv("LCX_PANEL_BLOCK_COLS", "512")                # several staging blocks
    x, kw = data(kind, n, v, 3)
    a, b = (Corex(n_hidden=3, seed=0, max_iter=2, x_storage=s, **kw).fit(x) for s in ("mx4", "dense"))
    dense = b._backend.download_x()
    got, want = a._backend.download_x().astype(np.float64), kept(dense)
    # the factor is rounded once and the product once; the 64-bit sums behind the factor count next to nothing
    assert (np.abs(got - want) <= 2.01 * 2.0 ** -24 * np.abs(want)).all()
    ms = (dense.astype(np.float64) ** 2).mean(axis=0)
    assert kind == "standard" or np.abs(ms - 1).max() > 1e-3             # what the factor has to keep
    # every value of a column has at most those two roundings, so its root mean square does
    assert (np.abs(np.sqrt((got ** 2).mean(axis=0)) - np.sqrt(ms)) <= 2.01 * 2.0 ** -24 * np.sqrt(ms)).all()


@pytest.mark.parametrize("kind", KINDS)
def test_fit_is_that_of_the_original_data_but_for_rounding_noise(kind):
    """the bars of the clean data's fit (test_mx4_fit_gpu.py): 5e-5 against a dense fit of X~, 15 % against one of the data themselves"""
    x, kw = data(kind, 400, 60, 3)
    a, b = (Corex(n_hidden=3, seed=0, x_storage=s, **kw).fit(x) for s in ("mx4", "dense"))
    c = Corex(n_hidden=3, seed=0, gaussianize="none").fit(kept(b._backend.download_x()).astype(np.float32))
    assert abs(a.tc - c.tc) <= 5e-5 * abs(c.tc), (a.tc, c.tc)
    assert abs(a.tc - b.tc) <= 0.15 * abs(b.tc), (a.tc, b.tc)
    # new rows are projected as they are: weights of a rescaled matrix would be off by the scale
    y, yd = a.transform(x), Corex.transform(c, b._backend.download_x())
    assert np.abs(y - yd).max() <= 0.02 * np.abs(yd).max()


def test_columns_without_a_value_and_columns_rounded_away():
    """a variable of zeros, one that is far below the others of its block (all of it rounds to zero), one huge"""
    x = np.random.RandomState(0).randn(90, 70).astype(np.float32)
    x[:, 3], x[:, 40] = 0.0, x[:, 40] * 1e-4
    x[:, 66] *= 2.0 ** 60
    be = HipBackend(90, 70, 2, np.float32, x_storage="mx4")
    try:
        be.upload_x(x)
        got, want = be.download_x().astype(np.float64), kept(x)
        assert not got[:, 3].any() and not got[:, 40].any() and got[:, 66].any() and not got[:, 64:66].any() and not got[:, 67:].any()
        assert (np.abs(got - want) <= 2.01 * 2.0 ** -24 * np.abs(want)).all()
    finally:
        be.close()


class BlockComm(ThreadComm):
    """ranks that are threads, cut as `linearcorex_amd.comm.Comm` cuts them"""

    def __init__(self, shared, rank, nv):
        c = Comm.__new__(Comm)
        c.world, c.bounds = shared.world, None
        self.cut = c
        super().__init__(shared, rank, [0] + [c.shard(nv, r, 32)[1] for r in range(shared.world)])

    def shard(self, nv, rank=None, unit=1):
        return self.cut.shard(nv, self.rank if rank is None else rank, unit)

    def gather_columns(self, local, nv, like, unit=1):
        assert local.shape[-1] == self.shard(nv, unit=unit)[1] - self.shard(nv, unit=unit)[0]
        return super().gather_columns(local, nv, like)


def _ranked(x, w0, iters, comm, out):
    n, v = x.shape
    model = Corex(n_hidden=len(w0), seed=None, tol=0.0, device=0, comm=comm, x_storage="mx4")
    c0, c1 = (0, v) if comm is None else comm.shard(v, unit=32)
    be = model._attach_shard(np.ascontiguousarray(x[:, c0:c1]), v)
    model.ws = w0
    out["x"] = be.download_x()
    out["history"] = _run_loop(model, iters)
    out["ws"] = model._gather(be.get_ws(0))
    be.close()


@pytest.mark.parametrize("world", [2, 3, 8])
@pytest.mark.parametrize("n,v,m", [(400, 260, 3), (900, 1111, 40)])
def test_the_fitted_matrix_does_not_depend_on_the_number_of_ranks(world, n, v, m):
    iters = 8
    x = O.preprocess(O.gen_planted(n, v, 3, seed=4)[0])[0].astype(np.float32)
    w0 = (np.random.RandomState(3).randn(m, v) * 0.004).astype(np.float32)
    one = {}
    _ranked(x, w0, iters, None, one)
    shared, results, errors = _Shared(world), [{} for _ in range(world)], []

    def main(r):
        try:
            torch.cuda.set_device(0)
            _ranked(x, w0, iters, BlockComm(shared, r, v), results[r])
        except BaseException as e:          # noqa: BLE001 - the others fail on the broken barrier
            errors.append(e)
            shared.barrier.abort()

    threads = [threading.Thread(target=main, args=(r,), daemon=True) for r in range(world)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(TIMEOUT)
    assert not errors, errors
    # X~ to the bit; the trajectory to float32 rounding (the bar of test_thread_ranks_gpu.py)
    assert np.array_equal(np.concatenate([r["x"] for r in results], axis=1), one["x"])
    for r in results:
        assert np.array_equal(r["history"], results[0]["history"]) and len(r["history"]) == len(one["history"]) == iters
        assert np.max(np.abs(r["history"] - one["history"]) / np.maximum(1.0, np.abs(one["history"]))) < 5e-5
        assert np.max(np.abs(r["ws"] - one["ws"])) < 1e-3 * np.max(np.abs(one["ws"]))


def test_kernel_names_are_in_the_trace_of_a_run():
    """`kernel_name` against the kernels that a profiler saw (a child process: the profiler stays attached to the one it ran in)"""
    code = r'''
import sys
sys.path.insert(0, %r)
import numpy as np
import torch
from torch.profiler import ProfilerActivity, profile
from linearcorex_amd.backend import HipBackend
for n, v, m in ((300, 200, 3), (2000, 3000, 30), (2000, 9000, 64), (700, 2000, 128), (20000, 2000, 64)):
    r = np.random.RandomState(0)
    be = HipBackend(n, v, m, np.float32, 0, x_storage="mx4")
    be.upload_x(r.randn(n, v).astype(np.float32))
    be.set_ws((r.randn(m, v) * 0.004).astype(np.float32))
    torch.cuda.synchronize()
    with profile(activities=[ProfilerActivity.CUDA]) as p:
        be.moments_a(0)
        be.moments_b(0, 0.3, False)
        be.moments_c(0)
        torch.cuda.synchronize()
    ran = {e.name.split("(")[0].replace("void ", "") for e in p.events()}
    for kind in (0, 1):
        assert be.kernel_name(kind) in ran, (n, v, m, be.kernel_name(kind), sorted(ran))
    be.close()
print("NAMES_OK")
''' % os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    p = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=110)
    assert p.returncode == 0 and "NAMES_OK" in p.stdout, (p.stdout[-500:], p.stderr[-2000:])


def test_fit_transform_is_fit_and_transform():
    """of the data as they are, not of the rounded ones"""
    x, kw = data("missing", 300, 100, 3)
    # (the seed is NumPy's global one, set when a model is made)
    a = Corex(n_hidden=3, seed=0, x_storage="mx4", **kw)
    y = a.fit_transform(x)
    b = Corex(n_hidden=3, seed=0, x_storage="mx4", **kw)
    yt = b.fit(x).transform(x)
    assert np.array_equal(a.ws, b.ws) and np.array_equal(y, yt)          # one process, one seed: the same launches
    want = O.preprocess(x.astype(np.float64), None, "standard", -999.0)[0] @ a.ws.T.astype(np.float64)
    s = np.abs(O.preprocess(x.astype(np.float64), None, "standard", -999.0)[0]) @ np.abs(a.ws.T.astype(np.float64))
    # float32: preprocessing (mean, scale, difference, quotient: 4 roundings of values up to |x - mean| + |mean|, |mean| < 1), 100 products and sums
    assert (np.abs(y - want) <= (100 + 8) * 2.0 ** -24 * s + 4 * 2.0 ** -24 * np.abs(a.ws).sum(axis=1)).all()
    rounded = kept(O.preprocess(x.astype(np.float64), None, "standard", -999.0)[0]) @ a.ws.T.astype(np.float64)
    assert np.abs(y - want).max() < 1e-3 * np.abs(rounded - want).max()
