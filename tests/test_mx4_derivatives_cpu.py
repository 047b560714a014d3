"""Derivatives, transforms and traced programs of the 4-bit products, the library's calls computed on the host (tests/mx4_derivatives.py)."""
import pytest

torch = pytest.importorskip("torch")
from linearcorex_amd import mx4                                          # noqa: E402
from tests import mx4_derivatives as D                                   # noqa: E402


@pytest.mark.parametrize("check", D.CHECKS, ids=lambda f: f.__name__)
def test_on_the_host(check, monkeypatch):
    monkeypatch.setattr(mx4, "_on_gpu", lambda t, what: None)
    monkeypatch.setattr(mx4, "_call", D.Emulator())
    monkeypatch.setattr(mx4, "_workspace_bytes", lambda *a: 0)
    check(mx4, "cpu")
