"""Derivatives, transforms and traced programs of the 4-bit products (tests/mx4_derivatives.py) on the GPU."""
import pytest

torch = pytest.importorskip("torch")
from tests import mx4_derivatives as D                                   # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("check", D.CHECKS, ids=lambda f: f.__name__)
def test_on_the_gpu(check):
    from linearcorex_amd import mx4
    check(mx4, "cuda")
