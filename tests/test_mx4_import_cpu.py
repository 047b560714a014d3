"""The library has to find the HIP runtime of torch's wheel: torch comes first, and mx4 says so where it did not."""
import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.parametrize("code,warns", [
    ("from linearcorex_amd import _abi; _abi.load(); import linearcorex_amd.mx4", True),
    ("from linearcorex_amd import _abi; _abi.load(); import torch; import linearcorex_amd.mx4", True),
    ("import torch; from linearcorex_amd import _abi; _abi.load(); import linearcorex_amd.mx4", False),
    ("import linearcorex_amd.mx4; from linearcorex_amd import _abi; _abi.load(); assert _abi.torch_first", False),
    ("from linearcorex_amd import Corex; import linearcorex_amd.mx4", False)])
def test_the_order_of_imports(code, warns):
    p = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True, timeout=120)
    assert p.returncode == 0, p.stderr[-1500:]
    assert ("import torch" in p.stderr and "RuntimeWarning" in p.stderr) == warns, p.stderr[-1500:]
