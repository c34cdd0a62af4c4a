"""CPU: the paged cache's Python surface."""
import subprocess
import sys

import mlz_b200
from tests.conftest import ROOT


def _python(code):
    return subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True, timeout=120)


def test_star_import_needs_no_torch():
    r = _python("import sys; sys.modules['torch'] = None\n"
                "from mlz_b200 import *\n"
                "assert callable(mul_mat) and ROPE_HALVES == 1")
    assert r.returncode == 0, r.stderr


def test_paged_calls_are_the_packages():
    from mlz_b200 import paged
    for name in paged.__all__:
        assert getattr(mlz_b200, name) is getattr(paged, name)
        assert name in dir(mlz_b200)
