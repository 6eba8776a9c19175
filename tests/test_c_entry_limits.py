"""The C entries of the adaLN passes and the 4-bit linear with what only a C caller can
pass: refused, or answered with 0, before any CUDA call.  Queries run in a process of
their own, so that one which ends its process is a failure and not the end of the run."""

import subprocess
import sys

import pytest

from sparsepr_b200 import build


@pytest.fixture(scope="module", autouse=True)
def library():
    build.build()


@pytest.mark.parametrize("name,sizes", [
    ("spr_adaln_backward_workspace_bytes", [(2 ** 40, 2 ** 40, 8, 0, 0), (2 ** 32, 2 ** 32, 8, 1, 1),
                                            (2 ** 31, 1, 8, 0, 0), (1, 2 ** 62, 8, 0, 1), (1, 4, 2 ** 30, 0, 0),
                                            (-1, 4, 8, 0, 0), (0, 4, 8, 0, 0)]),
    ("spr_int4_linear_workspace_bytes", [(2 ** 62, 8, 64, 32, 1), (2 ** 40, 2 ** 40, 64, 32, 1), (1, 8, 2 ** 36, 32, 1),
                                         (1, 8, 2 ** 37, 32, 1), (1, 8, 64, 2 ** 30, 1), (1, 8, 2 ** 36, 2 ** 30, 1),
                                         (1, 2 ** 62, 64, 32, 1), (1, 8, 64, 33, 1), (1, 8, 64, 0, 1)]),
    ("spr_int4_linear_grad_workspace_bytes", [(2 ** 62, 8, 64, 32, 1), (2 ** 40, 2 ** 40, 64, 32, 1),
                                              (1, 8, 2 ** 36, 32, 1), (1, 8, 2 ** 37, 32, 1), (1, 2 ** 62, 64, 32, 1),
                                              (1, 8, 2 ** 36, 2 ** 30, 1), (1, 8, 64, 48, 1)]),
])
def test_workspace_of_sizes_that_no_call_takes(name, sizes):
    script = f"from sparsepr_b200 import _lib\nfor s in {sizes!r}: print(_lib.query({name!r}, *s))"
    out = subprocess.run([sys.executable, "-c", script], capture_output=True, text=True, timeout=120)
    assert out.returncode == 0, (out.returncode, out.stderr)
    assert out.stdout.split() == ["0"] * len(sizes)
