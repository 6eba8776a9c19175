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


def _refused(msg, name, *args):
    from sparsepr_b200 import _lib

    with pytest.raises(RuntimeError, match=msg):
        _lib.call(name, *args)


def _adaln(**kw):
    from sparsepr_b200 import _lib

    o = _lib.SprAdaln(dtype=1, mod_dtype=0, batch=1, tokens=4, channels=8, eps=1e-6, scale_offset=1.0, x=256, h=256)
    for k, v in kw.items():
        setattr(o, k, v)
    return o


@pytest.mark.parametrize("kw,msg", [
    (dict(mean=256), "ARG.*rstd"), (dict(rstd=256), "ARG.*rstd"), (dict(x=257), "ALIGN"), (dict(h=255), "ALIGN"),
    (dict(y=257, z=256), "ALIGN"), (dict(y=256, z=257), "ALIGN"), (dict(shift=258), "ALIGN"),
    (dict(scale=258), "ALIGN"), (dict(y=256, z=256, gate=258), "ALIGN"), (dict(mean=258, rstd=256), "ALIGN"),
    (dict(mod_dtype=1, shift=257), "ALIGN"),
])
def test_adaln_forward_operands(kw, msg):
    import ctypes

    o = _adaln(**kw)
    _refused("SPR_ERR_" + msg, "spr_adaln_forward", ctypes.addressof(o), None)


@pytest.mark.parametrize("kw,msg", [
    (dict(dz=256), "ARG.*without a branch"), (dict(dh=257), "ALIGN"), (dict(dx=257), "ALIGN"),
    (dict(dshift=258), "ALIGN"), (dict(dscale=258), "ALIGN"), (dict(dscale=257), "ALIGN"),
])
def test_adaln_backward_operands(kw, msg):
    import ctypes

    from sparsepr_b200 import _lib

    o = _adaln(mean=256, rstd=256)
    g = _lib.SprAdalnGrad(**{**dict(dh=256, dx=256), **kw})
    _refused("SPR_ERR_" + msg, "spr_adaln_backward", ctypes.addressof(o), ctypes.addressof(g), 256, 1 << 30, None)


@pytest.mark.parametrize("kw", [dict(x=257), dict(scales=258), dict(bias=257), dict(y=257), dict(workspace=258)])
def test_int4_operands(kw):
    a = {**dict(x=256, scales=256, bias=None, y=256, workspace=None), **kw}
    _refused("SPR_ERR_ALIGN", "spr_int4_linear", a["x"], 64, 1, 1, 8, 64, 32, 256, a["scales"], 0, None, a["bias"],
             a["y"], a["workspace"], 1 << 30, None)
    if "bias" not in kw:
        _refused("SPR_ERR_ALIGN", "spr_int4_linear_grad", a["x"], 8, 1, 1, 8, 64, 32, 256, a["scales"], 0, None, a["y"],
                 a["workspace"] or 256, 1 << 30, None)


@pytest.mark.parametrize("current", [0, 1])
def test_workspace_is_sized_under_the_device_of_the_launch(monkeypatch, current):
    """Tensors on device 1: the size, the allocation and the launch all see device 1 as the current one."""
    import contextlib
    import types

    import torch

    from sparsepr_b200 import kernels as K

    state, seen = {"device": current}, []

    @contextlib.contextmanager
    def device(index):
        before, state["device"] = state["device"], index
        yield
        state["device"] = before

    monkeypatch.setattr(torch.cuda, "current_device", lambda: state["device"])
    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda index: 7 + index, raising=False)
    monkeypatch.setattr(K._lib, "query", lambda name, *a: seen.append((name, a, state["device"])) or 64)
    monkeypatch.setattr(K._lib, "call", lambda name, *a: seen.append((name, a, state["device"])))
    buffer = torch.empty(64, dtype=torch.uint8)
    like = types.SimpleNamespace(get_device=lambda: 1, new_empty=lambda n, dtype: buffer)
    K._launch_with_workspace(like, "query", (1, 2), "entry", 3, 4)
    assert seen == [("query", (1, 2), 1), ("entry", (3, 4, buffer.data_ptr(), 64, 8), 1)]
    assert state["device"] == current
