"""The recurrent block's entry points without a GPU: structures as the header has them, refusals on the host (no call reaches a launch: the
pointers are made-up numbers), workspaces from shapes alone."""
import ctypes as C
import re
from pathlib import Path

import pytest

from workloadsuite_b200 import _lib

ROOT = Path(__file__).resolve().parent.parent
P = 0x10000


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


@pytest.mark.parametrize("name,mirror", [("SsdGatedScanArgs", _lib.GatedScanArgs), ("SsdGatedStepArgs", _lib.GatedStepArgs),
                                         ("SsdNormArgs", _lib.NormArgs)])
def test_structures_mirror_the_header(name, mirror):
    header = (ROOT / "include" / "ssd_b200.h").read_text()
    body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (name, name), header, re.S).group(1)
    body = re.sub(r"/\*.*?\*/", "", body, flags=re.S)
    fields = []
    for decl in filter(None, (d.strip() for d in body.split(";"))):
        kind, names = re.match(r"((?:const )?\w+\s*\*?)\s*(.*)", decl, re.S).groups()
        for n in names.split(","):
            n, count = re.match(r"\s*\*?\s*(\w+)(?:\[(\d+)\])?", n).groups()
            one = 8 if "*" in kind or kind.split()[0] in ("int64_t", "size_t") else 4
            fields.append((n, one * int(count or 1)))
    assert fields == [(f[0], C.sizeof(f[1])) for f in mirror._fields_]


def scan(**kw):
    a = _lib.GatedScanArgs()
    for f in ("x", "input_gate", "decay_gate", "decay", "y", "pieces", "dy", "dx", "dinput_gate", "ddecay_gate", "ddecay", "workspace"):
        setattr(a, f, P)
    a.workspace_bytes, a.rate, a.batch, a.seqlen, a.channels, a.dtype = 1 << 40, 8.0, 2, 100, 64, _lib.DTYPE_BF16
    for k, v in kw.items():
        setattr(a, k, v)
    return C.byref(a)


def test_gated_scan_refuses_on_the_host(lib):
    for call in (lib.ssd_b200_gated_scan, lib.ssd_b200_gated_scan_backward):
        assert call(None, None) == -1
        for field in ("x", "input_gate", "decay_gate", "decay"):
            assert call(scan(**{field: None}), None) == -1, field
        for field in ("batch", "seqlen", "channels", "wait_limit_ms"):
            assert call(scan(**{field: -1}), None) == -2, field
        for rate in (0.0, -1.0, float("nan"), float("inf")):
            assert call(scan(rate=rate), None) == -2
        assert call(scan(dtype=9), None) == -4
        assert call(scan(seqlen=0x7fffffff), None) == -8
        assert call(scan(batch=1 << 20, seqlen=1 << 20, channels=1 << 12), None) == -8
    assert lib.ssd_b200_gated_scan(scan(y=None), None) == -1
    for field in ("pieces", "dy", "dx", "dinput_gate", "ddecay_gate", "ddecay"):
        assert lib.ssd_b200_gated_scan_backward(scan(**{field: None}), None) == -1, field
    # scratch: sequences of more than a tile, and every gradient
    need = lambda back, **kw: lib.ssd_b200_gated_scan_workspace_bytes(scan(**kw), back)
    assert need(0) == 0 and need(0, seqlen=1) == 0 and need(0, seqlen=1000) > 0 and need(1) > 0
    assert need(0, batch=0) == 0 and need(0, seqlen=1000, workspace=None) == need(0, seqlen=1000)
    for bad in (dict(workspace=None), dict(workspace_bytes=16), dict(workspace=P + 16)):
        assert lib.ssd_b200_gated_scan(scan(seqlen=1000, **bad), None) == -5
        assert lib.ssd_b200_gated_scan_backward(scan(**bad), None) == -5


def test_gated_step_refuses_on_the_host(lib):
    def step(**kw):
        a = _lib.GatedStepArgs()
        for f in ("x", "input_gate", "decay_gate", "decay", "state", "state_out", "y"):
            setattr(a, f, P)
        a.rate, a.batch, a.channels, a.dtype = 8.0, 2, 64, _lib.DTYPE_BF16
        for k, v in kw.items():
            setattr(a, k, v)
        return lib.ssd_b200_gated_step(C.byref(a), None)

    assert lib.ssd_b200_gated_step(None, None) == -1
    for f in ("x", "input_gate", "decay_gate", "decay", "state", "state_out", "y"):
        assert step(**{f: None}) == -1
    assert step(batch=0) == -2 and step(channels=-1) == -2 and step(rate=0.0) == -2 and step(dtype=5) == -4
    assert step(batch=0x7fffffff, channels=0x7fffffff) == -8


def test_norms_refuse_on_the_host(lib):
    def norm(**kw):
        a = _lib.NormArgs()
        for f in ("x", "weight", "residual", "y", "residual_out", "inv_rms", "inv_rms_post", "dy", "dx", "dresidual", "dweight", "workspace"):
            setattr(a, f, P)
        a.workspace_bytes, a.rows, a.d, a.groups, a.eps = 1 << 40, 4, 64, 1, 1e-6
        a.dtype = a.residual_dtype = _lib.DTYPE_F16
        for k, v in kw.items():
            setattr(a, k, v)
        return C.byref(a)

    plain, back = lib.ssd_b200_rms_norm, lib.ssd_b200_rms_norm_backward
    gated, gback = lib.ssd_b200_gated_rms_norm, lib.ssd_b200_gated_rms_norm_backward
    for call in (plain, back, gated, gback):
        z = dict(z=P, dz=P) if call in (gated, gback) else {}
        assert call(None, None) == -1
        assert call(norm(x=None, **z), None) == -1 and call(norm(weight=None, **z), None) == -1
        assert call(norm(rows=0, **z), None) == -2 and call(norm(d=0, **z), None) == -2 and call(norm(eps=-1.0, **z), None) == -2
        assert call(norm(d=16385, **z), None) == -8
        assert call(norm(dtype=3, **z), None) == -4
    assert plain(norm(y=None), None) == -1 and plain(norm(residual_out=None), None) == -1
    assert plain(norm(residual_dtype=_lib.DTYPE_BF16), None) == -4 and back(norm(residual_dtype=_lib.DTYPE_BF16), None) == -4
    assert plain(norm(residual=None, scale=P), None) == -4 and plain(norm(residual=None, post_weight=P), None) == -4
    assert back(norm(post_weight=P, inv_rms_post=None), None) == -1
    assert gated(norm(), None) == -1 and gback(norm(z=P), None) == -1      # z, dz missing
    assert gated(norm(z=P, groups=3), None) == -2 and gated(norm(z=P, groups=0), None) == -2
    for field in ("dy", "dx", "inv_rms"):
        assert back(norm(**{field: None}), None) == -1 and gback(norm(z=P, dz=P, **{field: None}), None) == -1
    for bad in (dict(workspace=None), dict(workspace_bytes=8), dict(workspace=P + 4)):
        assert back(norm(**bad), None) == -5 and gback(norm(z=P, dz=P, **bad), None) == -5
    size = lib.ssd_b200_norm_workspace_bytes
    assert size(norm()) >= 4 * 64 and size(norm(post_weight=P)) == 2 * size(norm()) and size(norm(rows=0)) == 0


def test_conv_gradient_refuses_on_the_host(lib):
    def grad(x=P, w=P, bias=P, dy=P, dx=P, dw=P, db=P, ws=P, nbytes=1 << 40, b=2, s=10, c=16, taps=4, dtype=_lib.DTYPE_BF16, strides=(160, 16) * 3):
        return lib.ssd_b200_conv1d_silu_backward(x, w, bias, dy, dx, dw, db, ws, nbytes, b, s, c, taps, dtype, *strides, None, None)

    for k in ("x", "w", "dy", "dx", "dw", "db"):
        assert grad(**{k: None}) == -1
    assert grad(b=0) == -2 and grad(c=12) == -4 and grad(taps=5) == -4 and grad(taps=1) == -4 and grad(dtype=7) == -4
    assert grad(ws=None) == -5 and grad(nbytes=4) == -5
    assert grad(x=P + 2) == -7 and grad(strides=(160, 17) + (160, 16) * 2) == -7
    size = lib.ssd_b200_conv1d_silu_workspace_bytes
    assert size(2, 10, 16, 4) >= 2 * 5 * 16 * 4 and size(0, 10, 16, 4) == 0


def test_python_refuses_what_is_not_on_a_gpu():
    import torch

    import workloadsuite_b200 as W

    x, d, w = torch.zeros(1, 4, 8), torch.zeros(8), torch.ones(8)
    for call in (lambda: W.gated_scan(x, x, x, d), lambda: W.gated_scan_step(x[:, 0], x[:, 0], x[:, 0], d, torch.zeros(1, 8)),
                 lambda: W.rms_norm(x, w), lambda: W.gated_rms_norm(x, x, w), lambda: W.conv1d_silu(x.requires_grad_(True), torch.zeros(8, 1, 4))):
        with pytest.raises(RuntimeError, match="no CPU path"):
            call()
