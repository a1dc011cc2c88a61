"""Calls of the recurrent block's entry points that have to be refused on the host, before anything is launched (the pointers are made-up
numbers)."""
import ctypes as C

import pytest

from workloadsuite_b200 import _lib

P = 0x10000


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def norm(**kw):
    a = _lib.NormArgs()
    for f in ("x", "weight", "residual", "y", "residual_out", "inv_rms", "inv_rms_post", "dy", "dx", "dresidual", "dweight", "workspace"):
        setattr(a, f, P)
    a.workspace_bytes, a.rows, a.d, a.groups, a.eps = 1 << 40, 4, 64, 1, 1e-6
    a.dtype = a.residual_dtype = _lib.DTYPE_F16
    for k, v in kw.items():
        setattr(a, k, v)
    return C.byref(a)


def test_a_norm_without_a_gate_takes_none(lib):
    """With a gate the workspace is asked for as the gated gradient's, which may be smaller than what the plain one writes: 5 000 rows of 16
    groups of 64 against 1 024 numbers, and a scale's sums beside the weight's."""
    shape = dict(rows=5000, d=1024, groups=16, post_weight=P)
    size = lib.ssd_b200_norm_workspace_bytes
    gated, plain = size(norm(z=P, **shape)), size(norm(**shape))
    assert gated < plain
    for nbytes in (gated, 1 << 40):
        assert lib.ssd_b200_rms_norm_backward(norm(z=P, dz=P, workspace_bytes=nbytes, **shape), None) == -4
        assert lib.ssd_b200_rms_norm(norm(z=P, workspace_bytes=nbytes, **shape), None) == -4
    assert lib.ssd_b200_rms_norm_backward(norm(workspace_bytes=gated, **shape), None) == -5
