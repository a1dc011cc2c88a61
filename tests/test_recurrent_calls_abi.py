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


def test_sizes_next_to_the_end_of_32_bits(lib):
    """Channels that rounding up to strips of 64 takes past 2^31, tokens that a run's rim does: too large, not a negative number of strips."""
    def scan(**kw):
        a = _lib.GatedScanArgs()
        for f in ("x", "input_gate", "decay_gate", "decay", "y", "pieces", "dy", "dx", "dinput_gate", "ddecay_gate", "ddecay", "workspace"):
            setattr(a, f, P)
        a.workspace_bytes, a.rate, a.batch, a.seqlen, a.channels, a.dtype = 1 << 62, 8.0, 1, 1, 64, _lib.DTYPE_BF16
        for k, v in kw.items():
            setattr(a, k, v)
        return C.byref(a)

    for channels in (0x7fffffff, 0x7fffffff - 60, 0x7fffff80):
        for call, back in ((lib.ssd_b200_gated_scan, 0), (lib.ssd_b200_gated_scan_backward, 1)):
            assert call(scan(channels=channels), None) == -8
            assert lib.ssd_b200_gated_scan_workspace_bytes(scan(channels=channels), back) == 0
    conv = lambda s, c: lib.ssd_b200_conv1d_silu_backward(P, P, P, P, P, P, P, P, 1 << 62, 1, s, c, 4, _lib.DTYPE_BF16, *(8, 8) * 3, None, None)
    assert conv(1, 0x7fffffff - 7) == -8 and conv(1, 64 * 65535 + 8) == -8
    assert conv(0x7fffffff, 8) == -8 and conv(0x7fffffff - 3, 8) == -8
    assert lib.ssd_b200_conv1d_silu(P, P, P, P, 1, 0x7fffffff - 3, 8, 4, _lib.DTYPE_BF16, *(8, 8) * 2, None) == -8
