"""Calls of the recurrent block's operators that the documentation allows and that once went wrong, each by itself.
Tolerances as in test_recurrent_gpu.py."""
import math

import pytest
import torch

from test_recurrent_gpu import DEV, DTYPES, W, _no_wait_ran_out, check, leaves, scan_inputs, scan_reference  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("aligned", [True, False])
@pytest.mark.parametrize("dtype", DTYPES)
def test_conv1d_silu_far_below_zero(dtype, aligned):
    """silu from -30 to 30 through the conv (taps 0, 1, so that what it is taken of is exact): rounded once, from 32 bits."""
    a = torch.linspace(-30, 30, 8 * 8192).to(dtype).reshape(1, -1, 8).to(DEV)
    w = torch.zeros(8, 1, 2, dtype=dtype, device=DEV)
    w[:, 0, 1] = 1
    if not aligned:
        a = torch.cat([a[..., :1], a], -1)[..., 1:]
        assert a.stride(1) == 9
    y = W().conv1d_silu(a, w)
    a6 = a.double()
    ref = a6 / (1 + torch.exp(-a6))
    check(y, ref, ref.abs(), 1, "silu")
