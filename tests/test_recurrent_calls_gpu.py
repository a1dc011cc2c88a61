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


@pytest.mark.parametrize("d", [64, 51])
@pytest.mark.parametrize("dtype", DTYPES)
def test_gated_scan_rounds_a_channel_whatever_its_neighbours_are(dtype, d):
    """A gate that is shut (a mask), one that is not a number, and a channel that decays fast are nothing to the bits of the other channels,
    nor to those of their gradients."""
    v = scan_inputs(2, 700, d, dtype, True, True, seed=31)

    def run(**new):
        w = dict(v, **new)
        ins = [w[k].detach().clone().requires_grad_(True) for k in ("x", "i", "r", "decay", "h")]
        y, fin = W().gated_scan(*ins[:4], initial_state=ins[4], reset=v["reset"], return_final_state=True)
        return [y.detach(), fin.detach(), *torch.autograd.grad([y, fin], ins, [v["dy"], v["dh"]])]

    want = run()
    c = 5
    others = torch.arange(d, device=DEV) != c
    for name, at, value in (("i", (0, slice(100, 300), c), -math.inf), ("i", (1, 3, c), -41.0), ("i", (1, 600, c), math.nan), ("x", (0, 9, c), math.inf),
                            ("r", (0, 50, c), math.nan), ("decay", (c,), 0.0), ("decay", (c,), 4.0), ("decay", (c,), math.nan)):
        changed = v[name].clone()
        changed[at] = value
        for n, (g, w) in enumerate(zip(run(**{name: changed}), want)):
            assert torch.equal(g[..., others], w[..., others]), (name, value, n)
