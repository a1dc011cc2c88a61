"""Calls of the recurrent block's operators that the documentation allows and that once went wrong, each by itself.
Tolerances as in test_recurrent_gpu.py."""
import math
import subprocess
import sys
from pathlib import Path

import pytest
import torch

from test_recurrent_gpu import DELTA, DEV, DTYPES, W, _no_wait_ran_out, check, leaves, scan_inputs, scan_reference  # noqa: F401

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


_FIRST_IN_A_CAPTURE = """
import torch
import workloadsuite_b200 as W
from workloadsuite_b200 import _lib

x = torch.randn(2, 40, 16, device="cuda", requires_grad=True)
w = torch.randn(16, 1, 4, device="cuda", requires_grad=True)
graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
torch.cuda.synchronize()
with torch.inference_mode(), torch.cuda.graph(torch.cuda.CUDAGraph(), stream=side):
    {first}
with torch.cuda.graph(graph, stream=side):
    y = W.conv1d_silu(x, w)
    torch.autograd.grad([y], [x, w], [torch.ones_like(y)])
word = _lib.fast().status_word(0)
assert (word == 0).all()
word[0] = 5
torch.cuda.synchronize()
graph.replay()
assert W.device_status() == 5 and W.device_status() == 0
"""

_FIRST_FROM_MANY_THREADS = """
import threading
import torch
import workloadsuite_b200 as W
from workloadsuite_b200 import _lib

_lib.fast()
x, w = torch.randn(2, 40, 16, device="cuda"), torch.randn(16, 1, 4, device="cuda")
gate, seen = threading.Barrier(8), []

def work(n):
    leaf = x.clone().requires_grad_(True)
    y = W.conv1d_silu(leaf, w).sum()
    torch.cuda.synchronize()
    gate.wait()
    if n % 2:
        y.backward()
    seen.append(_lib.fast().status_word(0).data_ptr())

threads = [threading.Thread(target=work, args=(n,)) for n in range(8)]
[t.start() for t in threads]
[t.join() for t in threads]
assert len(seen) == 8 and len(set(seen)) == 1, seen
"""


@pytest.mark.parametrize("program", [_FIRST_IN_A_CAPTURE.format(first="pass"), _FIRST_IN_A_CAPTURE.format(first="W.gated_scan(x, x, x, w[:, 0, 0])"),
                                     _FIRST_FROM_MANY_THREADS], ids=["a capture's backward", "a capture's forward", "threads"])
def test_the_status_word_is_made_once_and_outside_of_captures(program):
    """In processes that have not used it: its first use in a capture (of a backward pass, which another thread runs), or by many threads.  A
    status that nobody has read is there after a replay."""
    r = subprocess.run([sys.executable, "-c", program], cwd=Path(__file__).resolve().parent.parent, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]


def test_the_model_calls_layers_that_are_not_as_built_with_one_tensor():
    """A forward that is replaced on a layer or a norm (for offloading, recomputation, logging), or on their class, takes one tensor and gives
    one, as in the reference; so does what hooks on every module see.  Results: the sums are the same numbers, a norm in another place
    may round the other way (half a step, 2^-11, through two layers with a gain of some units)."""
    import torch.nn.modules.module as every
    from torch.utils.checkpoint import checkpoint

    from workloadsuite_b200 import mamba_model as M

    torch.manual_seed(6)
    model = M.Model(128, 3, 4, 128, 64, 2, 64, 4).to(DEV).eval()
    x = torch.randn(1, 128, 128, dtype=torch.float16, device=DEV)
    with torch.no_grad():
        want = model(x)
        same = lambda got: ((got - want).abs().max() <= 2.0 ** -8 * want.abs().max()).item()
        for module in (model.layers[1], model.layers[2].norm, model.final_norm):
            seen, old = [], module.forward
            module.forward = lambda u: (seen.append(u.shape), old(u))[1]
            assert same(model(x)) and seen == [x.shape]
            del module.forward
            module.forward = lambda u: checkpoint(old, u, use_reentrant=False)
            assert same(model(x))
            del module.forward
        for cls, calls in ((M.SSDLayer, 3), (M.RMSNorm, 4)):
            seen, old = [], cls.forward
            cls.forward = lambda self, u: (seen.append(u.shape), old(self, u))[1]
            try:
                assert same(model(x)) and len(seen) == calls
            finally:
                cls.forward = old
        seen = []
        hook = every.register_module_forward_hook(lambda m, a, out: seen.append((type(m).__name__, len(a), isinstance(out, torch.Tensor))))
        try:
            assert same(model(x))
        finally:
            hook.remove()
        assert all(n == 1 and one for _, n, one in seen) and [n for n, _, _ in seen].count("RMSNorm") == 4
        assert torch.equal(model(x), want)


def test_a_tangent_is_refused_and_not_dropped():
    """Whichever operand carries it, recorded for a backward gradient or not; outside of dual numbers the same call is made."""
    import torch.autograd.forward_ad as forward_ad

    v = scan_inputs(1, 9, 16, torch.float32, False, True, seed=3)
    x, w, cw, cb = v["x"], torch.ones(16, device=DEV), torch.randn(16, 1, 4, device=DEV), torch.zeros(16, device=DEV)
    calls = [("gated_scan", lambda *a: W().gated_scan(*a[:4], initial_state=a[4]), (x, v["i"], v["r"], v["decay"], v["h"])),
             ("rms_norm", lambda *a: W().rms_norm(a[0], a[1], residual=a[2], post_weight=a[3], scale=a[4]), (x, w, v["dy"], w, w)),
             ("rms_norm", W().rms_norm, (x, w)), ("gated_rms_norm", W().gated_rms_norm, (x, v["i"], w)), ("conv1d_silu", W().conv1d_silu, (x, cw, cb))]
    for name, call, args in calls:
        for records in (False, True):
            for n in range(len(args)):
                with forward_ad.dual_level():
                    other = [a.clone().requires_grad_(records and m != n) for m, a in enumerate(args)]
                    call(*other)
                    other[n] = forward_ad.make_dual(other[n], torch.ones_like(other[n]))
                    with pytest.raises(NotImplementedError, match=f"{name} has no forward-mode gradient"):
                        call(*other)


def test_the_model_s_norm_carries_what_pytorch_s_does():
    """Forward-mode tangents, function transforms and tensor subclasses go through PyTorch's operators, as with nn.RMSNorm."""
    import torch.autograd.forward_ad as forward_ad

    from workloadsuite_b200 import mamba_model as M

    class Sub(torch.Tensor):
        pass

    own, plain = M.RMSNorm(64).to(DEV), torch.nn.RMSNorm(64).to(DEV)
    with torch.no_grad():
        own.weight.uniform_(0.5, 1.5)
        plain.weight.copy_(own.weight)
    x, t = torch.randn(4, 5, 64, device=DEV), torch.randn(4, 5, 64, device=DEV)
    with forward_ad.dual_level():
        a, b = (forward_ad.unpack_dual(n(forward_ad.make_dual(x, t))) for n in (own, plain))
        assert torch.equal(a.primal, b.primal) and torch.equal(a.tangent, b.tangent)
        y, r = own(x, forward_ad.make_dual(x, t))
        assert torch.equal(forward_ad.unpack_dual(r).tangent, t) and forward_ad.unpack_dual(y).tangent is not None
    for transform in (torch.func.vmap, lambda f: torch.func.grad(lambda u: f(u).sum()), lambda f: lambda u: torch.func.jvp(f, (u,), (t,))[1]):
        assert torch.equal(transform(own)(x), transform(plain)(x))
    y = own(x.as_subclass(Sub))
    assert type(y) is Sub and torch.equal(y.as_subclass(torch.Tensor), plain(x))


@pytest.mark.parametrize("records", [False, True])
def test_conv1d_silu_says_the_same_whether_it_records_or_not(records):
    x = torch.randn(2, 30, 8, device=DEV).requires_grad_(records)
    w = torch.randn(8, 1, 4, device=DEV)
    for error, args in ((ValueError, (x, w, torch.zeros(7, device=DEV))), (ValueError, (x, w[:4])), (ValueError, (x, w.reshape(8, 2, 2))),
                        (ValueError, (x, w.cpu())), (ValueError, (x.transpose(1, 2), w)), (NotImplementedError, (x, w[..., :1])),
                        (NotImplementedError, (x[..., :7], w[:7])), (NotImplementedError, (x, w.repeat(1, 1, 2))), (W().SsdError, (x[:, :0], w))):
        with pytest.raises(error):
            W().conv1d_silu(*args)


@pytest.mark.parametrize("of", ["x", "w", "bias"])
def test_conv1d_silu_takes_tensor_subclasses(of):
    """The kernels read them, and gradients arrive at them."""
    class Sub(torch.Tensor):
        pass

    v = {"x": torch.randn(2, 30, 8, device=DEV), "w": torch.randn(8, 1, 4, device=DEV), "bias": torch.randn(8, device=DEV)}
    plain = {k: t.clone().requires_grad_(True) for k, t in v.items()}
    sub = {k: (t.clone().as_subclass(Sub) if k == of else t.clone()).requires_grad_(True) for k, t in v.items()}
    y, want = (W().conv1d_silu(*d.values()) for d in (sub, plain))
    assert torch.equal(y, want)
    dy = torch.randn_like(want)
    for a, b in zip(torch.autograd.grad([y], list(sub.values()), [dy]), torch.autograd.grad([want], list(plain.values()), [dy])):
        assert torch.equal(a.as_subclass(torch.Tensor), b)
    with torch.no_grad():
        assert torch.equal(W().conv1d_silu(*sub.values()), want)


def test_numbers_that_32_bits_do_not_hold_are_refused():
    """A limit of 2^32 milliseconds was taken as none, one of 2^70 and as many groups were a SystemError."""
    x, d, h = torch.randn(2, 300, 8, device=DEV), torch.zeros(8, device=DEV), torch.zeros(2, 8, device=DEV)
    for bad in (dict(wait_limit_ms=2 ** 31), dict(wait_limit_ms=2 ** 32), dict(wait_limit_ms=2 ** 70), dict(rate=1e39), dict(rate=1e-50)):
        with pytest.raises(ValueError):
            W().gated_scan(x, x, x, d, **bad)
    with pytest.raises(ValueError):
        W().gated_scan_step(x[:, 0], x[:, 0], x[:, 0], d, h, rate=1e39)
    for bad in (dict(groups=2 ** 33), dict(groups=2 ** 70), dict(groups=2 ** 32 + 1), dict(groups=0), dict(eps=1e39), dict(eps=-1e-60)):
        with pytest.raises(ValueError):
            W().gated_rms_norm(x, x, d, **bad)
    with pytest.raises(ValueError):
        W().rms_norm(x, d, eps=1e39)
    a, b = W().gated_scan(x, x, x, d, wait_limit_ms=2 ** 31 - 1), W().gated_scan(x, x, x, d)
    assert torch.equal(a, b) and torch.equal(W().rms_norm(x, d + 1, eps=1e-60), W().rms_norm(x, d + 1, eps=0.0))


def test_the_block_s_operators_take_tensor_subclasses():
    class Sub(torch.Tensor):
        pass

    sub = lambda t: t.detach().clone().as_subclass(Sub)
    same = lambda a, b: torch.equal(a.as_subclass(torch.Tensor), b)
    v = scan_inputs(2, 70, 16, torch.float16, True, True, seed=3)
    args, w = (v["x"], v["i"], v["r"], v["decay"]), torch.randn(16, device=DEV)
    want = W().gated_scan(*args, initial_state=v["h"], reset=v["reset"])
    for n in range(6):
        given = [sub(t) if m == n else t for m, t in enumerate((*args, v["h"], v["reset"]))]
        assert torch.equal(W().gated_scan(*given[:4], initial_state=given[4], reset=given[5]), want)
    out = sub(want)
    assert same(W().gated_scan(*args, initial_state=v["h"], reset=v["reset"], out=out.zero_()), want) and same(out, want)
    state, other = v["h"].clone(), sub(v["h"])
    y = W().gated_scan_step(*(t[:, 0] for t in args[:3]), args[3], state)
    assert torch.equal(W().gated_scan_step(*(sub(t[:, 0]) for t in args[:3]), sub(args[3]), other), y) and same(other, state)
    for call, ops in ((W().rms_norm, (v["x"], w)), (lambda x, w, r: W().rms_norm(x, w, residual=r)[0], (v["x"], w, v["dy"])),
                      (W().gated_rms_norm, (v["x"], v["i"], w))):
        plain, given = ([t.clone().requires_grad_(True) for t in ops], [sub(t).requires_grad_(True) for t in ops])
        want, got = call(*plain), call(*given)
        assert same(got, want)
        for a, b in zip(torch.autograd.grad([got], given, [v["dy"]]), torch.autograd.grad([want], plain, [v["dy"]])):
            assert same(a, b)


def test_a_backward_pass_notices_that_what_it_saved_was_written_over():
    """By `out`, or by a step's state: an error as for any operator that works in place, not a gradient of other numbers."""
    x, w, h = torch.randn(2, 16, device=DEV), torch.randn(16, device=DEV), torch.zeros(2, 16, device=DEV)
    cw = torch.randn(16, 1, 2, device=DEV)
    calls = {"gated_scan": lambda o: W().gated_scan(x[None], x[None], x[None], w, out=o[None]),
             "step's y": lambda o: W().gated_scan_step(x, x, x, w, h, out=o), "step's state": lambda o: W().gated_scan_step(x, x, x, w, o),
             "step's new state": lambda o: W().gated_scan_step(x, x, x, w, h, out_state=o), "rms_norm": lambda o: W().rms_norm(x, w, out=o),
             "gated_rms_norm": lambda o: W().gated_rms_norm(x, x, w, out=o), "conv1d_silu": lambda o: W().conv1d_silu(x[None], cw, out=o[None]),
             "conv1d_silu, the long way": lambda o: W().conv1d_silu(x[None], cw.double(), out=o[None])}
    for name, call in calls.items():
        leaf, saved = torch.ones(2, 16, device=DEV, requires_grad=True), torch.randn(2, 16, device=DEV)
        y = leaf * saved
        call(saved)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.sum().backward()
        with torch.inference_mode():
            call(torch.randn(2, 16, device=DEV))


def test_a_tile_that_is_lost_on_purpose_is_the_first_one():
    """Whichever CTA takes it: every such launch reports its waits (the first CTA may find no tile left, or one that nobody waits for)."""
    import ctypes as C

    from workloadsuite_b200 import _lib

    lib, (b, s, d) = _lib.load(), (1, 300, 64)
    v = scan_inputs(b, s, d, torch.bfloat16, False, False, seed=8)
    y, status = torch.zeros_like(v["x"]), torch.zeros(1, dtype=torch.int32, device=DEV)
    a = _lib.GatedScanArgs()
    a.x, a.input_gate, a.decay_gate, a.decay = (v[k].data_ptr() for k in ("x", "i", "r", "decay"))
    a.y, a.status = y.data_ptr(), status.data_ptr()
    a.rate, a.batch, a.seqlen, a.channels, a.dtype, a.wait_limit_ms, a.inject_lost_tile = 8.0, b, s, d, _lib.DTYPE_BF16, 5, 1
    for f in ("x", "input_gate", "decay_gate", "y"):
        setattr(a, f + "_stride", (C.c_int64 * 2)(s * d, d))
    ws = torch.empty(lib.ssd_b200_gated_scan_workspace_bytes(C.byref(a), 0), dtype=torch.uint8, device=DEV)
    a.workspace, a.workspace_bytes = ws.data_ptr(), ws.numel()
    side = torch.cuda.Stream()
    m = torch.randn(2048, 2048, device=DEV)
    for n in range(100):
        status.zero_()
        with torch.cuda.stream(side):
            m @ m
        assert lib.ssd_b200_gated_scan(C.byref(a), C.c_void_p(torch.cuda.current_stream().cuda_stream)) == 0
        torch.cuda.synchronize()
        assert status.item() == 8, n


@pytest.mark.parametrize("b,s", [(1, 1), (1, 5), (3, 1)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_conv1d_silu_gradient_of_rows_that_start_anywhere(dtype, b, s):
    """x and dy one number off the boundary of two, single rows among them: strides of one row may be anything, and it counts as contiguous."""
    d, taps = 24, 3
    gen = torch.Generator(device=DEV).manual_seed(b + s)
    rnd = lambda *n: torch.randn(*n, generator=gen, device=DEV).to(dtype)
    x, dy, w = rnd(b, s, d), rnd(b, s, d), rnd(d, 1, taps)

    def off(t, width):
        buf = torch.zeros(b, s, width, dtype=dtype, device=DEV)
        buf[..., 5:5 + d] = t
        return buf[..., 5:5 + d]

    def run(x, dy):
        ins = [x.detach().requires_grad_(True), w.detach().requires_grad_(True)]
        y = W().conv1d_silu(*ins)
        return [y.detach(), *torch.autograd.grad([y], ins, [dy])]

    want = run(x, dy)
    for width in (36, 37):
        for a, c in ((off(x, width), dy), (x, off(dy, width)), (off(x, width), off(dy, width))):
            for g, r in zip(run(a, c), want):
                near = 2 * torch.finfo(dtype).eps * r.abs() + 2 * DELTA * r.abs().max()
                assert ((g - r).abs() <= near).all()


@pytest.mark.parametrize("transform", [torch.func.vmap, lambda f: torch.func.grad(lambda t: f(t).sum()), lambda f: lambda t: torch.func.jvp(f, (t,), (t,))])
def test_function_transforms_are_refused_by_name(transform):
    w, decay = torch.ones(16, device=DEV), torch.zeros(16, device=DEV)
    x = torch.randn(3, 2, 9, 16, device=DEV)
    for name, call in (("gated_scan", lambda t: W().gated_scan(t, t, t, decay)), ("rms_norm", lambda t: W().rms_norm(t, w)),
                       ("gated_rms_norm", lambda t: W().gated_rms_norm(t, t, w)), ("conv1d_silu", lambda t: W().conv1d_silu(t, torch.ones(16, 1, 2, device=DEV)))):
        with pytest.raises(NotImplementedError, match=name):
            transform(call)(x if transform is torch.func.vmap else x[0])


_CAPTURE_BESIDE_AN_EAGER_GRAPH = """
import torch
import workloadsuite_b200 as W

x = torch.randn(2, 40, 16, device="cuda", requires_grad=True)
w = torch.ones(16, device="cuda", requires_grad=True)
alive, side = W.gated_scan(x, x, x, w), torch.cuda.Stream()      # recorded on another stream than the one that captures
torch.cuda.synchronize()
try:
    with torch.cuda.graph(torch.cuda.CUDAGraph(), stream=side):
        torch.autograd.grad([W.gated_scan(x, x, x, w)], [x, w], [torch.ones_like(x)])
except RuntimeError as e:
    print("raised", e)
"""

_BACKWARD_WITHOUT_MEMORY = """
import torch
import workloadsuite_b200 as W

x = torch.randn(4096, 4096, device="cuda", requires_grad=True)
w = torch.ones(4096, device="cuda", requires_grad=True)
calls = [W.rms_norm(x, w), W.gated_rms_norm(x, x, w), W.gated_scan(x[None], x[None], x[None], w)[0], W.conv1d_silu(x[None], torch.ones(4096, 1, 2, device="cuda"))[0]]
dy = torch.ones_like(x)
free = torch.cuda.memory_reserved()
torch.cuda.set_per_process_memory_fraction(free / torch.cuda.get_device_properties(0).total_memory)
keep = []
try:
    while True:
        keep.append(torch.empty(1 << 20, device="cuda"))
except torch.OutOfMemoryError:
    pass
raised = 0
for y in calls:
    try:
        torch.autograd.grad([y], [x], [dy])
    except torch.OutOfMemoryError:
        raised += 1
assert raised == len(calls), raised
del keep
torch.cuda.empty_cache()
torch.cuda.set_per_process_memory_fraction(1.0)
for y in (W.rms_norm(x, w),):
    torch.autograd.grad([y], [x], [dy])
print("raised")
"""


@pytest.mark.parametrize("program", [_CAPTURE_BESIDE_AN_EAGER_GRAPH, _BACKWARD_WITHOUT_MEMORY], ids=["capture", "memory"])
def test_what_a_backward_pass_runs_into_is_raised(program):
    """In processes of their own: a capture that PyTorch cannot make, an allocation that fails in autograd's thread."""
    r = subprocess.run([sys.executable, "-c", program], cwd=Path(__file__).resolve().parent.parent, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "raised" in r.stdout, (r.returncode, r.stdout[-500:], r.stderr[-2000:])
