"""The gated recurrence, the block norms and the gradient of conv1d + SiLU against their definitions in 64 bits.

Tolerances are counted, not fitted.  An output is rounded once to its type: half a step, ``finfo.eps / 2`` of its value (and half the
smallest step where float16 runs out of exponents).  What is computed in float32 before is off by at most ``DELTA`` of the sum of the
magnitudes it is made of, DELTA being 32 units of 2^-24: the functions of the special-function unit are good to 2^-22, four units each, and
no term passes more than eight of them or of the roundings between.  A number that s such steps follow one another in is allowed
1 + sqrt(s) times that (independent errors)."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
DELTA = 32 * 2.0 ** -24
DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def W():
    import workloadsuite_b200

    return workloadsuite_b200


@pytest.fixture(autouse=True)
def _no_wait_ran_out():
    yield
    assert W().device_status(DEV) == 0


def check(got, ref, mag, steps=1, what=""):
    info = torch.finfo(got.dtype)
    g, r, m = got.detach().double().cpu(), ref.detach().double().cpu(), mag.detach().double().cpu()
    assert g.shape == r.shape, (what, g.shape, r.shape)
    tol = info.eps / 2 * r.abs() + DELTA * (1 + math.sqrt(steps)) * m + info.smallest_normal * info.eps / 2
    bad = ~((g - r).abs() <= tol)
    if bad.any():
        i = int(((g - r).abs() - tol).nan_to_num(nan=math.inf).argmax())
        raise AssertionError(f"{what}: {int(bad.sum())} of {g.numel()} off, worst {g.flatten()[i]} for {r.flatten()[i]}, allowed {tol.flatten()[i]}")


# ---- gated recurrence -----------------------------------------------------------------------------------

def scan_inputs(b, s, d, dtype, reset, state, seed, strided=False):
    gen = torch.Generator().manual_seed(seed)
    rnd = lambda *n: torch.randn(*n, generator=gen)
    top = torch.rand(d, generator=gen) * 0.099 + 0.9
    v = {"decay": torch.log(torch.expm1(-torch.log(top) / 8.0)).to(DEV)}
    if strided:     # columns of one projection's output, an odd place between others
        buf = rnd(b, s, 3 * d + 5).to(dtype).to(DEV)
        v["x"], v["i"], v["r"] = buf[..., 1:d + 1], buf[..., d + 2:2 * d + 2], buf[..., 2 * d + 5:]
    else:
        v["x"], v["i"], v["r"] = (rnd(b, s, d).to(dtype).to(DEV) for _ in range(3))
    v["h"] = rnd(b, d).to(DEV) if state else None
    v["reset"] = (torch.rand(b, s, generator=gen) < 0.03).to(DEV) if reset else None
    v["dy"], v["dh"] = rnd(b, s, d).to(dtype).to(DEV), rnd(b, d).to(DEV)
    return v


def scan_reference(v, rate=8.0, grads=True):
    """The definition token by token in float64, gradients by autograd, and the magnitudes: the same sums of absolute values."""
    t = {k: None if v[k] is None else v[k].detach().double().cpu().requires_grad_(grads) for k in ("x", "i", "r", "decay", "h")}
    reset = None if v["reset"] is None else v["reset"].cpu()

    def run(x, i, r, decay, h):
        la = -rate * torch.nn.functional.softplus(decay, threshold=1e3) * torch.sigmoid(r)
        a, b = torch.exp(la), torch.sqrt(-torch.expm1(2 * la))
        keep = a if reset is None else torch.where(reset[..., None], torch.zeros_like(a), a)
        u = b * torch.sigmoid(i) * x
        h = torch.zeros_like(u[:, 0]) if h is None else h
        ys = []
        for n in range(x.shape[1]):
            h = torch.where(reset[:, n, None], u[:, n], a[:, n] * h + u[:, n]) if reset is not None else a[:, n] * h + u[:, n]
            ys.append(h)
        return torch.stack(ys, 1), h, la, a, b, keep

    y, fin, la, a, b, keep = run(**t)
    out = {"y": y, "fin": fin}
    with torch.no_grad():
        m, mfin, *_ = run(t["x"].abs(), t["i"], t["r"], t["decay"], None if t["h"] is None else t["h"].abs())
        out["m_y"], out["m_fin"] = m, mfin
    if grads:
        names = [k for k in t if t[k] is not None]
        got = torch.autograd.grad([y, fin], [t[k] for k in names], [v["dy"].double().cpu(), v["dh"].double().cpu()])
        out.update({"d" + k: g for k, g in zip(names, got)})
        with torch.no_grad():
            g, c = torch.empty_like(y), v["dh"].double().cpu().abs()
            for n in range(y.shape[1] - 1, -1, -1):
                g[:, n] = v["dy"][:, n].double().cpu().abs() + c
                c = keep[:, n] * g[:, n]
            before = torch.cat([(t["h"].abs() if t["h"] is not None else torch.zeros_like(mfin))[:, None], m[:, :-1]], 1)
            si, sr, x = torch.sigmoid(t["i"]), torch.sigmoid(t["r"]), t["x"].abs()
            dla = g * before * keep + g * si * x * a * a / b
            out["m_dx"], out["m_di"] = g * b * si, g * b * x * si
            out["m_dr"], out["m_dh"] = dla * la.abs(), c
            out["m_ddecay"] = rate * torch.sigmoid(t["decay"]) * (dla * sr).sum((0, 1))
    return out


def leaves(v, names):
    return [v[k].requires_grad_(True) for k in names if v[k] is not None]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("b,s,d,reset,state,strided", [
    (1, 1, 1, False, False, False), (2, 3, 5, True, True, False), (5, 1, 64, True, True, True), (3, 64, 64, False, True, False),
    (1, 65, 130, True, False, False), (2, 127, 63, False, False, True), (2, 128, 66, True, True, False), (2, 129, 64, False, True, False),
    (1, 777, 33, True, True, True), (2, 1100, 100, True, True, False), (1, 3001, 72, False, False, False), (70, 200, 8, True, False, False),
])
def test_gated_scan_and_its_gradient(dtype, b, s, d, reset, state, strided):
    v = scan_inputs(b, s, d, dtype, reset, state, seed=s + d, strided=strided)
    ref = scan_reference(v)
    for t in (v["x"], v["i"], v["r"]):
        assert t.stride(-1) == 1
    names = ["x", "i", "r", "decay", "h"]
    ins = [None if v[k] is None else v[k].detach().requires_grad_(True) for k in names]
    y, fin = W().gated_scan(*ins[:4], initial_state=ins[4], reset=v["reset"], return_final_state=True)
    check(y, ref["y"], ref["m_y"], s, "y")
    check(fin, ref["fin"], ref["m_fin"], s, "final state")
    got = torch.autograd.grad([y, fin], [t for t in ins if t is not None], [v["dy"], v["dh"]])
    for name, g in zip([k for k, t in zip(names, ins) if t is not None], got):
        check(g, ref["d" + name], ref["m_d" + name], s, "d" + name)
    with torch.no_grad():       # the call without a gradient is the same call
        y2, fin2 = W().gated_scan(*ins[:4], initial_state=ins[4], reset=v["reset"], return_final_state=True)
        assert torch.equal(y2, y) and torch.equal(fin2, fin)
        out = torch.zeros(b, s, 2 * d + 1, dtype=dtype, device=DEV)[..., 1:d + 1]
        assert W().gated_scan(*ins[:4], initial_state=ins[4], reset=v["reset"], out=out) is out and torch.equal(out, y)


def test_gated_scan_gradients_of_one_output_and_broadcast_gradients():
    v = scan_inputs(2, 150, 24, torch.float32, False, True, seed=5)
    ins = leaves(v, ["x", "i", "r", "decay", "h"])
    y, fin = W().gated_scan(*ins[:4], initial_state=ins[4], return_final_state=True)
    for k, grads in (("y", (torch.ones_like(v["dy"]), torch.zeros_like(v["dh"]))), ("fin", (torch.zeros_like(v["dy"]), torch.ones_like(v["dh"])))):
        w = dict(v, dy=grads[0], dh=grads[1])
        ref = scan_reference(w)
        got = torch.autograd.grad((y if k == "y" else fin).sum(), ins, retain_graph=True)     # an expanded gradient, the other one absent
        for name, g in zip(["x", "i", "r", "decay", "h"], got):
            check(g, ref["d" + name], ref["m_d" + name], 150, name)
    # the same tensor as x and as both gates: its gradients add up
    x = v["x"].detach().requires_grad_(True)
    decay = v["decay"].detach()
    got, = torch.autograd.grad(W().gated_scan(x, x, x, decay), [x], [v["dy"]])
    w = dict(v, x=x, i=x, r=x, h=None, dh=torch.zeros_like(v["dh"]))
    ref = scan_reference(w)
    check(got, ref["dx"] + ref["di"] + ref["dr"], ref["m_dx"] + ref["m_di"] + ref["m_dr"], 150, "shared leaf")


def test_gated_scan_gradient_against_differences():
    """Along a random direction, by a central difference: its error is e^2/6 of the third derivative (a few units, so 1e-5 at e = 4e-3)
    and the rounding of y over e (2^-24 * 40 values * 2 / 4e-3 = 2e-3, in the mean over signs 40^0.5 smaller)."""
    v = scan_inputs(1, 90, 16, torch.float32, True, True, seed=11)
    names = ["x", "i", "r", "decay", "h"]
    ins = leaves(v, names)
    gen = torch.Generator(device=DEV).manual_seed(3)
    wy = torch.randn(v["dy"].shape, generator=gen, device=DEV)

    def f(args):
        y, fin = W().gated_scan(*args[:4], initial_state=args[4], reset=v["reset"], return_final_state=True)
        return (y.double() * wy).sum() + fin.double().sum()

    grads = torch.autograd.grad(f(ins), ins)
    for n, (t, g) in enumerate(zip(ins, grads)):
        way = torch.randn(t.shape, generator=gen, device=DEV)
        e = 4e-3
        with torch.no_grad():
            up, down = ([u + s * e * way if m == n else u for m, u in enumerate(ins)] for s in (1, -1))
            diff = ((f(up) - f(down)) / (2 * e)).item()
        along = (g.double() * way).sum().item()
        scale = (g.double() * way).abs().sum().item()
        assert abs(diff - along) < 2e-3 * scale + 1e-3, (names[n], diff, along, scale)


@pytest.mark.parametrize("dtype", DTYPES)
def test_gated_scan_at_the_edges_of_its_gates(dtype):
    """Gates that are shut, open and infinite: a state that is kept, one that is dropped, gradients that vanish and no NaN."""
    inf = math.inf
    r = torch.tensor([-inf, -200.0, -100.0, -87.0, -30.0, 0.0, 30.0, 200.0, inf])
    i = torch.tensor([-inf, -100.0, 0.0, 100.0, inf])
    r, i = (t.reshape(-1) for t in torch.meshgrid(r, i, indexing="ij"))
    s = r.numel()
    gen = torch.Generator().manual_seed(2)
    d = 6
    v = {"x": torch.randn(1, s, d, generator=gen), "r": r[None, :, None].expand(1, s, d).clone(), "i": i[None, :, None].expand(1, s, d).clone(),
         "h": torch.randn(1, d, generator=gen), "reset": None, "decay": torch.tensor([-inf, -40.0, -6.0, 0.0, 5.0, 40.0])}
    v = {k: t if t is None else (t.to(dtype) if k in "xri" else t).to(DEV) for k, t in v.items()}
    ref = scan_reference(v, grads=False)
    ins = leaves(v, ["x", "i", "r", "decay", "h"])
    y = W().gated_scan(*ins[:4], initial_state=ins[4])
    assert torch.isfinite(y).all()
    check(y, ref["y"], ref["m_y"] + 1e-30, s, "y")
    grads = torch.autograd.grad([y], ins, [torch.ones_like(y)])
    for g in grads:
        assert torch.isfinite(g).all()
    dx, di, dr, _, _ = grads
    shut = (v["i"].float() == -inf)
    assert (dx[shut] == 0).all() and (di[shut] == 0).all() and (dr[v["r"].float().abs() == inf] == 0).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_off_16_bytes_through_many_tiles(dtype):
    """Rows that TMA cannot read, several tiles for every CTA: what the same numbers give where it can, bit by bit, and every time."""
    b, s, d = 54, 853, 151
    wide = scan_inputs(b, s, 152, dtype, True, True, seed=12)
    odd = {k: t[..., :d].contiguous() if k in ("x", "i", "r", "dy", "h", "dh", "decay") else t for k, t in wide.items()}

    def run(v):
        ins = [v[k].detach().requires_grad_(True) for k in ("x", "i", "r", "decay", "h")]
        y, fin = W().gated_scan(*ins[:4], initial_state=ins[4], reset=v["reset"], return_final_state=True)
        return [y.detach(), fin.detach(), *torch.autograd.grad([y, fin], ins, [v["dy"], v["dh"]])]

    want = run(wide)
    for _ in range(5):
        for g, w in zip(run(odd), want):
            assert torch.equal(g, w[..., :d])


def test_gated_scan_keeps_bad_numbers_where_they_are():
    """An infinity or a NaN reaches the tokens behind it in its own channel and row, up to a reset; everything else is as without it, and so
    are the gradients of what does not depend on it."""
    b, s, d = 2, 700, 40
    v = scan_inputs(b, s, d, torch.float32, False, True, seed=9)
    reset = torch.zeros(b, s, dtype=torch.bool, device=DEV)
    reset[0, 500] = True
    good = W().gated_scan(v["x"], v["i"], v["r"], v["decay"], initial_state=v["h"], reset=reset)
    for bad in (math.inf, -math.inf, math.nan):
        x = v["x"].clone()
        x[0, 130, 7] = bad
        ins = [x.requires_grad_(True), v["i"].detach().requires_grad_(True)]
        y = W().gated_scan(ins[0], ins[1], v["r"], v["decay"], initial_state=v["h"], reset=reset)
        hit = torch.zeros_like(reset[..., None].expand(b, s, d))
        hit[0, 130:500, 7] = True
        assert not torch.isfinite(y[hit]).any() and torch.equal(y[~hit], good[~hit])
        if not math.isnan(bad):
            assert (y[hit] == bad).all()
        dx, di = torch.autograd.grad([y], ins, [torch.ones_like(y)])
        assert torch.isfinite(dx).all()
        assert torch.isfinite(di[~hit]).all()
    for name in ("i", "r"):
        bad = {k: v[k].clone() for k in ("x", "i", "r")}
        bad[name][0, 130, 7] = math.nan
        y = W().gated_scan(bad["x"], bad["i"], bad["r"], v["decay"], initial_state=v["h"], reset=reset)
        assert torch.isnan(y[hit]).all() and torch.equal(y[~hit], good[~hit])
        step = W().gated_scan_step(bad["x"][:, 130], bad["i"][:, 130], bad["r"][:, 130], v["decay"], v["h"].clone())
        assert torch.isnan(step[0, 7]) and torch.isfinite(step).sum() == step.numel() - 1
    h = v["h"].clone()
    h[1, 3] = math.inf          # a state that is not finite, dropped at once
    reset[1, 0] = True
    y = W().gated_scan(v["x"], v["i"], v["r"], v["decay"], initial_state=h, reset=reset)
    assert torch.isfinite(y).all()


def test_gated_scan_is_the_same_in_pieces_and_token_by_token():
    v = scan_inputs(3, 333, 50, torch.bfloat16, True, True, seed=4)
    args = (v["x"], v["i"], v["r"])
    whole, fin = W().gated_scan(*args, v["decay"], initial_state=v["h"], reset=v["reset"], return_final_state=True)
    ref = scan_reference(v, grads=False)
    h = v["h"]
    for a, b in ((0, 0), (0, 1), (1, 130), (130, 333)):
        y, h = W().gated_scan(*(t[:, a:b] for t in args), v["decay"], initial_state=h, reset=v["reset"][:, a:b], return_final_state=True)
        check(y, ref["y"][:, a:b], ref["m_y"][:, a:b], 333, "piece")
    check(h, ref["fin"], ref["m_fin"], 333, "state")
    state, other = v["h"].clone(), torch.empty_like(v["h"])
    for n in range(40):
        cut = v["reset"][:, n, None]
        before = torch.where(cut, torch.zeros_like(state), state)
        kept = before.clone()
        y = W().gated_scan_step(*(t[:, n] for t in args), v["decay"], before, out_state=other)
        assert torch.equal(before, kept)
        y2 = W().gated_scan_step(*(t[:, n] for t in args), v["decay"], before)
        assert torch.equal(y, y2) and torch.equal(before, other)
        state = before
        check(y, ref["y"][:, n], ref["m_y"][:, n], n + 1, "step")


@pytest.mark.parametrize("b,d", [(1, 1), (3, 7), (64, 5120), (2, 66)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_gated_scan_step(dtype, b, d):
    v = scan_inputs(b, 1, d, dtype, False, True, seed=d)
    ref = scan_reference(v, grads=False)
    y = W().gated_scan_step(v["x"][:, 0], v["i"][:, 0], v["r"][:, 0], v["decay"].bfloat16().float(), v["h"].clone())
    assert y.shape == (b, d)
    wide = torch.zeros(b, d + 3, dtype=dtype, device=DEV)
    y = W().gated_scan_step(v["x"][:, 0], v["i"][:, 0], v["r"][:, 0], v["decay"], v["h"], out=wide[:, 1:d + 1])
    check(y, ref["y"][:, 0], ref["m_y"][:, 0], 1, "y")
    check(v["h"], ref["fin"], ref["m_fin"], 1, "state")
    assert (wide[:, 0] == 0).all() and (wide[:, d + 1:] == 0).all()


def test_views_of_any_layout_are_taken():
    """Channels that do not lie side by side, one channel of any stride, expanded batches, rows that do not lie at one distance."""
    v = scan_inputs(3, 70, 16, torch.float16, True, False, seed=6)
    want = W().gated_scan(v["x"], v["i"], v["r"], v["decay"], reset=v["reset"])
    turned = [v[k].transpose(1, 2).contiguous().transpose(1, 2) for k in ("x", "i", "r")]
    assert turned[0].stride(-1) != 1
    assert torch.equal(W().gated_scan(*turned, v["decay"].double().float(), reset=v["reset"].t().contiguous().t()), want)
    assert torch.equal(W().gated_scan_step(*(t[:, 5] for t in turned), v["decay"], torch.zeros(3, 16, device=DEV)),
                       W().gated_scan_step(*(v[k][:, 5] for k in ("x", "i", "r")), v["decay"], torch.zeros(3, 16, device=DEV)))
    one = [t[..., :1] for t in turned]
    assert one[0].stride(-1) != 1
    got = W().gated_scan(*one, v["decay"][:1], reset=v["reset"])
    assert ((got - want[..., :1]).abs() <= 2.0 ** -10 * want[..., :1].abs()).all()
    wide = [t[:1].expand(3, 70, 16) for t in (v["x"], v["i"], v["r"])]
    assert torch.equal(W().gated_scan(*wide, v["decay"])[2], W().gated_scan(*(t[:1] for t in wide), v["decay"])[0])
    x, w = torch.randn(4, 6, 24, device=DEV), torch.randn(24, device=DEV)
    n = W().rms_norm(x, w)
    assert torch.equal(W().rms_norm(x.transpose(0, 1), w), n.transpose(0, 1)) and torch.equal(W().rms_norm(x[:, ::2], w), n[:, ::2])
    assert torch.equal(W().rms_norm(x.transpose(1, 2).contiguous().transpose(1, 2), w), n)
    assert torch.equal(W().gated_rms_norm(x[:1].expand(4, 6, 24), x[1:2].expand(4, 6, 24), w)[3], W().gated_rms_norm(x[0], x[1], w))
    x = x.requires_grad_(True)
    a, = torch.autograd.grad(W().rms_norm(x.transpose(0, 1), w).sum(), [x])
    b, = torch.autograd.grad(W().rms_norm(x, w), [x], [torch.ones_like(n)])
    assert torch.equal(a, b)


def test_gradients_are_not_differentiable_and_say_so():
    v = scan_inputs(1, 8, 16, torch.float32, False, False, seed=2)
    x = v["x"].requires_grad_(True)
    w, cw = torch.ones(16, device=DEV, requires_grad=True), torch.ones(16, 1, 2, device=DEV)
    for y in (W().gated_scan(x, v["i"], v["r"], v["decay"]), W().rms_norm(x, w), W().rms_norm(x, w, residual=x)[0], W().gated_rms_norm(x, v["i"], w),
              W().conv1d_silu(x, cw)):
        g, = torch.autograd.grad(y.square().sum(), [x], create_graph=True)
        with pytest.raises(RuntimeError, match="not twice differentiable"):
            g.sum().backward()
    # an operand that is changed after the call is noticed
    a = x.detach().clone().requires_grad_(True)
    b = a * 1
    y = W().rms_norm(b, w)
    b.mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_gated_scan_of_no_tokens():
    x = torch.zeros(2, 0, 8, device=DEV)
    decay = torch.zeros(8, device=DEV)
    h = torch.randn(2, 8, device=DEV, requires_grad=True)
    y, fin = W().gated_scan(x, x, x, decay, initial_state=h, return_final_state=True)
    assert y.shape == (2, 0, 8) and torch.equal(fin, h)
    g, = torch.autograd.grad(fin.sum(), [h])
    assert (g == 1).all()
    y, fin = W().gated_scan(x, x, x, decay, return_final_state=True)
    assert (fin == 0).all()


def test_gated_scan_does_not_vary_and_leaves_its_neighbours():
    """Many tiles in flight, other work beside it: the same bits every time; nothing outside y is written."""
    b, s, d = 2, 20000, 200
    v = scan_inputs(b, s, d, torch.bfloat16, True, True, seed=21)
    ins = leaves(v, ["x", "i", "r", "decay", "h"])
    side = torch.cuda.Stream()
    first = None
    for n in range(6):
        with torch.cuda.stream(side):
            torch.randn(2000, 2000, device=DEV) @ torch.randn(2000, 2000, device=DEV)
        y, fin = W().gated_scan(*ins[:4], initial_state=ins[4], reset=v["reset"], return_final_state=True)
        now = [y, fin, *torch.autograd.grad([y, fin], ins, [v["dy"], v["dh"]])]
        if first is None:
            first = now
        assert all(torch.equal(p, q) for p, q in zip(first, now))
    buf = torch.full((b, s + 2, d + 2), 7.0, dtype=torch.bfloat16, device=DEV)
    with torch.no_grad():
        W().gated_scan(*ins[:4], initial_state=ins[4], reset=v["reset"], out=buf[:, 1:-1, 1:-1])
    assert torch.equal(buf[:, 1:-1, 1:-1], first[0])
    assert (buf[:, 0] == 7).all() and (buf[:, -1] == 7).all() and (buf[..., 0] == 7).all() and (buf[..., -1] == 7).all()
    torch.cuda.synchronize()


def test_two_gated_scans_at_once():
    """Two launches that share the chip, each waiting on its own tiles."""
    vs = [scan_inputs(1, 30000, 256, torch.float16, False, False, seed=n) for n in (1, 2)]
    want = [W().gated_scan(v["x"], v["i"], v["r"], v["decay"]) for v in vs]
    streams = [torch.cuda.Stream() for _ in vs]
    torch.cuda.synchronize()
    for _ in range(5):
        got = []
        for v, st in zip(vs, streams):
            with torch.cuda.stream(st):
                got.append(W().gated_scan(v["x"], v["i"], v["r"], v["decay"]))
        torch.cuda.synchronize()
        assert all(torch.equal(g, w) for g, w in zip(got, want))


def test_gated_scan_offsets_past_32_bits():
    s, d = 1_100_000, 2048          # 2.25e9 numbers a tensor
    gen = torch.Generator(device=DEV).manual_seed(1)
    base = torch.randn(1, 50_000, d, generator=gen, device=DEV, dtype=torch.float32).bfloat16()
    x = base.repeat(1, 22, 1)
    assert x.shape[1] == s
    decay = torch.rand(d, generator=gen, device=DEV) - 6
    y, fin = W().gated_scan(x, x, x, decay, return_final_state=True)
    at = s - 30_000
    _, h = W().gated_scan(x[:, :at], x[:, :at], x[:, :at], decay, return_final_state=True)
    tail, fin2 = W().gated_scan(x[:, at:], x[:, at:], x[:, at:], decay, initial_state=h, return_final_state=True)
    # tiles begin elsewhere, so sums are in another order: a rounding of the type apart at most
    scale = tail.float().abs().clamp_min(1e-3)
    assert ((y[:, at:].float() - tail.float()).abs() <= 2 * 2.0 ** -8 * scale).all()
    assert ((fin - fin2).abs() <= 1e-4 * fin2.abs().clamp_min(1e-2)).all()


def test_a_wait_between_tiles_that_runs_out_is_reported_and_the_next_call_is_fine():
    """Made on the host, without a fault: the first CTA leaves without working, so the tiles behind its own give up after 20 ms."""
    import ctypes as C

    from workloadsuite_b200 import _lib

    lib, (b, s, d) = _lib.load(), (2, 3000, 128)
    v = scan_inputs(b, s, d, torch.bfloat16, False, False, seed=8)
    y, status = torch.zeros_like(v["x"]), torch.zeros(1, dtype=torch.int32, device=DEV)
    pieces = torch.zeros(b, (s + 63) // 64, d, device=DEV)
    grads, dd = [torch.zeros_like(v["x"]) for _ in range(3)], torch.zeros(d, device=DEV)
    a = _lib.GatedScanArgs()
    a.x, a.input_gate, a.decay_gate, a.decay = (v[k].data_ptr() for k in ("x", "i", "r", "decay"))
    a.y, a.pieces, a.status, a.dy, a.ddecay = y.data_ptr(), pieces.data_ptr(), status.data_ptr(), v["dy"].data_ptr(), dd.data_ptr()
    a.dx, a.dinput_gate, a.ddecay_gate = (g.data_ptr() for g in grads)
    a.rate, a.batch, a.seqlen, a.channels, a.dtype, a.wait_limit_ms = 8.0, b, s, d, _lib.DTYPE_BF16, 20
    for f in ("x", "input_gate", "decay_gate", "y", "dy", "dx", "dinput_gate", "ddecay_gate"):
        setattr(a, f + "_stride", (C.c_int64 * 2)(s * d, d))
    stream = C.c_void_p(torch.cuda.current_stream().cuda_stream)
    for call, back in ((lib.ssd_b200_gated_scan, 0), (lib.ssd_b200_gated_scan_backward, 1)):
        ws = torch.empty(lib.ssd_b200_gated_scan_workspace_bytes(C.byref(a), back), dtype=torch.uint8, device=DEV)
        a.workspace, a.workspace_bytes = ws.data_ptr(), ws.numel()
        for inject, want in ((1, 8), (0, 0)):
            status.zero_()
            a.inject_lost_tile = inject
            assert call(C.byref(a), stream) == 0
            torch.cuda.synchronize()
            assert status.item() == want, (back, inject)
    ref = scan_reference(dict(v, dh=torch.zeros(b, d)))
    check(y, ref["y"], ref["m_y"], s, "y")
    check(grads[0], ref["dx"], ref["m_dx"], s, "dx")


# ---- norms ----------------------------------------------------------------------------------------------

def unit(v, eps):
    return v / torch.sqrt(v.square().mean(-1, keepdim=True) + eps)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,d,outer,res32,strided", [
    (1, 1, "both", False, False), (3, 8, "", False, False), (16, 2048, "", True, False), (5, 51, "both", True, True), (33, 256, "post", False, False),
    (7, 264, "scale", True, False), (9, 1537, "both", False, False), (600, 128, "both", False, True), (4, 5120, "both", True, False),
    (3, 8200, "post", False, False), (2, 16384, "both", True, False), (2, 16383, "both", False, False), (2000, 96, "", False, False),
])
def test_rms_norm_between_blocks_and_its_gradient(dtype, rows, d, outer, res32, strided):
    gen = torch.Generator().manual_seed(rows + d)
    rnd = lambda *n: torch.randn(*n, generator=gen)
    rt = torch.float32 if res32 else dtype
    eps = 1e-6
    wt = torch.float32 if d % 2 else dtype
    if strided:
        x = rnd(rows, d + 3).to(dtype).to(DEV)[:, 2:d + 2]
    else:
        x = rnd(rows, d).to(dtype).to(DEV)
    res, w = (2 * rnd(rows, d)).to(rt).to(DEV), (1 + 0.2 * rnd(d)).to(wt).to(DEV)
    post = (1 + 0.2 * rnd(d)).to(wt).to(DEV) if outer in ("post", "both") else None
    scale = (0.5 + 0.1 * rnd(d)).to(dtype).to(DEV) if outer in ("scale", "both") else None
    dy, dr = rnd(rows, d).to(dtype).to(DEV), rnd(rows, d).to(rt).to(DEV)
    ins = [t if t is None else t.detach().requires_grad_(True) for t in (x, res, w, post, scale)]
    y, r = W().rms_norm(ins[0], ins[2], eps=eps, residual=ins[1], post_weight=ins[3], scale=ins[4])
    got = torch.autograd.grad([y, r], [t for t in ins if t is not None], [dy, dr])

    t = [None if a is None else a.detach().double().cpu().requires_grad_(True) for a in ins]
    o = t[0] if post is None else unit(t[0], eps) * t[3]
    o = o if scale is None else o * t[4]
    r64 = t[1] + o
    check(r, r64, t[1].abs() + o.abs(), 1, "residual_out")
    # y is the norm of what is stored: the definition goes on from the tensor that came out
    stored = r64 + (r.detach().double().cpu() - r64.detach())
    y64 = unit(stored, eps) * t[2]
    check(y, y64, y64.abs(), 1, "y")
    ref = torch.autograd.grad([y64, stored], [a for a in t if a is not None], [dy.double().cpu(), dr.double().cpu()])
    # magnitudes: each term of the gradient by itself
    with torch.no_grad():
        rs = 1 / torch.sqrt(stored.square().mean(-1, keepdim=True) + eps)
        rh, g = stored * rs, dy.double().cpu() * t[2]
        m_r = dr.double().cpu().abs() + rs * (g.abs() + rh.abs() * (g * rh).abs().mean(-1, keepdim=True))
        mags = {"w": (dy.double().cpu() * rh).abs().sum(0), "res": m_r, "x": m_r}
        if outer:
            xs = t[0].detach() if post is None else unit(t[0].detach(), eps)
            both = (m_r * xs.abs()).sum(0)
            so = 1 if scale is None else t[4].detach().abs()
            po = 1 if post is None else t[3].detach().abs()
            mags["post"], mags["scale"] = both * so, both * po
            g2 = m_r * so * po
            if post is not None:
                s2 = 1 / torch.sqrt(t[0].detach().square().mean(-1, keepdim=True) + eps)
                mags["x"] = s2 * (g2 + xs.abs() * (g2 * xs.abs()).mean(-1, keepdim=True))
            else:
                mags["x"] = g2
    names = [n for n, a in zip(("x", "res", "w", "post", "scale"), ins) if a is not None]
    for name, a, b in zip(names, got, ref):
        check(a, b, mags[name], 1, "d" + name)
    with torch.no_grad():
        y2, r2 = W().rms_norm(x, w, eps=eps, residual=res, post_weight=post, scale=scale)
        assert torch.equal(y2, y) and torch.equal(r2, r)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(1, 1), (2, 3, 64), (5, 2048), (4, 1537), (2, 2, 2, 40)])
def test_rms_norm_alone_and_its_gradient(dtype, shape):
    gen = torch.Generator().manual_seed(shape[-1])
    x, w, dy = (torch.randn(*n, generator=gen).to(dtype).to(DEV) for n in (shape, shape[-1:], shape))
    x.requires_grad_(True), w.requires_grad_(True)
    y = W().rms_norm(x, w)
    eps = torch.finfo(torch.float32).eps
    x6, w6 = (t.detach().double().cpu().requires_grad_(True) for t in (x, w))
    y6 = unit(x6, eps) * w6
    check(y, y6, y6.abs(), 1, "y")
    dx, dw = torch.autograd.grad([y], [x, w], [dy])
    rx, rw = torch.autograd.grad([y6], [x6, w6], [dy.double().cpu()])
    rs = 1 / torch.sqrt(x6.detach().square().mean(-1, keepdim=True) + eps)
    g, xh = dy.double().cpu() * w6.detach(), x6.detach() * rs
    check(dx, rx, rs * (g.abs() + xh.abs() * (g * xh).abs().mean(-1, keepdim=True)), 1, "dx")
    check(dw, rw, (dy.double().cpu() * xh).abs().flatten(0, -2).sum(0), 1, "dw")
    assert torch.equal(W().rms_norm(x.detach().transpose(0, -1).contiguous().transpose(0, -1), w.detach()), y.detach())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("first", [False, True])
@pytest.mark.parametrize("rows,groups,d,strided", [(1, 1, 1, False), (3, 2, 16, False), (9, 8, 1024, True), (5, 1, 1537, False), (4, 3, 51 * 3, True),
                                                   (700, 4, 64 * 4, False), (2, 1, 8192, False), (3, 8, 8192, False), (2, 2, 16384, False)])
def test_gated_rms_norm_and_its_gradient(dtype, first, rows, groups, d, strided):
    gen = torch.Generator().manual_seed(rows * d)
    rnd = lambda *n: torch.randn(*n, generator=gen)
    if strided:
        buf = rnd(rows, 2 * d + 8).to(dtype).to(DEV)
        x, z = buf[:, :d], buf[:, d + 8:]
    else:
        x, z = rnd(rows, d).to(dtype).to(DEV), rnd(rows, d).to(dtype).to(DEV)
    w, dy, eps = (1 + 0.2 * rnd(d)).to(torch.float32 if rows % 2 else dtype).to(DEV), rnd(rows, d).to(dtype).to(DEV), 1e-5
    ins = [t.detach().requires_grad_(True) for t in (x, z, w)]
    y = W().gated_rms_norm(*ins, eps=eps, groups=groups, norm_first=first)
    got = torch.autograd.grad([y], ins, [dy])
    x6, z6, w6 = (t.detach().double().cpu().requires_grad_(True) for t in ins)
    gate = z6 * torch.sigmoid(z6)
    fold = lambda t: t.unflatten(-1, (groups, -1))
    v = fold(x6 if first else x6 * gate)
    y6 = unit(v, eps).flatten(-2) * w6 * (gate if first else 1)
    check(y, y6, y6.abs(), 1, "y")
    ref = torch.autograd.grad([y6], [x6, z6, w6], [dy.double().cpu()])
    with torch.no_grad():
        rs = 1 / torch.sqrt(v.square().mean(-1, keepdim=True) + eps)
        vh, g = (v * rs).abs(), dy.double().cpu().abs()
        sz = torch.sigmoid(z6)
        slope = sz * (1 + z6.abs() * (1 - sz))
        if first:
            gw = fold(g * w6.abs() * gate.abs())
            m_x = (rs * (gw + vh * (gw * vh).mean(-1, keepdim=True))).flatten(-2)
            mags = [m_x, g * vh.flatten(-2) * w6.abs() * slope, (g * vh.flatten(-2) * gate.abs()).sum(0)]
        else:
            gw = fold(g * w6.abs())
            m_v = (rs * (gw + vh * (gw * vh).mean(-1, keepdim=True))).flatten(-2)
            mags = [m_v * gate.abs(), m_v * x6.abs() * slope, (g * vh.flatten(-2)).sum(0)]
    for name, a, b, m in zip(("dx", "dz", "dw"), got, ref, mags):
        check(a, b, m, 1, name)


def test_norms_of_extreme_rows():
    """Rows of zeros, of the type's largest numbers' square roots, a row that is not finite: each row is its own."""
    d = 200
    x = torch.randn(6, d, device=DEV)
    x[0] = 0
    x[1] = 1e18
    x[2] = 1e-30
    x[3, 5] = math.nan
    x[4, 7] = math.inf
    w = torch.ones(d, device=DEV)
    x.requires_grad_(True)
    y = W().rms_norm(x, w, eps=1e-6)
    assert (y[0] == 0).all() and torch.allclose(y[1], torch.ones_like(y[1])) and torch.allclose(y[2], x[2] * 1e3)
    assert torch.isnan(y[3]).all() and torch.isnan(y[4, 7]) and torch.isfinite(y[5]).all()
    g, = torch.autograd.grad([y], [x], [torch.randn(6, d, device=DEV)])
    assert torch.isfinite(g[[0, 1, 2, 5]]).all()
    # a gate at its ends
    z = torch.tensor([-1e4, -200.0, 0.0, 200.0, 1e4], device=DEV).repeat_interleave(40)[None].expand(6, d)
    y = W().gated_rms_norm(x.detach()[[0, 5]], z[[0, 5]], w, eps=1e-6, norm_first=True)
    assert torch.isfinite(y).all() and (y[:, :80] == 0).all()


def test_norms_of_no_rows():
    x = torch.zeros(0, 16, device=DEV, requires_grad=True)
    w = torch.ones(16, device=DEV, requires_grad=True)
    for y in (W().rms_norm(x, w), W().rms_norm(x, w, residual=x)[0], W().gated_rms_norm(x, x, w)):
        assert y.shape == (0, 16)
        gx, gw = torch.autograd.grad(y.sum(), [x, w])
        assert gx.shape == (0, 16) and (gw == 0).all()


# ---- conv1d + SiLU's gradient ---------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("b,s,d,taps,bias,sliced", [(1, 1, 8, 4, True, False), (2, 2, 8, 4, False, False), (1, 7, 72, 3, True, True), (3, 64, 64, 2, True, False),
                                                    (2, 65, 136, 4, True, True), (1, 513, 40, 4, False, False), (2, 1030, 200, 3, True, False)])
def test_conv1d_silu_gradient(dtype, b, s, d, taps, bias, sliced):
    gen = torch.Generator().manual_seed(s + d)
    rnd = lambda *n: torch.randn(*n, generator=gen)
    x = rnd(b, s, d + 9).to(dtype).to(DEV)[..., 1:d + 1] if sliced else rnd(b, s, d).to(dtype).to(DEV)
    w, bs, dy = (0.5 * rnd(d, 1, taps)).to(dtype).to(DEV), (0.5 * rnd(d)).to(dtype).to(DEV) if bias else None, rnd(b, s, d).to(dtype).to(DEV)
    ins = [t if t is None else t.detach().requires_grad_(True) for t in (x, w, bs)]
    y = W().conv1d_silu(*ins)
    got = torch.autograd.grad([y], [t for t in ins if t is not None], [dy])
    with torch.no_grad():
        assert torch.equal(W().conv1d_silu(*ins), y)
    t = [None if a is None else a.detach().double().cpu().requires_grad_(True) for a in ins]

    def pre(xx, ww, bb):
        padded = torch.nn.functional.pad(xx, (0, 0, taps - 1, 0))
        p = sum(padded[:, k:k + s] * ww[:, 0, k] for k in range(taps))
        return p if bb is None else p + bb

    p6 = pre(*t)
    y6 = p6 * torch.sigmoid(p6)
    ref = torch.autograd.grad([y6], [a for a in t if a is not None], [dy.double().cpu()])
    with torch.no_grad():
        sg = torch.sigmoid(p6)
        big = pre(t[0].abs(), t[1].abs(), None if bs is None else t[2].abs())
        g = dy.double().cpu().abs() * (sg * (1 + p6.abs()) + big)      # (pre's own error passes through at a slope below one)
        padded = torch.nn.functional.pad(g, (0, 0, 0, taps - 1))
        m_x = sum(padded[:, taps - 1 - k:taps - 1 - k + s] * t[1][:, 0, k].abs() for k in range(taps))
        xp = torch.nn.functional.pad(t[0].abs(), (0, 0, taps - 1, 0))
        m_w = torch.stack([(g * xp[:, k:k + s]).sum((0, 1)) for k in range(taps)], -1)[:, None]
        mags = [m_x, m_w, g.sum((0, 1))]
    for name, a, r, m in zip(("dx", "dw", "dbias"), got, ref, mags):
        check(a, r, m, 1, name)


# ---- together -------------------------------------------------------------------------------------------

class _Block(torch.nn.Module):
    """A recurrent block as such models have it: norm, projections, conv, gated recurrence, gated norm, projection, residual."""

    def __init__(self, d, inner, taps=4):
        super().__init__()
        gen = torch.Generator().manual_seed(d)
        par = lambda *n, s=1.0: torch.nn.Parameter(s * torch.randn(*n, generator=gen))
        self.w, self.post, self.scale = par(d), par(d), par(d, s=0.3)
        self.into, self.outof = par(4 * inner, d, s=d ** -0.5), par(d, inner, s=inner ** -0.5)
        self.cw, self.cb, self.decay, self.gw = par(inner, 1, taps, s=0.5), par(inner, s=0.1), par(inner), par(inner)
        self.inner, self.taps = inner, taps

    def forward(self, x, residual, reset, ops):
        y, r = ops.rms_norm(x, self.w, eps=1e-6, residual=residual, post_weight=self.post, scale=self.scale)
        x, i, rg, z = (y @ self.into.T).split(self.inner, -1)
        x = ops.conv1d_silu(x, self.cw, self.cb)
        h = ops.gated_scan(x, i, rg, self.decay, reset=reset)
        return ops.gated_rms_norm(h, z, self.gw, eps=1e-6, groups=2) @ self.outof.T, r


class _Plain:
    @staticmethod
    def rms_norm(x, w, eps, residual, post_weight, scale):
        r = residual + unit(x, eps) * post_weight * scale
        return unit(r, eps) * w, r

    @staticmethod
    def conv1d_silu(x, w, b):
        p = torch.nn.functional.pad(x, (0, 0, w.shape[-1] - 1, 0))
        p = sum(p[:, k:k + x.shape[1]] * w[:, 0, k] for k in range(w.shape[-1])) + b
        return p * torch.sigmoid(p)

    @staticmethod
    def gated_scan(x, i, r, decay, reset):
        la = -8 * torch.nn.functional.softplus(decay) * torch.sigmoid(r)
        a = torch.where(reset[..., None], torch.zeros_like(la), torch.exp(la))
        u = torch.sqrt(-torch.expm1(2 * la)) * torch.sigmoid(i) * x
        h, out = torch.zeros_like(u[:, 0]), []
        for n in range(x.shape[1]):
            h = a[:, n] * h + u[:, n]
            out.append(h)
        return torch.stack(out, 1)

    @staticmethod
    def gated_rms_norm(x, z, w, eps, groups):
        return unit((x * z * torch.sigmoid(z)).unflatten(-1, (groups, -1)), eps).flatten(-2) * w


def test_two_blocks_together_and_their_gradients():
    """Two blocks in float32 against 64 bits, forward and backward.  Each of some twenty operations in line is good to DELTA and the two
    projections of 48 and 80 terms to that too; what follows multiplies an error by at most the block's gain (below 4 for these weights, four
    norms a pass): 20 * 4^2 * DELTA = 6e-4 of the largest number of a tensor."""
    d, inner, b, s = 48, 80, 2, 150
    blocks = torch.nn.ModuleList([_Block(d, inner), _Block(d, inner)])
    x, res, wy = torch.randn(b, s, d), torch.randn(b, s, d), torch.randn(b, s, d)
    reset = torch.rand(b, s) < 0.02

    def run(blocks, ops, x, res, reset, wy):
        x, res = x.requires_grad_(True), res.requires_grad_(True)
        o, r = blocks[0](x, res, reset, ops)
        o, r = blocks[1](o, r, reset, ops)
        pars = list(blocks.parameters())
        return [o, r, *torch.autograd.grad([(o * wy).sum() + r.sum()], [x, res, *pars])]

    import copy
    ref = run(copy.deepcopy(blocks).double(), _Plain, x.double(), res.double(), reset, wy.double())
    old = torch.backends.cuda.matmul.allow_tf32
    torch.backends.cuda.matmul.allow_tf32 = False
    try:
        got = run(copy.deepcopy(blocks).to(DEV), W(), x.to(DEV).detach(), res.to(DEV).detach(), reset.to(DEV), wy.to(DEV))
    finally:
        torch.backends.cuda.matmul.allow_tf32 = old
    for a, r in zip(got, ref):
        assert (a.cpu().double() - r).abs().max() <= 6e-4 * r.abs().max()


def test_the_model_adds_its_residuals_in_the_norms():
    """The drop-in Model against its own layers called one by one with the sums and norms in PyTorch.  The sums are the same numbers bit by bit
    and a norm's result may round the other way (half a step, 2^-11); two layers with a gain of some units pass that on: 2^-11 * 2 * 4."""
    from workloadsuite_b200 import mamba_model as M

    torch.manual_seed(5)
    model = M.Model(128, 3, 4, 128, 64, 2, 64, 4).to(DEV).eval()
    with torch.no_grad():
        for n in [layer.norm for layer in model.layers] + [model.final_norm]:
            n.weight.uniform_(0.5, 1.5)
    x = torch.randn(2, 256, 128, dtype=torch.float16, device=DEV)
    norm = torch.nn.functional.rms_norm
    with torch.inference_mode():
        got = model(x)
        u = x
        for layer in model.layers:
            assert torch.equal(layer.norm(u, u)[1], u + u)
            u = u + layer(u)
        want = norm(u, (128,), model.final_norm.weight)
        assert ((got - want).abs().max() <= 2.0 ** -8 * want.abs().max()).item()
        seen = []
        hook = model.layers[1].register_forward_hook(lambda m, a, out: seen.append((len(a), out.shape)))
        again = model(x)                       # a layer that is watched is called as before
        hook.remove()
        assert seen == [(1, x.shape)] and (again - want).abs().max() <= 2.0 ** -8 * want.abs().max()
    # gradients reach what they reached before: the residual stream and the norms
    x = x.clone().requires_grad_(True)
    y = model(x)
    gx, gw = torch.autograd.grad(y.float().sum(), [x, model.final_norm.weight])
    assert torch.isfinite(gx).all() and torch.isfinite(gw).all() and (gx != 0).any()
    cpu = M.RMSNorm(128, dtype=torch.float32)
    t = torch.randn(3, 128)
    assert torch.equal(cpu(t), torch.nn.functional.rms_norm(t, (128,), cpu.weight)) and torch.equal(cpu(t, t)[1], t + t)


def test_captured_forward_and_backward():
    """Two graphs, each with a forward and a backward of every operator, replayed in turn and beside each other on new inputs, while an eager
    graph of the same leaves is alive.  (PyTorch wants that one recorded on the stream that captures: its leaves' nodes keep the stream they were
    made on, and a capture cannot wait for another.)"""
    dt = torch.bfloat16
    b, s, d = 2, 300, 64

    class G:
        def __init__(self, seed):
            v = scan_inputs(b, s, d, dt, True, True, seed)
            self.v, self.par = v, leaves(v, ["x", "i", "r", "decay", "h"])
            gen = torch.Generator().manual_seed(seed)
            self.w = torch.randn(d, generator=gen).to(DEV).requires_grad_(True)
            self.cw = torch.randn(d, 1, 4, generator=gen).to(dt).to(DEV).requires_grad_(True)

        def run(self):
            x = W().conv1d_silu(self.par[0], self.cw)
            y, fin = W().gated_scan(x, *self.par[1:4], initial_state=self.par[4], reset=self.v["reset"], return_final_state=True)
            n, r = W().rms_norm(y, self.w, residual=self.v["dy"])
            g = W().gated_rms_norm(n, r, self.w)
            return [g, r, fin, *torch.autograd.grad([g, r, fin], [*self.par, self.w, self.cw], [self.v["dy"], self.v["dy"], self.v["dh"]])]

    gs = [G(1), G(2)]
    graphs, alive = [], []
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    for g in gs:
        with torch.cuda.stream(side):
            alive.append(g.run())
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = g.run()
        graphs.append((graph, out))
    for turn in range(3):
        for g in gs:
            with torch.no_grad():
                for t in g.par[:3]:
                    t.copy_(torch.randn(t.shape, device=DEV))
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            want = [[t.detach().clone() for t in g.run()] for g in gs]
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream(), torch.cuda.Stream()] if turn == 2 else [torch.cuda.current_stream()] * 2
        for (graph, _), st in zip(graphs, streams):
            with torch.cuda.stream(st):
                graph.replay()
        torch.cuda.synchronize()
        for (_, out), w in zip(graphs, want):
            assert all(torch.equal(a, c) for a, c in zip(out, w))
    assert len(alive) == 2


def test_other_stream_and_other_device():
    v = scan_inputs(1, 1000, 32, torch.float16, False, False, seed=3)
    w = torch.ones(32, device=DEV)
    want = W().gated_scan(v["x"], v["i"], v["r"], v["decay"])
    wn = W().gated_rms_norm(want, v["x"], w)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        y = W().gated_scan(v["x"], v["i"], v["r"], v["decay"])
        n = W().gated_rms_norm(y, v["x"], w)
    torch.cuda.synchronize()
    assert torch.equal(y, want) and torch.equal(n, wn)
    if torch.cuda.device_count() > 1:
        far = {k: t.to("cuda:1") for k, t in v.items() if t is not None}
        y = W().gated_scan(far["x"], far["i"], far["r"], far["decay"])
        assert y.device.index == 1 and torch.equal(y.cpu(), want.cpu())


def test_refusals_on_the_device():
    v = scan_inputs(2, 10, 16, torch.float32, False, True, seed=1)
    args = [v["x"], v["i"], v["r"], v["decay"]]
    for bad in (dict(initial_state=v["h"].half()), dict(initial_state=v["h"][:1]), dict(reset=torch.zeros(2, 10, device=DEV)),
                dict(reset=torch.zeros(2, 9, dtype=torch.bool, device=DEV)), dict(rate=0.0), dict(rate=-1.0), dict(rate=math.inf),
                dict(out=torch.empty(2, 10, 15, device=DEV)), dict(initial_state=v["h"].cpu()), dict(wait_limit_ms=-1)):
        with pytest.raises(ValueError):
            W().gated_scan(*args, **bad)
    with pytest.raises(ValueError):
        W().gated_scan(v["x"], v["i"].half(), v["r"], v["decay"])
    with pytest.raises(ValueError):
        W().gated_scan(v["x"], v["i"], v["r"], v["decay"][:3])
    with pytest.raises(ValueError):
        W().gated_scan(v["x"].detach().requires_grad_(True), *args[1:], out=torch.empty_like(v["x"]))
    with pytest.raises(ValueError):
        W().gated_scan_step(v["x"][:, 0], v["i"][:, 0], v["r"][:, 0], v["decay"], v["h"].t().contiguous().t())
    x, w = torch.randn(4, 24, device=DEV), torch.ones(24, device=DEV)
    for bad in (dict(residual=x[:3]), dict(residual=x.half()), dict(scale=w), dict(post_weight=w), dict(eps=-1.0), dict(residual=x, scale=w[:5]),
                dict(out=x.half())):
        with pytest.raises(ValueError):
            W().rms_norm(x, w, **bad)
    with pytest.raises(ValueError):
        W().gated_rms_norm(x, x, w, groups=5)
    with pytest.raises(ValueError):
        W().gated_rms_norm(x, x.half(), w)
    with pytest.raises(NotImplementedError):
        W().rms_norm(torch.zeros(1, 16385, device=DEV), torch.zeros(16385, device=DEV))
