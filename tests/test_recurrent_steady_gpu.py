"""The recurrent block's operators where their loops run more than once: several rows, tiles and blocks for every CTA, rings that are used
again, sums over a CTA's rows, ragged ends.  Against the definitions in 64 bits, with the tolerances of test_recurrent_gpu.py (their sums
over tokens or rows run 256 in line at most, errors of sqrt(256) units and so within DELTA), and against themselves, bit by bit."""
import pytest
import torch

from test_recurrent_gpu import DELTA, DEV, DTYPES, W, _no_wait_ran_out, check, scan_inputs, scan_reference, unit  # noqa: F401

pytestmark = pytest.mark.gpu
SMS = 148


def near(got, ref, mag, what):
    """check() of one step, on the device."""
    info = torch.finfo(got.dtype)
    assert got.shape == ref.shape, what
    tol = info.eps / 2 * ref.abs() + 2 * DELTA * mag + info.smallest_normal * info.eps / 2
    off = (got.detach().double() - ref).abs() - tol
    assert (off <= 0).all(), (what, int((~(off <= 0)).sum()), got.numel(), float(off.max()))


# ---- conv1d + SiLU's gradient: runs of 128 and 256 tokens ------------------------------------------------

def run_of(b, s, d, taps):
    """The tokens of a warp's run at least, from the workspace that the partial sums take: four runs a CTA."""
    from workloadsuite_b200 import _lib

    ctas = _lib.load().ssd_b200_conv1d_silu_workspace_bytes(b, s, d, taps) // (4 * b * (taps + 1) * d)
    return s // (4 * ctas)


@pytest.mark.parametrize("sliced", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("b,s,d,taps,bias", [(4, 2055, 2048, 4, True), (3, 4099, 1544, 3, False), (8, 2053, 2056, 2, True)])
def test_conv1d_silu_gradient_of_long_runs(b, s, d, taps, bias, dtype, sliced):
    assert run_of(b, s, d, taps) >= 64      # eight blocks of eight tokens and more: the ring's three or four places are filled again
    gen = torch.Generator(device=DEV).manual_seed(s)
    rnd = lambda *n: torch.randn(*n, generator=gen, device=DEV)
    x = rnd(b, s, d + 2).to(dtype)[..., 2:] if sliced else rnd(b, s, d).to(dtype)      # sliced: pairs, but no rows on 16 bytes
    w, bs, dy = (0.5 * rnd(d, 1, taps)).to(dtype), (0.5 * rnd(d)).to(dtype) if bias else None, rnd(b, s, d).to(dtype)
    ins = [t if t is None else t.detach().requires_grad_(True) for t in (x, w, bs)]
    given = [t for t in ins if t is not None]
    y = W().conv1d_silu(*ins)
    got = torch.autograd.grad([y], given, [dy])
    for a, c in zip(got, torch.autograd.grad([W().conv1d_silu(*ins)], given, [dy])):
        assert torch.equal(a, c)

    with torch.no_grad():
        x6, w6, g6 = x.double(), w.double()[:, 0], dy.double()
        before = lambda t, k: torch.nn.functional.pad(t, (0, 0, k, 0))[:, :s]         # t of k tokens ago
        after = lambda t, k: torch.nn.functional.pad(t, (0, 0, 0, k))[:, k:]
        pre, big = torch.zeros_like(x6), torch.zeros_like(x6)
        for k in range(taps):
            pre += before(x6, taps - 1 - k) * w6[:, k]
            big += (before(x6, taps - 1 - k) * w6[:, k]).abs()
        if bias:
            pre, big = pre + bs.double(), big + bs.double().abs()
        sg = torch.sigmoid(pre)
        near(y, pre * sg, (pre * sg).abs() + sg * big, "y")
        dpre, mag = g6 * sg * (1 + pre * (1 - sg)), g6.abs() * (sg * (1 + pre.abs()) + big)
        sums = lambda g, t: torch.stack([(g * before(t, taps - 1 - k)).sum((0, 1)) for k in range(taps)], -1)[:, None]
        back = lambda g, t: sum(after(g, taps - 1 - k) * t[:, k] for k in range(taps))
        near(got[0], back(dpre, w6), back(mag, w6.abs()), "dx")
        near(got[1], sums(dpre, x6), sums(mag, x6.abs()), "dw")
        if bias:
            near(got[2], dpre.sum((0, 1)), mag.sum((0, 1)), "dbias")


# ---- norms: more rows than the chip holds at a time -------------------------------------------------------

# Rows wider than a warp's 512 numbers are a CTA's; the SM holds 2 048 threads at most.  (A row's threads, eights of numbers a thread: 32 and 1;
# 64 and 2; 160 and 4, in the gradient 320 and 2; 128 and 2, one number at a time; 512 and 4.)
@pytest.mark.parametrize("outer,res32", [("", False), ("", True), ("both", True), ("post", False)])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,d,threads", [(9601, 96, 32), (9481, 51, 32), (4801, 1024, 64), (2003, 5120, 160), (2501, 1537, 128), (701, 16384, 512)])
def test_rms_norm_of_more_rows_than_the_chip_holds(rows, d, threads, dtype, outer, res32):
    assert rows > SMS * 2048 // threads
    gen = torch.Generator(device=DEV).manual_seed(d)
    rnd = lambda *n: torch.randn(*n, generator=gen, device=DEV)
    rt, eps = torch.float32 if res32 else dtype, 1e-6
    x, res, w = rnd(rows, d).to(dtype), (2 * rnd(rows, d)).to(rt), (1 + 0.2 * rnd(d)).to(dtype)
    post = (1 + 0.2 * rnd(d)).to(dtype) if outer else None
    scale = (0.5 + 0.1 * rnd(d)).to(dtype) if outer == "both" else None
    dy, dr = rnd(rows, d).to(dtype), rnd(rows, d).to(rt)
    ins = [t if t is None else t.detach().requires_grad_(True) for t in (x, res, w, post, scale)]
    given = [t for t in ins if t is not None]

    def call():
        y, r = W().rms_norm(ins[0], ins[2], eps=eps, residual=ins[1], post_weight=ins[3], scale=ins[4])
        return [y.detach(), r.detach(), *torch.autograd.grad([y, r], given, [dy, dr])]

    got = call()
    for a, c in zip(got, call()):
        assert torch.equal(a, c)
    with torch.no_grad():
        x6, w6, dy6 = x.double(), w.double(), dy.double()
        so, po = (1.0 if t is None else t.double() for t in (scale, post))
        s2 = 1 / torch.sqrt(x6.square().mean(-1, keepdim=True) + eps)
        xs = x6 if post is None else x6 * s2
        o = xs * po * so
        near(got[1], res.double() + o, res.double().abs() + o.abs(), "residual_out")
        r6 = got[1].double()                 # y is the norm of what is stored
        rs = 1 / torch.sqrt(r6.square().mean(-1, keepdim=True) + eps)
        rh, g = r6 * rs, dy6 * w6
        near(got[0], rh * w6, (rh * w6).abs(), "y")
        d_r = dr.double() + rs * (g - rh * (g * rh).mean(-1, keepdim=True))
        m_r = dr.double().abs() + rs * (g.abs() + rh.abs() * (g * rh).abs().mean(-1, keepdim=True))
        grads, mags = {"res": d_r, "w": (dy6 * rh).sum(0)}, {"res": m_r, "w": (dy6 * rh).abs().sum(0)}
        g2, m2 = d_r * so * po, m_r * (so if scale is None else so.abs()) * (po if post is None else po.abs())
        if post is not None:
            grads["post"], mags["post"] = (d_r * xs * so).sum(0), (m_r * xs.abs() * (so if scale is None else so.abs())).sum(0)
            g2, m2 = s2 * (g2 - xs * (g2 * xs).mean(-1, keepdim=True)), s2 * (m2 + xs.abs() * (m2 * xs.abs()).mean(-1, keepdim=True))
        if scale is not None:
            grads["scale"], mags["scale"] = (d_r * xs * po).sum(0), (m_r * (xs * po).abs()).sum(0)
        grads["x"], mags["x"] = g2, m2
        for name, a in zip([n for n, t in zip(("x", "res", "w", "post", "scale"), ins) if t is not None], got[2:]):
            near(a, grads[name], mags[name], "d" + name)


@pytest.mark.parametrize("first", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,groups,d,threads", [(1301, 8, 8 * 64, 32), (1211, 4, 4 * 1024, 64), (2501, 1, 1537, 128), (301, 2, 2 * 16384, 512),
                                                   (9601, 1, 200, 32)])
def test_gated_rms_norm_of_more_rows_than_the_chip_holds(rows, groups, d, threads, dtype, first):
    assert rows * groups > SMS * 2048 // threads
    gen = torch.Generator(device=DEV).manual_seed(d)
    rnd = lambda *n: torch.randn(*n, generator=gen, device=DEV)
    x, z, w, dy, eps = rnd(rows, d).to(dtype), rnd(rows, d).to(dtype), (1 + 0.2 * rnd(d)).to(dtype), rnd(rows, d).to(dtype), 1e-5
    ins = [t.requires_grad_(True) for t in (x, z, w)]

    def call():
        y = W().gated_rms_norm(*ins, eps=eps, groups=groups, norm_first=first)
        return [y.detach(), *torch.autograd.grad([y], ins, [dy])]

    got = call()
    for a, c in zip(got, call()):
        assert torch.equal(a, c)
    with torch.no_grad():
        x6, z6, w6, g6 = (t.double() for t in (x, z, w, dy))
        sz = torch.sigmoid(z6)
        gate, slope, m_slope = z6 * sz, sz * (1 + z6 * (1 - sz)), sz * (1 + z6.abs() * (1 - sz))
        fold, flat = lambda t: t.unflatten(-1, (groups, -1)), lambda t: t.flatten(-2)
        v = fold(x6 if first else x6 * gate)
        rs = 1 / torch.sqrt(v.square().mean(-1, keepdim=True) + eps)
        vh = v * rs
        y6 = flat(vh) * w6 * (gate if first else 1)
        gw = fold(g6 * w6 * (gate if first else 1))
        dv = flat(rs * (gw - vh * (gw * vh).mean(-1, keepdim=True)))
        m_v = flat(rs * (gw.abs() + vh.abs() * (gw * vh).abs().mean(-1, keepdim=True)))
        h = flat(vh)
        if first:
            pairs = [(dv, m_v), (g6 * h * w6 * slope, (g6 * h * w6).abs() * m_slope), ((g6 * h * gate).sum(0), (g6 * h * gate).abs().sum(0))]
        else:
            pairs = [(dv * gate, m_v * gate.abs()), (dv * x6 * slope, m_v * x6.abs() * m_slope), ((g6 * h).sum(0), (g6 * h).abs().sum(0))]
        near(got[0], y6, y6.abs(), "y")
        for name, a, (r, m) in zip(("dx", "dz", "dw"), got[1:], pairs):
            near(a, r, m, name)


# ---- gated scan: several tiles for every CTA, decays on either side of where the short form of the gates ends ---------------------

def decays(kind, d):
    """What a token's state keeps with an open gate: e^-k, k = 8 softplus(decay)."""
    k = torch.linspace(0.001, 0.1, d, dtype=torch.float64)
    if kind == "one fast channel a strip":
        k[::64] = 5.0
    elif kind == "around the border":
        k = torch.linspace(0.2, 1.2, d, dtype=torch.float64)
    elif kind == "fast":
        k = torch.logspace(-0.3, 1.5, d, dtype=torch.float64)
    return torch.log(torch.expm1(k / 8)).float().to(DEV)


def formulas(v, rate=8.0):
    """The gradients of the decay gate and of decay by their formulas in 64 bits.  (PyTorch differentiates expm1(x) as its result plus one, which
    is off by 2^-53 however small e^x is: of sqrt(1 - a^2), whose slope goes with a^2, nothing right is left once a is 1e-8.)"""
    x, i, r, decay, h, dy, dh = (v[k].detach().double().cpu() for k in ("x", "i", "r", "decay", "h", "dy", "dh"))
    reset = v["reset"].cpu()[..., None]
    si, sr = torch.sigmoid(i), torch.sigmoid(r)
    la = -rate * torch.nn.functional.softplus(decay, threshold=1e3) * sr
    a, b = torch.exp(la), torch.sqrt(-torch.expm1(2 * la))
    keep, u = torch.where(reset, torch.zeros_like(a), a), b * si * x
    before, g, c = torch.empty_like(u), torch.empty_like(u), dh
    for n in range(x.shape[1]):
        before[:, n] = h
        h = keep[:, n] * h + u[:, n]
    for n in range(x.shape[1] - 1, -1, -1):
        g[:, n] = dy[:, n] + c
        c = keep[:, n] * g[:, n]
    dla = g * (before * keep - si * x * a * a / b)
    return {"dr": dla * la * (1 - sr), "ddecay": -rate * torch.sigmoid(decay) * (dla * sr).sum((0, 1))}


@pytest.mark.parametrize("kind", ["mild", "one fast channel a strip", "around the border", "fast"])
@pytest.mark.parametrize("d", [136, 131])
@pytest.mark.parametrize("dtype", DTYPES)
def test_gated_scan_of_many_tiles(dtype, d, kind):
    b, s = 20, 1400
    units = b * 3
    assert units * ((s + 127) // 128) > 2 * 2 * SMS     # the widest tiles, two CTAs an SM: a third tile for some
    v = scan_inputs(b, s, d, dtype, True, True, seed=d)
    v["decay"] = decays(kind, d)
    ref = scan_reference(v)
    ref.update(formulas(v))
    names = ["x", "i", "r", "decay", "h"]
    ins = [v[k].detach().requires_grad_(True) for k in names]

    def call():
        y, fin = W().gated_scan(*ins[:4], initial_state=ins[4], reset=v["reset"], return_final_state=True)
        return [y.detach(), fin.detach(), *torch.autograd.grad([y, fin], ins, [v["dy"], v["dh"]])]

    got = call()
    for name, a in zip(["y", "fin"] + ["d" + k for k in names], got):
        check(a, ref[name], ref["m_" + name], s, name)
    for _ in range(3):
        assert all(torch.equal(a, c) for a, c in zip(got, call()))


def test_gradients_past_32_bits():
    """2.25e9 numbers a tensor (33 GB in all): the last rows, tokens and tiles are what the same numbers give by themselves."""
    s, d, n = 1_100_032, 2048, 30_080         # whole tiles ahead of the last ones, so that sums are in the same order
    gen = torch.Generator(device=DEV).manual_seed(1)
    base = lambda: torch.randn(50_000, d, generator=gen, device=DEV).bfloat16().repeat(23, 1)[:s]
    x, dy, w = base(), base(), (1 + 0.1 * torch.randn(d, generator=gen, device=DEV)).bfloat16()

    def of(call, outs, *ops):
        ins = [t.detach().requires_grad_(True) for t in ops]
        y = call(*ins)
        y = y if isinstance(y, tuple) else (y,)
        return [t.detach() for t in y] + list(torch.autograd.grad([y[k] for k in outs], ins, [dy[-y[0].shape[-2]:].view_as(y[k]) for k in outs]))

    def same(call, outs, *ops, skip=0):
        full, tail = of(call, outs, *ops), of(call, outs, *(t[-n:] if t.shape[0] == s else t for t in ops))
        for a, b in zip(full, tail):
            if a.numel() == s * d:
                assert torch.equal(a.view(s, d)[s - n + skip:], b.view(n, d)[skip:])
            assert torch.isfinite(a.flatten()[-d:]).all()

    same(lambda a, r, p: W().rms_norm(a, p, residual=r, post_weight=w, scale=w), (0, 1), x, x.flip(1), w)
    same(lambda a, z, p: W().gated_rms_norm(a, z, p, groups=4), (0,), x, x.flip(1), w)
    same(lambda a, c: W().conv1d_silu(a[None], c), (0,), x, (0.5 * torch.randn(d, 4, generator=gen, device=DEV)).bfloat16(), skip=3)
    decay = torch.rand(d, generator=gen, device=DEV) - 6
    with torch.no_grad():
        _, h = W().gated_scan(*[x[None, :-n]] * 3, decay, return_final_state=True)
    same(lambda a, i, r: W().gated_scan(a[None], i[None], r[None], decay, initial_state=h if a.shape[0] == n else None), (0,), x, x, x)
