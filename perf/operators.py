"""The operators of a recurrent block beside the SSD core, measured: a per-channel gated linear recurrence with its
gradient and its single-token form, the block's RMS norms (with residual, scales and gate) with theirs, and the gradient of
the causal conv1d + SiLU.

``run`` computes the plain form (elementary torch operations in 32 bits) while ``own`` is false, and calls the package's
operators while it is true.  ``exact`` is the definition in 64 bits.
"""
from __future__ import annotations

import math

import torch

own = False

_DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_EPS = 1e-6
_RATE = 8.0


def listed():
    return [
        # one decoded token for each of 64 requests in flight, the old state kept: latency, and the state's round trip
        {"name": "scan_step_b64", "op": "step", "b": 64, "d": 5120, "dtype": "bf16"},
        # a prompt of odd length and width in fp32, behind an earlier state, two documents in one row
        {"name": "scan_prompt_f32", "op": "scan", "b": 2, "s": 777, "d": 1537, "dtype": "f32", "reset": True, "state": True},
        # one long document, forward only: a few strips of channels, so the sequence itself is what is cut
        {"name": "scan_long_bf16", "op": "scan", "b": 1, "s": 131072, "d": 2048, "dtype": "bf16", "reset": False, "state": False},
        # a training step's worth of one layer
        {"name": "scan_train_bf16", "op": "scan_train", "b": 8, "s": 2048, "d": 2048, "dtype": "bf16", "reset": False, "state": False},
        # packed documents, state handed in and out with its gradient (a sequence trained on piece by piece)
        {"name": "scan_train_packed_f16", "op": "scan_train", "b": 3, "s": 1021, "d": 1536, "dtype": "f16", "reset": True, "state": True},
        # between two blocks, a token for each of 16 requests: latency
        {"name": "norm_decode", "op": "norm", "rows": 16, "d": 2048, "dtype": "f16", "res32": False, "post": False},
        # between two blocks of the 24-layer model: batch 8, 2048 tokens
        {"name": "norm_between_blocks", "op": "norm", "rows": 16384, "d": 2048, "dtype": "f16", "res32": False, "post": False},
        # the same in training, with a norm and a scale behind the block and the residual stream in fp32
        {"name": "norm_train_post_res32", "op": "norm_train", "rows": 8192, "d": 2560, "dtype": "bf16", "res32": True, "post": True},
        # the gated norm ahead of the output projection, eight groups of channels, in training
        {"name": "gated_norm_train", "op": "gnorm_train", "rows": 8192, "d": 8192, "groups": 8, "first": False, "dtype": "bf16"},
        # an odd width in fp32, normalised before the gate
        {"name": "gated_norm_train_odd", "op": "gnorm_train", "rows": 1021, "d": 1537, "groups": 1, "first": True, "dtype": "f32"},
        # conv1d + SiLU in training at the 2.7B layer's shape
        {"name": "conv_train_bf16", "op": "conv_train", "b": 4, "s": 8192, "d": 5120, "taps": 4, "dtype": "bf16"},
        # many short ragged sequences in fp32, three taps
        {"name": "conv_train_short_f32", "op": "conv_train", "b": 16, "s": 125, "d": 1544, "taps": 3, "dtype": "f32"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["step", "scan", "scan", "scan_train", "scan_train", "norm", "norm_train", "gnorm_train", "conv_train"])
    case = {"op": op, "dtype": rng.choice(["bf16", "bf16", "f16", "f32"])}
    width = rng.choice([rng.randrange(1, 129) * 64, rng.randrange(1, 1024) * 8, _log(rng, 17, 8191)])
    case["d"] = width
    if op == "step":
        case["b"] = _log(rng, 1, 256)
    elif op in ("scan", "scan_train"):
        most = (1 << 27) if op == "scan" else (1 << 25)
        case["s"] = _log(rng, 1, 131072)
        case["b"] = max(1, min(_log(rng, 1, 64), most // (case["s"] * width)))
        case["s"] = max(1, min(case["s"], most // (case["b"] * width)))
        case["reset"], case["state"] = rng.random() < 0.5, rng.random() < 0.5
    elif op in ("norm", "norm_train"):
        case["rows"] = max(1, min(_log(rng, 1, 32768), (1 << 25) // width))
        case["res32"], case["post"] = rng.random() < 0.5, rng.random() < 0.5
    elif op == "gnorm_train":
        case["rows"] = max(1, min(_log(rng, 1, 32768), (1 << 26) // width))
        case["groups"] = rng.choice([g for g in (1, 1, 2, 4, 8) if width % g == 0])
        case["first"] = rng.random() < 0.3
    else:
        case["d"] = 8 * max(1, width // 8)
        case["s"] = _log(rng, 1, 16384)
        case["b"] = max(1, min(_log(rng, 1, 64), (1 << 26) // (case["s"] * case["d"])))
        case["s"] = max(1, min(case["s"], (1 << 26) // (case["b"] * case["d"])))
        case["taps"] = rng.choice([2, 3, 4, 4])
    return case


# ---- inputs ---------------------------------------------------------------------------------------------

def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt, d, op = _DT[case["dtype"]], case["d"], case["op"]

    def randn(*shape, dtype=dt, scale=1.0, shift=0.0):
        t = torch.randn(*shape, generator=gen, device="cuda", dtype=torch.float32)
        return t.mul_(scale).add_(shift).to(dtype)

    st = {"case": case}
    if op in ("step", "scan", "scan_train"):
        # decays of a fully open gate between 0.9 and 0.999 a token, as such layers are initialised
        top = torch.rand(d, generator=gen, device="cuda") * 0.099 + 0.9
        st["decay"] = torch.log(torch.expm1(-torch.log(top) / _RATE))
        lead = (case["b"],) if op == "step" else (case["b"], case["s"])
        st["x"], st["i"], st["r"] = randn(*lead, d), randn(*lead, d), randn(*lead, d)
        if op == "step":
            st["h"] = randn(case["b"], d, dtype=torch.float32)
            st["h_next"] = torch.empty_like(st["h"])    # the token may yet be taken back: the old state stays
        else:
            st["h"] = randn(case["b"], d, dtype=torch.float32) if case["state"] else None
            st["reset"] = None
            if case["reset"]:   # documents of some 300 tokens
                st["reset"] = torch.rand(*lead, generator=gen, device="cuda") < 1.0 / 300
        if op == "scan_train":
            st["dy"] = randn(*lead, d)
            st["dh"] = randn(case["b"], d, dtype=torch.float32) if case["state"] else None
            leaves = ["x", "i", "r", "decay"] + (["h"] if case["state"] else [])
    elif op in ("norm", "norm_train"):
        rows, rt = case["rows"], torch.float32 if case["res32"] else dt
        st["x"], st["res"] = randn(rows, d), randn(rows, d, dtype=rt, scale=2.0)
        st["w"] = randn(d, scale=0.2, shift=1.0)
        st["post"] = randn(d, scale=0.2, shift=1.0) if case["post"] else None
        st["scale"] = randn(d, scale=0.1, shift=0.5) if case["post"] else None
        if op == "norm_train":
            st["dy"], st["dres"] = randn(rows, d), randn(rows, d, dtype=rt)
            leaves = ["x", "res", "w"] + (["post", "scale"] if case["post"] else [])
    elif op == "gnorm_train":
        rows = case["rows"]
        st["x"], st["z"], st["w"], st["dy"] = randn(rows, d), randn(rows, d), randn(d, scale=0.2, shift=1.0), randn(rows, d)
        leaves = ["x", "z", "w"]
    else:
        b, s, taps = case["b"], case["s"], case["taps"]
        st["x"], st["dy"] = randn(b, s, d), randn(b, s, d)
        st["w"], st["bias"] = randn(d, 1, taps, scale=0.5), randn(d, scale=0.5)
        leaves = ["x", "w", "bias"]
    if op.endswith("_train"):
        st["leaves"] = leaves
        for name in leaves:
            st[name].requires_grad_(True)
    return st


# ---- one pass -------------------------------------------------------------------------------------------

def run(state):
    op = state["case"]["op"]
    if own:
        return _own(op, state)
    with torch.no_grad():
        return {"step": _plain_step, "scan": _plain_scan, "scan_train": _plain_scan_train, "norm": _plain_norm,
                "norm_train": _plain_norm_train, "gnorm_train": _plain_gnorm_train, "conv_train": _plain_conv_train}[op](state)


def _own(op, st):
    import workloadsuite_b200 as W

    leaves = [st[n] for n in st.get("leaves", ())]
    if op == "step":
        y = W.gated_scan_step(st["x"], st["i"], st["r"], st["decay"], st["h"], out_state=st["h_next"], rate=_RATE)
        return [y, st["h_next"]]
    if op == "scan":
        return list(W.gated_scan(st["x"], st["i"], st["r"], st["decay"], initial_state=st["h"], reset=st["reset"],
                                 return_final_state=True, rate=_RATE))
    if op == "scan_train":
        y, fin = W.gated_scan(st["x"], st["i"], st["r"], st["decay"], initial_state=st["h"], reset=st["reset"],
                              return_final_state=True, rate=_RATE)
        outs, grads = ([y, fin], [st["dy"], st["dh"]]) if st["dh"] is not None else ([y], [st["dy"]])
        return [y.detach(), fin.detach(), *torch.autograd.grad(outs, leaves, grads)]
    if op == "norm":
        return list(W.rms_norm(st["x"], st["w"], eps=_EPS, residual=st["res"], post_weight=st["post"], scale=st["scale"]))
    if op == "norm_train":
        y, r = W.rms_norm(st["x"], st["w"], eps=_EPS, residual=st["res"], post_weight=st["post"], scale=st["scale"])
        return [y.detach(), r.detach(), *torch.autograd.grad([y, r], leaves, [st["dy"], st["dres"]])]
    if op == "gnorm_train":
        y = W.gated_rms_norm(st["x"], st["z"], st["w"], eps=_EPS, groups=st["case"]["groups"], norm_first=st["case"]["first"])
        return [y.detach(), *torch.autograd.grad([y], leaves, [st["dy"]])]
    y = W.conv1d_silu(st["x"], st["w"], st["bias"])
    return [y.detach(), *torch.autograd.grad([y], leaves, [st["dy"]])]


# ---- the plain forms ------------------------------------------------------------------------------------

def _gates(x, i, r, decay):
    """Rate of decay per channel, the gates, log a, a, b = sqrt(1 - a^2), and what enters the state."""
    k = -_RATE * torch.log1p(torch.exp(-decay.abs())) - _RATE * decay.clamp_min(0)
    sr, si = torch.sigmoid(r.float()), torch.sigmoid(i.float())
    la = k * sr
    b = torch.sqrt(-torch.expm1(2 * la))
    return k, sr, si, la, torch.exp(la), b, b * si * x.float()


def _running(a, u):
    """h_t = a_t h_{t-1} + u_t along axis 1 from zero, by doubling (u and a are overwritten)."""
    step, s = 1, u.shape[1]
    while step < s:
        u[:, step:] += a[:, step:] * u[:, :-step]
        a[:, step:] = a[:, step:] * a[:, :-step]
        step *= 2
    return u


def _plain_step(st):
    _, _, _, _, a, _, u = _gates(st["x"], st["i"], st["r"], st["decay"])
    h = a * st["h"] + u
    return [h.to(st["x"].dtype), h]


def _forward32(st):
    k, sr, si, la, a, b, u = _gates(st["x"], st["i"], st["r"], st["decay"])
    keep = a if st["reset"] is None else a.masked_fill(st["reset"][..., None], 0.0)
    h0 = st["h"]
    first = u.clone()
    if h0 is not None:
        first[:, 0] += keep[:, 0] * h0
    h = _running(keep.clone(), first)
    return k, sr, si, la, a, b, keep, h


def _plain_scan(st):
    h = _forward32(st)[-1]
    return [h.to(st["x"].dtype), h[:, -1].clone()]


def _plain_scan_train(st):
    k, sr, si, la, a, b, keep, h = _forward32(st)
    x, dt = st["x"].float(), st["x"].dtype
    g = st["dy"].float()
    if st["dh"] is not None:
        g[:, -1] += st["dh"]
    # g_t = dy_t + a_{t+1} g_{t+1}
    back = torch.zeros_like(keep)
    back[:, 1:] = keep[:, 1:].flip(1)
    g = _running(back, g.flip(1)).flip(1)
    before = torch.zeros_like(h)
    before[:, 1:] = h[:, :-1]
    if st["h"] is not None:
        before[:, 0] = st["h"]
    dx = g * b * si
    di = g * b * x * si * (1 - si)
    dla = g * before * keep - torch.where(b > 0, g * si * x * a * a / b, torch.zeros_like(b))
    dr = dla * la * (1 - sr)
    ddecay = (dla * sr).sum((0, 1)) * -_RATE * torch.sigmoid(st["decay"])
    out = [h.to(dt), h[:, -1].clone(), dx.to(dt), di.to(dt), dr.to(dt), ddecay]
    if st["h"] is not None:
        out.append(keep[:, 0] * g[:, 0])
    return out


def _rms(v):
    return torch.rsqrt((v * v).mean(-1, keepdim=True) + _EPS)


def _norm32(st):
    x, res = st["x"].float(), st["res"]
    s, xh = None, x
    if st["post"] is not None:
        s = _rms(x)
        xh = x * s
        o = xh * st["post"].float() * st["scale"].float()
    else:
        o = x
    r = (res.float() + o).to(res.dtype)      # the residual as it is stored: what the norm is of
    rf = r.float()
    rs = _rms(rf)
    return s, xh, r, rf * rs, rs


def _plain_norm(st):
    _, _, r, rh, _ = _norm32(st)
    return [(rh * st["w"].float()).to(st["x"].dtype), r]


def _through_rms(g, vh, rs):
    """Gradient of v * rms(v) against v, g that of the normalised row vh."""
    return rs * (g - vh * (g * vh).mean(-1, keepdim=True))


def _plain_norm_train(st):
    s, xh, r, rh, rs = _norm32(st)
    dt, w, dy = st["x"].dtype, st["w"].float(), st["dy"].float()
    dr = st["dres"].float() + _through_rms(dy * w, rh, rs)
    dw = (dy * rh).sum(0)
    out = [(rh * w).to(dt), r]
    if st["post"] is None:
        return out + [dr.to(dt), dr.to(r.dtype), dw.to(dt)]
    post, scale = st["post"].float(), st["scale"].float()
    both = (dr * xh).sum(0)
    dx = _through_rms(dr * scale * post, xh, s)
    return out + [dx.to(dt), dr.to(r.dtype), dw.to(dt), (both * scale).to(dt), (both * post).to(dt)]


def _plain_gnorm_train(st):
    groups, first, dt = st["case"]["groups"], st["case"]["first"], st["x"].dtype
    rows, d = st["x"].shape
    cut = lambda t: t.reshape(rows, groups, d // groups)
    x, z, dy, w = st["x"].float(), st["z"].float(), st["dy"].float(), st["w"].float()
    sz = torch.sigmoid(z)
    gate, slope = z * sz, sz * (1 + z * (1 - sz))
    v = cut(x if first else x * gate)
    rs = _rms(v)
    vh = (v * rs)
    flat = vh.reshape(rows, d)
    if first:
        y = flat * w * gate
        dw = (dy * flat * gate).sum(0)
        dx = _through_rms(cut(dy * w * gate), vh, rs).reshape(rows, d)
        dz = dy * flat * w * slope
    else:
        y = flat * w
        dw = (dy * flat).sum(0)
        dv = _through_rms(cut(dy * w), vh, rs).reshape(rows, d)
        dx, dz = dv * gate, dv * x * slope
    return [y.to(dt), dx.to(dt), dz.to(dt), dw.to(dt)]


def _plain_conv_train(st):
    taps, dt = st["case"]["taps"], st["x"].dtype
    x, dy, w = st["x"].float(), st["dy"].float(), st["w"].float().reshape(-1, taps)
    s = x.shape[1]
    pre = st["bias"].float().expand_as(x).clone()
    for k in range(taps):
        back = taps - 1 - k
        if back < s:
            pre[:, back:] += x[:, :s - back] * w[:, k]
    sg = torch.sigmoid(pre)
    y = pre * sg
    dpre = dy * sg * (1 + pre * (1 - sg))
    dx, dw = torch.zeros_like(x), torch.zeros_like(w)
    for k in range(taps):
        back = taps - 1 - k
        if back < s:
            dx[:, :s - back] += dpre[:, back:] * w[:, k]
            dw[:, k] = (dpre[:, back:] * x[:, :s - back]).sum((0, 1))
    return [y.to(dt), dx.to(dt), dw.reshape(st["w"].shape).to(dt), dpre.sum((0, 1)).to(dt)]


# ---- what a pass cannot do without ----------------------------------------------------------------------

def work(case):
    d, op = case["d"], case["op"]
    e = 4 if case["dtype"] == "f32" else 2
    if op == "step":
        n = case["b"] * d
        return {"bytes": n * (4 * e + 8) + 4 * d, "flops": 14 * n}
    if op in ("scan", "scan_train"):
        n, states = case["b"] * case["s"] * d, case["b"] * d * 4
        marks = case["b"] * case["s"] if case["reset"] else 0
        if op == "scan":
            return {"bytes": 4 * n * e + marks + 4 * d + states * (2 if case["state"] else 1), "flops": 14 * n}
        return {"bytes": 8 * n * e + marks + 8 * d + states * (4 if case["state"] else 1), "flops": 45 * n}
    if op in ("norm", "norm_train"):
        n, r = case["rows"] * d, 4 if case["res32"] else e
        p = 3 if case["post"] else 1
        if op == "norm":
            return {"bytes": n * (2 * e + 2 * r) + p * d * e, "flops": (9 if case["post"] else 5) * n}
        return {"bytes": n * (4 * e + 4 * r) + 2 * p * d * e, "flops": (30 if case["post"] else 15) * n}
    if op == "gnorm_train":
        n = case["rows"] * d
        return {"bytes": 6 * n * e + 2 * d * e, "flops": 32 * n}
    n, taps = case["b"] * case["s"] * d, case["taps"]
    return {"bytes": 4 * n * e + 2 * d * (taps + 1) * e, "flops": (6 * taps + 14) * n}


# ---- the definitions in 64 bits -------------------------------------------------------------------------

def exact(case, seed):
    st = prepare(case, seed)
    op = case["op"]
    v = {k: t.detach().double() for k, t in st.items() if isinstance(t, torch.Tensor) and t.is_floating_point()}
    for name in st.get("leaves", ()):
        v[name].requires_grad_(True)
    leaves = [v[n] for n in st.get("leaves", ())]

    if op in ("step", "scan", "scan_train"):
        la = -_RATE * torch.nn.functional.softplus(v["decay"], threshold=1e3) / (1 + torch.exp(-v["r"]))
        a = torch.exp(la)
        u = torch.sqrt(-torch.expm1(2 * la)) * v["x"] / (1 + torch.exp(-v["i"]))
        if op == "step":
            h = a * v["h"] + u
            return [h, h]
        if st["reset"] is not None:
            a = torch.where(st["reset"][..., None], torch.zeros_like(a), a)
        h = v["h"] if "h" in v else torch.zeros_like(u[:, 0])
        if op == "scan":
            hs = torch.empty_like(u)
            for t in range(case["s"]):
                h = torch.addcmul(u[:, t], a[:, t], h, out=hs[:, t])
            return [hs, h]
        if case["s"] > 16384:
            return None
        steps = []
        for at, ut in zip(a.unbind(1), u.unbind(1)):
            h = torch.addcmul(ut, at, h)
            steps.append(h)
        hs = torch.stack(steps, 1)
        outs, grads = ([hs, h], [v["dy"], v["dh"]]) if st["dh"] is not None else ([hs], [v["dy"]])
        return [hs.detach(), h.detach(), *torch.autograd.grad(outs, leaves, grads)]

    unit = lambda t: t / torch.sqrt(t.square().mean(-1, keepdim=True) + _EPS)
    if op in ("norm", "norm_train"):
        o = v["x"] if st["post"] is None else unit(v["x"]) * v["post"] * v["scale"]
        r = v["res"] + o
        # the norm is of the residual as it is stored; its gradient passes the rounding unchanged
        r = r + (r.detach().to(st["res"].dtype).double() - r.detach())
        y = unit(r) * v["w"]
        if op == "norm":
            return [y, r]
        return [y.detach(), r.detach(), *torch.autograd.grad([y, r], leaves, [v["dy"], v["dres"]])]
    if op == "gnorm_train":
        gate = v["z"] / (1 + torch.exp(-v["z"]))
        fold = lambda t: t.unflatten(-1, (case["groups"], -1))
        y = unit(fold(v["x"])).flatten(-2) * v["w"] * gate if case["first"] else unit(fold(v["x"] * gate)).flatten(-2) * v["w"]
        return [y.detach(), *torch.autograd.grad([y], leaves, [v["dy"]])]
    padded = torch.nn.functional.pad(v["x"], (0, 0, case["taps"] - 1, 0))
    pre = v["bias"] + sum(padded[:, k:k + case["s"]] * v["w"][:, 0, k] for k in range(case["taps"]))
    y = pre / (1 + torch.exp(-pre))
    return [y.detach(), *torch.autograd.grad([y], leaves, [v["dy"]])]
