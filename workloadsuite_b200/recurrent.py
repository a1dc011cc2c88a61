"""A recurrent block's pieces beside the SSD core, with their gradients: a per-channel gated linear recurrence
(``gated_scan``, ``gated_scan_step``) and the block's RMS norms (``rms_norm``, ``gated_rms_norm``).

The reference has the norms as ``nn.RMSNorm`` with a residual sum of its own (``model_ref.py:49-66, 165-204``) and no
counterpart of the recurrence.  All run in the kernels of ``csrc/ssd_gated_scan.cu`` and ``csrc/ssd_norm.cu`` on the current
CUDA stream, without a CPU path, and never synchronise the host.  Gradients are backward ones, recorded by autograd; an operand with a
forward-mode tangent or under a function transform (``torch.func``) is refused (NotImplementedError).
"""
from __future__ import annotations

import ctypes
import math
from typing import Optional

import torch

from . import _lib
from .ssd import _DTYPES, _check_out, _no_tangents, _plain, _same_device


def _records(*tensors) -> bool:
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


def _need_cuda(name: str, x: torch.Tensor):
    if not x.is_cuda:
        raise RuntimeError(f"{name} needs CUDA tensors (there is no CPU path)")


def _rows(t: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    """A tensor whose channels do not lie side by side is copied once; anything else stays the view it is."""
    t = _plain(t)
    return t if t is None or t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _real(v: float) -> float:
    """As the kernels get it, in 32 bits."""
    return ctypes.c_float(v).value


def _done(got, name: str):
    if got is None:
        raise NotImplementedError(f"{name}: sizes or strides outside what the kernels cover")
    return got


# ---- gated recurrence -----------------------------------------------------------------------------------

def _check_gates(name, x, input_gate, decay_gate, decay, dims, rate):
    _need_cuda(name, x)
    if x.dim() != dims:
        raise ValueError(f"x must be [{'b,s,d' if dims == 3 else 'b,d'}]")
    _same_device(x, input_gate=input_gate, decay_gate=decay_gate, decay=decay)
    if x.dtype not in _DTYPES:
        raise TypeError("x must be float32, float16 or bfloat16")
    for what, t in (("input_gate", input_gate), ("decay_gate", decay_gate)):
        if t.shape != x.shape or t.dtype != x.dtype:
            raise ValueError(f"{what} must have the shape and dtype of x")
    if decay.shape != x.shape[-1:] or decay.dtype not in _DTYPES:
        raise ValueError("decay must be a floating point [d]")
    if not 0 < _real(rate) < math.inf:
        raise ValueError("rate must be positive and finite in float32")


def _check_state(name, t, x):
    want = (x.shape[0], x.shape[-1])
    if t.shape != want or t.dtype != torch.float32:
        raise ValueError(f"{name} must be float32 [b,d]")


def gated_scan(x: torch.Tensor, input_gate: torch.Tensor, decay_gate: torch.Tensor, decay: torch.Tensor,
               initial_state: Optional[torch.Tensor] = None, reset: Optional[torch.Tensor] = None,
               return_final_state: bool = False, rate: float = 8.0, out: Optional[torch.Tensor] = None,
               wait_limit_ms: int = 0):
    """Per-channel gated linear recurrence over a sequence, on the current CUDA stream, with its gradient::

        log a[t] = -rate * softplus(decay) * sigmoid(decay_gate[t])
        h[t]     = a[t] * h[t-1] + sqrt(1 - a[t]^2) * sigmoid(input_gate[t]) * x[t],      y = h

    x, input_gate, decay_gate [b,s,d] in one dtype of float32/float16/bfloat16 (views with contiguous channels, such as columns of
    a projection's output, are read where they lie); decay [d], one number per channel, float32 or any of those;
    initial_state float32 [b,d] or None for zeros; reset bool [b,s]: a token that is marked starts anew, as if the state
    before it were zero, whatever it was (documents packed into one row); the factor sqrt(1 - a^2) stays, which published blocks of this
    kind drop at a document's first token.  Gates, decays and the state are float32
    throughout; y is rounded once, to x's dtype.  Sequences of no tokens are allowed.

    Returns y [b,s,d], with ``return_final_state`` also the float32 state [b,d] behind the last token (the
    ``initial_state`` of a call that goes on, or the ``state`` of ``gated_scan_step``).  Differentiable in x, both gates, decay and
    initial_state, through y and through the final state; the gradient makes the states again in float32 from those of
    every 64th token, which the forward then keeps (d / 16 bytes a token).  ``out`` receives y where no gradient is recorded.
    Results and gradients do not vary from run to run.  Waits between the CTAs of a launch are bounded as in ``ssd_forward``
    (``device_status`` 8).
    """
    rate = float(rate)
    got = _lib.fast().gated_scan(x, input_gate, decay_gate, decay, initial_state, reset, out, rate, 0) \
        if 0 < rate < math.inf and wait_limit_ms == 0 else None
    if got is not None:
        return got if return_final_state else got[0]
    _check_gates("gated_scan", x, input_gate, decay_gate, decay, 3, rate)
    _no_tangents("gated_scan", x, input_gate, decay_gate, decay, initial_state)
    _same_device(x, initial_state=initial_state, reset=reset, out=out)
    if not 0 <= wait_limit_ms < 1 << 31:
        raise ValueError("wait_limit_ms must not be negative, nor 2^31 and more")
    if initial_state is not None:
        _check_state("initial_state", initial_state, x)
        initial_state = _plain(initial_state).contiguous()
    if reset is not None and (reset.shape != x.shape[:2] or reset.dtype != torch.bool):
        raise ValueError("reset must be bool [b,s]")
    if out is not None:
        if _records(x, input_gate, decay_gate, decay, initial_state):
            raise ValueError("out cannot be given where a gradient is recorded")
        _check_out(out, x)
    x, input_gate, decay_gate, decay = _rows(x), _rows(input_gate), _rows(decay_gate), _plain(decay).float().contiguous()
    reset, out = _plain(reset), _plain(out)
    if x.numel() == 0:      # no tokens: the state stays what it was
        y = (x + input_gate + decay_gate) * decay.to(x.dtype) if out is None else out
        fin = x.new_zeros((x.shape[0], x.shape[2]), dtype=torch.float32) if initial_state is None else initial_state.clone()
    else:
        y, fin = _done(_lib.fast().gated_scan(x, input_gate, decay_gate, decay, initial_state, reset, out, rate, int(wait_limit_ms)), "gated_scan")
    return (y, fin) if return_final_state else y


def gated_scan_step(x: torch.Tensor, input_gate: torch.Tensor, decay_gate: torch.Tensor, decay: torch.Tensor, state: torch.Tensor,
                    rate: float = 8.0, out: Optional[torch.Tensor] = None, out_state: Optional[torch.Tensor] = None) -> torch.Tensor:
    """One token of ``gated_scan`` on the current CUDA stream, the state carried in place (decode-style use).

    x, input_gate, decay_gate [b,d] in one dtype, decay [d], state float32 [b,d] contiguous, updated in place, or left as it
    is where ``out_state`` (the same shape) receives the new one: a token that may yet be taken back.  Returns y [b,d].
    Records no gradient.
    """
    rate = float(rate)
    got = _lib.fast().gated_step(x, input_gate, decay_gate, decay, state, out_state, out, rate) if 0 < rate < math.inf else None
    if got is not None:
        return got
    _check_gates("gated_scan_step", x, input_gate, decay_gate, decay, 2, rate)
    _same_device(x, state=state, out_state=out_state, out=out)
    for name, t in (("state", state), ("out_state", out_state)):
        if t is not None:
            _check_state(name, t, x)
            if not t.is_contiguous():
                raise ValueError(f"{name} must be contiguous")
    if out is not None:
        _check_out(out, x)
    if x.numel() == 0:
        return torch.empty_like(x) if out is None else out
    return _done(_lib.fast().gated_step(_rows(x), _rows(input_gate), _rows(decay_gate), _plain(decay).detach().float().contiguous(), _plain(state),
                                        _plain(out_state), _plain(out), rate), "gated_scan_step")


# ---- norms ----------------------------------------------------------------------------------------------

_EPS = torch.finfo(torch.float32).eps     # what nn.RMSNorm takes where none is given


def _flat(t: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    """[..., d] whose rows do not lie at one distance is copied once."""
    t = _plain(t)
    if t is None or t.dim() < 2:
        return t if t is None or t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()
    try:
        t.view(-1, t.shape[-1])
    except RuntimeError:
        return t.contiguous()
    return _rows(t)


def _check_norm(name, x, eps, vectors, rows, groups=1):
    _need_cuda(name, x)
    if x.dim() < 1 or x.dtype not in _DTYPES:
        raise TypeError("x must be [...,d] of float32, float16 or bfloat16")
    _same_device(x, **vectors, **rows)
    for what, t in vectors.items():
        if t is not None and (t.shape != x.shape[-1:] or t.dtype not in (torch.float32, x.dtype)):
            raise ValueError(f"{what} must be [d], float32 or in x's dtype")
    for what, t in rows.items():
        if t is not None and t.shape != x.shape:
            raise ValueError(f"{what} must have the shape of x")
    if x.shape[-1] == 0:
        raise ValueError("rows must not be empty")
    if not 0 <= _real(eps) < math.inf or eps < 0:
        raise ValueError("eps must be finite in float32 and not negative")
    if groups <= 0 or x.shape[-1] % groups != 0:
        raise ValueError("groups must divide d")


def rms_norm(x: torch.Tensor, weight: torch.Tensor, eps: Optional[float] = None, residual: Optional[torch.Tensor] = None,
             post_weight: Optional[torch.Tensor] = None, scale: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None):
    """RMS norm ahead of a block, with what lies between two blocks in the same pass, on the current CUDA stream, and its gradient.

    Without ``residual``: ``x * rms(x) * weight``, ``rms(v) = 1 / sqrt(mean(v^2) + eps)``, the ``nn.RMSNorm`` of
    ``model_ref.py:49-66``.  With ``residual`` x is what the block before has put out, and the call returns (y, residual_out)::

        o = x,  or with post_weight  x * rms(x) * post_weight  (a norm behind the block);   o *= scale  when given
        residual_out = residual + o,         y = residual_out * rms(residual_out) * weight

    x [...,d] of float32/float16/bfloat16 (rows may be views); residual and residual_out in x's dtype or float32; weight, post_weight and
    scale [d], float32 or in x's dtype; d up to 16384.  Sums are float32 and everything is rounded once; y is the norm of
    residual_out as it is stored.  ``eps`` None is float32's, as in ``nn.RMSNorm``.  ``out`` receives y where no gradient is recorded.
    """
    eps = _EPS if eps is None else float(eps)
    got = _lib.fast().rms_norm(x, weight, residual, post_weight, scale, out, eps) if 0 <= eps < math.inf else None
    if got is not None:
        return got[0] if residual is None else got
    _check_norm("rms_norm", x, eps, dict(weight=weight, post_weight=post_weight, scale=scale), dict(residual=residual, out=out))
    _no_tangents("rms_norm", x, weight, residual, post_weight, scale)
    if residual is None and (post_weight is not None or scale is not None):
        raise ValueError("post_weight and scale apply to what is added to residual: give one")
    if residual is not None and residual.dtype not in (torch.float32, x.dtype):
        raise ValueError("residual must be float32 or in x's dtype")
    if out is not None:
        if _records(x, weight, residual, post_weight, scale):
            raise ValueError("out cannot be given where a gradient is recorded")
        _check_out(out, x)
        out = _plain(out)
        if _flat(out) is not out:
            raise ValueError("out: rows must lie at one distance from each other")
    weight, post_weight, scale = (None if t is None else _plain(t).contiguous() for t in (weight, post_weight, scale))
    x, residual = _flat(x), _flat(residual)
    if x.numel() == 0:
        for t in (post_weight, scale):
            x = x if t is None else x * t.to(x.dtype)
        y = x * weight.to(x.dtype) if out is None else out
        return y if residual is None else (y, residual + x.to(residual.dtype))
    y, r = _done(_lib.fast().rms_norm(x, weight, residual, post_weight, scale, out, eps), "rms_norm")
    return y if residual is None else (y, r)


def gated_rms_norm(x: torch.Tensor, z: torch.Tensor, weight: torch.Tensor, eps: Optional[float] = None, groups: int = 1,
                   norm_first: bool = False, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """RMS norm and gate ahead of a block's output projection, on the current CUDA stream, with its gradient:
    ``(x * silu(z)) * rms(x * silu(z)) * weight``, or with ``norm_first`` ``x * rms(x) * weight * silu(z)``, rms over each of
    ``groups`` equal parts of a row.

    x and z [...,d] in one dtype of float32/float16/bfloat16 (rows may be views, such as columns of a projection's output); weight [d],
    float32 or in x's dtype; d / groups up to 16384.  float32 inside, one rounding.  ``eps`` and ``out`` as in ``rms_norm``.
    """
    eps = _EPS if eps is None else float(eps)
    groups, norm_first = int(groups), bool(norm_first)
    got = _lib.fast().gated_rms_norm(x, z, weight, out, eps, groups, norm_first) if 0 <= eps < math.inf else None
    if got is not None:
        return got
    _check_norm("gated_rms_norm", x, eps, dict(weight=weight), dict(z=z, out=out), groups)
    _no_tangents("gated_rms_norm", x, z, weight)
    if z.dtype != x.dtype:
        raise ValueError("z must be in x's dtype")
    if out is not None:
        if _records(x, z, weight):
            raise ValueError("out cannot be given where a gradient is recorded")
        _check_out(out, x)
        out = _plain(out)
        if _flat(out) is not out:
            raise ValueError("out: rows must lie at one distance from each other")
    x, z, weight = _flat(x), _flat(z), _plain(weight).contiguous()
    if x.numel() == 0:
        return x * z * weight.to(x.dtype) if out is None else out
    return _done(_lib.fast().gated_rms_norm(x, z, weight, out, eps, groups, norm_first), "gated_rms_norm")
