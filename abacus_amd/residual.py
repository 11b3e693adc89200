"""The residual stream between two blocks of the decoder: a block's output added to it, and the next block's norm.

``residual_norm`` takes the two steps of transformer_block.py:98-100 and norm.py:26-31, x + f and RMSNorm, in one pass
each way (csrc/residual_norm.hip), with a norm of the block's output, a gate and a residual scale where a model has
them.  CPU tensors take the same steps in torch's operations.
"""

from __future__ import annotations

import ctypes

import torch
from torch.autograd import forward_ad

from . import _lib
from .kv_cache import _call
from .moe import _contig

__all__ = ["residual_norm"]


def _norm(v, weight, eps: float):
    return weight * v * torch.rsqrt(v.square().mean(dim=-1, keepdim=True) + eps)


def _plain(x, y, gamma, post_gamma, gate, scale: float, eps: float):
    """(r, h) in torch's operations, in fp32 (fp64 for fp64 tensors); h of r rounded to x's type."""
    wide = torch.promote_types(x.dtype, torch.float32)
    branch = y.to(wide)
    if post_gamma is not None:
        branch = _norm(branch, post_gamma.to(wide), eps)
    if gate is not None:
        branch = gate.to(wide) * branch
    r = (x.to(wide) + scale * branch).to(x.dtype)
    return r, _norm(r.to(wide), gamma.to(wide), eps).to(x.dtype)


def _gate_kind(gate: torch.Tensor | None) -> int:
    return 0 if gate is None else 1 if gate.dim() == 1 else 2


def _at(t: torch.Tensor | None) -> int | None:
    """The address of an operand that _contig has seen, or of a new tensor."""
    return None if t is None else t.data_ptr()


def _forward(x, y, gamma, post_gamma, gate, scale: float, eps: float, keep: bool):
    """(r, h, rstd, y_rstd) of contiguous tensors; the last two None where they are not kept."""
    D, dev = x.shape[-1], x.device
    rows = x.numel() // D
    r, h = torch.empty_like(x), torch.empty_like(x)
    rstd = torch.empty(rows, dtype=torch.float32, device=dev) if keep else None
    y_rstd = torch.empty(rows, dtype=torch.float32, device=dev) if keep and post_gamma is not None else None
    _call(dev, "abacus_residual_norm_fwd", x.data_ptr(), y.data_ptr(), gamma.data_ptr(), _at(post_gamma), _at(gate),
          _gate_kind(gate), rows, D, scale, eps, _lib.dtype_code(x.dtype), r.data_ptr(), h.data_ptr(), _at(rstd), _at(y_rstd))
    return r, h, rstd, y_rstd


def _recorded(ctx, grads, dr, dh, y, gamma, post_gamma, gate, r):
    """grads, tied to what they were formed from where the running backward is itself recorded: dx and dgamma to r (which
    leads on to x and y) and gamma, the others to dx and the branch's own operands."""
    from .transformer import _KernelGradient

    dx, dy, dgamma, dpost, dgate = grads
    d_out = torch.stack([torch.zeros_like(r) if d is None else d for d in (dr, dh)])
    dx, dgamma = _KernelGradient.apply(lambda r, gamma: torch.stack((r, _norm(r, gamma, ctx.eps))), (dx, dgamma), d_out, r,
                                       gamma)
    if post_gamma is None and gate is None:
        return dx, ctx.scale * dx, dgamma, None, None

    def branch(y, *rest):
        rest = list(rest)
        b = y if post_gamma is None else _norm(y, rest.pop(0), ctx.eps)
        return ctx.scale * (b if gate is None else rest.pop(0) * b)

    formed = iter(_KernelGradient.apply(branch, tuple(d for d in (dy, dpost, dgate) if d is not None), dx,
                                        *(t for t in (y, post_gamma, gate) if t is not None)))
    return dx, next(formed), dgamma, *(None if d is None else next(formed) for d in (dpost, dgate))


class _ResidualNorm(torch.autograd.Function):
    """residual_norm and its gradients, one kernel each way and the sums over rows."""

    @staticmethod
    def forward(ctx, x, y, gamma, post_gamma, gate, scale: float, eps: float):
        ctx.set_materialize_grads(False)
        ctx.scale, ctx.eps = scale, eps
        c = [None if t is None else _contig(t) for t in (x, y, gamma, post_gamma, gate)]
        r, h, rstd, y_rstd = _forward(*c, scale, eps, True)
        ctx.save_for_backward(None if post_gamma is None and gate is None else y, gamma, post_gamma, gate, r, rstd, y_rstd)
        return r, h

    @staticmethod
    def backward(ctx, dr, dh):
        if dr is None and dh is None:
            return (None,) * 7
        *leaves, rstd, y_rstd = ctx.saved_tensors
        if not torch.is_grad_enabled():
            return (*_ResidualNorm.gradients(ctx, dr, dh, *leaves, rstd, y_rstd, ctx.needs_input_grad[2:5]), None, None)
        with torch.no_grad():
            grads = _ResidualNorm.gradients(ctx, dr, dh, *leaves, rstd, y_rstd)
        return (*_recorded(ctx, grads, dr, dh, *leaves), None, None)

    @staticmethod
    def gradients(ctx, dr, dh, y, gamma, post_gamma, gate, r, rstd, y_rstd, want=(True, True, True)):
        """(dx, dy, dgamma, dpost, dgate); want: which of the last three are formed, where there is one."""
        D, dev, dt = r.shape[-1], r.device, _lib.dtype_code(r.dtype)
        rows = r.numel() // D
        r, rstd = _contig(r), rstd.contiguous()
        y_rstd = None if y_rstd is None else y_rstd.contiguous()
        dr, dh, y, gamma, post_gamma, gate = [None if t is None else _contig(t) for t in (dr, dh, y, gamma, post_gamma, gate)]
        dx = torch.empty_like(r)
        same = post_gamma is None and gate is None and ctx.scale == 1.0  # dy is dx
        dy = None if same else torch.empty_like(r)
        dgamma, dpost, dgate = (torch.empty_like(t) if w and t is not None else None
                                for t, w in zip((gamma, post_gamma, gate), want))
        kind = _gate_kind(gate)
        nbytes = _lib.query("abacus_residual_norm_bwd_ws_bytes", rows, D, int(post_gamma is not None), kind)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
        _call(dev, "abacus_residual_norm_bwd", _at(dr), _at(dh), r.data_ptr(), _at(y), gamma.data_ptr(), _at(post_gamma),
              _at(gate), kind, rstd.data_ptr(), _at(y_rstd), rows, D, ctx.scale, dt, dx.data_ptr(), _at(dy), _at(dgamma),
              _at(dpost), _at(dgate), ws.data_ptr(), nbytes)
        return dx, dx if same else dy, dgamma, dpost, dgate


def residual_norm(x: torch.Tensor, y: torch.Tensor, gamma: torch.Tensor, post_gamma: torch.Tensor | None = None,
                  gate: torch.Tensor | None = None, scale: float = 1.0, eps: float = 1e-5):
    """(r, h): r = x + scale * gate * b, the stream x with a block's output y in it, and h = gamma * r / rms(r).

    x and y (..., D); gamma, post_gamma (D,); gate (D,) or x's shape.  b is y, or with post_gamma
    post_gamma * y / rms(y); rms(v) = sqrt(mean(v^2) + eps).  All in fp32, r rounded once and h, once more, of r as it
    is returned: without post_gamma, gate and scale, the bits of ``x + y`` and RMSNorm.
    """
    D = x.shape[-1] if x.dim() else 0
    if D < 1 or y.shape != x.shape:
        raise ValueError(f"residual_norm takes x and y of one shape (..., D), got {tuple(x.shape)} and {tuple(y.shape)}")
    for name, t in (("gamma", gamma), ("post_gamma", post_gamma)):
        if t is not None and t.shape != (D,):
            raise ValueError(f"{name} has {D} values, got {tuple(t.shape)}")
    if gate is not None and gate.shape not in ((D,), x.shape):
        raise ValueError(f"gate has {D} values or x's shape {tuple(x.shape)}, got {tuple(gate.shape)}")
    grad = x.requires_grad
    for name, t in (("y", y), ("gamma", gamma), ("post_gamma", post_gamma), ("gate", gate)):
        if t is None:
            continue
        if t.dtype != x.dtype:
            raise TypeError(f"residual_norm takes tensors of one type: x is {x.dtype} and {name} {t.dtype}")
        if t.device != x.device:
            raise ValueError(f"residual_norm takes tensors on one device: x is on {x.device} and {name} on {t.device}")
        grad = grad or t.requires_grad
    if x.device.type == "cpu" or x.numel() == 0:
        return _plain(x, y, gamma, post_gamma, gate, scale, eps)
    least, most = (8, 8192) if _lib.dtype_code(x.dtype, x.device) == _lib.BF16 else (4, 4096)
    if not least <= D <= most:
        raise ValueError(f"residual_norm takes a dim of {least} to {most} for {x.dtype} on the GPU, got {D}")
    scale = ctypes.c_float(scale).value  # as the kernels have it: whether it is 1 is asked on both sides
    if grad and torch.is_grad_enabled() or forward_ad._current_level >= 0:  # (which refuses a tangent)
        return _ResidualNorm.apply(x, y, gamma, post_gamma, gate, scale, float(eps))
    operands = [None if t is None else _contig(t) for t in (x, y, gamma, post_gamma, gate)]
    return _forward(*operands, scale, float(eps), False)[:2]
