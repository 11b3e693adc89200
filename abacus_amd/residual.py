"""The residual stream between two blocks of the decoder: a block's output added to it, and the next block's norm.

``residual_norm`` takes the two steps of transformer_block.py:98-100 and norm.py:26-31, x + f and RMSNorm, in one pass
each way (csrc/residual_norm.hip), with a norm of the block's output, a gate and a residual scale where a model has
them.  CPU tensors take the same steps in torch's operations.
"""

from __future__ import annotations

import torch

from . import _lib
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


def _forward(x, y, gamma, post_gamma, gate, scale: float, eps: float, keep: bool):
    """(r, h, rstd, y_rstd) of contiguous tensors; the last two None where they are not kept."""
    D, dev = x.shape[-1], x.device
    rows = x.numel() // D
    r, h = torch.empty_like(x), torch.empty_like(x)
    rstd = torch.empty(rows, dtype=torch.float32, device=dev) if keep else None
    y_rstd = torch.empty(rows, dtype=torch.float32, device=dev) if keep and post_gamma is not None else None
    _lib.call("abacus_residual_norm_fwd", _lib.ptr(x), _lib.ptr(y), _lib.ptr(gamma), _lib.ptr(post_gamma), _lib.ptr(gate),
              _gate_kind(gate), rows, D, scale, eps, _lib.dtype_code(x.dtype), _lib.ptr(r), _lib.ptr(h), _lib.ptr(rstd),
              _lib.ptr(y_rstd), _lib.stream_of(dev))
    return r, h, rstd, y_rstd


class _ResidualNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, y, gamma, post_gamma, gate, scale: float, eps: float):
        c = [None if t is None else _contig(t) for t in (x, y, gamma, post_gamma, gate)]
        r, h, rstd, y_rstd = _forward(*c, scale, eps, True)
        ctx.save_for_backward(x, y, gamma, post_gamma, gate, r, rstd, y_rstd)
        ctx.scale, ctx.eps = scale, eps
        ctx.set_materialize_grads(False)
        return r, h

    @staticmethod
    def backward(ctx, dr, dh):
        from .transformer import _KernelGradient

        if dr is None and dh is None:
            return (None,) * 7
        x, y, gamma, post_gamma, gate, r, rstd, y_rstd = ctx.saved_tensors
        with torch.no_grad():
            grads = _ResidualNorm.gradients(ctx, dr, dh, y, gamma, post_gamma, gate, r, rstd, y_rstd)
        if torch.is_grad_enabled():
            there = [t is not None for t in (post_gamma, gate)]

            def op(x, y, gamma, *rest):  # r and h side by side: one output
                rest = list(rest)
                post, gt = (rest.pop(0) if t else None for t in there)
                branch = y if post is None else _norm(y, post, ctx.eps)
                r = x + ctx.scale * (branch if gt is None else gt * branch)
                return torch.stack((r, _norm(r, gamma, ctx.eps)))

            leaves = [t for t in (x, y, gamma, post_gamma, gate) if t is not None]
            d_out = torch.stack([torch.zeros_like(r) if d is None else d for d in (dr, dh)])
            formed = iter(_KernelGradient.apply(op, tuple(g for g in grads if g is not None), d_out, *leaves))
            grads = tuple(None if g is None else next(formed) for g in grads)
        return (*grads, None, None)

    @staticmethod
    def gradients(ctx, dr, dh, y, gamma, post_gamma, gate, r, rstd, y_rstd):
        D, dev = r.shape[-1], r.device
        rows = r.numel() // D
        same = post_gamma is None and gate is None and ctx.scale == 1.0  # dy is dx
        dr, dh, y, gamma, post_gamma, gate = (None if t is None else _contig(t) for t in (dr, dh, y, gamma, post_gamma, gate))
        dx = torch.empty_like(r)
        dy = None if same else torch.empty_like(r)
        dgamma, dpost, dgate = (None if t is None else torch.empty_like(t) for t in (gamma, post_gamma, gate))
        kind = _gate_kind(gate)
        nbytes = _lib.query("abacus_residual_norm_bwd_ws_bytes", rows, D, int(post_gamma is not None), kind)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
        _lib.call("abacus_residual_norm_bwd", _lib.ptr(dr), _lib.ptr(dh), _lib.ptr(r), _lib.ptr(y), _lib.ptr(gamma),
                  _lib.ptr(post_gamma), _lib.ptr(gate), kind, _lib.ptr(rstd), _lib.ptr(y_rstd), rows, D, ctx.scale,
                  _lib.dtype_code(r.dtype), _lib.ptr(dx), _lib.ptr(dy), _lib.ptr(dgamma), _lib.ptr(dpost), _lib.ptr(dgate),
                  _lib.ptr(ws), nbytes, _lib.stream_of(dev))
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
    tensors = [t for t in (y, gamma, post_gamma, gate) if t is not None]
    if any(t.dtype != x.dtype for t in tensors):
        raise TypeError(f"residual_norm takes tensors of one type, got {x.dtype} and {', '.join(str(t.dtype) for t in tensors)}")
    if any(t.device != x.device for t in tensors):
        raise ValueError("residual_norm takes tensors on one device")
    if x.device.type == "cpu" or x.numel() == 0:
        return _plain(x, y, gamma, post_gamma, gate, scale, eps)
    least, most = (8, 8192) if _lib.dtype_code(x.dtype, x.device) == _lib.BF16 else (4, 4096)
    if not least <= D <= most:
        raise ValueError(f"residual_norm takes a dim of {least} to {most} for {x.dtype} on the GPU, got {D}")
    if torch.is_grad_enabled() and any(t.requires_grad for t in (x, *tensors)):
        return _ResidualNorm.apply(x, y, gamma, post_gamma, gate, float(scale), float(eps))
    operands = [None if t is None else _contig(t) for t in (x, y, gamma, post_gamma, gate)]
    return _forward(*operands, float(scale), float(eps), False)[:2]
