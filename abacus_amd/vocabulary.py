"""The decoder's two ends over the vocabulary: the embedding of tokens, and the loss of the head's product.

``embedding`` is embedding.py's indexing with a scale; its gradient adds the rows of each token in fp32, by tokens
sorted by id (csrc/embedding.hip).

``linear_cross_entropy`` is the cross-entropy of ``x @ w`` without its logits in memory: they stay in the registers they are
formed in, and with gradients the probabilities are in memory a piece of the rows at a time, from which the products of both
operands' gradients are taken (csrc/linear_cross_entropy.hip).  The reference takes the
two steps one after the other (transformer_moe.py:75, kernels/liger.py:12-47).

CPU tensors take the same steps in torch's operations.
"""

from __future__ import annotations

import ctypes

import torch
import torch.nn.functional as F
from torch.autograd import forward_ad

from . import _lib
from .kv_cache import _call
from .moe import _contig

__all__ = ["embedding", "linear_cross_entropy"]

_REDUCTIONS = {"none": 0, "sum": 1, "mean": 2}  # ABACUS_LOSS_ROWS, _SUM, _MEAN


def _plain_loss(x_TD, w_DV, targets_T, ignore_index: int, reduction: str):
    """The loss in torch's operations, fp32 (fp64 for fp64 operands)."""
    wide = torch.promote_types(x_TD.dtype, torch.float32)
    return F.cross_entropy(x_TD.to(wide) @ w_DV.to(wide), targets_T, ignore_index=ignore_index, reduction=reduction)


def _loss_op(x_TD, w_DV, targets_T, ignore_index: int, reduction: str):
    """What the kernels' gradients are the gradients of, for second derivatives: ignored rows are left out before the product,
    whatever they hold, and a target outside the vocabulary (whose loss is NaN) is none."""
    kept = targets_T != ignore_index
    known = kept & (targets_T >= 0) & (targets_T < w_DV.shape[1])
    logits = torch.where(kept[:, None], x_TD, 0.0) @ w_DV
    picked = logits.gather(1, torch.where(known, targets_T, 0)[:, None])[:, 0]
    rows = torch.where(kept, torch.logsumexp(logits, -1) - torch.where(known, picked, 0.0), 0.0)
    return rows if reduction == "none" else rows.sum() / (kept.sum().clamp(min=1) if reduction == "mean" else 1)


def _loss_call(x_TD, w_DV, targets_T, ignore_index: int, reduction: str, row_grad=None, want=(False, False), want_loss=True):
    """(loss or None, dx or None, dw or None) of one call of the kernels, of operands of any strides."""
    T, D = x_TD.shape
    if x_TD.stride(1) != 1 or x_TD.stride(0) < D:
        x_TD = x_TD.contiguous()
    targets_T = targets_T.contiguous()
    V = w_DV.shape[1]
    dev, dt = x_TD.device, _lib.dtype_code(x_TD.dtype, x_TD.device)
    loss = torch.empty((T,) if reduction == "none" else (), dtype=torch.float32, device=dev) if want_loss else None
    dx = torch.empty(T, D, dtype=x_TD.dtype, device=dev) if want[0] else None
    dw = torch.empty(D, V, dtype=w_DV.dtype, device=dev) if want[1] else None
    nbytes = _lib.query("abacus_linear_cross_entropy_ws_bytes", T, D, V, dt, int(any(want)))
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    w = _contig(w_DV)
    _call(dev, "abacus_linear_cross_entropy", x_TD.data_ptr(), x_TD.stride(0), _lib.ptr(w), targets_T.data_ptr(), T, D, V,
          ignore_index, dt, _REDUCTIONS[reduction], _lib.ptr(row_grad), _lib.ptr(loss), _lib.ptr(dx), _lib.ptr(dw),
          _lib.ptr(ws), nbytes)
    return loss, dx, dw


def _capture(dev: torch.device) -> int:
    """The number of the graph that dev's current stream records, 0 where it records none."""
    if dev.index == torch._C._cuda_getDevice() and not torch.cuda.is_current_stream_capturing():  # (the current device's)
        return 0
    number = ctypes.c_int64()
    _call(dev, "abacus_capture_id", ctypes.addressof(number))
    return number.value


class _LinearCrossEntropy(torch.autograd.Function):
    """Loss and gradients in one pass over the logits: of a mean or a sum the forward forms both gradients, and the
    backward multiplies them by the loss's own (they are left alone, on the device, where that is 1).  In between they are
    saved tensors, which hooks may move and checkpointing drops.  The losses of rows
    have gradients a row that only the backward knows, so it makes the pass once more; so does a second
    backward of a mean or a sum, and one that is not recorded into the graph its forward is in (each of the two may be
    replayed without the other)."""

    @staticmethod
    def forward(ctx, x_TD, w_DV, targets_T, ignore_index: int, reduction: str):
        ctx.args = ignore_index, reduction
        now = ctx.needs_input_grad[:2] if reduction != "none" else (False, False)
        ctx.capture = _capture(x_TD.device)
        loss, *grads = _loss_call(x_TD, w_DV, targets_T, ignore_index, reduction, want=now)
        ctx.formed = any(now)
        ctx.save_for_backward(x_TD, w_DV, targets_T, *grads)
        return loss

    @staticmethod
    def backward(ctx, g):
        x, w, targets, *grads = ctx.saved_tensors
        if not torch.is_grad_enabled():
            return (*_LinearCrossEntropy.gradients(ctx, g, x, w, targets, grads), None, None, None)
        from .transformer import _by_kernel

        op = lambda x, w: _loss_op(x, w, targets, *ctx.args)
        wanted = lambda: tuple(torch.zeros_like(t) if d is None else d
                               for t, d in zip((x, w), _LinearCrossEntropy.gradients(ctx, g, x, w, targets, grads)))
        return (*_by_kernel(op, wanted, g, x, w), None, None, None)

    @staticmethod
    def gradients(ctx, g, x, w, targets, grads):
        ignore_index, reduction = ctx.args
        g = g.contiguous()
        if reduction == "none":
            return _loss_call(x, w, targets, ignore_index, reduction, g, ctx.needs_input_grad[:2], want_loss=False)[1:]
        formed, ctx.formed = ctx.formed, False
        if not formed or ctx.capture != _capture(x.device):  # handed over by an earlier backward, or another's to write
            grads = _loss_call(x, w, targets, ignore_index, reduction, want=ctx.needs_input_grad[:2])[1:]
        else:  # (what becomes of them is the caller's: versions of their own, so that a retained graph does not mind)
            grads = [None if d is None else _contig(d.data) for d in grads]
        sizes = [0 if t is None else t.numel() for t in grads]
        _call(x.device, "abacus_scale_by", _lib.ptr(grads[0]), sizes[0], _lib.ptr(grads[1]), sizes[1], _lib.dtype_code(x.dtype),
              g.data_ptr())
        return tuple(grads)


def linear_cross_entropy(x: torch.Tensor, w_DV: torch.Tensor, targets: torch.Tensor, ignore_index: int = -100,
                         reduction: str = "mean") -> torch.Tensor:
    """cross_entropy(x @ w_DV, targets) without the logits in memory: x (..., D), w_DV (D, V), targets (...) int64.

    The loss is fp32, the mean over (or the sum of) the rows whose target is not ignore_index, or each row's loss
    ("none", 0 where ignored).  A mean of no rows is NaN and its gradients are 0.  A target outside [0, V) other than
    ignore_index makes its row's loss NaN, as train.cross_entropy on the GPU has it (on the CPU torch raises); nothing
    waits on the host.  Logits and sums are fp32, whatever the operands' type; ignored rows cost no products.

    Where a gradient is recorded, a mean's or sum's forward forms both and the backward hands them over (times the loss's
    own, rounded once more where that is not 1).  The losses of rows have the logits formed again by the backward.  Besides the
    gradients a call holds a copy of x (of all rows: how many are kept is known on the device alone) and, with gradients, the
    probabilities in w's type of one piece of the rows after the other: up to 1 GiB, or 256 rows where those are more.  Where
    the rows take several pieces dw's sums in fp32 (4 D V bytes) come to it, and up to 128 MiB of partial sums where the
    products are small: 2.3 GiB in all for 16384 x 4096 x 65536 in bf16.  A w of other strides than a contiguous one's, or of an
    odd vocabulary for over 64 rows, is copied.
    """
    if reduction not in _REDUCTIONS:
        raise ValueError(f"reduction is one of {', '.join(_REDUCTIONS)}, got {reduction!r}")
    if x.dim() < 1 or w_DV.dim() != 2 or x.shape[-1] != w_DV.shape[0] or 0 in w_DV.shape:
        raise ValueError(f"linear_cross_entropy takes x (..., D) and w (D, V), got {tuple(x.shape)} and {tuple(w_DV.shape)}")
    if targets.shape != x.shape[:-1] or targets.dtype != torch.int64:
        raise ValueError(f"linear_cross_entropy takes int64 targets {tuple(x.shape[:-1])}, got {targets.dtype} "
                         f"{tuple(targets.shape)}")
    if w_DV.dtype != x.dtype:
        raise TypeError(f"x is {x.dtype} and w is {w_DV.dtype}")
    if not x.device == w_DV.device == targets.device:
        raise ValueError(f"x, w and targets are on {x.device}, {w_DV.device} and {targets.device}")
    x_TD, targets_T = x.reshape(-1, x.shape[-1]), targets.reshape(-1)
    if x.device.type == "cpu" or x_TD.shape[0] == 0:
        loss = _plain_loss(x_TD, w_DV, targets_T, ignore_index, reduction)
    else:
        _lib.dtype_code(x.dtype, x.device)  # refuses other types
        # (forward mode too, where torch refuses a tangent that the kernels would drop)
        if torch.is_grad_enabled() and (x.requires_grad or w_DV.requires_grad) or forward_ad._current_level >= 0:
            loss = _LinearCrossEntropy.apply(x_TD, w_DV, targets_T, int(ignore_index), reduction)
        else:
            loss = _loss_call(x_TD, w_DV, targets_T, int(ignore_index), reduction)[0]
    return loss.view(targets.shape) if reduction == "none" else loss


class _Embedding(torch.autograd.Function):
    """scale * w[tokens] and its gradient, the rows of each token added in a fixed order."""

    @staticmethod
    def forward(ctx, tokens, w_VD, scale: float):
        ctx.save_for_backward(tokens)
        ctx.shape, ctx.scale = w_VD.shape, scale
        return _embed_call(tokens, w_VD, scale)

    @staticmethod
    def backward(ctx, d_out):
        (tokens,) = ctx.saved_tensors
        if torch.is_grad_enabled():  # (it is to be differentiated itself)
            return None, _EmbeddingGradient.apply(d_out, tokens, ctx.shape, ctx.scale), None
        return None, _embed_gradient(d_out, tokens, ctx.shape, ctx.scale), None


class _EmbeddingGradient(torch.autograd.Function):
    """The gradient is linear in d_out, and its own derivative the embedding again."""

    @staticmethod
    def forward(ctx, d_out, tokens, shape, scale: float):
        ctx.save_for_backward(tokens)
        ctx.scale = scale
        return _embed_gradient(d_out, tokens, shape, scale)

    @staticmethod
    def backward(ctx, d_dw):
        (tokens,) = ctx.saved_tensors
        return _Embedding.apply(tokens, d_dw, ctx.scale), None, None, None


def _embed_gradient(d_out, tokens, shape, scale: float):
    V, D = shape
    T, dev = tokens.numel(), d_out.device
    dw = torch.empty(V, D, dtype=d_out.dtype, device=dev)
    nbytes = _lib.query("abacus_embedding_bwd_ws_bytes", T, V, D)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    tokens, d_out = tokens.contiguous(), _contig(d_out)
    _call(dev, "abacus_embedding_bwd", tokens.data_ptr(), d_out.data_ptr(), T, V, D, scale, _lib.dtype_code(d_out.dtype),
          dw.data_ptr(), ws.data_ptr(), nbytes)
    return dw


def _embed_call(tokens, w_VD, scale: float):
    V, D = w_VD.shape
    tokens, w = tokens.contiguous(), _contig(w_VD)
    out = torch.empty(*tokens.shape, D, dtype=w.dtype, device=w.device)
    _call(w.device, "abacus_embedding_fwd", tokens.data_ptr(), w.data_ptr(), tokens.numel(), V, D, scale,
          _lib.dtype_code(w.dtype), out.data_ptr())
    return out


def embedding(tokens: torch.Tensor, w_VD: torch.Tensor, scale: float = 1.0) -> torch.Tensor:
    """scale * w_VD[tokens] (embedding.py:20-23): tokens (...) int64, w_VD (V, D), out (..., D).

    Negative tokens count from the end, as in torch's indexing.  A token outside [-V, V) gives a row of NaN and no
    gradient on the GPU (on the CPU torch raises); nothing waits on the host.  The gradient of a row is the sum of its
    tokens' in fp32, times the scale, rounded once, and the same bits every run.

    Text repeats tokens, and the gradient's time hardly depends on how often.  It does on the table: past some 2^18 rows every
    2^18 more have all tokens read once more (csrc/embedding.hip), and indexing, whose time is that of the most frequent token, is
    faster for tokens that are all different.
    """
    if tokens.dtype != torch.int64:
        raise ValueError(f"embedding takes int64 tokens, got {tokens.dtype}")
    if w_VD.dim() != 2 or 0 in w_VD.shape:
        raise ValueError(f"embedding takes a table (V, D), got {tuple(w_VD.shape)}")
    if tokens.device != w_VD.device:
        raise ValueError(f"tokens are on {tokens.device}, the table on {w_VD.device}")
    if w_VD.device.type == "cpu":
        return w_VD[tokens] if scale == 1.0 else w_VD[tokens] * scale
    _lib.dtype_code(w_VD.dtype, w_VD.device)  # refuses other types
    if torch.is_grad_enabled() and w_VD.requires_grad or forward_ad._current_level >= 0:  # (which refuses a tangent)
        return _Embedding.apply(tokens, w_VD, float(scale))
    return _embed_call(tokens, w_VD, float(scale))
