"""The root-mean-square norm of a block's residual stream, on the library.

``model/transformer.py:14-24`` norms in float32 and casts to the compute dtype; the block
adds what it computed to its input first (``:82-95``).  :class:`RMSNorm` does both in one
launch (``hmoe_add_rms_norm``) and is differentiable (``hmoe_add_rms_norm_bwd``).
"""
from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from . import kernels as K
from .moe import Param, _aligned, _refuse_tangents


class RMSNorm:
    """``y = total * rsqrt(mean(total^2) + eps) * scale`` of ``total = x + residual`` over the
    last dimension.  ``scale`` is a float32 :class:`hanuman_amd.moe.Param` of ones."""

    def __init__(self, d_model: int, eps: float = 1e-6, *, device: str | torch.device | None = None):
        dev = torch.device(device) if device is not None else torch.device("cuda")
        self.eps = eps
        self.scale = Param(torch.ones(d_model, dtype=torch.float32, device=dev))

    def rows(self, x: torch.Tensor, residual: torch.Tensor | None = None, *, out_dtype=None,
             quant: str | None = None) -> K.NormOut:
        """:func:`hanuman_amd.kernels.add_rms_norm` of all leading dimensions as rows, outside
        autograd."""
        return _rows(x.detach(), None if residual is None else residual.detach(), self.scale.value.detach(), self.eps,
                     out_dtype, quant)

    def with_sum(self, x: torch.Tensor, residual: torch.Tensor | None = None, *, out_dtype=None):
        """``(y, total)`` in ``x``'s shape; ``total`` is ``x`` without a residual.

        A graph that captures gradients takes them with ``torch.autograd.grad``, or while no
        autograd graph of the same leaves from before the capture is alive: autograd adds into a
        leaf's ``.grad`` on the stream of the first of them, which may not be captured.
        Second and forward-mode derivatives are refused."""
        w = self.scale.value
        _refuse_tangents("RMSNorm", x, residual, w)
        if residual is not None and residual.shape != x.shape:
            raise ValueError(f"residual must have x's shape {tuple(x.shape)} (got {tuple(residual.shape)})")
        tracked = x.requires_grad or w.requires_grad or (residual is not None and residual.requires_grad)
        if torch.is_grad_enabled() and tracked:
            if residual is None:
                return _AddRmsNorm.apply(self.eps, out_dtype, x, w, None), x
            return _AddRmsNorm.apply(self.eps, out_dtype, x, w, residual)
        r = self.rows(x, residual, out_dtype=out_dtype)
        return r.y.view(x.shape), x if residual is None else r.sum.view(x.shape)

    def __call__(self, x: torch.Tensor, *, out_dtype=None) -> torch.Tensor:
        """``norm(x)`` in ``out_dtype`` (``x``'s by default)."""
        return self.with_sum(x, None, out_dtype=out_dtype)[0]


def _rows(x, residual, w, eps, out_dtype, quant=None) -> K.NormOut:
    D = x.shape[-1]
    if residual is not None:
        if residual.shape != x.shape:
            raise ValueError(f"residual must have x's shape {tuple(x.shape)} (got {tuple(residual.shape)})")
        residual = _aligned(residual.reshape(-1, D).contiguous())
    return K.add_rms_norm(_aligned(x.reshape(-1, D).contiguous()), _aligned(w.contiguous()), residual, eps,
                          out_dtype=out_dtype, quant=quant)


class _AddRmsNorm(torch.autograd.Function):
    """``(y, total)``, or ``y`` alone without a residual."""

    @staticmethod
    def forward(ctx, eps, out_dtype, x, w, residual):
        r = _rows(x, residual, w, eps, out_dtype)
        ctx.set_materialize_grads(False)
        ctx.types = x.dtype, None if residual is None else residual.dtype, w.dtype
        y = r.y.view(x.shape)
        if residual is None:
            ctx.save_for_backward(x, w, r.rstd)
            return y
        total = r.sum.view(x.shape)
        ctx.save_for_backward(total, w, r.rstd)
        return y, total

    @staticmethod
    @once_differentiable
    def backward(ctx, d_y, d_total=None):
        total, w, rstd = ctx.saved_tensors
        x_type, r_type, w_type = ctx.types
        need_x, need_w, need_r = ctx.needs_input_grad[2:]
        shape, D = total.shape, total.shape[-1]
        if d_y is None:
            dx, dw = d_total, None
        else:
            d_sum = None
            if d_total is not None:
                d_sum = _aligned(d_total.to(total.dtype).reshape(-1, D).contiguous())
            dx, dw = K.add_rms_norm_bwd(_aligned(d_y.reshape(-1, D).contiguous()),
                                        _aligned(total.reshape(-1, D).contiguous()), _aligned(w.contiguous()), rstd,
                                        d_sum, need_weight=need_w)
            dx = dx.view(shape)
        return (None, None, dx.to(x_type) if need_x and dx is not None else None,
                dw.to(w_type) if need_w and dw is not None else None,
                dx.to(r_type) if need_r and dx is not None else None)
