"""Layer norm and RMS norm with learned weight and bias, as one autograd op each.

``n = (x - mean) * rstd``, ``y = n * w + b`` (RMS norm: no mean, no bias), computed in fp32 and rounded
once to ``x``'s dtype.  This is not the model's eager ``models.layers.rms_norm``, which also
rounds ``n`` before the weight multiplies it.

The backward returns ``dx`` and the fully reduced ``dw`` / ``db`` (fp32 sums in a fixed order: the same
bits every time).  With ``kept8=True`` the input is kept in 8 bits (:mod:`pan2_b200.ops.kept8`) and the
backward reads ``n`` from those, with the exact input's ``mean`` and ``rstd``.  There are no second
derivatives: a backward with ``create_graph=True`` raises.

CUDA tensors (bf16 or fp32; any width, any leading dims, strided rows without a copy) run the
sm_100a kernels of ``csrc/norm_ops.cu``; CPU tensors run plain PyTorch with the same math.
"""
from __future__ import annotations

from typing import Optional

import torch

from ._ext import ext
from .kept8 import _keep_cpu, _values_cpu, check_activation, refuse_create_graph, wide_dtype


class _NormCPU(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, b, eps, layer, kept8):
        y, stats = _forward_cpu(x, w, b, eps, layer)
        codes, scales = _keep_cpu(x) if kept8 else (None, None)
        ctx.save_for_backward(None if kept8 else x, codes, scales, stats, w)
        ctx.layer = layer
        ctx.w_dtype = w.dtype if w is not None else b.dtype if b is not None else x.dtype
        return y

    @staticmethod
    def backward(ctx, dy):
        refuse_create_graph("layer_norm" if ctx.layer else "rms_norm")
        x, codes, scales, stats, w = ctx.saved_tensors
        grads = _backward_cpu(dy, x, codes, scales, stats, w, ctx.layer, ctx.w_dtype)
        return *(g if need else None for g, need in zip(grads, ctx.needs_input_grad)), None, None, None


def _forward_cpu(x, w, b, eps, layer):
    v = x.detach().to(wide_dtype(x.dtype))
    mean = v.mean(-1, keepdim=True) if layer else v.new_zeros(*v.shape[:-1], 1)
    rstd = torch.rsqrt((v - mean).square().mean(-1, keepdim=True) + eps)
    y = (v - mean) * rstd
    if w is not None:
        y = y * w.to(y.dtype)
    if b is not None:
        y = y + b.to(y.dtype)
    return y.to(x.dtype), torch.cat([mean, rstd], -1)


def _backward_cpu(dy, x, codes, scales, stats, w, layer, w_dtype):
    d = dy.to(wide_dtype(dy.dtype))
    v = x.to(d.dtype) if codes is None else _values_cpu(codes, scales, dy.shape[-1], d.dtype).view(dy.shape)
    mean, rstd = stats[..., :1], stats[..., 1:]
    n = (v - mean) * rstd
    g = d if w is None else d * w.to(d.dtype)
    dx = g - n * (g * n).mean(-1, keepdim=True)
    if layer:
        dx = dx - g.mean(-1, keepdim=True)
    rows = tuple(range(dy.dim() - 1))
    total = (lambda t: t.sum(rows) if rows else t)
    return (dx * rstd).to(dy.dtype), total(d * n).to(w_dtype), total(d).to(w_dtype)


def _check(x, w, b, eps):
    check_activation(x, "x")
    for name, t in (("weight", w), ("bias", b)):
        if t is None:
            continue
        if t.dim() != 1 or t.shape[0] != x.shape[-1]:
            raise ValueError(f"{name} {tuple(t.shape)} does not fit rows of width {x.shape[-1]}")
        if t.device != x.device:
            raise ValueError(f"{name} is on {t.device}, x on {x.device}")
    if w is not None and b is not None and w.dtype != b.dtype:
        raise TypeError(f"weight and bias have different dtypes: {w.dtype} and {b.dtype}")
    if not eps >= 0:
        raise ValueError(f"eps={eps} is negative")


def _norm(x, w, b, eps, layer, kept8):
    if getattr(x, "is_cuda", False):  # the binding makes the same checks
        return ext().norm(x, w, b, eps, layer, kept8)
    _check(x, w, b, eps)
    return _NormCPU.apply(x, w, b, float(eps), layer, bool(kept8))


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
               eps: float = 1e-6, kept8: bool = False) -> torch.Tensor:
    """``(x - mean) * rsqrt(var + eps) * weight + bias`` over the last dim (biased variance)."""
    return _norm(x, weight, bias, eps, True, kept8)


def rms_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, eps: float = 1e-6,
             kept8: bool = False) -> torch.Tensor:
    """``x * rsqrt(mean(x^2) + eps) * weight`` over the last dim."""
    return _norm(x, weight, None, eps, False, kept8)
