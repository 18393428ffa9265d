"""Activations kept in 8 bits between the forward and the backward, and the operators that use them.

Training memory between a forward and its backward is mostly activations that the backward reads
once.  Held in 8 bits they take 1.03 bytes a value instead of 2 (bf16) or 4 (fp32); only what is
*kept* is approximate, the forward computes with the exact tensors:

* :func:`keep8` / :func:`restore8` store and reload any activation (block checkpoints);
* :func:`kept8_linear` is ``x W^T + b`` whose weight gradient reads the kept input;
* :func:`kept8_swiglu` is ``silu(gate) * value`` whose backward reads both kept inputs;
* :func:`kept8_swiglu_ffn` is the SwiGLU MLP ``w2(silu(w1 x) * (w3 x))`` that keeps ``x``, gate and value
  only, and recomputes the product for the weight gradient of ``w2``;
* :func:`pan2_b200.ops.norm.layer_norm` / ``rms_norm`` take ``kept8=True``.

Format: every row is cut into blocks of 32 consecutive channels; a block has one power-of-two step
``2^s``, ``s = clamp(floor(log2(max |x|)) - 6, -126, 121)``, and 32 codes
``clamp(round_half_even(x / 2^s), -127, 127)`` (the OCP microscaling MXINT8 layout).  A value
``code * 2^s`` is exact in bf16, so the reload adds no rounding of its own; the error is at most half a step, i.e.
``2^-7`` of the block's largest value (twice that for an fp32 value that clamps).  Blocks with an
infinity or a NaN read back as NaN, so a non-finite activation still reaches the gradients.

Gradients are those of the formulas evaluated at the kept values; the store itself is treated as the
identity (no gradient flows through the rounding).  There are no second derivatives: a backward with
``create_graph=True`` raises, since codes and statistics carry no graph.  CUDA tensors run the sm_100a kernels of
``csrc/kept8_ops.cu`` and ``csrc/gemm_sm100.cu``; CPU tensors run plain PyTorch with the same math.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from ._ext import ext
from .gemm import mm_nn, mm_nt

BLOCK = 32


class Kept8:
    """An activation held in 8 bits: ``codes`` int8 ``[rows, C rounded up to 32]``, ``scales`` uint8
    ``[rows, blocks rounded up to 4]`` (exponent byte of each block), and the ``shape`` / ``dtype`` it
    came from."""

    __slots__ = ("codes", "scales", "shape", "dtype")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, shape, dtype: torch.dtype):
        self.codes, self.scales, self.shape, self.dtype = codes, scales, torch.Size(shape), dtype

    @property
    def nbytes(self) -> int:
        return self.codes.numel() + self.scales.numel()

    def __repr__(self) -> str:
        return f"Kept8({tuple(self.shape)}, {self.dtype}, {self.nbytes} bytes)"


# --------------------------------------------------------------------------------------------
# checks and the CPU restatement of the format
# --------------------------------------------------------------------------------------------

def check_activation(x: torch.Tensor, name: str) -> None:
    """Raise unless ``x`` is an activation the operators of this module take."""
    if not isinstance(x, torch.Tensor):
        raise TypeError(f"{name} must be a tensor, got {type(x).__name__}")
    if x.is_cuda:
        if x.dtype not in (torch.bfloat16, torch.float32):
            raise TypeError(f"{name} must be bf16 or fp32 on CUDA, got {x.dtype}")
    elif not x.is_floating_point():
        raise TypeError(f"{name} must be a floating tensor, got {x.dtype}")
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"{name} needs a last dimension of at least 1, got shape {tuple(x.shape)}")


def _check_match(a: torch.Tensor, b: torch.Tensor, names: str) -> None:
    if a.shape != b.shape or a.dtype != b.dtype or a.device != b.device:
        raise ValueError(f"{names} differ: {tuple(a.shape)} {a.dtype} {a.device} and "
                         f"{tuple(b.shape)} {b.dtype} {b.device}")


def refuse_create_graph(name: str) -> None:
    """Raise in a backward that is itself to be differentiated (what it reads carries no graph)."""
    if torch.is_grad_enabled():
        raise RuntimeError(f"{name} has no second derivative: run its backward without create_graph")


def wide_dtype(dtype: torch.dtype) -> torch.dtype:
    """The dtype CPU paths compute in: fp32, or fp64 for fp64 inputs."""
    return torch.float64 if dtype == torch.float64 else torch.float32


def _keep_cpu(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    C = x.shape[-1]
    rows = x.numel() // C
    v = torch.nn.functional.pad(x.detach().reshape(rows, C).to(wide_dtype(x.dtype)), (0, -C % BLOCK))
    v = v.view(rows, v.shape[1] // BLOCK, BLOCK)
    top = v.abs().amax(-1)
    finite = torch.isfinite(top)
    # frexp: top = m * 2^e with m in [1/2, 1), so floor(log2(top)) = e - 1; of 0 it gives e = 0
    byte = (torch.frexp(torch.where(finite, top, torch.ones_like(top)))[1] + 126).clamp(7, 254)
    byte = torch.where(top == 0, torch.full_like(byte, 7), byte)
    step = torch.ldexp(torch.ones_like(top), byte - 133)
    codes = torch.round(v / step.unsqueeze(-1)).clamp(-127, 127)
    codes = torch.where(finite.unsqueeze(-1), codes, torch.zeros_like(codes)).to(torch.int8).flatten(1)
    byte = torch.where(finite, byte, torch.full_like(byte, 255)).to(torch.uint8)
    return codes, torch.nn.functional.pad(byte, (0, -byte.shape[1] % 4), value=127)


def _values_cpu(codes: torch.Tensor, scales: torch.Tensor, C: int, dtype: torch.dtype) -> torch.Tensor:
    """``[rows, C]`` values of the codes in ``dtype``."""
    rows, nb = codes.shape[0], codes.shape[1] // BLOCK
    byte = scales[:, :nb].to(torch.int32)
    step = torch.ldexp(torch.ones(byte.shape, dtype=wide_dtype(dtype)), byte - 133)
    step = torch.where(byte == 255, torch.full_like(step, float("nan")), step)
    v = codes.view(rows, nb, BLOCK).to(step.dtype) * step.unsqueeze(-1)
    return v.flatten(1)[:, :C].to(dtype)


def keep_codes(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """``(codes, scales)`` of the rows of ``x``."""
    return ext().keep8(x) if x.is_cuda else _keep_cpu(x)


# --------------------------------------------------------------------------------------------
# store and reload
# --------------------------------------------------------------------------------------------

def keep8(x: torch.Tensor) -> Kept8:
    """``x`` (any leading dims and strides) held in 8 bits.  Not differentiable."""
    if not getattr(x, "is_cuda", False):  # the binding makes the same checks
        check_activation(x, "x")
    return Kept8(*keep_codes(x), x.shape, x.dtype)


def restore8(kept: Kept8, dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """The values of ``kept`` as a contiguous tensor of its shape, in its dtype (or ``dtype``)."""
    if not isinstance(kept, Kept8):
        raise TypeError(f"restore8 takes what keep8 returned, got {type(kept).__name__}")
    dtype = kept.dtype if dtype is None else dtype
    if kept.codes.is_cuda:
        if dtype not in (torch.bfloat16, torch.float32):
            raise TypeError(f"restore8 gives bf16 or fp32 on CUDA, not {dtype}")
        return ext().restore8_new(kept.codes, kept.scales, kept.shape, dtype == torch.float32)
    return _values_cpu(kept.codes, kept.scales, kept.shape[-1], dtype).view(kept.shape)


# --------------------------------------------------------------------------------------------
# linear
# --------------------------------------------------------------------------------------------

def weight_grad8(g: torch.Tensor, codes: torch.Tensor, scales: torch.Tensor, K: int, dtype) -> torch.Tensor:
    """``g^T x`` in ``dtype``, ``x [rows, K]`` the kept matrix and ``g [rows, N]``: the weight gradient of a
    projection that read ``x``."""
    if codes.is_cuda:
        return ext().linear8_weight_grad(g, codes, scales, K, dtype != torch.bfloat16).to(dtype)
    x = _values_cpu(codes, scales, K, wide_dtype(g.dtype))
    return (g.to(x.dtype).t() @ x).to(dtype)


def row_sum(g: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    """``g [rows, N]`` summed over its rows in fp32, in a fixed order (bias gradients)."""
    if g.is_cuda:
        return ext().row_sum(g, dtype == torch.float32).to(dtype)
    return g.to(wide_dtype(g.dtype)).sum(0).to(dtype)


def _project(x2: torch.Tensor, w: torch.Tensor) -> torch.Tensor:
    """``x2 [rows, K] @ w^T`` (no autograd)."""
    if not x2.is_cuda:
        return _project_cpu(x2, w, None)
    if x2.shape[0] == 0:
        return x2.new_empty(0, w.shape[0])
    return mm_nt(ext().gemm_operand(x2, False), ext().gemm_operand(w, True))[:, :w.shape[0]]


def _project_cpu(x2: torch.Tensor, w: torch.Tensor, b: Optional[torch.Tensor]) -> torch.Tensor:
    wide = wide_dtype(x2.dtype)
    y = x2.to(wide) @ w.to(wide).t()
    return (y if b is None else y + b.to(wide)).to(x2.dtype)


def _input_grad(*pairs: Tuple[torch.Tensor, torch.Tensor]) -> torch.Tensor:
    """Sum of ``g2 [rows, N] @ w [N, K]`` over the pairs.  On CUDA the sum so far is bf16 between the products (one
    rounding more than an fp32 sum, at half its traffic); the next one is added to it in fp32."""
    out = None
    for g2, w in pairs:
        if not g2.is_cuda:
            wide = wide_dtype(g2.dtype)
            y = (g2.to(wide) @ w.to(wide)).to(g2.dtype)
            out = y if out is None else out + y
        elif g2.shape[0] == 0:
            out = g2.new_empty(0, w.shape[1])
        else:
            out = mm_nn(ext().gemm_operand(g2, False), ext().gemm_operand(w, True), out=out, accumulate=out is not None)
    return out[:, :pairs[0][1].shape[1]]


def _check_linear(x: torch.Tensor, w: torch.Tensor, b: Optional[torch.Tensor]) -> None:
    check_activation(x, "x")
    if w.dim() != 2 or w.shape[1] != x.shape[-1] or w.shape[0] < 1:
        raise ValueError(f"weight {tuple(w.shape)} does not fit an input of width {x.shape[-1]}")
    if b is not None and (b.dim() != 1 or b.shape[0] != w.shape[0]):
        raise ValueError(f"bias {tuple(b.shape)} does not fit a weight {tuple(w.shape)}")
    for name, t in (("weight", w), ("bias", b)):
        if t is not None and t.device != x.device:
            raise ValueError(f"{name} is on {t.device}, the input on {x.device}")


class _Kept8LinearCPU(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, b):
        x2 = x.reshape(-1, x.shape[-1])
        y = _project_cpu(x2, w, b)
        codes, scales = _keep_cpu(x2) if ctx.needs_input_grad[1] else (None, None)
        ctx.save_for_backward(codes, scales, w)
        ctx.shape, ctx.b_dtype = x.shape, None if b is None else b.dtype
        return y.reshape(*x.shape[:-1], w.shape[0])

    @staticmethod
    def backward(ctx, gy):
        refuse_create_graph("kept8_linear")
        codes, scales, w = ctx.saved_tensors
        g2 = gy.reshape(-1, gy.shape[-1])
        gx = _input_grad((g2, w)).reshape(ctx.shape) if ctx.needs_input_grad[0] else None
        gw = weight_grad8(g2, codes, scales, w.shape[1], w.dtype) if ctx.needs_input_grad[1] else None
        gb = row_sum(g2, ctx.b_dtype) if ctx.b_dtype is not None and ctx.needs_input_grad[2] else None
        return gx, gw, gb


def kept8_linear(x: torch.Tensor, w: torch.Tensor, b: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``x @ w^T + b`` that keeps ``x`` in 8 bits for the weight gradient ``dy^T x``.

    CUDA inputs compute in bf16 with fp32 accumulation, like :func:`pan2_b200.ops.gemm.linear`; any
    widths work (those that are not multiples of 8 are padded)."""
    if getattr(x, "is_cuda", False):  # the binding makes the same checks
        return ext().linear8(x, w, b)
    _check_linear(x, w, b)
    return _Kept8LinearCPU.apply(x, w, b)


# --------------------------------------------------------------------------------------------
# SwiGLU
# --------------------------------------------------------------------------------------------

def _swiglu_forward(gate, value):
    """``(h, codes and scales of gate, of value)``."""
    if gate.is_cuda:
        return ext().swiglu8_fwd(gate, value, True)
    wide = wide_dtype(gate.dtype)
    g = gate.to(wide)
    h = (g * torch.sigmoid(g) * value.to(wide)).to(gate.dtype)
    return [h, *_keep_cpu(gate), *_keep_cpu(value)]


def _swiglu_backward(dh, kept, want_h: bool):
    """``[dgate, dvalue(, h)]`` from the kept codes."""
    if dh.is_cuda:
        return ext().swiglu8_bwd(dh, *kept, want_h)
    wide, C = wide_dtype(dh.dtype), dh.shape[-1]
    g = _values_cpu(kept[0], kept[1], C, wide).view(dh.shape)
    v = _values_cpu(kept[2], kept[3], C, wide).view(dh.shape)
    d, s = dh.to(wide), torch.sigmoid(g)
    out = [d * v * s * (1 + g * (1 - s)), d * g * s] + ([g * s * v] if want_h else [])
    return [t.to(dh.dtype) for t in out]


class _Kept8SwiGLUCPU(torch.autograd.Function):
    @staticmethod
    def forward(ctx, gate, value):
        h, *kept = _swiglu_forward(gate, value)
        ctx.save_for_backward(*kept)
        return h

    @staticmethod
    def backward(ctx, dh):
        refuse_create_graph("kept8_swiglu")
        return tuple(_swiglu_backward(dh, ctx.saved_tensors, False))


def kept8_swiglu(gate: torch.Tensor, value: torch.Tensor) -> torch.Tensor:
    """``silu(gate) * value``, computed in fp32 and rounded once, whose backward reads ``gate`` and
    ``value`` from 8 bits."""
    if getattr(gate, "is_cuda", False) and getattr(value, "is_cuda", False):  # the binding makes the same checks
        return ext().swiglu8(gate, value)
    check_activation(gate, "gate")
    check_activation(value, "value")
    _check_match(gate, value, "gate and value")
    return _Kept8SwiGLUCPU.apply(gate, value)


class _Kept8SwiGLUFFN(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w1, w3, w2):
        K = x.shape[-1]
        x2 = x.reshape(-1, K)
        h, *kept = _swiglu_forward(_project(x2, w1), _project(x2, w3))
        ctx.save_for_backward(*keep_codes(x2), *kept, w1, w3, w2)
        ctx.shape = x.shape
        return _project(h, w2).reshape(*x.shape[:-1], w2.shape[0])

    @staticmethod
    def backward(ctx, gy):
        refuse_create_graph("kept8_swiglu_ffn")
        codes, scales, *kept, w1, w3, w2 = ctx.saved_tensors
        need_x, need_1, need_3, need_2 = ctx.needs_input_grad
        g2 = gy.reshape(-1, gy.shape[-1])
        dgate, dvalue, *h = _swiglu_backward(_input_grad((g2, w2)).contiguous(), kept, need_2)
        gx = gw1 = gw3 = gw2 = None
        if need_2:
            gw2 = _dense_weight_grad(g2, h[0], w2.dtype)
        if need_x:
            gx = _input_grad((dgate, w1), (dvalue, w3)).reshape(ctx.shape)
        if need_1:
            gw1 = weight_grad8(dgate, codes, scales, w1.shape[1], w1.dtype)
        if need_3:
            gw3 = weight_grad8(dvalue, codes, scales, w3.shape[1], w3.dtype)
        return gx, gw1, gw3, gw2


def _dense_weight_grad(g2: torch.Tensor, h: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    if g2.is_cuda:
        return ext().weight_grad(g2, h, dtype != torch.bfloat16).to(dtype)
    wide = wide_dtype(g2.dtype)
    return (g2.to(wide).t() @ h.to(wide)).to(dtype)


def kept8_swiglu_ffn(x: torch.Tensor, w1: torch.Tensor, w3: torch.Tensor, w2: torch.Tensor) -> torch.Tensor:
    """Bias-free SwiGLU MLP ``w2(silu(w1 x) * (w3 x))`` that keeps ``x``, ``w1 x`` and ``w3 x`` in 8 bits
    (their product is recomputed in the backward).  CUDA inputs compute in bf16."""
    for w in (w1, w3):
        _check_linear(x, w, None)
    if w1.shape != w3.shape:
        raise ValueError(f"gate and value weights differ: {tuple(w1.shape)} and {tuple(w3.shape)}")
    if w2.dim() != 2 or w2.shape[1] != w1.shape[0] or w2.device != x.device:
        raise ValueError(f"output weight {tuple(w2.shape)} on {w2.device} does not fit a hidden width of {w1.shape[0]}")
    if x.is_cuda:
        x = x.to(torch.bfloat16)
    if not (torch.is_grad_enabled() and any(t.requires_grad for t in (x, w1, w3, w2))):  # nothing to keep
        x2 = x.reshape(-1, x.shape[-1])
        h = kept8_swiglu(_project(x2, w1), _project(x2, w3))
        return _project(h, w2).reshape(*x.shape[:-1], w2.shape[0])
    return _Kept8SwiGLUFFN.apply(x, w1, w3, w2)
