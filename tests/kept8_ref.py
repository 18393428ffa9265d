"""64-bit definitions of the 8-bit format, the norms and SwiGLU for the tests (no framework code)."""
import math

import torch

F32 = 2.0 ** -24  # unit roundoff of fp32
BF16 = 2.0 ** -9  # ... of bf16


def unit(dtype):
    return BF16 if dtype == torch.bfloat16 else F32


def kept_values(x):
    """What ``x`` reads back as, in fp64, one block of 32 at a time."""
    rows = x.detach().cpu().double().reshape(-1, x.shape[-1])
    out = torch.empty_like(rows)
    for a in range(0, rows.shape[1], 32):
        blk = rows[:, a:a + 32]
        top = blk.abs().amax(1)
        bad = ~torch.isfinite(top)
        s = torch.floor(torch.log2(torch.where(bad | (top == 0), torch.ones_like(top), top))) - 6
        # log2 of a number just below a power of two may round up to it
        s = torch.where(2.0 ** (s + 6) > top, s - 1, s)
        s = torch.where(top == 0, torch.zeros_like(s), s).clamp(-126, 121)
        step = (2.0 ** s).unsqueeze(1)
        val = torch.round(blk / step).clamp(-127, 127) * step
        val[bad] = float("nan")
        out[:, a:a + 32] = val
    return out.reshape(x.shape)


def norm(x, w, b, dy, eps, layer, kept):
    """``(y, dx, dw, db)`` and the absolute sums of the terms of dw and db, fp64 on the CPU."""
    x64, d = x.detach().cpu().double(), dy.cpu().double()
    C = x.shape[-1]
    w64 = torch.ones(C, dtype=torch.double) if w is None else w.detach().cpu().double()
    mean = x64.mean(-1, keepdim=True) if layer else torch.zeros_like(x64[..., :1])
    std = ((x64 - mean).square().mean(-1, keepdim=True) + eps).sqrt()
    y = (x64 - mean) / std * w64
    if b is not None:
        y = y + b.detach().cpu().double()
    n = ((kept_values(x) if kept else x64) - mean) / std
    g = d * w64
    dx = g - n * (g * n).mean(-1, keepdim=True)
    if layer:
        dx = dx - g.mean(-1, keepdim=True)
    rows = (d * n).reshape(-1, C), d.reshape(-1, C)
    return dict(y=y, dx=dx / std, dw=rows[0].sum(0), db=rows[1].sum(0), dw_abs=rows[0].abs().sum(0),
                db_abs=rows[1].abs().sum(0))


def swiglu(gate, value, dh):
    g, v, d = (t.detach().cpu().double() for t in (gate, value, dh))
    h = g * torch.sigmoid(g) * v
    kg, kv = kept_values(gate), kept_values(value)
    s = torch.sigmoid(kg)
    return dict(h=h, dgate=d * kv * s * (1 + kg * (1 - s)), dvalue=d * kg * s, kept_h=kg * s * kv)


def check(out, ref, dtype, terms, what):
    """``out`` is ``ref`` rounded to ``dtype`` (half an ulp, doubled for an fp32 value that lands on the
    other side of a rounding boundary) after fp32 arithmetic whose error is at most ``terms``."""
    out = out.detach().cpu().double()
    assert out.shape == ref.shape, f"{what}: {tuple(out.shape)} != {tuple(ref.shape)}"
    assert bool((torch.isnan(out) == torch.isnan(ref)).all()), f"{what}: NaNs in other places"
    bound = 2 * unit(dtype) * ref.abs() + terms
    off = ((out - ref).abs() - bound)[~torch.isnan(ref)]
    assert off.numel() == 0 or float(off.max()) <= 0, f"{what}: {float(off.max()):.3e} over the bound"


def activations(*shape, seed=0, dtype=torch.float32, device="cpu"):
    """Hidden states with a per-row gain and a few loud channels."""
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(*shape, generator=gen) * (torch.rand(*shape[:-1], 1, generator=gen) + 0.5)
    x[..., ::37] *= 12
    return x.to(dtype).to(device)


def sqrt_terms(n):
    return math.sqrt(max(1, n))
