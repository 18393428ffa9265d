"""Measured cases of the memory-lean training operators: 8-bit kept activations and the operators
whose backward reads them (layer / RMS norm, linear, SwiGLU).

Every case is one pass of one operator as a training step makes it: the 8-bit store and its reload,
or a forward and its backward.  ``run`` computes it in plain torch arithmetic, or through
``pan2_b200.ops`` where ``own`` is set; ``exact`` states the same definitions in 64 bits.

The 8-bit format ("kept8"): rows are cut into blocks of 32 consecutive channels (the last block may be
short).  A block's step is ``2^s`` with ``s = clamp(floor(log2(max |x|)) - 6, -126, 121)``, its codes are
``clamp(round_half_even(x / 2^s), -127, 127)`` and its values ``code * 2^s``; every step of that is exact
in 32 bits, so the values do not depend on who computes them.  A block that holds an infinity or a NaN
reads back as NaN.
"""
import math

import torch

own = False

BLOCK = 32
DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


# ------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # block checkpoint of one short image sample: 256 tokens, hidden size 4096
        dict(name="checkpoint_image", op="checkpoint", rows=256, cols=4096, dtype="bf16"),
        # block checkpoint at the pretraining configuration's joint token budget
        dict(name="checkpoint_budget", op="checkpoint", rows=110576, cols=4096, dtype="bf16"),
        # fp32 activations whose width ends inside a block
        dict(name="checkpoint_ragged", op="checkpoint", rows=18993, cols=1001, dtype="fp32"),
        # layer norm of a single conditioning row: launch latency
        dict(name="norm_one_row", op="norm", kind="layer", rows=1, heads=1, cols=4096, dtype="bf16", kept8=False),
        # caption encoder's pre-norm over a full caption budget, input kept in 8 bits
        dict(name="norm_caption", op="norm", kind="rms", rows=4096, heads=1, cols=4096, dtype="bf16", kept8=True),
        # q norm of the caption encoder: head dim 128 inside the fused [tokens, 3, heads, 128] projection
        dict(name="norm_heads", op="norm", kind="rms", rows=4096, heads=32, cols=128, dtype="bf16", kept8=False),
        # five packed clips of video tokens, input kept in 8 bits
        dict(name="norm_video", op="norm", kind="layer", rows=94960, heads=1, cols=4096, dtype="bf16", kept8=True),
        # fp32 rows of odd width
        dict(name="norm_ragged", op="norm", kind="layer", rows=1537, heads=1, cols=1001, dtype="fp32", kept8=False),
        # caption encoder's fused qkv projection over a full caption budget
        dict(name="linear_caption", op="linear", rows=4096, k=4096, n=12288, bias=False),
        # one odd-length caption through a small projection with bias
        dict(name="linear_ragged", op="linear", rows=777, k=1000, n=1032, bias=True),
        # caption encoder's SwiGLU (mlp ratio 4) over a full caption budget
        dict(name="swiglu_caption", op="swiglu", rows=4096, cols=16384, dtype="bf16"),
        # fp32, odd width
        dict(name="swiglu_ragged", op="swiglu", rows=333, cols=1001, dtype="fp32"),
    ]


def _spread(rng, lo, hi):
    """A number in [lo, hi], its logarithm uniform: 1, 8 or 64 times an odd one, so that every alignment comes up."""
    v = int(math.exp(rng.uniform(math.log(lo), math.log(hi))))
    unit = max(u for u in (1, rng.choice([1, 8, 64])) if u <= max(v, 1))
    v = v // unit
    v = (v - 1 if v % 2 == 0 else v) * unit
    return v if lo <= v <= hi else lo


def draw(rng):
    op = rng.choice(["checkpoint", "norm", "norm", "linear", "swiglu"])
    dtype = rng.choice(["bf16", "bf16", "fp32"])
    if op == "checkpoint":
        cols = _spread(rng, 8, 16384)
        return dict(op=op, rows=_spread(rng, 1, min(200000, 200_000_000 // cols)), cols=cols, dtype=dtype)
    if op == "norm":
        kind, kept8 = rng.choice(["layer", "rms"]), rng.random() < 0.5
        if rng.random() < 0.25:
            heads, cols = rng.choice([4, 16, 32, 40]), rng.choice([64, 80, 128, 256])
            return dict(op=op, kind=kind, rows=_spread(rng, 1, 8192), heads=heads, cols=cols, dtype=dtype, kept8=kept8)
        cols = _spread(rng, 32, 16384)
        return dict(op=op, kind=kind, rows=_spread(rng, 1, min(200000, 120_000_000 // cols)), heads=1, cols=cols,
                    dtype=dtype, kept8=kept8)
    if op == "linear":
        k, n = _spread(rng, 32, 8192), _spread(rng, 32, 12288)
        rows = _spread(rng, 1, max(1, min(32768, 4096 * 4096 * 12288 // (2 * k * n))))
        return dict(op=op, rows=rows, k=k, n=n, bias=rng.random() < 0.5)
    cols = _spread(rng, 16, 32768)
    return dict(op=op, rows=_spread(rng, 1, min(65536, 36_000_000 // cols)), cols=cols, dtype=dtype)


def work(case):
    """Bytes that have to move and operations that have to run in one pass."""
    if case["op"] == "linear":
        l, k, n = case["rows"], case["k"], case["n"]
        # forward: x, W read, y and the codes written; backward: dy, W, codes read, dx, dW (and the bias, db) written
        by = 2 * l * k + 2 * n * k + 2 * l * n + _kept_bytes(l, k)
        by += 2 * l * n + 2 * n * k + _kept_bytes(l, k) + 2 * l * k + 2 * n * k + (4 * n if case["bias"] else 0)
        return {"bytes": by, "flops": 6 * l * k * n}
    e = 2 if case["dtype"] == "bf16" else 4
    if case["op"] == "checkpoint":
        l, c = case["rows"], case["cols"]
        return {"bytes": 2 * e * l * c + 2 * _kept_bytes(l, c), "flops": 4 * l * c}
    if case["op"] == "norm":
        l, c = case["rows"] * case["heads"], case["cols"]
        kept = _kept_bytes(l, c)
        forward = 2 * e * l * c + (kept if case["kept8"] else 0)
        backward = 2 * e * l * c + (kept if case["kept8"] else e * l * c)
        vectors = (2 if case["kind"] == "layer" else 1) * e * c
        return {"bytes": forward + backward + 3 * vectors, "flops": 20 * l * c}
    l, c = case["rows"], case["cols"]
    # forward: gate, value read, h and both codes written; backward: dh and the codes read, both gradients written
    return {"bytes": 3 * e * l * c + 2 * _kept_bytes(l, c) + 3 * e * l * c + 2 * _kept_bytes(l, c), "flops": 25 * l * c}


def _kept_bytes(rows, cols):
    """Codes and one scale byte for each block."""
    return rows * cols + rows * (-(-cols // BLOCK))


# ----------------------------------------------------------------------------------------- inputs
def _activations(gen, shape, dtype):
    """Hidden states: unit scale, a per-row gain, and a few channels that run an order of magnitude larger."""
    x = torch.randn(shape, generator=gen, device="cuda")
    x *= torch.rand(shape[:-1] + (1,), generator=gen, device="cuda") * 1.5 + 0.25
    loud = torch.rand(shape[-1], generator=gen, device="cuda") < 0.004
    x = torch.where(loud, x * 20, x)
    return x.to(dtype)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed) * 7919 + 17)
    s = dict(case)
    if case["op"] == "linear":
        l, k, n = case["rows"], case["k"], case["n"]
        bf = torch.bfloat16
        s["x"] = _activations(gen, (l, k), bf).requires_grad_(True)
        s["w"] = (torch.randn(n, k, generator=gen, device="cuda") * k ** -0.5).to(bf).requires_grad_(True)
        s["b"] = (torch.randn(n, generator=gen, device="cuda") * 0.1).to(bf).requires_grad_(True) if case["bias"] else None
        s["dy"] = (torch.randn(l, n, generator=gen, device="cuda") * 0.01).to(bf)
        return s
    dt, c = DTYPES[case["dtype"]], case["cols"]
    if case["op"] == "checkpoint":
        s["x"] = _activations(gen, (case["rows"], c), dt)
        return s
    if case["op"] == "norm":
        if case["heads"] > 1:  # the q third of a fused projection: rows are not adjacent in memory
            fused = _activations(gen, (case["rows"], 3, case["heads"], c), dt)
            s["x"] = fused[:, 0].detach().requires_grad_(True)
        else:
            s["x"] = _activations(gen, (case["rows"], c), dt).requires_grad_(True)
        s["w"] = (1 + 0.2 * torch.randn(c, generator=gen, device="cuda")).to(dt).requires_grad_(True)
        s["b"] = None
        if case["kind"] == "layer":
            s["b"] = (0.2 * torch.randn(c, generator=gen, device="cuda")).to(dt).requires_grad_(True)
        s["eps"] = 1e-6 if case["kind"] == "layer" else 1e-5
        s["dy"] = (torch.randn(s["x"].shape, generator=gen, device="cuda") * 0.01).to(dt)
        return s
    s["gate"] = _activations(gen, (case["rows"], c), dt).requires_grad_(True)
    s["value"] = _activations(gen, (case["rows"], c), dt).requires_grad_(True)
    s["dh"] = (torch.randn(case["rows"], c, generator=gen, device="cuda") * 0.01).to(dt)
    return s


# ------------------------------------------------------------------------------------- one pass
def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(s):
    if s["op"] == "checkpoint":
        from pan2_b200.ops.kept8 import keep8, restore8
        return {"x": restore8(keep8(s["x"]))}
    if s["op"] == "norm":
        from pan2_b200.ops.norm import layer_norm, rms_norm
        if s["kind"] == "layer":
            y = layer_norm(s["x"], s["w"], s["b"], s["eps"], kept8=s["kept8"])
            dx, dw, db = torch.autograd.grad(y, (s["x"], s["w"], s["b"]), s["dy"])
            return {"y": y, "dx": dx, "dw": dw, "db": db}
        y = rms_norm(s["x"], s["w"], s["eps"], kept8=s["kept8"])
        dx, dw = torch.autograd.grad(y, (s["x"], s["w"]), s["dy"])
        return {"y": y, "dx": dx, "dw": dw}
    if s["op"] == "linear":
        from pan2_b200.ops.kept8 import kept8_linear
        y = kept8_linear(s["x"], s["w"], s["b"])
        wrt = ("x", "w", "b") if s["b"] is not None else ("x", "w")
        grads = torch.autograd.grad(y, [s[i] for i in wrt], s["dy"])
        return {"y": y, **{"d" + i: g for i, g in zip(wrt, grads)}}
    from pan2_b200.ops.kept8 import kept8_swiglu
    h = kept8_swiglu(s["gate"], s["value"])
    dgate, dvalue = torch.autograd.grad(h, (s["gate"], s["value"]), s["dh"])
    return {"h": h, "dgate": dgate, "dvalue": dvalue}


def _kept_values(x):
    """The values that ``x`` [..., C] reads back as after being held in 8 bits, in fp32."""
    c = x.shape[-1]
    v = torch.nn.functional.pad(x.float(), (0, -c % BLOCK)).unflatten(-1, (-1, BLOCK))
    top = v.abs().amax(-1, keepdim=True)
    fine = torch.isfinite(top)
    s = (torch.frexp(torch.where(fine, top, 1.0))[1] - 7).clamp(-126, 121)  # frexp: top = m 2^e, m in [1/2, 1)
    code = torch.clamp(torch.round(v * _power_of_two(-s)), -127, 127)
    back = torch.where(fine, code * _power_of_two(s), float("nan"))
    return back.flatten(-2)[..., :c]


def _power_of_two(s):
    """``2^s`` in fp32 from its bits (``-126 <= s <= 127``)."""
    return ((s + 127) << 23).to(torch.int32).view(torch.float32)


@torch.no_grad()
def _run_plain(s):
    if s["op"] == "checkpoint":
        return {"x": _kept_values(s["x"]).to(s["x"].dtype)}
    if s["op"] == "norm":
        x, w, dy, dt = s["x"].float(), s["w"].float(), s["dy"].float(), s["x"].dtype
        layer = s["kind"] == "layer"
        mean = x.mean(-1, keepdim=True) if layer else 0.0
        rstd = torch.rsqrt((x - mean).square().mean(-1, keepdim=True) + s["eps"])
        y = (x - mean) * rstd * w
        if layer:
            y = y + s["b"].float()
        n = ((_kept_values(s["x"]) if s["kept8"] else x) - mean) * rstd
        g = dy * w
        dx = g - n * (g * n).mean(-1, keepdim=True)
        if layer:
            dx = dx - g.mean(-1, keepdim=True)
        rows = tuple(range(x.dim() - 1))
        out = {"y": y.to(dt), "dx": (dx * rstd).to(dt), "dw": (dy * n).sum(rows).to(dt)}
        if layer:
            out["db"] = dy.sum(rows).to(dt)
        return out
    if s["op"] == "linear":
        x, w, dy, dt = s["x"].float(), s["w"].float(), s["dy"].float(), s["x"].dtype
        y = x @ w.t()
        out = {"y": (y if s["b"] is None else y + s["b"].float()).to(dt), "dx": (dy @ w).to(dt),
               "dw": (dy.t() @ _kept_values(s["x"])).to(dt)}
        if s["b"] is not None:
            out["db"] = dy.sum(0).to(dt)
        return out
    gate, value, dh, dt = s["gate"].float(), s["value"].float(), s["dh"].float(), s["gate"].dtype
    h = gate / (1 + torch.exp(-gate)) * value
    g, v = _kept_values(s["gate"]), _kept_values(s["value"])
    sig = 1 / (1 + torch.exp(-g))
    return {"h": h.to(dt), "dgate": (dh * v * sig * (1 + g * (1 - sig))).to(dt), "dvalue": (dh * g * sig).to(dt)}


# --------------------------------------------------------------------------------- 64 bits
def _kept_exact(x):
    """``_kept_values`` from the format's definition, the exponent read from the bits of the 64-bit maximum."""
    rows, c = x.shape[0], x.shape[-1]
    out = torch.empty(x.shape, dtype=torch.float64, device=x.device)
    full = c - c % BLOCK
    for lo, hi, width in ((0, full, BLOCK), (full, c, c - full)):
        if hi == lo or rows == 0:
            continue
        v = x[..., lo:hi].double().reshape(-1, width)
        top = v.abs().amax(1)
        s = torch.clamp((top.view(torch.int64) >> 52) - 1023 - 6, -126, 121)
        step = ((s + 1023) << 52).view(torch.float64)[:, None]
        out[..., lo:hi] = ((v / step).round().clamp(-127, 127) * step).reshape(x[..., lo:hi].shape)
    return out


@torch.no_grad()
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "checkpoint":
        return {"x": _kept_exact(s["x"])}
    if case["op"] == "norm":
        x, w, dy = s["x"].double(), s["w"].double(), s["dy"].double()
        lead, c = tuple(range(x.dim() - 1)), x.shape[-1]
        mean = x.sum(-1, keepdim=True) / c if case["kind"] == "layer" else torch.zeros_like(x[..., :1])
        var = ((x - mean) ** 2).sum(-1, keepdim=True) / c
        std = torch.sqrt(var + s["eps"])
        out = {"y": (x - mean) / std * w}
        n = ((_kept_exact(s["x"]) if case["kept8"] else x) - mean) / std
        g = dy * w
        dx = g - n * ((g * n).sum(-1, keepdim=True) / c)
        if case["kind"] == "layer":
            out["y"] = out["y"] + s["b"].double()
            out["db"] = dy.sum(lead)
            dx = dx - g.sum(-1, keepdim=True) / c
        return {**out, "dx": dx / std, "dw": (dy * n).sum(lead)}
    if case["op"] == "linear":
        x, w, dy = s["x"].double(), s["w"].double(), s["dy"].double()
        y = torch.einsum("lk,nk->ln", x, w)
        out = {"dx": torch.einsum("ln,nk->lk", dy, w), "dw": torch.einsum("ln,lk->nk", dy, _kept_exact(s["x"]))}
        if case["bias"]:
            y, out["db"] = y + s["b"].double(), dy.sum(0)
        return {**out, "y": y}
    gate, value, dh = s["gate"].double(), s["value"].double(), s["dh"].double()
    h = gate * torch.sigmoid(gate) * value
    g, v = _kept_exact(s["gate"]), _kept_exact(s["value"])
    sig = torch.sigmoid(g)
    return {"h": h, "dgate": dh * v * (sig + g * sig * (1 - sig)), "dvalue": dh * g * sig}
