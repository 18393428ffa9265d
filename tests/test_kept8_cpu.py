"""8-bit kept activations, norms and SwiGLU on the CPU: the format, gradients, refusals."""
import pytest
import torch

import kept8_ref as R
from pan2_b200.ops.kept8 import (Kept8, keep8, kept8_linear, kept8_swiglu, kept8_swiglu_ffn, restore8)
from pan2_b200.ops.norm import layer_norm, rms_norm


@pytest.mark.parametrize("shape", [(1, 1), (3, 31), (2, 32), (5, 33), (2, 3, 100), (0, 40), (7, 128)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_store_reads_back_the_defined_values(shape, dtype):
    x = R.activations(*shape, dtype=dtype)
    kept = keep8(x)
    assert kept.shape == x.shape and kept.dtype == dtype
    back = restore8(kept)
    assert back.dtype == dtype and back.shape == x.shape
    assert torch.equal(back.double(), R.kept_values(x))


def test_error_is_within_a_step_of_the_block_maximum():
    x = R.activations(64, 96)
    blocks = x.view(64, 3, 32)
    err = (restore8(keep8(x)) - x).abs().view(64, 3, 32)
    assert bool((err <= blocks.abs().amax(-1, keepdim=True) * 2.0 ** -6).all())
    bf = x.bfloat16()  # bf16 inputs never lose more than half a step when they clamp
    err = (restore8(keep8(bf)).double() - bf.double()).abs().view(64, 3, 32)
    assert bool((err <= bf.double().view(64, 3, 32).abs().amax(-1, keepdim=True) * 2.0 ** -7).all())


def test_values_are_exact_in_bf16_and_storing_twice_changes_nothing():
    x = R.activations(16, 200)
    back = restore8(keep8(x))
    assert torch.equal(back.bfloat16().float(), back)
    again = restore8(keep8(back))
    # the largest code of a block is 64 .. 127, so its values lead to the same step again
    assert torch.equal(again, back)


def test_special_values():
    x = torch.zeros(6, 64)
    x[1, 3] = float("inf")
    x[2, 40] = float("nan")
    x[3, :32] = 1e-42                      # subnormal block: flushes below half the smallest step
    x[4, 0] = torch.finfo(torch.float32).max
    x[4, 1] = -torch.finfo(torch.float32).max
    x[5, 0] = 2.0 ** -120
    back = restore8(keep8(x))
    assert bool((back[0] == 0).all())
    assert bool(torch.isnan(back[1, :32]).all()) and bool((back[1, 32:] == 0).all())
    assert bool((back[2, :32] == 0).all()) and bool(torch.isnan(back[2, 32:]).all())
    assert bool((back[3] == 0).all())
    assert torch.isfinite(back[4]).all() and back[4, 0] == -back[4, 1] and back[4, 0] > 3.3e38
    assert back[5, 0] == 2.0 ** -120


def test_bytes():
    kept = keep8(torch.randn(10, 4096))
    assert kept.nbytes == 10 * 4096 + 10 * 128


@pytest.mark.parametrize("layer", [True, False], ids=["layer", "rms"])
def test_norm_gradients_against_differences(layer):
    x = R.activations(3, 4, 24).double().requires_grad_(True)
    w = torch.randn(24, dtype=torch.double, requires_grad=True)
    b = torch.randn(24, dtype=torch.double, requires_grad=True)
    if layer:
        assert torch.autograd.gradcheck(lambda *a: layer_norm(*a, 1e-3), (x, w, b))
        assert torch.autograd.gradcheck(lambda a: layer_norm(a, eps=1e-3), (x,))
    else:
        assert torch.autograd.gradcheck(lambda *a: rms_norm(*a, 1e-3), (x, w))


def test_swiglu_and_linear_gradients_against_differences_where_storing_is_exact():
    # whole numbers up to 127 with a 64 in every block keep a step of 1: the store is the identity
    gen = torch.Generator().manual_seed(3)
    x = torch.randint(-127, 128, (5, 64), generator=gen).double()
    x[:, ::32] = 64
    assert torch.equal(restore8(keep8(x)), x)
    w = torch.randn(6, 64, dtype=torch.double, requires_grad=True)
    b = torch.randn(6, dtype=torch.double, requires_grad=True)
    x.requires_grad_(True)
    assert torch.autograd.gradcheck(lambda *a: kept8_linear(*a), (x, w, b))
    g = (x.detach() / 128).requires_grad_(True)  # 64 / 128 .. 127 / 128: the same codes, a step of 1 / 128
    v = (x.detach().flip(0) / 64).requires_grad_(True)
    # the backward is that of the kept values: compare with differences at a point the store leaves alone
    h = kept8_swiglu(g, v)
    dh = torch.randn(h.shape, dtype=torch.double, generator=gen)
    dg, dv = torch.autograd.grad(h, (g, v), dh)
    eps = 1e-6
    f = lambda a, c: (a * torch.sigmoid(a) * c * dh).sum(-1)  # noqa: E731
    for i in (0, 17, 63):
        e = torch.zeros(64, dtype=torch.double)
        e[i] = eps
        assert torch.allclose((f(g + e, v) - f(g - e, v)) / (2 * eps), dg[:, i], rtol=1e-6, atol=1e-8)
        assert torch.allclose((f(g, v + e) - f(g, v - e)) / (2 * eps), dv[:, i], rtol=1e-6, atol=1e-8)


@pytest.mark.parametrize("rows,C", [(1, 1), (4, 40), (0, 33), (9, 130)])
@pytest.mark.parametrize("layer", [True, False], ids=["layer", "rms"])
@pytest.mark.parametrize("kept", [True, False], ids=["kept8", "exact"])
def test_norm_against_64_bits(rows, C, layer, kept):
    x = R.activations(rows, C, seed=rows).requires_grad_(True)
    w, b = (torch.randn(C, requires_grad=True) for _ in range(2))
    dy = torch.randn(rows, C)
    y = layer_norm(x, w, b, 1e-6, kept8=kept) if layer else rms_norm(x, w, 1e-6, kept8=kept)
    got = torch.autograd.grad(y, (x, w) + ((b,) if layer else ()), dy)
    ref = R.norm(x, w, b if layer else None, dy, 1e-6, layer, kept)
    for t, name in zip((y,) + got, ("y", "dx", "dw", "db")):
        scale = float(ref[name].abs().max()) if ref[name].numel() else 0.0
        R.check(t, ref[name], torch.float32, 64 * R.F32 * (scale + float(ref["dw_abs"].max())), name)


def test_ffn_matches_its_parts():
    x = R.activations(6, 48).requires_grad_(True)
    w1, w3 = (torch.randn(96, 48, requires_grad=True) for _ in range(2))
    w2 = torch.randn(20, 96, requires_grad=True)
    dy = torch.randn(6, 20)
    whole = kept8_swiglu_ffn(x, w1, w3, w2)
    got = torch.autograd.grad(whole, (x, w1, w3, w2), dy)
    parts = torch.nn.functional.linear(kept8_swiglu(kept8_linear(x, w1), kept8_linear(x, w3)), w2)
    assert torch.allclose(whole, parts, rtol=1e-5, atol=1e-4)
    want = torch.autograd.grad(parts, (x, w1, w3, w2), dy)
    for a, c, name in zip(got, want, ("x", "w1", "w3", "w2")):
        tol = 2e-2 if name == "w2" else 1e-5  # w2's gradient reads the product recomputed from 8 bits
        assert float((a - c).norm() / c.norm()) < tol, name


def test_gradients_only_where_needed():
    x = torch.randn(4, 64, requires_grad=True)
    w = torch.randn(8, 64)
    kept8_linear(x, w).sum().backward()
    assert x.grad is not None and w.grad is None
    y = rms_norm(torch.randn(4, 64), torch.ones(64, requires_grad=True), kept8=True)
    y.sum().backward()


def test_refusals():
    x = torch.randn(4, 64)
    with pytest.raises(TypeError, match="floating"):
        keep8(torch.zeros(4, 4, dtype=torch.int32))
    with pytest.raises(TypeError, match="tensor"):
        keep8([1.0, 2.0])
    with pytest.raises(ValueError, match="last dimension"):
        keep8(torch.zeros(4, 0))
    with pytest.raises(ValueError, match="last dimension"):
        keep8(torch.tensor(1.0))
    with pytest.raises(TypeError, match="keep8 returned"):
        restore8(x)
    with pytest.raises(ValueError, match="does not fit"):
        kept8_linear(x, torch.randn(8, 32))
    with pytest.raises(ValueError, match="does not fit"):
        kept8_linear(x, torch.randn(8, 64), torch.randn(9))
    with pytest.raises(ValueError, match="differ"):
        kept8_swiglu(x, torch.randn(4, 32))
    with pytest.raises(ValueError, match="differ"):
        kept8_swiglu(x, x.double())
    with pytest.raises(ValueError, match="differ"):
        kept8_swiglu_ffn(x, torch.randn(8, 64), torch.randn(9, 64), torch.randn(64, 8))
    with pytest.raises(ValueError, match="does not fit"):
        kept8_swiglu_ffn(x, torch.randn(8, 64), torch.randn(8, 64), torch.randn(64, 9))
    with pytest.raises(ValueError, match="does not fit"):
        layer_norm(x, torch.ones(32))
    with pytest.raises(ValueError, match="does not fit"):
        layer_norm(x, torch.ones(64), torch.ones(1, 64))
    with pytest.raises(TypeError, match="different dtypes"):
        layer_norm(x, torch.ones(64), torch.ones(64, dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="negative"):
        rms_norm(x, eps=-1.0)
    with pytest.raises(ValueError, match="negative"):
        rms_norm(x, eps=float("nan"))
    assert isinstance(keep8(x), Kept8)


def kept_calls(dtype, device, grad=True):
    """Every operator with a backward, on small inputs: ``name -> (call, inputs)``."""
    t = lambda *s: R.activations(*s, seed=len(s), dtype=dtype, device=device).requires_grad_(grad)  # noqa: E731
    return {
        "layer_norm": (layer_norm, (t(4, 64), t(64), t(64))),
        "layer_norm kept8": (lambda *a: layer_norm(*a, kept8=True), (t(4, 64), t(64), t(64))),
        "rms_norm": (rms_norm, (t(4, 64), t(64))),
        "rms_norm kept8": (lambda *a: rms_norm(*a, kept8=True), (t(4, 64), t(64))),
        "kept8_linear": (kept8_linear, (t(4, 64), t(8, 64))),
        "kept8_swiglu": (kept8_swiglu, (t(4, 64), t(4, 64))),
        "kept8_swiglu_ffn": (kept8_swiglu_ffn, (t(4, 64), t(96, 64), t(96, 64), t(64, 96))),
    }


def refuses_second_derivatives(dtype, device):
    for name, (call, inputs) in kept_calls(dtype, device).items():
        y = call(*inputs)
        with pytest.raises(RuntimeError, match="no second derivative"):
            torch.autograd.grad(y.float().sum(), inputs, create_graph=True)
        grads = torch.autograd.grad(call(*inputs).float().sum(), inputs)  # as before without
        assert all(g.shape == i.shape and not g.requires_grad for g, i in zip(grads, inputs)), name


@pytest.mark.parametrize("dtype", [torch.float32, torch.float64])
def test_second_derivatives_are_refused(dtype):
    """The backward reads statistics and codes that carry no graph, so what it returns must not be differentiated."""
    refuses_second_derivatives(dtype, "cpu")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float64])
def test_scale_bytes(dtype):
    """Exponent of the block's largest value, 7 for blocks of zeros and subnormals, 255 for non-finite ones, 127 for padding."""
    x = torch.zeros(1, 6 * 32, dtype=dtype)
    x[0, 32], x[0, 64 + 31], x[0, 96], x[0, 128], x[0, 160] = 1.0, -3.0, 2.0 ** -130, float("inf"), 2.0 ** -126
    assert keep8(x).scales.tolist() == [[7, 127, 128, 7, 255, 7, 127, 127]]
