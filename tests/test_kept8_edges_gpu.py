"""8-bit operators on a B200 where a call comes in an unusual form: views at odd addresses, empty batches, widths of
the forms that other tests do not reach, threads."""
import pytest
import torch

import kept8_ref as R
from pan2_b200.ops.kept8 import keep8, kept8_linear, kept8_swiglu, kept8_swiglu_ffn
from pan2_b200.ops.norm import layer_norm, rms_norm

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _no_device_errors():
    from pan2_b200.ops._ext import ext
    yield
    torch.cuda.synchronize()
    assert ext().error_flag(True) == 0, "a kernel recorded a bounded-wait timeout"


def odd_copy(t, by=1):
    """``t`` contiguous at an address ``by`` elements past a 16-byte boundary."""
    flat = torch.empty(t.numel() + 16, dtype=t.dtype, device=t.device)
    view = flat[by:by + t.numel()].view(t.shape)
    view.copy_(t)
    assert view.is_contiguous() and view.data_ptr() % 16 == by * t.element_size() % 16
    return view


def bf16(*shape, seed, scale=1.0):
    gen = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=gen) * scale).bfloat16().cuda()


@pytest.mark.parametrize("N", [8, 264, 1032])
@pytest.mark.parametrize("by", [1, 3, 4])
def test_linear_with_a_bias_at_an_odd_address(N, by):
    from pan2_b200.ops.gemm import grouped_linear, linear
    x, w, b = bf16(300, 64, seed=1), bf16(N, 64, seed=2, scale=0.125), bf16(N, seed=3)
    odd = odd_copy(b, by)
    for fn in (kept8_linear, linear):
        assert torch.equal(fn(x, w, odd), fn(x, w, b)), fn.__name__
    y64 = x.cpu().double() @ w.cpu().double().t()
    # 64 roundings of the terms' absolute sum: the tensor core adds blocks of terms with a truncation each
    terms = 64 * R.F32 * (x.cpu().double().abs() @ w.cpu().double().t().abs())
    R.check(kept8_linear(x, w, odd), y64 + b.cpu().double(), torch.bfloat16, terms, "y")
    two, odd_two = torch.stack([b, b + 1]), odd_copy(torch.stack([b, b + 1]), by)
    ww = torch.stack([w, w])
    assert torch.equal(grouped_linear(x, ww, odd_two, [0, 100, 300]), grouped_linear(x, ww, two, [0, 100, 300]))


# Views that are neither aligned nor contiguous: one element at a time, by groups of a warp (to 256 columns), of 256
# threads (to 2048) and of 512 or 1024 (to 8192), then by sweeps.
SINGLE = [(9, 200), (37, 257), (21, 1001), (300, 2048), (13, 2049), (8, 8191), (5, 9001), (3, 16400)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("layer", [True, False], ids=["layer", "rms"])
@pytest.mark.parametrize("kept", [False, True], ids=["exact", "kept8"])
@pytest.mark.parametrize("rows,C", SINGLE)
def test_norm_of_views_of_every_width(rows, C, dtype, layer, kept):
    view = lambda t: t[:, 1:1 + C]  # noqa: E731
    base = R.activations(rows, C + 5, seed=C, dtype=dtype, device="cuda")
    x = view(base).detach().requires_grad_(True)
    gen = torch.Generator().manual_seed(C)
    w = (1 + 0.3 * torch.randn(C, generator=gen)).to(dtype).cuda().requires_grad_(True)
    b = (0.3 * torch.randn(C, generator=gen)).to(dtype).cuda().requires_grad_(True)
    dy = view(torch.randn(rows, C + 5, generator=gen).to(dtype).cuda())
    y = layer_norm(x, w, b, 1e-6, kept8=kept) if layer else rms_norm(x, w, 1e-6, kept8=kept)
    wrt = (x, w, b) if layer else (x, w)
    got = dict(zip(("dx", "dw", "db"), torch.autograd.grad(y, wrt, dy)), y=y)
    ref = R.norm(x, w, b if layer else None, dy, 1e-6, layer, kept)
    for name, t in got.items():
        if name in ("y", "dx"):  # fp32 sums of at most 96 sequential terms and their tree, by the row's largest value
            terms = 128 * R.F32 * ref[name].abs().amax(-1, keepdim=True)
        else:  # at most 1024 sequential additions of terms that are off by some roundings
            terms = 1024 * R.F32 * ref[name + "_abs"]
        R.check(t, ref[name], dtype, terms, name)


@pytest.mark.parametrize("by", [1, 2, 3])
@pytest.mark.parametrize("C", [264, 1024, 4096])
def test_norm_at_odd_addresses(C, by):
    x, w, b, dy = bf16(40, C, seed=C), bf16(C, seed=1), bf16(C, seed=2), bf16(40, C, seed=3)
    for kept in (False, True):
        ref = R.norm(x, w, b, dy, 1e-6, True, kept)
        for odd in ("x", "w", "dy", "all"):
            args = {n: odd_copy(t, by) if odd in (n, "all") else t for n, t in (("x", x), ("w", w), ("b", b), ("dy", dy))}
            xs, ws, bs = (args[n].detach().requires_grad_(True) for n in ("x", "w", "b"))
            y = layer_norm(xs, ws, bs, kept8=kept)
            got = dict(zip(("dx", "dw", "db"), torch.autograd.grad(y, (xs, ws, bs), args["dy"])), y=y)
            for name, t in got.items():
                terms = (128 * R.F32 * ref[name].abs().amax(-1, keepdim=True) if name in ("y", "dx")
                         else 1024 * R.F32 * ref[name + "_abs"])
                R.check(t, ref[name], torch.bfloat16, terms, f"{name}, {odd} odd")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
def test_second_derivatives_are_refused(dtype):
    from test_kept8_cpu import refuses_second_derivatives
    refuses_second_derivatives(dtype, "cuda")


def test_swiglu_refuses_shapes_that_only_have_as_many_rows():
    gate = torch.randn(4, 64, device="cuda", requires_grad=True)
    for shape in ((2, 2, 64), (1, 4, 64)):
        for pair in ((gate, torch.randn(shape, device="cuda")), (torch.randn(shape, device="cuda"), gate)):
            with pytest.raises(ValueError, match="differ"):
                kept8_swiglu(*pair)
            with pytest.raises(ValueError, match="differ"):  # as the CPU path does
                kept8_swiglu(*(t.cpu() for t in pair))


def product_terms(a, b):
    """Bound on the fp32 accumulation error of ``a @ b``: the terms' absolute sum, 64 roundings."""
    return 64 * R.F32 * (a.abs() @ b.abs())


def d(t):
    return t.detach().cpu().double()


@pytest.mark.parametrize("w_dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("rows,K,H,N", [(260, 96, 328, 96), (77, 100, 171, 45), (300, 33, 1001, 64), (1, 64, 8, 200),
                                        (0, 64, 96, 40)])
def test_swiglu_ffn_against_64_bits(rows, K, H, N, w_dtype):
    """Each step against 64 bits, given the inputs that the step before it makes: the same kernels on the same
    operands as inside the FFN, so its bf16 intermediates are at hand."""
    from pan2_b200.ops._ext import ext
    x = bf16(rows, K, seed=1).requires_grad_(True)
    # values of bf16 in either type: fp32 weights are read as bf16
    w1, w3 = (bf16(H, K, seed=s, scale=K ** -0.5).to(w_dtype).requires_grad_(True) for s in (2, 3))
    w2 = bf16(N, H, seed=4, scale=H ** -0.5).to(w_dtype).requires_grad_(True)
    dy = bf16(rows, N, seed=5)
    y = kept8_swiglu_ffn(x, w1, w3, w2)
    dx, dw1, dw3, dw2 = torch.autograd.grad(y, (x, w1, w3, w2), dy)
    assert [t.dtype for t in (y, dx, dw1, dw3, dw2)] == [torch.bfloat16] * 2 + [w_dtype] * 3
    gate, value = kept8_linear(x, w1).detach(), kept8_linear(x, w3).detach()
    h, *kept = ext().swiglu8_fwd(gate, value, True)
    R.check(y, d(h) @ d(w2).t(), torch.bfloat16, product_terms(d(h), d(w2).t()), "y")
    hh = h.clone().requires_grad_(True)
    (dh,) = torch.autograd.grad(kept8_linear(hh, w2), hh, dy)
    dgate, dvalue = ext().swiglu8_bwd(dh, *kept, False)
    k64 = R.kept_values(x)
    for got, by, name in ((dw1, dgate, "dw1"), (dw3, dvalue, "dw3")):
        R.check(got, d(by).t() @ k64, w_dtype, product_terms(d(by).t(), k64), name)
    one, two = d(dgate) @ d(w1), d(dvalue) @ d(w3)
    # the first product is rounded to bf16 before the second is added to it
    R.check(dx, one + two, torch.bfloat16,
            2 * R.BF16 * one.abs() + product_terms(d(dgate), d(w1)) + product_terms(d(dvalue), d(w3)), "dx")
    # the product of the kept values, rounded to bf16: a handful of fp32 roundings before that
    h64 = R.swiglu(gate, value, dh)["kept_h"] if rows else torch.zeros(0, H, dtype=torch.double)
    off = 2 * R.BF16 * h64.abs() + 32 * R.F32 * (R.kept_values(gate) * R.kept_values(value)).abs()
    R.check(dw2, d(dy).t() @ h64, w_dtype, d(dy).abs().t() @ off + product_terms(d(dy).t(), h64), "dw2")


def test_swiglu_ffn_at_odd_addresses():
    x, dy = bf16(120, 64, seed=1), bf16(120, 40, seed=5)
    w1, w3, w2 = bf16(96, 64, seed=2, scale=0.125), bf16(96, 64, seed=3, scale=0.125), bf16(40, 96, seed=4, scale=0.125)

    def run(*args):
        *args, g = args
        args = [a.detach().requires_grad_(True) for a in args]
        y = kept8_swiglu_ffn(*args)
        return (y, *torch.autograd.grad(y, args, g))
    want = run(x, w1, w3, w2, dy)
    names = ("x", "w1", "w3", "w2", "dy")
    for which in names + ("all",):
        args = [odd_copy(t, 3) if which in (n, "all") else t for n, t in zip(names, (x, w1, w3, w2, dy))]
        for a, b, name in zip(want, run(*args), ("y", "dx", "dw1", "dw3", "dw2")):
            assert torch.equal(a, b), (which, name)
    wide = bf16(120, 130, seed=1)  # a column slice with rows at odd addresses
    for a, b in zip(run(wide[:, 1:65].contiguous(), w1, w3, w2, dy), run(wide[:, 1:65], w1, w3, w2, dy)):
        assert torch.equal(a, b)
    with torch.no_grad():
        assert torch.equal(kept8_swiglu_ffn(odd_copy(x), w1, w3, w2), want[0])


def test_norms_of_many_widths_from_several_threads():
    import threading
    widths = [1101, 1535, 2901, 3501, 5001, 7001, 8191, 12001]
    data = {}
    for C in widths:
        x = R.activations(64, C, seed=C, device="cuda").requires_grad_(True)
        w = torch.linspace(0.5, 1.5, C, device="cuda").requires_grad_(True)
        data[C] = (x, w, torch.ones_like(x))

    def run(C):
        x, w, dy = data[C]
        y = rms_norm(x, w, kept8=True)
        return (y, *torch.autograd.grad(y, (x, w), dy))
    failed, got = [], {}

    def work(i):
        try:
            for C in widths[i:] + widths[:i]:
                got[i, C] = run(C)
        except Exception as e:  # noqa: BLE001 - reported below
            failed.append(e)
    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(widths))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not failed, failed
    for C in widths:
        want = run(C)
        for i in range(len(widths)):
            assert all(torch.equal(a, b) for a, b in zip(got[i, C], want)), (i, C)


@pytest.mark.parametrize("C", [128, 1001], ids=["aligned", "odd"])
def test_swiglu_of_fp32_is_fp32_arithmetic(C):
    """h, dgate and dvalue to a few fp32 roundings of themselves, far into the sigmoid's tails too."""
    rows = 60
    gate = torch.empty(rows, C, device="cuda")
    # whole numbers times a power of two, at most 127 of them: what the store reads back is the gate itself
    step = torch.tensor([2.0 ** (-r % 9 - 6) for r in range(rows)], device="cuda")[:, None]
    gen = torch.Generator().manual_seed(C)
    gate.copy_(torch.randint(-110, 100, (rows, C), generator=gen))
    gate[:, ::32] = 64
    gate *= step * 32
    gate[:6] = gate[:6] / gate[:6].abs().amax() * 86  # no longer whole numbers: the forward's only
    value = torch.randn(rows, C, generator=gen).cuda()
    gate.requires_grad_(True), value.requires_grad_(True)
    dh = torch.randn(rows, C, generator=gen).cuda()
    h = kept8_swiglu(gate, value)
    dg, dv = torch.autograd.grad(h, (gate, value), dh)
    ref = R.swiglu(gate, value, dh)
    g, kv = R.kept_values(gate), R.kept_values(value)
    assert float(d(gate).min()) < -80 and bool((g[6:] == d(gate)[6:]).all())
    # exp good to 2 ulp (4 roundings), a sum, a quotient, four products; terms that vanish below the smallest normal
    tiny = 2.0 ** -126
    R.check(h, ref["h"], torch.float32, 14 * R.F32 * ref["h"].abs() + tiny, "h")
    R.check(dv, ref["dvalue"], torch.float32, 14 * R.F32 * ref["dvalue"].abs() + tiny, "dvalue")
    s = torch.sigmoid(g)
    terms = (d(dh) * kv * s).abs() * (1 + g.abs() * torch.sigmoid(-g))  # what the slope adds up
    R.check(dg, ref["dgate"], torch.float32, 18 * R.F32 * terms + tiny, "dgate")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
def test_swiglu_at_the_ends_of_the_range(dtype):
    g = torch.tensor([-1e30, -1000.0, -120.0, -104.0, -89.0, -88.0, -87.5, 0.0, -0.0, 88.0, 89.0, 120.0, 1e30], device="cuda")
    gate = torch.zeros(len(g), 64, device="cuda", dtype=dtype)
    gate[:, 0] = g.to(dtype)  # a block of its own: kept to half a step
    value, dh = torch.ones_like(gate), torch.ones_like(gate)
    gate.requires_grad_(True), value.requires_grad_(True)
    h = kept8_swiglu(gate, value)
    dg, dv = torch.autograd.grad(h, (gate, value), dh)
    ref = R.swiglu(gate, value, dh)
    # results below 2^-119 may vanish: the sigmoid's smallest normal value times |g| < 128
    for t, name in ((h, "h"), (dg, "dgate"), (dv, "dvalue")):
        assert bool(torch.isfinite(t).all()), name
        R.check(t, ref[name], dtype, 32 * R.F32 * ref[name].abs() + 2.0 ** -119, name)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("C", [96, 97, 104], ids=["aligned", "odd", "short block"])
def test_blocks_of_zeros_hold_the_same_bytes_as_on_the_cpu(C, dtype):
    x = R.activations(70, C, dtype=dtype)
    x[::3, :32], x[1::3, 64:], x[5] = 0, 0, 0
    cpu, gpu = keep8(x), keep8(x.cuda())
    assert torch.equal(cpu.codes, gpu.codes.cpu()) and torch.equal(cpu.scales, gpu.scales.cpu())


@pytest.mark.parametrize("rows,K,N", [(32769, 64, 72), (70001, 33, 20), (65536, 520, 264)])
def test_linear_of_more_rows_than_are_reloaded_at_once(rows, K, N):
    """The weight gradient reloads 32768 rows at a time and adds the later ones in fp32."""
    for w_dtype in (torch.bfloat16, torch.float32):
        x = bf16(rows, K, seed=rows)
        w = bf16(N, K, seed=1).to(w_dtype).requires_grad_(True)
        dy = bf16(rows, N, seed=2)
        (dw,) = torch.autograd.grad(kept8_linear(x, w), w, dy)
        k64 = R.kept_values(x)
        R.check(dw, d(dy).t() @ k64, w_dtype, product_terms(d(dy).t(), k64), "dw")


def test_linear_repeats_bit_for_bit():
    """On a busy GPU, on another stream, after other work: sums run in one order."""
    x, w, b = bf16(4099, 1024, seed=1), bf16(1544, 1024, seed=2, scale=0.03), bf16(1544, seed=3)
    dy = bf16(4099, 1544, seed=4)
    args = [t.requires_grad_(True) for t in (x, w, b)]

    def run():
        y = kept8_linear(*args)
        return (y.detach(), *torch.autograd.grad(y, args, dy))
    first, junk, side = run(), torch.empty(1 << 26, device="cuda"), torch.cuda.Stream()
    for i in range(12):
        if i % 3 == 1:
            junk.normal_()
        if i % 3 == 2:
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                got = run()
            torch.cuda.current_stream().wait_stream(side)
        else:
            got = run()
        assert all(torch.equal(p, q) for p, q in zip(first, got)), i


def test_linear_of_views():
    base, wide_w, dys = bf16(4, 50, 3, 96, seed=1), bf16(80, 120, seed=2, scale=0.1), bf16(400, 160, seed=3)
    inputs = {"aligned columns": base[..., 8:72], "odd columns": base[..., 3:67], "odd width": base[..., 5:38],
              "middle index": base[:, :, 1, :64], "transposed": base.transpose(0, 2)[..., :64],
              "three levels": base[::2, ::3, ::2, :64], "last dim strided": base[..., ::2],
              "expanded": base[:1, :, :, :64].expand(3, -1, -1, -1), "odd address": odd_copy(base[..., :64], 5),
              "one row": base[0, 0, 0, :64]}
    for name, x in inputs.items():
        K, rows = x.shape[-1], x.numel() // x.shape[-1]
        weights = {"columns": wide_w[:40, 8:8 + K], "odd columns": wide_w[:40, 1:1 + K],
                   "transposed": bf16(K, 40, seed=5, scale=0.1).t(), "odd address": odd_copy(wide_w[:33, :K])}
        for w_name, w in weights.items():
            N = w.shape[0]
            dy = dys[:, 3:3 + N].repeat(3, 1)[:rows].reshape(*x.shape[:-1], N)

            def run(x, w, dy):
                x, w = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
                y = kept8_linear(x, w)
                return (y, *torch.autograd.grad(y, (x, w), dy))
            want = run(x.contiguous(), w.contiguous(), dy.contiguous())
            for a, b in zip(want, run(x, w, dy)):
                assert a.shape == b.shape and torch.equal(a, b), (name, w_name)


NORM_FORMS = [(50, 1024), (50, 384), (50, 12288), (50, 77), (50, 1101), (50, 7001), (9, 20001), (0, 64)]


@pytest.mark.parametrize("rows,C", NORM_FORMS + [(40, -300), (40, -1500), (40, -9000)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("kept", [False, True], ids=["exact", "kept8"])
def test_norm_gradients_one_at_a_time(rows, C, dtype, kept):
    """Any subset of the gradients is the same as in all of them; a negative width is a view at an odd address."""
    x = R.activations(rows, abs(C) + 1, seed=1, dtype=dtype, device="cuda")
    x = x[:, :C].contiguous() if C > 0 else x[:, 1:]
    C = abs(C)
    w, b = (torch.linspace(lo, lo + 1, C, device="cuda").to(dtype) for lo in (0.5, -0.5))
    dy = torch.randn(rows, C, generator=torch.Generator().manual_seed(3)).to(dtype).cuda()

    def run(*need):
        args = [t.detach().requires_grad_(n) for t, n in zip((x, w, b), need)]
        y = layer_norm(*args, kept8=kept)
        wrt = [a for a in args if a.requires_grad]
        grads = iter(torch.autograd.grad(y, wrt, dy) if wrt else ())
        return y, [next(grads) if n else None for n in need]
    y, full = run(True, True, True)
    for mask in range(7):
        need = tuple(bool(mask >> i & 1) for i in range(3))
        z, some = run(*need)
        assert torch.equal(y, z), need
        for a, c in zip(full, some):
            assert c is None or torch.equal(a, c), need
