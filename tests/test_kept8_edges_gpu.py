"""8-bit operators on a B200 where a call comes in an unusual form: views at odd addresses, empty batches, widths of
the forms that other tests do not reach, threads."""
import pytest
import torch

import kept8_ref as R
from pan2_b200.ops.kept8 import kept8_linear

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
