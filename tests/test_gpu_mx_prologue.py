"""The MX8 prologue's row statistic and its launch shapes on a B200, value by value.

With a weight of one, normed is RN(fl32(x * r)), r = fl32(1 / sqrt(mean x^2 + eps)).  The
mean is summed in 64 bits and its root taken there, which leaves the rounding of r, 2^-24
relative, the fp32 product's, another 2^-24 where the type is narrower than fp32, and the
rounding to the type, half of its step at the value.  `check_unit` holds every value to that
sum; nothing is averaged.  A row whose squares leave fp32's range is scaled by 2^-64 or 2^64
before the product, which is exact but for elements that become subnormal there: at most
2^-145 of the result."""
from __future__ import annotations

import pytest
import torch

from easyinfra_b200 import ops

pytestmark = pytest.mark.gpu
bf = torch.bfloat16


def gen(device, seed):
    return torch.Generator(device=device).manual_seed(seed)


def check_unit(nm, x, eps):
    """nm against x / sqrt(mean x^2 + eps) in 64 bits (a weight of one)."""
    d = x.double()
    e = d / torch.sqrt(d.square().mean(-1, keepdim=True) + eps)
    digits, tiny, extra = (8, -133, 2.001) if x.dtype == bf else (24, -149, 1.001)
    exponent = torch.frexp(e.abs() * (1 + 2.0 ** -22)).exponent.double()     # |e| = m 2^exponent, m in [0.5, 1)
    half = torch.exp2((exponent - digits).clamp_min(tiny) - 1)
    half = torch.where(e == 0, torch.zeros_like(half), half)
    err = (nm.double() - e).abs()
    tol = half + extra * 2.0 ** -24 * e.abs() + 2.0 ** -145
    assert torch.isfinite(nm).all() and (err <= tol).all(), (int((err > tol).sum()), float((err / tol).max()))


def run(x, add, eps, weight=None, **kw):
    """The prologue of rows x, as residual + hidden with half of the rows in either."""
    w = torch.ones(x.shape[1], dtype=x.dtype, device=x.device) if weight is None else weight
    if not add:
        return ops.add_rmsnorm_mx8(x, None, w, eps, **kw)
    first = (torch.arange(x.shape[0], device=x.device) % 2 == 0)[:, None]
    return ops.add_rmsnorm_mx8(torch.where(first, x, 0), torch.where(first, 0, x), w, eps, **kw)


@pytest.mark.parametrize("dtype", [bf, torch.float32])
@pytest.mark.parametrize("T", [333, 4801])
@pytest.mark.parametrize("add", [True, False])
def test_statistic_under_a_loud_channel(cuda_device, T, dtype, add):
    """One loud channel, beside it channels whose squares are just under half a unit in the
    last place of its square in fp32: a sum in fp32 loses every one of them.  (The others give
    every row a root of its own, so that some bf16 values lie next to a border.)"""
    d, H = cuda_device, 1024
    g = gen(d, T)
    x = 0.03 * torch.randn(T, H, generator=g, device=d)
    V = 8 if dtype == bf else 4
    s = 0.99609375 * 2.0 ** -8 if dtype == bf else (1 - 2.0 ** -12) * 2.0 ** -8
    x.view(T, H // V, V)[:, ::32] = s
    x[:, 0] = 16 + 0.125 * torch.randint(0, 49, (T,), generator=g, device=d)  # squares in [256, 512): units of 2^-15
    x = x.to(dtype)
    ro, nm, q = run(x, add, 1e-6)
    assert torch.equal(ro, x)
    check_unit(nm, x, 1e-6)
    assert torch.equal(q.buf, ops.quantize_mx8(nm).buf)


@pytest.mark.parametrize("dtype", [bf, torch.float32])
@pytest.mark.parametrize("eps", [0.0, 1e-6])
def test_rows_beyond_the_squares_of_fp32(cuda_device, dtype, eps):
    """Finite rows from the smallest to the largest magnitudes, whose squares overflow or
    vanish in fp32."""
    d, H = cuda_device, 512
    x = torch.randn(64, H, generator=gen(d, 9), device=d).clamp(-3.9, 3.9).double()
    scale = torch.linspace(-126, 126, 64, device=d).round()
    x = (x * torch.exp2(scale.double())[:, None]).to(dtype)
    x[5, 7] = torch.finfo(dtype).max              # one value over all others
    x[6] = torch.finfo(dtype).max
    x[7] = torch.finfo(dtype).smallest_normal
    assert torch.isfinite(x).all()
    for add in (False, True):
        ro, nm, q = run(x, add, eps)
        assert torch.equal(ro, x)
        check_unit(nm, x, eps)
        assert torch.equal(q.buf, ops.quantize_mx8(nm).buf)


def test_rows_that_are_not_finite(cuda_device):
    """An infinity makes the row's mean infinite and a NaN makes all of it NaN, as the formula
    says; the other rows are as without them."""
    d = cuda_device
    x = torch.randn(9, 256, generator=gen(d, 1), device=d).to(bf)
    want = run(x, False, 1e-6)[1]
    x[2, 5], x[4, 9], x[6, 0] = float("inf"), float("nan"), float("-inf")
    nm = run(x, False, 1e-6)[1]
    rest = [0, 1, 3, 5, 7, 8]
    assert torch.equal(nm[rest], want[rest])
    assert torch.isnan(nm[4]).all()
    for r, c in ((2, 5), (6, 0)):
        assert torch.isnan(nm[r, c]) and int((nm[r] == 0).sum()) == 255


# 1201 tokens are more than eight per SM, which takes four vectors a thread instead of one;
# wide rows take two or four at any batch.
@pytest.mark.parametrize("dtype", [bf, torch.float32])
@pytest.mark.parametrize("T,H", [(1201, 32), (1201, 96), (1201, 1408), (1201, 4096), (1300, 8192), (2, 8192), (3, 16384)])
@pytest.mark.parametrize("add", [True, False])
def test_launch_shapes(cuda_device, T, H, dtype, add):
    if dtype == torch.float32 and H > 8192:
        pytest.skip("rows of up to 32 KB")
    d = cuda_device
    g = gen(d, T + H)
    x = (2 * torch.randn(T, H, generator=g, device=d)).to(dtype)
    ro, nm, q = run(x, add, 1e-6)
    assert torch.equal(ro, x)
    check_unit(nm, x, 1e-6)
    assert torch.equal(q.buf, ops.quantize_mx8(nm).buf)           # codes, scales and padding
    # another weight: the same unit row, one product and one rounding (exact in 64 bits)
    w = (1 + 0.2 * torch.randn(H, generator=g, device=d)).to(dtype)
    nm2, q2 = run(x, add, 1e-6, w)[1:]
    assert torch.equal(nm2, (nm.double() * w.double()).to(dtype))
    assert torch.equal(q2.buf, ops.quantize_mx8(nm2).buf)
    # without normed rows, and in place
    ro3, none, q3 = run(x, add, 1e-6, w, norm=False)
    assert none is None and torch.equal(q3.buf, q2.buf) and torch.equal(ro3, x)
    z = x.clone()
    ro4, _, q4 = ops.add_rmsnorm_mx8(z, None, w, 1e-6, residual_out=z)
    assert ro4 is z and torch.equal(z, x) and torch.equal(q4.buf, q2.buf)
