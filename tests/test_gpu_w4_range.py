"""4-bit products of bf16 x at the ends of its range against the formula in 64 bits.

Tolerance: the sums t of x (16 + c) and X of x, whose multiple 16 + z comes off, have terms of
at most 31 |x|, each of up to 128 additions off by 2^-23 of what it has reached; then one
addition a group, slice and wave; y is rounded once more, half a step."""
import pytest
import torch
from test_gpu_w4 import BF16, given, spread, value

pytestmark = pytest.mark.gpu
EPS = torch.finfo(BF16).eps / 2


def run(pkg, dev, x, c, s, z, group):
    w = pkg.w4.w4_pack(c.to(dev), s.to(dev), z.to(dev), group)
    y = pkg.w4.w4_linear(x.to(dev), w).double().cpu()
    k = c.shape[1]
    want = x.double() @ value(c, s, z, group).T
    reach = 31 * (x.double().abs() @ spread(s.double(), group, k).T)
    return y, want, EPS * want.abs() + (2 * 131 + -(-k // group) + 16) * 2.0 ** -23 * reach


@pytest.mark.parametrize("m,n,k,group", [(1, 40, 512, 128), (16, 40, 512, 32), (30, 33, 264, 64),
                                         (64, 40, 512, 128), (9, 100, 24576, 128)])
def test_largest_values_of_x(pkg, lib, dev, m, n, k, group):
    """x up to the largest of its type, with scales that keep y far inside: no infinity comes of
    a sum before its scale."""
    c, s, z = given(n, k, group, BF16, seed=n)
    s = s * 2.0 ** -12
    x = torch.finfo(BF16).max * (torch.rand(m, k, generator=torch.Generator().manual_seed(m)) * 2 - 1)
    x = x.to(BF16)
    x[0] = torch.finfo(BF16).max
    y, want, tol = run(pkg, dev, x, c, s, z, group)
    assert float(want.abs().max()) < 2.0 ** 126
    assert bool(y.isfinite().all()) and bool(((y - want).abs() <= tol).all())


@pytest.mark.parametrize("m", [1, 16, 30, 64])
def test_a_large_value_at_weights_of_zero(pkg, lib, dev, m):
    """Where code and zero point agree the term is 0, up to the rounding of the sums."""
    c, s, z = given(40, 264, 64, BF16, seed=m)
    c[:, 5] = z[:, 0]
    x = torch.randn(m, 264, generator=torch.Generator().manual_seed(m)).to(BF16)
    x[:, 5] = 2.0 ** 127
    y, want, tol = run(pkg, dev, x, c, s, z, 64)
    assert bool(y.isfinite().all()) and bool(((y - want).abs() <= tol).all())


@pytest.mark.parametrize("m", [1, 16, 30, 64])
@pytest.mark.parametrize("e", [-100, -114, -122])
def test_small_values_of_x(pkg, lib, dev, m, e):
    """x of at least 2^(e - 3), down to the least normal number: what is summed may be 2^-8 of it,
    multiples of 2^-145; each of the five groups' parts of y is rounded, at 2^-138."""
    c, s, z = given(40, 264, 64, BF16, seed=m)
    x = torch.randn(m, 264, generator=torch.Generator().manual_seed(m))
    x = torch.where(x.abs() < 2.0 ** -3, 1.0, x) * 2.0 ** e
    y, want, tol = run(pkg, dev, x.to(BF16), c, s, z, 64)
    assert bool(((y - want).abs() <= tol + 5 * 2.0 ** -138).all())


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_a_bad_value_stays_in_its_row(pkg, lib, dev, bad):
    c, s, z = given(40, 264, 64, BF16, seed=7)
    x = torch.randn(18, 264, generator=torch.Generator().manual_seed(7)).to(BF16)
    good, want, tol = run(pkg, dev, x, c, s, z, 64)
    x[3, 100] = x[17, 7] = bad
    y, _, _ = run(pkg, dev, x, c, s, z, 64)
    rest = [i for i in range(18) if i not in (3, 17)]
    assert torch.equal(y[rest], good[rest]) and bool(y[[3, 17]].isnan().all())
    assert bool(((y - want).abs() <= tol)[rest].all())
