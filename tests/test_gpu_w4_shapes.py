"""4-bit products at sizes that choose every number of tiles of a workgroup (2, 3 and 6) in each
class of rows, with tile counts that it does not divide, whole and with K cut in slices, in
every group size and type.  Sums are exact as in test_gpu_w4, so y is held bit for bit."""
import pytest
import torch
from test_gpu_w4 import BF16, F16, given, value

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("m", [13, 29, 61])
@pytest.mark.parametrize("n,k", [
    (8313, 136),                  # 520 tiles by 3
    (16529, 136),                 # 1034 tiles by 6
    (590, 12312),                 # 37 tiles by 2, eight slices of 97 blocks
    (600, 24584),                 # 38 tiles by 3, sixteen slices
    (2150, 12312)])               # 135 tiles by 6, eight slices
def test_exact_sums(pkg, lib, dev, m, n, k, group, dt):
    c, s, z = given(n, k, group, dt, seed=m + n + k, exact=True)
    x = torch.randint(-4, 5, (m, k), generator=torch.Generator().manual_seed(k)).to(dt).to(dev)
    c, s, z = c.to(dev), s.to(dev), z.to(dev)
    y = pkg.w4.w4_linear(x, pkg.w4.w4_pack(c, s, z, group))
    v = value(c, s, z, group)
    # units of 2^-7: below 2^24 of them every sum is exact
    assert float((x.abs().double() @ v.abs().t().contiguous()).max()) * 128 < 2 ** 24
    assert torch.equal(y, (x.double() @ v.t().contiguous()).to(dt))
