"""4-bit projections (w4.py) against their formulas in 64 bits.

With small integers for x and powers of two for the scales every sum is exact in fp32,
so y is RN of the exact product, bit for bit.  With ordinary values: a group's sums t and
X have up to 128 terms of at most 31 |x|, each addition off by at most 2^-23 of what it
has reached (the matrix unit need not round to nearest), then one addition a group and
wave; y is rounded once more, half a step."""
import pytest
import torch

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


def spread(x, group, k):
    return x.repeat_interleave(group, 1)[:, :k]


def given(n, k, group, dt, zeros=True, seed=0, exact=False):
    g = torch.Generator().manual_seed(seed)
    kg = -(-k // group)
    c = torch.randint(0, 16, (n, k), generator=g, dtype=torch.uint8)
    z = torch.randint(0, 16, (n, kg), generator=g, dtype=torch.uint8) if zeros else None
    s = 2.0 ** -torch.randint(5, 8, (n, kg), generator=g) if exact else \
        (torch.rand(n, kg, generator=g) + 0.5) * 0.2 * max(k, 1) ** -0.5
    return c, s.to(dt), z


def value(c, s, z, group):
    k = c.shape[1]
    z = torch.full(s.shape, 8.0) if z is None else z.double()
    return (c.double() - spread(z.double(), group, k)) * spread(s.double(), group, k)


SIZES = [(1, 16, 128), (1, 1, 8), (2, 17, 136), (5, 100, 1000), (16, 48, 64), (17, 33, 2048),
         (33, 40, 264), (64, 300, 3000), (64, 15, 8), (3, 2112, 6144)]


@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("m,n,k", SIZES)
def test_exact_sums(pkg, lib, dev, m, n, k, group, dt):
    c, s, z = given(n, k, group, dt, zeros=(n + group) % 3 > 0, seed=m + n + k, exact=True)
    g = torch.Generator().manual_seed(k)
    x = torch.randint(-4, 5, (m, k), generator=g).to(dt)
    w = pkg.w4.w4_pack(c.to(dev), s.to(dev), None if z is None else z.to(dev), group)
    y = pkg.w4.w4_linear(x.to(dev), w)
    # units of 2^-7: below 2^24 of them every sum is exact
    assert float((x.abs().double() @ value(c, s, z, group).abs().T).max()) * 128 < 2 ** 24
    want = (x.double() @ value(c, s, z, group).T).to(dt)
    assert y.dtype == dt and torch.equal(y.cpu(), want)


@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("m,n,k,group", [(1, 700, 24576, 128), (4, 2112, 6144, 64), (64, 500, 6144, 128),
                                         (31, 97, 4104, 32)])
def test_ordinary_values(pkg, lib, dev, m, n, k, group, dt):
    c, s, z = given(n, k, group, dt, seed=n)
    x = torch.randn(m, k, generator=torch.Generator().manual_seed(m)).to(dt)
    w = pkg.w4.w4_pack(c.to(dev), s.to(dev), z.to(dev), group)
    y = pkg.w4.w4_linear(x.to(dev), w).double().cpu()
    want = x.double() @ value(c, s, z, group).T
    reach = 31 * (x.double().abs() @ spread(s.double(), group, k).T)
    tol = torch.finfo(dt).eps / 2 * want.abs() + (2 * 131 + -(-k // group) + 16) * 2.0 ** -23 * reach
    assert bool(((y - want).abs() <= tol).all())
    # and far closer than that on the whole: errors that add like a random walk
    rms = (y - want).pow(2).mean().sqrt() / want.pow(2).mean().sqrt()
    assert rms <= torch.finfo(dt).eps / 2


@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("n,k,group", [(1, 8, 32), (17, 136, 128), (33, 1000, 64), (100, 264, 32)])
def test_pack_and_dequant(pkg, lib, dev, n, k, group, dt):
    """Every code and zero point comes back, high bits of a given code are not looked at."""
    c, s, z = given(n, k, group, dt, seed=k)
    w = pkg.w4.w4_pack((c | 0xa0).to(dev), s.to(dev), z.to(dev), group)
    assert torch.equal(pkg.w4.w4_dequant(w).cpu(), value(c, s, z, group).to(dt))


def quantised(w, group, symmetric):
    n, k = w.shape
    kg = -(-k // group)
    v = torch.zeros(n, kg * group, dtype=torch.float64)
    v[:, :k] = w.double()
    v = v.view(n, kg, group)
    lo, hi = v.amin(2).clamp(max=0), v.amax(2).clamp(min=0)
    s = torch.maximum(hi / 7, -lo / 8) if symmetric else (hi - lo) / 15
    s = s.float().to(w.dtype).double().clamp_min(2.0 ** -24 if w.dtype == F16 else 2.0 ** -126)
    z = torch.full_like(s, 8) if symmetric else torch.round(-lo / s).clamp(0, 15)
    c = (torch.round(v / s[:, :, None]) + z[:, :, None]).clamp(0, 15)
    return ((c - z[:, :, None]) * s[:, :, None]).view(n, -1)[:, :k].to(w.dtype)


@pytest.mark.parametrize("symmetric", [False, True])
@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("n,k,group", [(1, 8, 128), (16, 128, 128), (50, 1000, 64), (130, 264, 32),
                                       (64, 6144, 128)])
def test_quantize(pkg, lib, dev, n, k, group, dt, symmetric):
    g = torch.Generator().manual_seed(n + k)
    w = torch.randn(n, k, generator=g) * torch.rand(n, 1, generator=g)
    w[:, : k // 3] += 0.7       # groups on one side of 0
    w = (w * (1e-6 if n == 50 else 1.0)).to(dt)   # fp16: subnormal weights and scales
    w[0] = 0                    # a range of nothing
    if n > 1:
        w[1, :] = torch.finfo(dt).max
        w[1, 1::2] = -torch.finfo(dt).max
    got = pkg.w4.w4_dequant(pkg.w4.w4_quantize(w.to(dev), group, symmetric))
    assert torch.equal(got.cpu(), quantised(w, group, symmetric))


def test_quantised_weights_multiply(pkg, lib, dev):
    g = torch.Generator().manual_seed(3)
    w, x = torch.randn(200, 1024, generator=g).half().to(dev), torch.randn(7, 1024, generator=g).half().to(dev)
    q = pkg.w4.w4_quantize(w)
    y = pkg.w4.w4_linear(x, q)
    want = x.double() @ pkg.w4.w4_dequant(q).double().T   # weights rounded to fp16 there
    reach = x.double().abs() @ w.double().abs().T
    assert bool(((y.double() - want).abs() <= 2.0 ** -10 * want.abs() + 2.0 ** -11 * reach).all())


def test_strided_unaligned_and_given_output(pkg, lib, dev):
    c, s, z = given(40, 256, 128, F16, seed=4, exact=True)
    x = torch.randint(-4, 5, (6, 256)).half()
    want = (x.double() @ value(c, s, z, 128).T).half()
    w = pkg.w4.w4_pack(c.t().contiguous().t().to(dev), s.to(dev), z.to(dev))
    wide = torch.full((6, 300), float("nan"), dtype=F16, device=dev)
    for at in (0, 8, 9, 3):
        v = wide[:, at:at + 256]
        v.copy_(x)
        assert torch.equal(pkg.w4.w4_linear(v, w).cpu(), want)
    one = torch.empty(257, dtype=F16, device=dev)[1:].view(1, 256)   # one row off 16 bytes
    one.copy_(x[:1])
    out = torch.full((1, 40), 7.0, dtype=F16, device=dev)
    assert pkg.w4.w4_linear(one, w, out) is out and torch.equal(out.cpu(), want[:1])


def test_infinities_stay_in_their_row(pkg, lib, dev):
    c, s, z = given(40, 256, 128, F16, seed=5, exact=True)
    x = torch.randint(-4, 5, (18, 256)).half()
    want = (x.double() @ value(c, s, z, 128).T).half()
    w = pkg.w4.w4_pack(c.to(dev), s.to(dev), z.to(dev))
    x[3, 100], x[17, 7] = float("nan"), float("inf")
    y = pkg.w4.w4_linear(x.to(dev), w).cpu()
    rest = [i for i in range(18) if i not in (3, 17)]
    assert torch.equal(y[rest], want[rest]) and not bool(torch.isfinite(y[[3, 17]]).any())


def test_empty(pkg, lib, dev):
    w = pkg.w4.w4_quantize(torch.randn(8, 64, device=dev).half())
    assert pkg.w4.w4_linear(torch.empty(0, 64, dtype=F16, device=dev), w).shape == (0, 8)
    w = pkg.w4.w4_quantize(torch.empty(0, 64, dtype=F16, device=dev))
    assert pkg.w4.w4_linear(torch.ones(2, 64, dtype=F16, device=dev), w).shape == (2, 0)
    w = pkg.w4.w4_quantize(torch.empty(8, 0, dtype=F16, device=dev))
    assert pkg.w4.w4_linear(torch.ones(2, 0, dtype=F16, device=dev), w).tolist() == [[0.0] * 8] * 2
    assert pkg.w4.w4_dequant(w).shape == (8, 0)


def test_captured_and_other_stream(pkg, lib, dev):
    c, s, z = given(100, 512, 64, BF16, seed=6, exact=True)
    w = pkg.w4.w4_pack(c.to(dev), s.to(dev), z.to(dev), 64)
    x = torch.zeros(5, 512, dtype=BF16, device=dev)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        pkg.w4.w4_linear(x, w)
    st.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = pkg.w4.w4_linear(x, w)
    for i in range(4):
        v = torch.randint(-4, 5, (5, 512), generator=torch.Generator().manual_seed(i)).to(BF16)
        x.copy_(v)
        graph.replay()
        eager = pkg.w4.w4_linear(x, w)
        torch.cuda.synchronize()
        assert torch.equal(y, eager)
        assert torch.equal(y.cpu(), (v.double() @ value(c, s, z, 64).T).to(BF16))
