"""Tree attention with scores far past the range in which a softmax weighs anything but the
largest: whole numbers whose dot products are exact in fp32, under scales from 1e3 to
1e30, and rows and pieces that see nothing under such a scale.

Scores differ by whole units, so every weight is 0 or that of the largest: o is the value
of the largest key (or the mean of several equal ones), exact but for one rounding of it
to fp16 and, where several are joined, of 1 / l; lse = scale max + ln count, to 2^-22 of
its size (fp32: log2 e times the scale, the product, ln 2 times it, half a step each)."""
import math

import pytest
import torch
from test_gpu_mla_tree import H16, call, make

pytestmark = pytest.mark.gpu


def case(lens, counts, H, kv, seed):
    c = make(lens, counts, H, 16, kv, seed=seed)
    g = torch.Generator().manual_seed(seed)
    n = c["rows"].shape[0]
    lat = torch.randint(-8, 9, (n, 576), generator=g).half()
    if kv == "fp8":  # whole numbers under a scale of 1
        one = torch.ones(n, 4).view(torch.uint8)
        c["rows"] = torch.cat([lat[:, :512].float().to(torch.float8_e4m3fn).view(torch.uint8), one,
                               lat[:, 512:].contiguous().view(torch.uint8)], 1)
    else:
        c["rows"] = lat
    c["q"] = torch.randint(-8, 9, c["q"].shape, generator=g).half()
    return c, lat.double()


def expected(c, lat, scale):
    T, H = c["q"].shape[:2]
    o, lse = torch.zeros(T, H, 512, dtype=torch.float64), torch.full((T, H), -math.inf, dtype=torch.float64)
    for r in range(len(c["seq"])):
        a, b, L = int(c["cu"][r]), int(c["cu"][r + 1]), int(c["seq"][r])
        for t in range(a, b):
            ctx = L - (b - a)
            see = [p for p in range(L) if p < ctx or int(c["mask"][t]) >> (p - ctx) & 1]
            if not see:
                continue
            p = torch.tensor(see)
            K = lat[c["bt"][r].long()[p // 16] * 16 + p % 16]
            s = c["q"][t].double() @ K.T * math.copysign(1, scale)
            top = s == s.amax(1, keepdim=True)
            o[t] = top.double() @ K[:, :512] / top.sum(1, keepdim=True)
            lse[t] = s.amax(1) * abs(scale) + top.sum(1).double().log()
    return o, lse


@pytest.mark.parametrize("kv", ["fp16", "fp8"])
@pytest.mark.parametrize("scale", [1e3, 1e6, -1e6, 3e8, 1e30])
def test_the_largest_alone(pkg, lib, dev, kv, scale):
    c, lat = case([200, 33, 5, 1500], [5, 3, 5, 2], 16, kv, 61)
    c["mask"][8] = 0  # no context and no token: nothing
    o, lse = call(pkg, c, dev, scale)
    wo, wl = expected(c, lat, scale)
    o, lse = o.double().cpu(), lse.double().cpu()
    assert bool(torch.isinf(wl[8]).all()) and bool((o[8] == 0).all()) and bool((lse[8] == -math.inf).all())
    live = torch.arange(15) != 8
    assert bool(((o - wo).abs() <= (H16 + 2.0 ** -22) * wo.abs()).all())
    assert bool(((lse - wl)[live].abs() <= 2.0 ** -22 * wl[live].abs() + 1e-6).all())


@pytest.mark.parametrize("kv", ["fp16", "fp8"])
def test_pieces_that_see_nothing(pkg, lib, dev, kv):
    """Most of a cut context has no pages."""
    c, lat = case([3000], [2], 16, kv, 62)
    c["bt"][0, 3:180] = -1
    keep = c["bt"].clone()
    o, lse = call(pkg, c, dev, 1e30)
    p = torch.arange(3000)
    p = p[(p // 16 < 3) | (p // 16 >= 180)]
    for t in range(2):
        see = p[(p < 2998) | ((c["mask"][t] >> (p - 2998).clamp(0)) & 1 == 1)]
        K = lat[keep[0].long()[see // 16] * 16 + see % 16]
        s = c["q"][t].double() @ K.T
        top = s == s.amax(1, keepdim=True)
        want = top.double() @ K[:, :512] / top.sum(1, keepdim=True)
        assert bool(((o[t].double().cpu() - want).abs() <= (H16 + 2.0 ** -22) * want.abs()).all())
        assert bool(torch.isfinite(lse[t]).all())
