"""Tree attention over contexts of many keys that each weigh next to nothing beside one
heavy key, their values of one sign, so that what they lose adds up.

Bound: that of test_gpu_mla_tree with its 2^-25 n max |v| for subnormal weights 2^6 times
smaller: P stands 2^6 above the running maximum, so the largest P is 2^6 or more, and
half a step of a subnormal, 2^-25, is at most 2^-31 of it."""
import math

import pytest
import torch
from test_gpu_mla_tree import SCALE, call, check, make, oracle, quantise

pytestmark = pytest.mark.gpu


def tight(c):
    """oracle's bounds with 2^-31 n max |v| in place of 2^-25 n max |v|."""
    o, lse, tol, ltol = oracle(c)
    n, vmax = float(c["seq"].max()), 1.0  # the scores' dims are rope dims: in no value
    return o, lse, tol - n * vmax * 2.0 ** -25 * (1 - 2.0 ** -6), ltol


def rows(c, kv, lat):
    """Writes the latents of request 0 through its block table."""
    p = torch.arange(lat.shape[0])
    at = c["bt"][0].long()[p // c["page"]] * c["page"] + p % c["page"]
    c["rows"][at] = quantise(lat) if kv == "fp8" else lat.half()


def everywhere(pkg, c, dev):
    """The call for one request alone, cut in pieces (each with a maximum of its own), and
    for 256 copies of it, one workgroup each: whole contexts with one running maximum."""
    n = 256
    many = dict(c, q=torch.zeros(n, 128, 576).half(), bt=c["bt"].expand(n, -1).contiguous(),
                seq=c["seq"].expand(n).contiguous(), cu=torch.arange(n + 1, dtype=torch.int32),
                mask=torch.ones(n, dtype=torch.int64))
    H = c["q"].shape[1]
    many["q"][:, :H] = c["q"]
    o, lse = call(pkg, many, dev)
    assert torch.equal(o, o[:1].expand_as(o)) and torch.equal(lse, lse[:1].expand_as(lse))
    want = tight(c)
    check((o[:1, :H], lse[:1, :H]), want)
    check(call(pkg, c, dev), want)
    return want


@pytest.mark.parametrize("kv", ["fp16", "fp8"])
@pytest.mark.parametrize("n,heavy", [(5000, 0), (40000, 0), (40000, 20000), (40000, 39998)])
def test_one_heavy_key(pkg, lib, dev, kv, n, heavy):
    """Every other key at 2^-25.2 (or 2^-24) of the heavy one, values 1: at 40000 keys they
    make o = 0.00104, with 0 where they are lost."""
    c = make([n], [1], 2, 64, kv, seed=41)
    lat = torch.zeros(n, 576)
    lat[:, :512] = 1.0
    lat[heavy, :512] = 0.0
    lat[heavy, 512] = 16.0
    rows(c, kv, lat)
    c["q"].zero_()
    c["q"][:, 0, 512] = 25.2 * math.log(2.0) / SCALE / 16
    c["q"][:, 1, 512] = 24.0 * math.log(2.0) / SCALE / 16
    want = everywhere(pkg, c, dev)
    assert 1e-4 < float(want[0][0, 0, 5]) < 2e-3


@pytest.mark.parametrize("kv", ["fp16", "fp8"])
def test_weights_of_all_sizes(pkg, lib, dev, kv):
    """Scores spread evenly over 40 octaves, heaviest first, last or in between."""
    n = 20000
    c = make([n], [1], 3, 64, kv, seed=42)
    lat = torch.ones(n, 576)
    x = torch.linspace(-1, 1, n)
    lat[:, 512], lat[:, 513], lat[:, 514] = x, -x, 1 - 2 * x.abs()
    rows(c, kv, lat)
    c["q"].zero_()
    for h in range(3):
        c["q"][:, h, 512 + h] = 20.0 * math.log(2.0) / SCALE
    everywhere(pkg, c, dev)


def test_long_context(pkg, lib, dev):
    n = 184320
    c = make([n], [1], 2, 64, "fp16", seed=43)
    lat = torch.ones(n, 576)
    lat[:, 512] = 0.0
    lat[0, :512] = 0.0
    lat[0, 512] = 16.0
    rows(c, "fp16", lat)
    c["q"].zero_()
    c["q"][:, :, 512] = 25.2 * math.log(2.0) / SCALE / 16
    check(call(pkg, c, dev), tight(c))
