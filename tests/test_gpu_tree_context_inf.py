"""Infinities in context rows, which every row of a request sees, count as numbers do: a
score of -inf weighs nothing.  Also where the context's last keys share a tile with drafted
tokens, whose own bad rows are NaN to those that see them."""
import math

import pytest
import torch
from test_gpu_mla_tree import call, check, make, oracle

pytestmark = pytest.mark.gpu


def put(c, r, pos, v):
    """v into rope dim 7 of position pos."""
    row = int(c["bt"][r, pos // c["page"]]) * c["page"] + pos % c["page"]
    if c["rows"].dtype == torch.uint8:
        c["rows"][row, 528:].view(torch.float16)[7] = v
    else:
        c["rows"][row, 519] = v


@pytest.mark.parametrize("kv", ["fp16", "fp8"])
@pytest.mark.parametrize("H", [3, 64])
@pytest.mark.parametrize("pos", [3, 31, 32, 40, 53])
def test_minus_infinity_weighs_nothing(pkg, lib, dev, kv, H, pos):
    """As a score far below the others, bit for bit; 54 context keys, so that those from 32
    on are in the first drafted token's tile."""
    c = make([60, 33], [6, 2], H, 16, kv, seed=51)
    check(call(pkg, c, dev), oracle(c))
    c["q"][:, :, 519] = 4.0
    put(c, 0, pos, -30000.0)  # times 4 times the scale: -8660
    far = call(pkg, c, dev)
    assert bool(torch.isfinite(far[0]).all())
    put(c, 0, pos, -math.inf)
    got = call(pkg, c, dev)
    assert torch.equal(got[0], far[0]) and torch.equal(got[1], far[1])
    put(c, 0, 55, -math.inf)  # drafted token 1: NaN to itself and to those below it
    o = call(pkg, c, dev)[0]
    see = (c["mask"][:6] >> 1) & 1 == 1
    assert bool(torch.isnan(o[:6][see]).all()) and bool(see[1])
    assert torch.equal(o[:6][~see], got[0][:6][~see]) and torch.equal(o[6:], got[0][6:])


@pytest.mark.parametrize("kv", ["fp16", "fp8"])
@pytest.mark.parametrize("pos", [3, 40])
@pytest.mark.parametrize("v", [math.inf, math.nan])
def test_infinity_and_nan_are_seen_by_all(pkg, lib, dev, kv, pos, v):
    c = make([60, 33], [6, 2], 16, 16, kv, seed=52)
    c["q"][:, :, 519] = 4.0
    want = oracle(c)
    put(c, 0, pos, v)
    o, lse = call(pkg, c, dev)
    assert bool(torch.isnan(o[:6]).all())
    live = torch.tensor([False] * 6 + [True] * 2)
    check((o, lse), want, live)
