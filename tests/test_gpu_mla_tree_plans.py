"""Tree attention where its work is cut in other ways than by cells of one segment: more
row groups than workgroups, uneven lengths, block tables longer than a segment, and
drafted tokens over several tiles.  Bounds as in test_gpu_mla_tree."""
import math

import pytest
import torch
from test_gpu_mla_tree import SCALE, cache, call, check, make, oracle

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kv", ["fp16", "fp8"])
def test_more_groups_than_workgroups(pkg, lib, dev, kv):
    """300 requests, one or two groups each: every workgroup takes several pieces."""
    lens = [(53 * i) % 310 for i in range(300)]
    counts = [min(1 + (7 * i) % 9, n) for i, n in enumerate(lens)]
    c = make(lens, counts, 16, 16, kv, seed=31)
    check(call(pkg, c, dev), oracle(c))


@pytest.mark.parametrize("kv", ["fp16", "fp8"])
def test_long_request_among_many_short_ones(pkg, lib, dev, kv):
    """Groups cut into many pieces of the line of tiles."""
    c = make([6000] + [40 + i % 7 for i in range(270)], [16] + [1] * 270, 64, 64, kv, seed=32,
             spread=2.0)
    check(call(pkg, c, dev), oracle(c))


@pytest.mark.parametrize("kv", ["fp16", "fp8"])
def test_a_page_for_every_key(pkg, lib, dev, kv):
    """Pages of one key: a workgroup's block table does not fit at once.  The same rows in
    pages of 64 give the same bits."""
    n, H = 8, 128
    c = make([70000], [n], H, 64, kv, seed=33)
    a = call(pkg, c, dev)
    one = dict(c, page=1)
    p = torch.arange(70000)
    one["bt"] = (c["bt"][0].long()[p // 64] * 64 + p % 64).int()[None]
    b = call(pkg, one, dev)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    few = dict(c, q=c["q"][:, ::43])
    assert few["q"].shape[1] == 3
    check((a[0][:, ::43], a[1][:, ::43]), oracle(few))


@pytest.mark.parametrize("kv", ["fp16", "fp8"])
@pytest.mark.parametrize("H", [1, 5, 32])
@pytest.mark.parametrize("n", [33, 64])
def test_bad_rows_in_trees_over_several_tiles(pkg, lib, dev, kv, H, n):
    """NaN and infinities in drafted rows of two or three tiles: rows that see one are NaN,
    the others as if it were not there."""
    c = make([n + 20, n, 200], [n, n, n], H, 16, kv, seed=34 + n)
    want = oracle(c)
    g = torch.Generator().manual_seed(n)
    hit = torch.zeros(3 * n, dtype=torch.bool)
    for r, L in enumerate(c["seq"].tolist()):
        for i in torch.randperm(n - 1, generator=g)[:4].tolist():
            i += 1  # not the first token: some rows see none of them
            pos = L - n + i
            row = int(c["bt"][r, pos // 16]) * 16 + pos % 16
            v = [math.nan, math.inf, -math.inf][i % 3]
            if kv == "fp8":
                c["rows"][row, 512 + 4 * (i % 4):516 + 4 * (i % 4)].view(torch.float32)[0] = v
            else:
                c["rows"][row, (97 * i) % 576] = v
            for j in range(n):
                hit[r * n + j] |= bool((int(c["mask"][r * n + j]) >> i) & 1)
    o, lse = call(pkg, c, dev)
    assert bool(torch.isnan(o[hit].float().sum(2)).all()) and bool(torch.isnan(lse[hit]).all())
    assert 0 < int(hit.sum()) < 3 * n
    check((o, lse), want, ~hit)


def test_two_streams_at_once(pkg, lib, dev):
    """Calls that overlap on two streams, each with its own workspace."""
    c = [make([5000, 77], [5, 9], 64, 64, "fp16", seed=35),
         make([3000, 4000], [8, 3], 32, 16, "fp8", seed=36)]
    args = [[x["q"].to(dev), cache(x, dev), x["bt"].to(dev), x["seq"].to(dev), x["cu"].to(dev),
             x["mask"].to(dev), SCALE] for x in c]
    f = pkg.mla_tree.tree_attention
    want = [f(*a) for a in args]
    st = [torch.cuda.Stream() for _ in c]
    torch.cuda.synchronize()
    got = []
    for k in range(12):
        with torch.cuda.stream(st[k % 2]):
            got.append(f(*args[k % 2]))
    torch.cuda.synchronize()
    for k, (o, lse) in enumerate(got):
        assert torch.equal(o, want[k % 2][0]) and torch.equal(lse, want[k % 2][1])
