"""A request's result does not depend on the requests beside it: alone, among copies of
itself and among other lengths, however the work is then divided (cells of keys, runs of
the line of tiles with partials on both sides).  Each is held to the definition's bounds,
and the same batch twice gives the same bits."""
import pytest
import torch
from test_gpu_mla_tree import call, check, make, oracle

pytestmark = pytest.mark.gpu


def batch(one, lens, counts, at, H, kv, seed):
    """Requests of `lens` and `counts` with `one` put in at the places `at`; the cache holds
    the pages of all of them."""
    c = make(lens, counts, H, one["page"], kv, seed=seed)
    n = c["rows"].shape[0] // c["page"]
    bt1 = torch.where(one["bt"] >= 0, one["bt"] + n, one["bt"])
    width = max(c["bt"].shape[1], bt1.shape[1])

    def wide(t):
        return torch.cat([t, torch.full((t.shape[0], width - t.shape[1]), -1, dtype=torch.int32)], 1)

    q, bt, seq, mask, cnt, places = [], [], [], [], [], []
    cu = c["cu"].tolist()
    for i in range(len(lens) + len(at)):
        if i in at:
            places.append(sum(cnt))
            q.append(one["q"])
            bt.append(wide(bt1))
            seq.append(int(one["seq"][0]))
            mask.append(one["mask"])
            cnt.append(one["q"].shape[0])
        else:
            r = i - sum(1 for a in at if a < i)
            q.append(c["q"][cu[r]:cu[r + 1]])
            bt.append(wide(c["bt"][r:r + 1]))
            seq.append(lens[r])
            mask.append(c["mask"][cu[r]:cu[r + 1]])
            cnt.append(counts[r])
    out = dict(q=torch.cat(q), rows=torch.cat([c["rows"], one["rows"]]), page=c["page"],
               bt=torch.cat(bt), seq=torch.tensor(seq, dtype=torch.int32), mask=torch.cat(mask),
               cu=torch.tensor([sum(cnt[:i]) for i in range(len(cnt) + 1)], dtype=torch.int32))
    return out, places


@pytest.mark.parametrize("kv", ["fp16", "fp8"])
@pytest.mark.parametrize("H", [16, 64])
def test_alone_and_among_others(pkg, lib, dev, H, kv):
    one = make([3000], [5], H, 64, kv, seed=71)
    want = oracle(one)
    alone = call(pkg, one, dev)
    check(alone, want)
    for lens, counts, at in (
            ([], [], [0, 1, 2]),                                      # copies only, cells
            ([77, 0, 900], [9, 2, 1], [1, 4]),                        # others, cells
            ([40 + i % 90 for i in range(270)], [1 + i % 3 for i in range(270)], [0, 135, 271, 272]),
            ([6000] + [33] * 300, [16] + [1] * 300, [150, 301]),      # the line's runs
            ([4000], [64], [0])):
        c, places = batch(one, lens, counts, at, H, kv, 72) if lens else (None, None)
        if c is None:
            n = len(at)
            c = dict(one, q=one["q"].repeat(n, 1, 1), bt=one["bt"].repeat(n, 1), seq=one["seq"].repeat(n),
                     mask=one["mask"].repeat(n), cu=torch.arange(n + 1, dtype=torch.int32) * 5)
            places = [0, 5, 10]
        o, lse = call(pkg, c, dev)
        for p in places:
            check((o[p:p + 5], lse[p:p + 5]), want)
        again = call(pkg, c, dev)
        assert torch.equal(o, again[0]) and torch.equal(lse, again[1])
