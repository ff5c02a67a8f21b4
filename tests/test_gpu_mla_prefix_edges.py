"""Attention over a shared prefix where keys of one request stand beside those of others:
rows that are not finite, requests without a token, lengths past the table, own keys in several
segments.  Oracle and tolerances as in test_gpu_mla_prefix."""
import math

import pytest
import torch
from test_gpu_mla_prefix import call, check, make, oracle

pytestmark = pytest.mark.gpu
I32 = torch.int32


def row_of(c, r, p):
    return int(c["bt"][r, p // c["page"]]) * c["page"] + p % c["page"]


def spoil(c, rows, bad):
    """Every value of the rows, or (fp8) their scales and rope values."""
    if c["rows"].dtype == torch.uint8:
        c["rows"][rows, 512:528] = torch.full((4,), bad).view(torch.uint8)
        c["rows"][rows, 528:] = torch.full((64,), bad, dtype=torch.float16).view(torch.uint8)
    else:
        c["rows"][rows] = bad


def bf16_rope(c):
    """The cache's rope values as bf16, and (first) the case that the oracle sees."""
    b = c["rows"][:, 528:].contiguous().view(torch.float16).to(torch.bfloat16)
    seen = dict(c, rows=c["rows"].clone())
    seen["rows"][:, 528:] = b.to(torch.float16).view(torch.uint8)
    c["rows"][:, 528:] = b.view(torch.uint8)
    return seen, c


@pytest.mark.parametrize("kv", ["fp16", "fp8", "bf16 rope"])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("H", [4, 16])
def test_whole_tiles_of_bad_rows(pkg, lib, dev, kv, bad, H):
    """A request whose own rows are all bad, in front of others' rows in one line of tiles, six
    tiles long, with waves that have no rows; then a bad tile in the middle of it."""
    for first, sizes in [(0, [40, 70, 50, 60]), (1, [30, 40, 70, 60])]:
        c = make([(64, [(n, 1) for n in sizes])], H, 16, "fp16" if kv == "fp16" else "fp8", seed=first)
        seen, c = bf16_rope(c) if kv == "bf16 rope" else (c, c)
        want = oracle(seen)
        rows = [row_of(c, first, p) for p in range(64, 64 + sizes[first])]
        spoil(c, torch.tensor(rows), bad)
        if kv == "bf16 rope":
            c["rows"][torch.tensor(rows), 528:] = torch.full((64,), bad, dtype=torch.bfloat16).view(torch.uint8)
        more = dict(pe_dtype=torch.bfloat16) if kv == "bf16 rope" else {}
        got = call(pkg, c, dev, **more)
        check(got, want, torch.arange(4) != first)
        assert not bool(got[0][first].isfinite().any()) and bool(got[1][first].isnan().all())


@pytest.mark.parametrize("kv", ["fp16", "fp8"])
@pytest.mark.parametrize("H", [4, 32])
def test_first_requests_without_a_token(pkg, lib, dev, kv, H):
    """Groups whose first requests take no part in the step: ended, with no page left, or short,
    with fewer pages than the others share."""
    c = make([(320, [(9, 0), (70, 2), (5, 1), (12, 3)]), (64, [(9, 0)]), (96, [(3, 0), (4, 0), (40, 1)]),
              (200, [(20, 2), (6, 1)])], H, 16, kv, seed=2)
    c["bt"][0], c["seq"][0] = -1, 0
    c["bt"][5, 2:], c["seq"][5] = -1, 32
    c["bt"][6], c["seq"][6] = -1, 0
    check(call(pkg, c, dev), oracle(c))


@pytest.mark.parametrize("kv", ["fp16", "fp8"])
@pytest.mark.parametrize("H", [4, 32])
@pytest.mark.parametrize("n", [1, 3])
def test_lengths_near_2_31(pkg, lib, dev, kv, H, n):
    """Lengths past the table, of requests behind others in a row group: every key that the table
    holds is context."""
    c = make([(16, [(90, n), (20, n), (40, n)]), (0, [(35, 1), (50, n)])], H, 16, kv, seed=3)
    c["seq"][1], c["seq"][2], c["seq"][4] = 2 ** 31 - 1, 2 ** 31 - 60, 2 ** 31 - 1
    check(call(pkg, c, dev), oracle(c))


def pooled(sets, H, page, seed):
    """As make, with the pages of all requests out of a pool of 256."""
    g = torch.Generator().manual_seed(seed)
    lens = [P + n for P, reqs in sets for n in reqs]
    W = max(-(-n // page) for n in lens)
    bt = torch.randint(0, 256, (len(lens), W), generator=g).int()
    cs = [0]
    for P, reqs in sets:
        bt[cs[-1]:cs[-1] + len(reqs), :P // page] = bt[cs[-1], :P // page].clone()
        cs.append(cs[-1] + len(reqs))
    R = len(lens)
    return dict(q=torch.randn(R, H, 576, generator=g).half(), page=page, bt=bt,
                rows=torch.randn(256 * page, 576, generator=g).half(), seq=torch.tensor(lens, dtype=I32),
                mask=torch.ones(R, dtype=torch.int64), cu=torch.arange(R + 1, dtype=I32),
                cs=torch.tensor(cs, dtype=I32), shared=torch.tensor([P for P, _ in sets], dtype=I32))


@pytest.mark.parametrize("sets,H", [
    ([(0, [2500 + i % 9])for i in range(300)], 1),              # one request's keys
    ([(16, [900, 870 + i % 60, 905]) for i in range(300)], 4),  # keys of three
    ([(0, [4100, 40, 70 + i % 30]) for i in range(130)], 32)])  # many of one, then others'
def test_more_own_keys_than_a_segment_takes(pkg, lib, dev, sets, H):
    """A workgroup's piece holds more than the 64 tiles of own keys that are resolved at a time."""
    c = pooled(sets, H, 16, seed=H)
    check(call(pkg, c, dev), oracle(c))
