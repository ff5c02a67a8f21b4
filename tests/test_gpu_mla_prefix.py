"""Attention over a shared prefix (mla_prefix.shared_prefix_attention) against its definition
in 64 bits on the CPU.  To the definition a request is one of tree attention: it sees its
context and its drafted tokens, whoever else holds the same rows; oracle, tolerances
and their derivation are those of tree attention's tests.  One rounding comes on top where a
row's pieces are joined in fp32, which their 2^-21 holds."""
import math

import pytest
import torch
from test_gpu_mla_tree import SCALE, cache, check, oracle, quantise

pytestmark = pytest.mark.gpu
I32 = torch.int32


def make(sets, H, page, kv, seed=0, spread=1.0):
    """sets: for each (shared positions, [(own positions, drafted tokens), ..]), the own ones
    with the drafted ones among them; pages in random order, random trees."""
    g = torch.Generator().manual_seed(seed)
    lens, counts, rows, shared, cu = [], [], [], [], [0]
    pages = lambda n: -(-n // page)  # noqa: E731
    need = sum(P // page + sum(pages(P % page + n) for n, _ in reqs) for P, reqs in sets)
    order = torch.randperm(need + 2, generator=g).tolist()
    for P, reqs in sets:
        lead = [order.pop() for _ in range(P // page)]   # whole pages are shared
        shared.append(P // page * page)
        for n, k in reqs:
            lens.append(P + n)
            counts.append(k)
            rows.append(lead + [order.pop() for _ in range(pages(P % page + n))])
        cu.append(cu[-1] + len(reqs))
    W = max(1, max(len(r) for r in rows))
    bt = torch.tensor([r + [-1] * (W - len(r)) for r in rows], dtype=I32)
    lat = torch.randn((need + 2) * page, 576, generator=g)
    mask = []
    for n in counts:
        anc = []
        for j in range(n):
            p = int(torch.randint(-1, max(j, 0), (1,), generator=g)) if j else -1
            anc.append((anc[p] if p >= 0 else 0) | 1 << j)
        mask += anc
    T = sum(counts)
    return dict(q=torch.randn(T, H, 576, generator=g).half() * spread,
                rows=quantise(lat) if kv == "fp8" else lat.half(), page=page, bt=bt,
                seq=torch.tensor(lens, dtype=I32), mask=torch.tensor(mask, dtype=torch.int64),
                cu=torch.tensor([sum(counts[:i]) for i in range(len(counts) + 1)], dtype=I32),
                cs=torch.tensor(cu, dtype=I32), shared=torch.tensor(shared, dtype=I32))


def args(c, dev, scale=SCALE, tree=None):
    """tree: with the drafted tokens' tensors (default: where a request has several)."""
    one = bool((c["cu"] == torch.arange(c["cu"].numel())).all()) and c["q"].shape[0] == c["bt"].shape[0]
    more = {} if (one if tree is None else not tree) else \
        dict(cu_seqlens_q=c["cu"].to(dev), tree_mask=c["mask"].to(dev))
    return [c["q"].to(dev), cache(c, dev), c["bt"].to(dev), c["seq"].to(dev), c["cs"].to(dev),
            c["shared"].to(dev), scale], more


def call(pkg, c, dev, scale=SCALE, tree=None, **kw):
    a, more = args(c, dev, scale, tree)
    return pkg.mla_prefix.shared_prefix_attention(*a, **more, **kw)


CASES = [
    # sets, heads, page
    ([(0, [(1, 1)])], 1, 64),                                        # one row, one key
    ([(64, [(1, 1), (2, 1), (33, 1), (5, 1)])], 16, 16),             # decode, 8 requests a group
    ([(96, [(40, 1), (1, 1), (64, 1)])], 64, 32),                    # 2 requests a group
    ([(128, [(40, 1), (1, 1), (64, 1)])], 128, 64),                  # each its own group
    ([(33, [(7, 3), (50, 2), (9, 9), (3, 1)])], 20, 1),              # rows that straddle groups
    ([(48, [(20, 2), (100, 1)]), (0, [(70, 5)]), (160, [(1, 1), (3, 2), (30, 4)])], 8, 16),
    ([(500, [(12, 1)] * 40)], 3, 7),                                 # 40 requests in one group
    ([(320, [(2, 1), (70, 0), (5, 2)]), (64, [(9, 0)])], 32, 64),    # requests without a token
    ([(16, [(1 + (7 * i) % 60, 1 + i % 3) for i in range(90)])], 5, 16),
    ([(32, [(2, 1), (3, 1)])] * 70, 4, 16),                          # more sets than lanes
    ([(0, [(5, 1)]), (64, [(1, 1)] * 3), (0, [(200, 8), (3, 2)])], 130, 64),
]


@pytest.mark.parametrize("kv", ["fp16", "fp8"])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_matches_definition(pkg, lib, dev, case, kv):
    sets, H, page = CASES[case]
    c = make(sets, H, page, kv, seed=case)
    check(call(pkg, c, dev), oracle(c))


def test_one_token_with_and_without_the_tree(pkg, lib, dev):
    c = make([(96, [(40, 1), (1, 1), (64, 1)]), (16, [(9, 1), (2, 1)])], 24, 16, "fp16", seed=1)
    a, b = call(pkg, c, dev, tree=False), call(pkg, c, dev, tree=True)
    check(a, oracle(c))
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.parametrize("kv", ["fp16", "fp8"])
def test_long_prefix_is_cut(pkg, lib, dev, kv):
    """Cells of one set, of sets of unequal lengths, and rows that pass the pages resolved
    at a time."""
    for sets, H, page in [([(6000, [(40, 1), (200, 1), (1, 1)])], 32, 16),
                          ([(7000, [(30, 2), (9, 1)]), (800, [(5, 1)] * 6)], 16, 64),
                          ([(4500, [(700, 1), (1, 1)])], 4, 1)]:
        c = make(sets, H, page, kv, seed=len(sets) + H, spread=2.0)
        check(call(pkg, c, dev), oracle(c))


def test_equal_runs(pkg, lib, dev):
    """More row groups than workgroups, and uneven ones: runs that hold whole groups and
    pieces of several, segments that begin inside a request's own keys."""
    sets = [(64, [(1 + (37 * i + s) % 150, 1) for i in range(9)]) for s in range(30)]
    c = make(sets, 128, 16, "fp16", seed=2)           # 270 groups
    check(call(pkg, c, dev), oracle(c))
    sets = [(320 * (s % 3), [(1 + (401 * i + s) % 600, 1) for i in range(20)]) for s in range(10)]
    c = make(sets, 96, 16, "fp16", seed=3)            # 150 groups of two requests' rows
    check(call(pkg, c, dev), oracle(c))


@pytest.mark.parametrize("n,size", [(1100, 1100), (600, 1), (40, 30)])
def test_many_requests(pkg, lib, dev, n, size):
    """More requests, sets and row groups than the division holds in LDS: one set of many
    requests, many sets of one, and more row groups than a workgroup has threads."""
    sets = [(16, [(1 + (7 * i + s) % 40, 1) for i in range(size)]) for s in range(n // size if size > 30 else n)]
    c = make(sets, 2 if size != 30 else 110, 16, "fp16", seed=n)
    check(call(pkg, c, dev), oracle(c))


def test_the_same_rows_whatever_is_said_to_be_shared(pkg, lib, dev):
    """Less than what is shared, none, too much (clamped to the shortest request's context),
    negative; one group, or each request alone."""
    c = make([(256, [(40, 2), (3, 3), (64, 1)])], 16, 16, "fp16", seed=4)
    want = oracle(c)
    for n in (0, 1, 31, 100, 255, 256, -5):
        c["shared"][0] = n
        check(call(pkg, c, dev), want)
    c["shared"] = torch.tensor([9, 256, 10 ** 9], dtype=I32)
    c["cs"] = torch.tensor([0, 1, 2, 3], dtype=I32)
    check(call(pkg, c, dev), want)
    c = make([(256, [(2, 2), (3, 3), (9, 9)])], 16, 16, "fp16", seed=5)
    c["shared"][0] = 10 ** 9                          # all contexts end at 256
    check(call(pkg, c, dev), oracle(c))


def test_requests_of_no_group_stay(pkg, lib, dev):
    c = make([(64, [(4, 1), (5, 2)]), (32, [(9, 1), (1, 1), (7, 3)])], 16, 16, "fp16", seed=6)
    want = oracle(c)
    for cs, shared, live in [([1, 2, 4], [0, 32], slice(1, 5)), ([0, 0, 2], [7, 64], slice(0, 3)),
                             ([2, 9], [32], slice(3, 8)), ([5], [], slice(0, 0))]:
        c["cs"], c["shared"] = torch.tensor(cs, dtype=I32), torch.tensor(shared, dtype=I32)
        out = torch.full((8, 16, 512), 7.0, dtype=torch.float16, device=dev)
        lse = torch.full((8, 16), 7.0, device=dev)
        got = call(pkg, c, dev, out=out, lse=lse)
        assert got[0] is out and got[1] is lse
        sel = torch.zeros(8, dtype=torch.bool)
        sel[live] = True
        check(got, want, sel)
        assert bool((out.cpu()[~sel] == 7).all()) and bool((lse.cpu()[~sel] == 7).all())


@pytest.mark.parametrize("kv", ["fp16", "fp8"])
def test_empty_masks_lengths_and_pages(pkg, lib, dev, kv):
    c = make([(64, [(3, 3), (50, 4)]), (0, [(6, 2), (2, 2)])], 16, 16, kv, seed=7)
    c["mask"][0] = 0            # the shared keys alone
    c["mask"][7] = 0            # the context alone
    c["mask"][9:] = 0           # no context, no bit: sees nothing
    c["bt"][0, 1] = -1          # a shared page that is missing: not seen by any of the set
    c["bt"][1, 1] = -1
    c["bt"][1, 5] = 1 << 20     # past the cache
    want = oracle(c)
    assert bool(torch.isinf(want[1][9:]).all())
    check(call(pkg, c, dev), want)
    c["seq"][:] = torch.tensor([40, 2, -3, 100])      # below the tree, none, past the table
    check(call(pkg, c, dev), oracle(c))
    c["seq"][:] = 0
    got = call(pkg, c, dev)
    assert bool((got[0] == 0).all()) and bool((got[1] == -math.inf).all())


@pytest.mark.parametrize("kv", ["fp16", "fp8"])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("H", [4, 16, 64])
def test_infinities_of_others_rows(pkg, lib, dev, kv, bad, H):
    """An own row (context or drafted) that is not finite reaches its request's rows alone."""
    c = make([(64, [(9, 2), (70, 3), (5, 1), (40, 4)])], H, 16, kv, seed=8)
    want = oracle(c)
    p = 64 + 20                                        # of request 1: context
    row = int(c["bt"][1, p // 16]) * 16 + p % 16
    if kv == "fp8":
        c["rows"][row, 528:].view(torch.float16)[5] = bad
        c["rows"][row, 512:516].view(torch.float32)[0] = bad
    else:
        c["rows"][row, 3] = bad
    p = 64 + 40 - 3                                    # of request 3: drafted token 1
    c["mask"][6:] = torch.tensor([1, 3, 5, 13])        # seen by itself only
    want3 = oracle(c)
    row = int(c["bt"][3, p // 16]) * 16 + p % 16
    if kv == "fp8":
        c["rows"][row, 528:].view(torch.float16)[5] = bad
    else:
        c["rows"][row, 100] = bad
    used = set()                                       # whatever else is in the pages
    for r, n in enumerate(c["seq"].tolist()):
        used |= {int(c["bt"][r, i // 16]) * 16 + i % 16 for i in range(n)}
    c["rows"][torch.tensor([i not in used for i in range(c["rows"].shape[0])])] = \
        0x7f if kv == "fp8" else math.nan
    got = call(pkg, c, dev)
    live = torch.ones(10, dtype=torch.bool)
    live[2:5] = live[7] = False
    check(got, [torch.where((torch.arange(10) < 6).view(-1, *[1] * (a.dim() - 1)), a, b)
                for a, b in zip(want, want3)], live)
    assert bool(torch.isnan(got[0][7]).all()) and bool(torch.isnan(got[1][7]).all())
    assert not bool(torch.isfinite(got[0][2:5, :, 3 if kv == "fp16" else 0]).any()) or bad == -math.inf


def test_a_shared_infinity_counts_for_all(pkg, lib, dev):
    c = make([(64, [(9, 1), (70, 1)]), (32, [(4, 1)])], 16, 16, "fp16", seed=9)
    want = oracle(c)
    c["rows"][int(c["bt"][0, 1]) * 16 + 3, 7] = math.nan
    got = call(pkg, c, dev)
    assert bool(torch.isnan(got[0][:2]).all())
    check(got, want, torch.tensor([False, False, True]))


def test_nan_query_stays_in_its_row(pkg, lib, dev):
    c = make([(64, [(9, 1), (70, 1), (3, 1)])], 16, 16, "fp16", seed=10)
    want = oracle(c)
    c["q"][1, 4] = math.nan
    o, lse = call(pkg, c, dev)
    assert bool(torch.isnan(o[1, 4]).all()) and math.isnan(float(lse[1, 4]))
    o[1, 4], lse[1, 4] = want[0][1, 4].half().to(dev), want[1][1, 4].float().to(dev)
    check((o, lse), want)


@pytest.mark.parametrize("H", [4, 32, 64])
def test_nan_queries_of_a_request(pkg, lib, dev, H):
    """All rows of a wave, or some: their scores of every key are NaN, the keys are not."""
    c = make([(64, [(9, 1), (70, 1), (3, 2)])], H, 16, "fp16", seed=20)
    want = oracle(c)
    c["q"][1] = math.nan
    got = call(pkg, c, dev)
    assert bool(torch.isnan(got[0][1]).all()) and bool(torch.isnan(got[1][1]).all())
    check(got, want, torch.tensor([True, False, True, True]))


@pytest.mark.parametrize("scale", [0.0, -0.07, 1.5])
def test_scales(pkg, lib, dev, scale):
    c = make([(48, [(9, 1), (70, 1), (3, 1)])], 16, 16, "fp16", seed=11, spread=0.3)
    check(call(pkg, c, dev, scale), oracle(c, scale))


def test_bf16_rope_values(pkg, lib, dev):
    """Rope values written as bf16 count as the fp16 values that reading them back gives."""
    c = make([(96, [(9, 1), (40, 1), (3, 1)]), (0, [(50, 1)])], 16, 16, "fp8", seed=12)
    b = c["rows"][:, 528:].contiguous().view(torch.float16).to(torch.bfloat16)
    c["rows"][:, 528:] = b.to(torch.float16).view(torch.uint8)
    want = oracle(c)
    c["rows"][:, 528:] = b.view(torch.uint8)
    check(call(pkg, c, dev, pe_dtype=torch.bfloat16), want)


def test_deterministic_and_like_tree_attention(pkg, lib, dev):
    c = make([(3000, [(40, 3), (7, 1), (90, 2)])], 16, 64, "fp16", seed=13)
    a, b = call(pkg, c, dev), call(pkg, c, dev)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    want = oracle(c)
    check(a, want)
    check(pkg.mla_tree.tree_attention(c["q"].to(dev), cache(c, dev), c["bt"].to(dev), c["seq"].to(dev),
                                      c["cu"].to(dev), c["mask"].to(dev), SCALE), want)


def test_strided_inputs(pkg, lib, dev):
    c = make([(64, [(9, 1), (70, 1)])], 16, 16, "fp16", seed=14)
    (q, kv, bt, seq, cs, sh, scale), _ = args(c, dev)
    wide = torch.empty(2, 32, 576, dtype=torch.float16, device=dev)[:, ::2]
    wide.copy_(q)

    def every_other(x):
        y = torch.zeros(*x.shape[:-1], 2 * x.shape[-1], dtype=x.dtype, device=dev)[..., ::2]
        return y.copy_(x)

    got = pkg.mla_prefix.shared_prefix_attention(wide, kv, every_other(bt), every_other(seq),
                                                 every_other(cs), every_other(sh), scale)
    check(got, oracle(c))


def test_other_stream_and_graph(pkg, lib, dev):
    """On a side stream, and captured with two calls in one graph, replayed with new inputs,
    other lengths and eager work between the replays."""
    c1 = make([(900, [(5, 1), (40, 1), (9, 1)])], 16, 64, "fp16", seed=15)
    c2 = make([(48, [(9, 3), (20, 4)])], 32, 16, "fp8", seed=16)
    w1, w2 = oracle(c1), oracle(c2)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        got = call(pkg, c1, dev)
    st.synchronize()
    check(got, w1)
    (a1, m1), (a2, m2) = args(c1, dev), args(c2, dev)
    f = pkg.mla_prefix.shared_prefix_attention
    f(*a1, **m1), f(*a2, **m2)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        r1, r2 = f(*a1, **m1), f(*a2, **m2)
    q1 = a1[0].clone()
    short = dict(c1, seq=torch.tensor([903, 917, 906], dtype=I32))
    ws = oracle(short)
    for k in range(4):
        a1[0].copy_(q1)
        a1[3].copy_(c1["seq"] if k % 2 == 0 else short["seq"])
        g.replay()
        eager = call(pkg, c2, dev)  # the program's own work between replays
        torch.cuda.synchronize()
        check(eager, w2)
        check(r2, w2)
        check(r1, w1 if k % 2 == 0 else ws)


@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("H,n", [(5, 3), (1, 1), (33, 1), (16, 9)])
def test_a_bad_last_query_row(pkg, lib, dev, H, n, bad):
    """The last row of a set in a wave that it does not fill: the others keep their bits."""
    c = make([(96, [(20, 1)] * n), (32, [(3, 1)] * 2)], H, 16, "fp16", seed=8)
    want = call(pkg, c, dev)
    c["q"][n - 1, H - 1, -4:] = bad
    got = call(pkg, c, dev)
    rest = torch.ones(n + 2, H, dtype=torch.bool, device=dev)
    rest[n - 1, H - 1] = False
    assert torch.equal(got[0][rest], want[0][rest]) and torch.equal(got[1][rest], want[1][rest])
    assert not bool(got[1][n - 1, H - 1].isfinite()) or bad == math.inf
