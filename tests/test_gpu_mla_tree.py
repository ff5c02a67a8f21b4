"""GPU parity of tree attention (mla_tree.tree_attention) against its definition in
64 bits on the CPU.

Tolerances.  With A = sum p |v| / sum p of a row and dim, ds the largest error of
a score and n the keys: rounding P to fp16 costs at most half a step, 2^-11 A, and
where p is subnormal 2^-25 a key (the running maximum keeps the largest p at 1 or
more); scores off by ds change every weight by ds, twice over with the sum; o is
rounded once more, 2^-11 |o|.  A score is 576 products summed in fp32: ds <= 600
2^-24 scale sum |q k|, and the exponential and its argument add 2^-21.  lse: ds,
and n 2^-24 of the sum."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

H16 = 2.0 ** -11
SCALE = 192 ** -0.5


def quantise(lat):
    n = lat.shape[0]
    t = lat[:, :512].float().view(n, 4, 128)
    s = (t.abs().amax(2) / 448.0).clamp_min(torch.finfo(torch.float32).tiny)
    q = (t / s[:, :, None]).to(torch.float8_e4m3fn).view(torch.uint8).view(n, 512)
    return torch.cat([q, s.view(torch.uint8).view(n, 16),
                      lat[:, 512:].half().view(torch.uint8).view(n, 128)], 1)


def values(rows):
    """Cache rows as the fp16 values the attention uses, in fp64."""
    if rows.dtype != torch.uint8:
        return rows.double()
    n = rows.shape[0]
    v = rows[:, :512].contiguous().view(torch.float8_e4m3fn).float().view(n, 4, 128)
    v = v * rows[:, 512:528].contiguous().view(torch.float32)[:, :, None]
    return torch.cat([v.view(n, 512).half(), rows[:, 528:].contiguous().view(torch.float16)],
                     1).double()


def make(lens, counts, H, page, kv, seed=0, spread=1.0, parents=None):
    """A paged cache in random page order with random trees on the last positions."""
    g = torch.Generator().manual_seed(seed)
    R, T = len(lens), sum(counts)
    need = [max(1, -(-n // page)) for n in lens]
    perm = torch.randperm(sum(need) + 2, generator=g).int()
    bt = torch.full((R, max(need)), -1, dtype=torch.int32)
    at = 0
    for r, k in enumerate(need):
        bt[r, :k] = perm[at:at + k]
        at += k
    lat = torch.randn((sum(need) + 2) * page, 576, generator=g)
    rows = quantise(lat) if kv == "fp8" else lat.half()
    mask = []
    for r, n in enumerate(counts):
        anc = []
        for j in range(n):
            p = int(torch.randint(-1, max(j, 0), (1,), generator=g)) if j else -1
            anc.append((anc[p] if p >= 0 else 0) | (1 << j) % 2 ** 64)
        mask += [a - 2 ** 64 if a >> 63 else a for a in anc]
    q = torch.randn(T, H, 576, generator=g).half() * spread
    cu = torch.tensor([sum(counts[:i]) for i in range(R + 1)], dtype=torch.int32)
    return dict(q=q, rows=rows, page=page, bt=bt, seq=torch.tensor(lens, dtype=torch.int32), cu=cu,
                mask=torch.tensor(mask, dtype=torch.int64))


def oracle(c, scale=SCALE):
    """o, lse, and the bounds on their errors, in fp64."""
    T, H = c["q"].shape[:2]
    o, A = torch.zeros(T, H, 512, dtype=torch.float64), torch.zeros(T, H, 512, dtype=torch.float64)
    lse = torch.full((T, H), -math.inf, dtype=torch.float64)
    ds = torch.zeros(T, H, dtype=torch.float64)
    ns, vmax = torch.zeros(T, H, dtype=torch.float64), torch.zeros(T, H, dtype=torch.float64)
    n_rows, page, width = c["rows"].shape[0], c["page"], c["bt"].shape[1] * c["page"]
    for r in range(c["bt"].shape[0]):
        lo, hi = int(c["cu"][r]), int(c["cu"][r + 1])
        n, L = hi - lo, int(c["seq"][r])
        p = torch.arange(min(max(L, 0), width))
        row = c["bt"][r].long()[p // page] * page + p % page
        ok = (c["bt"][r].long()[p // page] >= 0) & (row < n_rows)
        K = values(c["rows"][row.clamp(0, n_rows - 1)])
        for j in range(n):
            m = int(c["mask"][lo + j])
            d = p - (L - n)
            bit = torch.tensor([x < 0 or (x < 64 and (m >> int(x)) & 1 == 1) for x in d.tolist()],
                               dtype=torch.bool)
            see = ok & bit
            if not bool(see.any()):
                continue
            k = K[see]
            q = c["q"][lo + j].double()
            s = q @ k.T * scale
            mx = s.amax(1, keepdim=True)
            e = (s - mx).exp()
            l = e.sum(1, keepdim=True)
            o[lo + j], A[lo + j] = e @ k[:, :512] / l, e @ k[:, :512].abs() / l
            lse[lo + j] = (mx + l.log())[:, 0]
            ds[lo + j] = 600 * 2.0 ** -24 * abs(scale) * (q.abs() @ k.abs().T).amax(1)
            ns[lo + j], vmax[lo + j] = k.shape[0], k[:, :512].abs().max()
    ds = ds + 2.0 ** -21
    tol = (H16 * 1.01 + 2 * ds[:, :, None]) * A + H16 * o.abs() \
        + (ns * vmax * 2.0 ** -25)[:, :, None] + 2.0 ** -25
    ltol = ds + ns * 2.0 ** -24 + 2.0 ** -22 * lse.abs().clamp(1, 1e3)
    return o, lse, tol, ltol


def cache(c, dev):
    return c["rows"].view(-1, c["page"], c["rows"].shape[1]).to(dev)


def call(pkg, c, dev, scale=SCALE, **kw):
    return pkg.mla_tree.tree_attention(c["q"].to(dev), cache(c, dev), c["bt"].to(dev),
                                       c["seq"].to(dev), c["cu"].to(dev), c["mask"].to(dev), scale,
                                       **kw)


def check(got, want, live=None):
    o, lse = got[0].double().cpu(), got[1].double().cpu()
    wo, wl, tol, ltol = want
    live = torch.ones(o.shape[0], dtype=torch.bool) if live is None else live
    o, lse, wo, wl, tol, ltol = (x[live] for x in (o, lse, wo, wl, tol, ltol))
    none = torch.isinf(wl)
    assert torch.equal(none, lse == -math.inf)
    assert bool((o[none] == 0).all())
    assert bool(((lse - wl)[~none].abs() <= ltol[~none]).all()), (lse - wl)[~none].abs().max()
    worst = ((o - wo).abs() / tol).max() if o.numel() else 0
    assert worst <= 1, f"{float(worst)} of the tolerance"


CASES = [
    # lens, counts, heads, page
    ([1], [1], 1, 64),
    ([4], [4], 16, 64),
    ([31, 32, 33], [1, 2, 3], 8, 16),
    ([64, 65, 97], [5, 1, 33], 20, 48),
    ([500], [4], 16, 64),
    ([130, 3, 0, 700], [7, 3, 1, 2], 64, 64),
    ([300, 200], [64, 17], 3, 1),
    ([2500], [9], 64, 128),
    ([40, 41, 42, 43, 44], [2, 2, 2, 2, 2], 128, 7),
]


@pytest.mark.parametrize("kv", ["fp16", "fp8"])
@pytest.mark.parametrize("lens,counts,H,page", CASES)
def test_matches_definition(pkg, lib, dev, lens, counts, H, page, kv):
    c = make(lens, counts, H, page, kv, seed=sum(lens) + H)
    check(call(pkg, c, dev), oracle(c))


@pytest.mark.parametrize("kv", ["fp16", "fp8"])
def test_many_requests(pkg, lib, dev, kv):
    """More requests than lanes, lengths of every remainder, some without tokens."""
    lens = [(37 * i) % 190 for i in range(150)]
    counts = [min((5 * i) % 7, n) for i, n in enumerate(lens)]
    c = make(lens, counts, 4, 16, kv, seed=3)
    check(call(pkg, c, dev), oracle(c))


def test_long_context_is_split(pkg, lib, dev):
    c = make([9000, 70], [3, 2], 2, 64, "fp16", seed=5, spread=2.0)
    check(call(pkg, c, dev), oracle(c))


@pytest.mark.parametrize("kv", ["fp16", "fp8"])
def test_empty_masks_and_bits_past_the_tree(pkg, lib, dev, kv):
    c = make([3, 50], [3, 4], 16, 16, kv, seed=6)
    c["mask"][0] = 0            # no context, no bit: sees nothing
    c["mask"][1] = ~7           # only bits past its tree
    c["mask"][4] = 0            # the context alone
    c["mask"][5] = -1           # every drafted token, later ones too
    want = oracle(c)
    assert bool(torch.isinf(want[1][0]).all()) and bool(torch.isinf(want[1][1]).all())
    check(call(pkg, c, dev), want)


def test_more_tokens_than_a_mask_names(pkg, lib, dev):
    """Drafted tokens from the 65th on are seen by none; as queries they work."""
    c = make([90], [70], 2, 16, "fp16", seed=7)
    c["mask"][:] = -1
    check(call(pkg, c, dev), oracle(c))


@pytest.mark.parametrize("scale", [0.0, -0.07, 1.5])
def test_scales(pkg, lib, dev, scale):
    c = make([77, 5], [3, 5], 16, 16, "fp16", seed=8, spread=0.3)
    check(call(pkg, c, dev, scale), oracle(c, scale))


@pytest.mark.parametrize("kv", ["fp16", "fp8"])
def test_unresolved_pages_are_not_seen(pkg, lib, dev, kv):
    c = make([200, 150], [3, 2], 16, 16, kv, seed=9)
    c["bt"][0, 2] = -1
    c["bt"][0, 5] = 1 << 20     # past the cache
    c["bt"][1, :] = -5          # nothing of request 1 resolves
    want = oracle(c)
    assert bool(torch.isinf(want[1][3:]).all())
    check(call(pkg, c, dev), want)


def test_lengths_past_the_table_and_below_the_tree(pkg, lib, dev):
    c = make([64, 64], [3, 5], 16, 16, "fp16", seed=10)
    c["seq"][0] = 100           # the table has 64 positions; the tree stands past it
    c["seq"][1] = 2             # two of five drafted tokens have a position: the last two
    check(call(pkg, c, dev), oracle(c))
    c["seq"][0] = -3
    check(call(pkg, c, dev), oracle(c))


@pytest.mark.parametrize("kv", ["fp16", "fp8"])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_infinities_and_nan_in_masked_places(pkg, lib, dev, kv, bad):
    """Not visible drafted tokens and cache rows outside the sequences may hold
    anything; a row that sees such a token is NaN."""
    c = make([70, 40], [6, 4], 16, 16, kv, seed=11)
    c["mask"][:6] = torch.tensor([1, 3, 4, 12, 16, 33])   # token 2 is seen by 2 and 3 only
    want = oracle(c)
    p = 70 - 6 + 2
    row = int(c["bt"][0, p // 16]) * 16 + p % 16
    if kv == "fp8":  # rope values, and a tile scale
        c["rows"][row, 528:].view(torch.float16)[5] = bad
        c["rows"][row, 512:516].view(torch.float32)[0] = bad
    else:
        c["rows"][row, 3] = bad
    used = set()
    for r, n in enumerate([70, 40]):
        used |= {int(c["bt"][r, i // 16]) * 16 + i % 16 for i in range(n)}
    free = torch.tensor([i not in used for i in range(c["rows"].shape[0])])
    c["rows"][free] = 0x7f if kv == "fp8" else math.nan
    got = call(pkg, c, dev)
    live = torch.ones(10, dtype=torch.bool)
    live[2] = live[3] = False
    check(got, want, live)
    assert bool(torch.isnan(got[0][2:4]).all()) and bool(torch.isnan(got[1][2:4]).all())


def test_rows_of_no_request_stay(pkg, lib, dev):
    """Rows before the first and behind the last request, and requests of no token."""
    c = make([40, 30, 20], [3, 0, 2], 16, 16, "fp16", seed=12)
    want = oracle(c)
    pad = torch.full((2, 16, 576), math.nan).half()
    c["q"] = torch.cat([pad, c["q"], pad])
    c["mask"] = torch.cat([torch.full((2,), -1), c["mask"], torch.full((2,), -1)])
    c["cu"] = c["cu"] + 2
    out = torch.full((9, 16, 512), 7.0, dtype=torch.float16, device=dev)
    lse = torch.full((9, 16), 7.0, device=dev)
    got = call(pkg, c, dev, out=out, lse=lse)
    assert got[0] is out and got[1] is lse
    check((out[2:7], lse[2:7]), want)
    for x in (out[:2], out[7:], lse[:2], lse[7:]):
        assert bool((x == 7).all())


def test_nan_query_stays_in_its_row(pkg, lib, dev):
    c = make([60], [3], 16, 16, "fp16", seed=13)
    want = oracle(c)
    c["q"][1, 4] = math.nan
    o, lse = call(pkg, c, dev)
    assert bool(torch.isnan(o[1, 4]).all()) and math.isnan(float(lse[1, 4]))
    o[1, 4], lse[1, 4] = want[0][1, 4].half().to(dev), want[1][1, 4].float().to(dev)
    check((o, lse), want)


@pytest.mark.parametrize("kv", ["fp16", "fp8"])
def test_growing_scores(pkg, lib, dev, kv):
    """Scores that climb along the context, so that the running maximum moves often,
    up to where early keys weigh nothing."""
    c = make([400], [2], 16, 16, kv, seed=14)
    lat = torch.randn(400, 576) * 0.1
    lat[:, 0] = torch.linspace(-40, 40, 400)
    c["q"][:, :, :] = 0
    c["q"][:, :, 0] = torch.linspace(-3, 3, 32).view(2, 16).half()
    for i in range(400):
        row = int(c["bt"][0, i // 16]) * 16 + i % 16
        c["rows"][row] = quantise(lat[i:i + 1])[0] if kv == "fp8" else lat[i].half()
    check(call(pkg, c, dev), oracle(c))


def test_same_result_alone_and_in_a_batch_of_copies(pkg, lib, dev):
    """Deterministic: the same call twice gives the same bits."""
    c = make([3000, 77], [5, 9], 64, 64, "fp16", seed=15)
    a, b = call(pkg, c, dev), call(pkg, c, dev)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_other_stream_and_graph(pkg, lib, dev):
    """On a side stream, and captured with two calls in one graph, replayed with new
    inputs and eager work between the replays."""
    c1, c2 = make([900], [5], 16, 64, "fp16", seed=16), make([50, 60], [3, 4], 32, 16, "fp8", seed=17)
    w1, w2 = oracle(c1), oracle(c2)
    st = torch.cuda.Stream()
    with torch.cuda.stream(st):
        got = call(pkg, c1, dev)
    st.synchronize()
    check(got, w1)

    def args(c):
        return [c["q"].to(dev), cache(c, dev), c["bt"].to(dev), c["seq"].to(dev), c["cu"].to(dev),
                c["mask"].to(dev), SCALE]

    a1, a2 = args(c1), args(c2)
    f = pkg.mla_tree.tree_attention
    f(*a1), f(*a2)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        r1, r2 = f(*a1), f(*a2)
    q1 = a1[0].clone()
    for k in range(4):
        a1[0].copy_(q1 * (1 if k % 2 == 0 else 0.5))
        g.replay()
        eager = call(pkg, c2, dev)  # the program's own work between replays
        torch.cuda.synchronize()
        check(eager, w2)
        check(r2, w2)
        if k % 2 == 0:
            check(r1, w1)
        else:
            e = f(*a1)
            assert torch.equal(e[0], r1[0]) and torch.equal(e[1], r1[1])


def test_strided_inputs(pkg, lib, dev):
    c = make([300, 40], [4, 3], 16, 16, "fp16", seed=18)
    q = torch.empty(7, 32, 576, dtype=torch.float16, device=dev)[:, ::2]
    q.copy_(c["q"])
    bt = torch.empty(2, 2 * c["bt"].shape[1], dtype=torch.int32, device=dev)[:, ::2]
    bt.copy_(c["bt"])
    got = pkg.mla_tree.tree_attention(q, cache(c, dev), bt, c["seq"].to(dev), c["cu"].to(dev),
                                      c["mask"].to(dev), SCALE)
    check(got, oracle(c))


def test_agrees_with_dense_decode(pkg, lib, dev, ops):
    """One drafted token of a request sees what sm70_mla_decode sees."""
    c = make([400, 33, 1, 129], [1, 1, 1, 1], 32, 64, "fp16", seed=19, spread=0.5)
    c["mask"][:] = 1
    o, lse = call(pkg, c, dev)
    do, dl = torch.empty_like(o), torch.empty_like(lse)
    ops.sm70_mla_decode(do, dl, c["q"].to(dev), cache(c, dev), c["bt"].to(dev), c["seq"].to(dev),
                        SCALE)
    torch.testing.assert_close(o.float(), do.float(), rtol=2e-3, atol=2e-3)
    torch.testing.assert_close(lse, dl, rtol=0, atol=2e-3)
