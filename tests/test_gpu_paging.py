"""Block tables and slot maps (paging.py) against whole numbers on the CPU, request by
request and page by page.  Everything is an integer: equal, or wrong."""
import pytest
import torch

pytestmark = pytest.mark.gpu
I32 = torch.int32


def pages(n, page):
    return -(-n // page)


def extend(bt, seq, new, free, count, page, T):
    """The definition, on lists that it changes; returns slots, positions, cu, granted, count."""
    W, at, wanted, avail = len(bt[0]) if bt else 0, 0, 0, count
    slots, pos, cu, granted = [-1] * T, [-1] * T, [0], []
    for r, (n, k) in enumerate(zip(seq, new)):
        n, k = max(n, 0), max(k, 0)
        need = pages(n + k, page) - pages(n, page)
        fits = pages(n + k, page) <= W and at + k <= T
        wanted += need if fits else 0
        ok = fits and (need == 0 or wanted <= avail)
        if ok:
            for i in range(pages(n, page), pages(n + k, page)):
                count -= 1
                bt[r][i] = free[count]
            seq[r] = n + k
            for i in range(k):
                e = bt[r][(n + i) // page]
                pos[at + i] = n + i
                slots[at + i] = e * page + (n + i) % page if e >= 0 else -1
        granted.append(ok)
        at += k
        cu.append(min(at, T))
    return slots, pos, cu, granted, count


def truncate(bt, seq, keep, free, count, page):
    out = []
    for r, (n, k) in enumerate(zip(seq, keep)):
        k = min(max(k, 0), max(n, 0))
        for i in range(min(pages(k, page), len(bt[r])), min(pages(max(n, 0), page), len(bt[r]))):
            if bt[r][i] >= 0:
                out.append(bt[r][i])
            bt[r][i] = -1
        seq[r] = k if n > k else n
    for j, x in enumerate(out):
        at = count + len(out) - 1 - j
        if at < len(free):
            free[at] = x
    return min(count + len(out), len(free))


class Both:
    """The state on the GPU and as lists, stepped together."""

    def __init__(self, pkg, dev, lens, W, page, spare, seed=0):
        g = torch.Generator().manual_seed(seed)
        self.pkg, self.dev, self.page, self.R, self.W = pkg, dev, page, len(lens), W
        held = [min(pages(n, page), W) for n in lens]
        order = torch.randperm(sum(held) + spare, generator=g).tolist()
        self.bt = [[-1] * W for _ in lens]
        for r, k in enumerate(held):
            self.bt[r][:k] = [order.pop() for _ in range(k)]
        self.count = len(order)
        self.free = order + [-1] * sum(held)
        self.seq = list(lens)
        self.d = dict(bt=torch.tensor(self.bt, dtype=I32).view(self.R, W).to(dev),
                      seq=torch.tensor(self.seq, dtype=I32, device=dev),
                      free=torch.tensor(self.free, dtype=I32, device=dev),
                      count=torch.tensor([self.count], dtype=I32, device=dev))

    def same(self):
        assert self.d["bt"].cpu().tolist() == self.bt
        assert self.d["seq"].tolist() == self.seq
        assert self.d["free"].tolist() == self.free
        assert self.d["count"].tolist() == [self.count]

    def extend(self, new, T):
        d = self.d
        got = self.pkg.paging.extend_tables(d["bt"], d["seq"],
                                            torch.tensor(new, dtype=I32, device=self.dev), d["free"],
                                            d["count"], self.page, T)
        *want, self.count = extend(self.bt, self.seq, new, self.free, self.count, self.page, T)
        for a, b, dt in zip(got, want, (I32, I32, I32, torch.bool)):
            assert a.dtype == dt and a.tolist() == b
        self.same()
        return want[3]

    def truncate(self, keep):
        d = self.d
        self.pkg.paging.truncate_tables(d["bt"], d["seq"],
                                        torch.tensor(keep, dtype=I32, device=self.dev), d["free"],
                                        d["count"], self.page)
        self.count = truncate(self.bt, self.seq, keep, self.free, self.count, self.page)
        self.same()


@pytest.mark.parametrize("page", [1, 16, 48, 64])
@pytest.mark.parametrize("R", [1, 3, 65, 300])
def test_steps(pkg, lib, dev, page, R):
    """Decode, drafts partly rejected, idle and ended requests, a prefill chunk."""
    lens = [(37 * i) % 190 for i in range(R)]
    W = pages(190 + 400, page)
    b = Both(pkg, dev, lens, W, page, R * pages(400, page) + R, seed=R + page)
    b.extend([1] * R, R)
    assert all(b.extend([(5 * i) % 7 for i in range(R)], 6 * R + 3))
    b.truncate([n - (3 * i) % 5 for i, n in enumerate(b.seq)])
    b.truncate([0 if i % 3 == 0 else n + 9 for i, n in enumerate(b.seq)])
    assert all(b.extend([133 if i % 3 == 0 else 1 for i in range(R)], 134 * R))
    b.extend([0] * R, 0)
    b.truncate([0] * R)
    assert b.count == len(b.free) and b.seq == [0] * R


def test_more_requests_than_the_workgroup_has_threads(pkg, lib, dev):
    R = 2500
    b = Both(pkg, dev, [i % 50 for i in range(R)], 8, 16, 3 * R, seed=1)
    assert all(b.extend([i % 4 for i in range(R)], 2 * R))        # tokens by the second launch
    assert all(b.extend([1] * R, R))                              # and by the first
    b.truncate([max(n - 2, 0) for n in b.seq])


def test_extend_and_cut_back_leave_the_stack(pkg, lib, dev):
    b = Both(pkg, dev, [5, 64, 127, 0, 30], 40, 16, 60, seed=2)
    was = [list(b.free), b.count, [list(x) for x in b.bt], list(b.seq)]
    b.extend([20, 0, 100, 33, 2], 200)
    b.truncate(was[3])
    assert [b.free[:b.count], b.count, b.bt, b.seq] == [was[0][:was[1]], *was[1:]]


@pytest.mark.parametrize("T", [60, 5000])  # one launch, two launches
def test_refusals_on_the_device(pkg, lib, dev, T):
    """Pages run out in the middle: requests in order, those that need none go on."""
    b = Both(pkg, dev, [15, 30, 16, 7, 48], 6, 16, 3, seed=3)
    # 15 + 2, 16 + 30 and 48 + 1 need 1, 2 and 1 pages
    assert b.extend([2, 2, 30, 3, 1], T) == [True, True, True, True, False]
    b = Both(pkg, dev, [15, 30, 16, 7, 48], 6, 16, 2, seed=3)
    assert b.extend([2, 2, 30, 3, 1], T) == [True, True, False, True, False]
    # the table's width, the rows
    b = Both(pkg, dev, [60, 10, 3], 4, 16, 50, seed=4)
    assert b.extend([5, 2, 1], T) == [False, True, True]
    b = Both(pkg, dev, [6, 10, 3], 4000, 2, 8000, seed=4)
    assert b.extend([5, T - 5, 1], T) == [True, True, False]
    b = Both(pkg, dev, [6, 10, 3], 4000, 2, 8000, seed=4)
    assert b.extend([5, T, 1], T) == [True, False, False]


def test_no_pages_and_odd_lengths(pkg, lib, dev):
    b = Both(pkg, dev, [16, 20, 0], 4, 16, 0, seed=5)
    assert b.extend([1, 3, 0], 9) == [False, True, True]
    b.d["seq"][2] = b.seq[2] = -7       # a negative length counts as none
    b.d["count"][0] = b.count = -3      # and so does a negative count
    b.count = 0
    assert b.extend([0, -5, 2], 9) == [True, True, False]
    b.truncate([-4, 18, 5])
    b = Both(pkg, dev, [2 ** 31 - 3, 40], 4, 16, 9, seed=6)   # sums past 31 bits
    assert b.extend([2 ** 31 - 1, 2], 40) == [False, False]
    assert b.extend([2, 2], 40) == [False, True]
    b.truncate([5, 0])


def test_missing_entries(pkg, lib, dev):
    """Entries that are -1 already: no slot, and nothing given back."""
    b = Both(pkg, dev, [40, 300, 17], 30, 16, 9, seed=7)
    for r, k in ((0, 2), (1, 3), (1, 17)):
        b.bt[r][k] = -1
        b.d["bt"][r, k] = -1
    b.extend([3, 2, 1], 6)
    b.truncate([1, 7, 17])


def test_a_full_stack_drops(pkg, lib, dev):
    b = Both(pkg, dev, [100, 50], 8, 16, 4, seed=8)
    b.d["free"], b.free = b.d["free"][:7].clone(), b.free[:7]
    b.truncate([10, 0])
    assert b.count == 7


def test_no_request(pkg, lib, dev):
    b = Both(pkg, dev, [], 4, 16, 5)
    b.extend([], 7)
    b.truncate([])
    t, n = pkg.paging.token_tables(b.d["bt"], b.d["seq"], torch.zeros(1, dtype=I32, device=dev), 3)
    assert t.tolist() == [[-1] * 4] * 3 and n.tolist() == [0] * 3
    cu = torch.zeros(3, dtype=I32, device=dev)
    assert pkg.paging.shared_lengths(b.d["bt"], b.d["seq"], cu, 16).tolist() == [0, 0]


def test_feeds_the_cache_writer(pkg, lib, dev):
    """Slots as the writers take them: every token's row, padded ones skipped."""
    b = Both(pkg, dev, [10, 33], 8, 16, 9, seed=9)
    slots, pos, cu, _ = pkg.paging.extend_tables(b.d["bt"], b.d["seq"],
                                                 torch.tensor([2, 3], dtype=I32, device=dev),
                                                 b.d["free"], b.d["count"], 16, 7)
    cache = torch.zeros(20, 16, 576, dtype=torch.float16, device=dev)
    kv = torch.randn(7, 576, device=dev).half()
    one = torch.ones((), device=dev)
    pkg._cache_ops.concat_and_cache_mla(kv[:, :512].contiguous(), kv[:, 512:].contiguous(), cache,
                                        slots, "auto", one)
    rows = pkg._cache_ops.gather_latent_cache(cache, b.d["bt"], cu, 5,
                                              starts=torch.tensor([10, 33], dtype=I32, device=dev))
    assert torch.equal(rows, kv[:5])
    assert pos.tolist() == [10, 11, 33, 34, 35, -1, -1]
    assert int((cache != 0).any(2).sum()) == 5


@pytest.mark.parametrize("T,cols", [(0, 5), (1, 1), (7, 0), (30, 6), (31, 8), (300, 8)])
@pytest.mark.parametrize("W,cut", [(8, 0), (9, 1), (5000, 1)])
def test_token_tables(pkg, lib, dev, T, cols, W, cut):
    """Rows of no request in front and behind, requests without a token, strided tables."""
    g = torch.Generator().manual_seed(T + cols)
    cols = min(cols, W) if W < 5000 else W - 3 * (cols % 3)
    counts = [3, 0, 11, 1, 9]
    cu, seq = [2], [40, 7, 11, 0, 2 ** 31 - 1]
    for n in counts:
        cu.append(cu[-1] + n)
    bt = torch.randint(-1, 1 << 30, (5, W + cut), generator=g).int()[:, :W]
    rows, lens = pkg.paging.token_tables(
        bt.to(dev) if not cut else torch.cat([bt, bt[:, :1]], 1).to(dev)[:, :W],
        torch.tensor(seq, dtype=I32, device=dev), torch.tensor(cu, dtype=I32, device=dev), T, cols)
    wr, wl = torch.full((T, cols), -1, dtype=I32), [0] * T
    for t in range(T):
        for r, n in enumerate(counts):
            if cu[r] <= t < cu[r + 1]:
                wr[t], wl[t] = bt[r, :cols], max(0, seq[r] - n + t - cu[r] + 1)
    assert torch.equal(rows.cpu(), wr) and lens.tolist() == wl


@pytest.mark.parametrize("page,W", [(1, 3000), (16, 9), (64, 2100)])
def test_shared_lengths(pkg, lib, dev, page, W):
    g = torch.Generator().manual_seed(W)
    R = 12
    bt = torch.randint(0, 1 << 20, (1, W), generator=g).int().repeat(R, 1)
    seq = [W * page - 3 * i for i in range(R)]
    cuts = {1: 0, 2: W // 2, 4: W - 1, 5: W // 2 + 1, 9: 1}    # first page that differs
    for r, k in cuts.items():
        bt[r, k:] += 1
    seq[7] = 0
    cu = [0, 2, 3, 3, 7, 9, 10, 12]
    got = pkg.paging.shared_lengths(bt.to(dev), torch.tensor(seq, dtype=I32, device=dev),
                                    torch.tensor(cu, dtype=I32, device=dev), page)
    want = []
    for a, b in zip(cu, cu[1:]):
        n = [min(seq[r], page * next((k for k in range(W) if bt[r, k] != bt[a, k]), W))
             for r in range(a, b)]
        want.append(min(n) if n else 0)
    assert got.tolist() == want


@pytest.mark.parametrize("T", [64, 6000])
def test_captured(pkg, lib, dev, T):
    """A step and its cut in a graph, replayed on moving lengths with eager work between."""
    b = Both(pkg, dev, [3, 60, 17], 40, 16, 60, seed=10)
    other = Both(pkg, dev, [9, 9], 40, 16, 60, seed=11)
    new = torch.tensor([2, 1, 9], dtype=I32, device=dev)
    back = torch.tensor([7, 200, 0], dtype=I32, device=dev)
    cu = torch.tensor([0, 2, 3], dtype=I32, device=dev)
    d, P = b.d, pkg.paging

    def step():
        s, p, c, k = P.extend_tables(d["bt"], d["seq"], new, d["free"], d["count"], 16, T)
        rows = P.token_tables(d["bt"], d["seq"], c, T, 7)
        sh = P.shared_lengths(d["bt"], d["seq"], cu, 16)
        return s, p, c, k, *rows, sh

    keep = {k: v.clone() for k, v in d.items()}
    step(), P.truncate_tables(d["bt"], d["seq"], back, d["free"], d["count"], 16)
    torch.cuda.synchronize()
    for k, v in keep.items():
        d[k].copy_(v)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
        P.truncate_tables(d["bt"], d["seq"], back, d["free"], d["count"], 16)
    for i in range(4):
        n = [2 + i, 1, 9]
        new.copy_(torch.tensor(n, dtype=I32))
        graph.replay()
        other.extend([1, 2], 3)  # the program's own work
        torch.cuda.synchronize()
        s, p, c, k, count = extend(b.bt, b.seq, n, b.free, b.count, 16, T)
        assert [x.tolist() for x in out[:4]] == [s, p, c, k]
        for t in range(sum(n)):
            r = next(r for r in range(3) if c[r] <= t < c[r + 1])
            assert out[4][t].tolist() == b.bt[r][:7]
            assert out[5][t] == b.seq[r] - n[r] + t - c[r] + 1
        b.count = truncate(b.bt, b.seq, [7, 200, 0], b.free, count, 16)
        b.same()


def test_other_stream(pkg, lib, dev):
    b = Both(pkg, dev, [3, 60, 17], 40, 16, 60, seed=12)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        b.extend([4, 5, 600], 20)
        b.truncate([1, 62, 0])
