"""Sizes whose offsets pass 32 bits, and calls of two streams at once: shared-prefix
attention, block tables and 4-bit weights against what the same calls give alone or at
small sizes."""
import pytest
import torch
from test_gpu_mla_prefix import SCALE, cache, make

pytestmark = pytest.mark.gpu
I32 = torch.int32


@pytest.mark.parametrize("kv", ["fp16", "fp8"])
def test_cache_rows_past_4_gib(pkg, lib, dev, kv):
    c = make([(96, [(40, 2), (5, 1)]), (32, [(7, 3)])], 16, 16, kv, seed=3)
    near = cache(c, dev)
    n, more = near.shape[0], -(-(5 << 30) // (near[0].numel() * near.element_size()))
    far = torch.empty(n + more, *near.shape[1:], dtype=near.dtype, device=dev)
    far[more:] = near
    bt = c["bt"].to(dev)
    rest = [c[k].to(dev) for k in ("seq", "cs", "shared")]
    tree = [c[k].to(dev) for k in ("cu", "mask")]
    run = pkg.mla_prefix.shared_prefix_attention
    want = run(c["q"].to(dev), near, bt, *rest, SCALE, *tree)
    got = run(c["q"].to(dev), far, torch.where(bt >= 0, bt + more, bt), *rest, SCALE, *tree)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert bool(want[0].isfinite().all()) and bool(want[0].any())


def test_token_tables_of_more_than_2_31_entries(pkg, lib, dev):
    T, W, R = 200_000, 11_520, 3
    bt = torch.arange(R * W, dtype=I32, device=dev).view(R, W)
    cu = torch.tensor([0, 70_001, 70_001, 199_990], dtype=I32, device=dev)
    seq = torch.full((R,), 180_000, dtype=I32, device=dev)
    rows, lens = pkg.paging.token_tables(bt, seq, cu, T)
    for t, r in ((0, 0), (70_000, 0), (70_001, 2), (190_000, 2), (199_989, 2)):
        assert torch.equal(rows[t], bt[r]), t
    assert bool((rows[199_990:] == -1).all()) and lens[199_990:].tolist() == [0] * 10
    assert lens[199_989].item() == 180_000 and lens[0].item() == 180_000 - 70_001 + 1


def test_4_bit_weights_of_more_than_2_31_values(pkg, lib, dev):
    N, K, last = 131_072, 24_576, 64
    g = torch.Generator(device=dev).manual_seed(1)
    w = torch.randn(1024, K, generator=g, device=dev).half()
    small = pkg.w4.w4_quantize(w[-last:].contiguous(), 128)
    big = pkg.w4.w4_quantize(w.repeat(N // 1024, 1), 128)
    assert torch.equal(big.q[-last // 16:], small.q) and torch.equal(big.sz[-last // 16:], small.sz)
    v = pkg.w4.w4_dequant(big)
    assert torch.equal(v[-last:], pkg.w4.w4_dequant(small))
    x = torch.randn(2, K, generator=g, device=dev).half()
    y = pkg.w4.w4_linear(x, big)
    want = x.double() @ v[-last:].double().T
    A = x.double().abs() @ v[-last:].double().abs().T
    # weights enter unrounded, v rounds each: half a step of 2^-10; fp32 sums, y's own half step
    tol = (2.0 ** -11 + 2.0 ** -20) * A + 2.0 ** -11 * want.abs()
    assert bool(((y[:, -last:].double() - want).abs() <= tol).all())


def test_two_streams_at_once(pkg, lib, dev):
    """Each stream its own states; the calls overlap as they will, and give what they give alone."""
    W = torch.randn(512, 24_576, generator=torch.Generator().manual_seed(4)).half().to(dev)
    w = pkg.w4.w4_quantize(W, 64)

    def state(seed):
        c = make([(400, [(30, 1), (9, 1), (70, 1)]), (64, [(5, 1)])], 32, 16, "fp16", seed=seed)
        g = torch.Generator().manual_seed(seed)
        return dict(a=[c["q"].to(dev), cache(c, dev), c["bt"].to(dev), c["seq"].to(dev), c["cs"].to(dev),
                       c["shared"].to(dev)],
                    x=torch.randn(64, 24_576, generator=g).half().to(dev),
                    bt=torch.full((40, 9), -1, dtype=I32, device=dev),
                    seq=torch.zeros(40, dtype=I32, device=dev),
                    new=torch.randint(0, 30, (40,), generator=g).int().to(dev),
                    free=torch.randperm(400, generator=g).int().to(dev),
                    count=torch.tensor([400], dtype=I32, device=dev))

    def step(s):
        o, lse = pkg.mla_prefix.shared_prefix_attention(*s["a"], SCALE)
        y = pkg.w4.w4_linear(s["x"], w)
        out = pkg.paging.extend_tables(s["bt"], s["seq"], s["new"], s["free"], s["count"], 16, 1200)
        sh = pkg.paging.shared_lengths(s["bt"], s["seq"], s["a"][4][:2], 16)
        pkg.paging.truncate_tables(s["bt"], s["seq"], s["new"] // 2, s["free"], s["count"], 16)
        return [o, lse, y, *out, sh, s["bt"].clone(), s["free"].clone(), s["count"].clone()]

    want = [[step(s) for _ in range(3)] for s in (state(1), state(2))]
    both = [state(1), state(2)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(3):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got[i].append(step(both[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for a, b in zip(got[i], want[i]):
            for u, v in zip(a, b):
                assert torch.equal(u, v)


def test_two_graphs_of_one_pool(pkg, lib, dev):
    """Two captured calls whose workspaces share a memory pool, replayed in both orders with
    eager calls between."""
    w = pkg.w4.w4_quantize(torch.randn(512, 24_576, generator=torch.Generator().manual_seed(5)).half().to(dev))
    c = make([(300, [(30, 1), (9, 1), (70, 1)])], 32, 16, "fp16", seed=5)
    a = [c[k].to(dev) for k in ("bt", "seq", "cs", "shared")]
    kv, q = cache(c, dev), c["q"].to(dev)
    x = torch.randn(64, 24_576, generator=torch.Generator().manual_seed(6)).half().to(dev)

    def one():
        return pkg.mla_prefix.shared_prefix_attention(q, kv, *a, SCALE)

    def two():
        return pkg.w4.w4_linear(x, w), pkg.paging.shared_lengths(a[0], a[1], a[2], 16)

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        one(), two()
    torch.cuda.synchronize()
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1):
        out1 = one()
    with torch.cuda.graph(g2, pool=g1.pool()):
        out2 = two()
    for i in range(4):
        q.copy_(c["q"].to(dev) * (i + 1) / 2)
        x.mul_(-0.5)
        for g in ((g1, g2), (g2, g1))[i % 2]:
            g.replay()
        torch.cuda.synchronize()
        for u, v in zip((*out1, *out2), (*one(), *two())):
            assert torch.equal(u, v), i
