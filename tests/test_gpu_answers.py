"""Several answers to one prompt, step by step: tables and slots from the lengths, 4-bit
projections, rotation and cache write, the shared length found in the tables, attention over the
shared prompt, the way back -- each step's attention held to its definition in 64 bits on
what the cache holds (tolerances as in test_gpu_verify_tree), the rest to what the operators
give one by one."""
import pytest
import torch
from test_gpu_verify_tree import P, PAGE, PARENTS, V, check_attention, layer, step, write_context

pytestmark = pytest.mark.gpu
I32 = torch.int32
D = 256  # hidden


class Server:
    """A layer, its pages and its 4-bit projections: q, (kv_c | k_pe) and the output."""

    def __init__(self, pkg, dev, H, fp8, n_req, seed=1):
        self.pkg, self.dev, self.H = pkg, dev, H
        self.L = layer(pkg, dev, H, fp8, blocks=80, seed=seed)
        g = torch.Generator().manual_seed(seed)

        def w(n, k):
            return pkg.w4.w4_quantize((torch.randn(n, k, generator=g) * k ** -0.5).half().to(dev), 64)

        self.wq, self.wkv, self.wo = w(H * (P + 64), D), w(576, D), w(D, H * V)
        self.tab = pkg.rope.rotary_table(64, 512, device=dev)
        self.bt = torch.full((n_req, 30), -1, dtype=I32, device=dev)
        self.seq = torch.zeros(n_req, dtype=I32, device=dev)
        self.free = torch.randperm(80, generator=g).int().to(dev)
        self.count = torch.tensor([80], dtype=I32, device=dev)
        self.cs = torch.tensor([0, n_req], dtype=I32, device=dev)

    def extend(self, new, T):
        return self.pkg.paging.extend_tables(self.bt, self.seq, new, self.free, self.count, PAGE, T)

    def step(self, x, new, mask=None):
        """x [T, D] of new tokens a request (one each without a mask) -> [T, D]."""
        p, T = self.pkg, x.shape[0]
        slots, pos, cu, granted = self.extend(new, T)
        q = p.w4.w4_linear(x, self.wq).view(T, self.H, P + 64)
        kv = p.w4.w4_linear(x, self.wkv)
        q = p._cache_ops.rope_concat_and_cache_mla(pos, self.tab, kv[:, :512], kv[:, 512:],
                                                   self.L.latent_cache, slots, self.L.kv_dtype, q=q,
                                                   q_offset=P)
        ql = p.dsa_layer.q_latent(q, self.L.w)
        shared = p.paging.shared_lengths(self.bt, self.seq, self.cs, PAGE)
        more = {} if mask is None else dict(cu_seqlens_q=cu, tree_mask=mask)
        o, lse = p.mla_prefix.shared_prefix_attention(ql, self.L.latent_cache, self.bt, self.seq, self.cs,
                                                      shared, self.L.w.scale, **more)
        self.ql, self.o, self.lse, self.shared, self.cu = ql, o, lse, shared, cu
        return p.w4.w4_linear(p.dsa_layer.v_up(o, self.L.w), self.wo)

    def check(self, see):
        """o and lse of every token against the keys that see(request, token) names."""
        seq, cu = self.seq.tolist(), self.cu.tolist()
        starts = [0]
        for n in seq:
            starts.append(starts[-1] + n)
        kv = self.pkg._cache_ops.gather_latent_cache(
            self.L.latent_cache, self.bt, torch.tensor(starts, dtype=I32, device=self.dev), starts[-1])
        kv, ql = kv.double().cpu(), self.ql.double().cpu()
        for r in range(len(seq)):
            for t in range(cu[r], cu[r + 1]):
                K = kv[starts[r]:starts[r + 1]][see(r, t - cu[r])]
                s = ql[t] @ K.T * self.L.w.scale
                p = s.softmax(1)
                want, A = p @ K[:, :512], p @ K[:, :512].abs()
                ds = 600 * 2.0 ** -24 * self.L.w.scale * (ql[t].abs() @ K.abs().T).amax(1) + 2.0 ** -21
                tol = (1.01 * 2.0 ** -11 + 2 * ds[:, None]) * A + 2.0 ** -11 * want.abs() \
                    + K.shape[0] * 2.0 ** -25 * K.abs().max() + 2.0 ** -25
                assert bool(((self.o[t].double().cpu() - want).abs() <= tol).all()), (r, t)


def prompt(s, n, g):
    """The prompt's rows written for request 0, its whole pages given to all the others, who
    write the rest of it themselves."""
    R = s.seq.numel()
    new = torch.zeros(R, dtype=I32, device=s.dev)
    new[0] = n
    slots, pos, _, granted = s.extend(new, n)
    assert bool(granted.all())
    x = torch.randn(n, 576, generator=g).half().to(s.dev)
    one = torch.ones((), device=s.dev)
    write = s.pkg._cache_ops.concat_and_cache_mla
    write(x[:, :512], x[:, 512:], s.L.latent_cache, slots, s.L.kv_dtype, one)
    whole = n // PAGE * PAGE
    s.bt[1:, :n // PAGE] = s.bt[0, :n // PAGE]
    s.seq[1:] = whole
    new = torch.full((R,), n - whole, dtype=I32, device=s.dev)
    new[0] = 0
    slots, _, cu, granted = s.extend(new, (R - 1) * (n - whole))
    assert bool(granted.all())
    tail = x[whole:].repeat(R - 1, 1)
    write(tail[:, :512], tail[:, 512:], s.L.latent_cache, slots, s.L.kv_dtype, one)


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("H,n", [(16, 100), (64, 96), (3, 13)])
def test_answers(pkg, lib, dev, H, n, fp8):
    g = torch.Generator().manual_seed(H)
    R = 5
    s = Server(pkg, dev, H, fp8, R)
    prompt(s, n, g)
    for k in range(20):
        x = torch.randn(R, D, generator=g).half().to(dev)
        y = s.step(x, torch.ones(R, dtype=I32, device=dev))
        assert y.shape == (R, D) and bool(torch.isfinite(y).all())
        assert s.seq.tolist() == [n + k + 1] * R
        if k in (0, 5, 19):
            assert s.shared.tolist() == [n // PAGE * PAGE]
            s.check(lambda r, j: slice(None))
    # two drafted tokens each, a third of them rejected; then two requests end
    left = int(s.count)
    mask = torch.tensor([1, 3] * R, device=dev)
    s.step(torch.randn(2 * R, D, generator=g).half().to(dev), torch.full((R,), 2, dtype=I32, device=dev), mask)
    s.check(lambda r, j: slice(0, n + 21 + j))
    keep = torch.tensor([n + 20 + (r % 3 > 0) + (r % 3 > 1) for r in range(R)], dtype=I32, device=dev)
    pkg.paging.truncate_tables(s.bt, s.seq, keep, s.free, s.count, PAGE)
    assert s.seq.tolist() == keep.tolist()
    y = s.step(torch.randn(R, D, generator=g).half().to(dev), torch.ones(R, dtype=I32, device=dev))
    s.check(lambda r, j: slice(None))
    whole = torch.tensor([n // PAGE * PAGE], dtype=I32, device=dev).expand(R).contiguous()
    pkg.paging.truncate_tables(s.bt, s.seq, whole, s.free, s.count, PAGE)  # the prompt's pages stay
    assert int(s.count) == 80 - n // PAGE and int(s.count) >= left
    assert len(set(s.free[:80 - n // PAGE].tolist()) | set(s.bt[0, :n // PAGE].tolist())) == 80


def test_a_captured_decode_loop(pkg, lib, dev):
    """One graph, replayed: every replay is the next step, as eager steps give it."""
    g = torch.Generator().manual_seed(4)
    R, n = 4, 40
    a, b = (Server(pkg, dev, 16, True, R, seed=2) for _ in range(2))
    for s in (a, b):
        prompt(s, n, torch.Generator().manual_seed(5))
    new = torch.ones(R, dtype=I32, device=dev)
    x = torch.zeros(R, D, dtype=torch.float16, device=dev)
    keep = [t.clone() for t in (a.bt, a.seq, a.free, a.count, a.L.latent_cache)]
    a.step(x, new)
    torch.cuda.synchronize()
    for t, k in zip((a.bt, a.seq, a.free, a.count, a.L.latent_cache), keep):
        t.copy_(k)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = a.step(x, new)
    for _ in range(40):
        x.copy_(torch.randn(R, D, generator=g).half())
        graph.replay()
        want = b.step(x, new)
        torch.cuda.synchronize()
        assert torch.equal(y, want) and torch.equal(a.seq, b.seq) and torch.equal(a.bt, b.bt)
    assert torch.equal(a.L.latent_cache, b.L.latent_cache) and int(a.seq[0]) == n + 40


@pytest.mark.parametrize("fp8,dtype", [(False, torch.float16), (True, torch.bfloat16)])
def test_verify_tree_of_a_shared_prompt(pkg, lib, dev, fp8, dtype):
    """DsaLayer.verify_tree told of the shared rows: what it gives without, and the
    definition; caches alike."""
    g = torch.Generator().manual_seed(6)
    H, ctx = 16, [70, 64, 99]
    pages = torch.randperm(36, generator=g).int()
    bt = torch.full((3, 12), 0, dtype=I32)
    bt[:, :4] = pages[:4]                 # 64 positions in common
    bt[:, 4:] = pages[4:28].view(3, 8)
    tab = pkg.rope.rotary_table(64, 256, device=dev)
    A, B = (layer(pkg, dev, H, fp8) for _ in range(2))
    write_context(pkg, dev, A, tab, ctx, bt, dtype, g)
    B.latent_cache.copy_(A.latent_cache)
    a = step(pkg, dev, ctx, PARENTS, bt, H, dtype, g)
    cs = torch.tensor([0, 3], dtype=I32, device=dev)
    shared = pkg.paging.shared_lengths(a["block_table"], a["seq_lens"], cs, PAGE)
    assert shared.tolist() == [64]
    out = A.verify_tree(table=tab, cu_shared=cs, shared_lens=shared, **a)
    check_attention(pkg, dev, A, a, ctx, PARENTS, tab)
    assert torch.equal(out, pkg.dsa_layer.v_up(A.last_o, A.w))
    B.verify_tree(table=tab, **a)
    assert torch.equal(A.latent_cache, B.latent_cache) and torch.equal(A.idx_k_cache, B.idx_k_cache)


@pytest.mark.parametrize("backend", ["eager", "aot_eager"])
def test_compiled(pkg, lib, dev, backend):
    """The operators in one compiled function, a whole graph: the eager results, bit for bit,
    and the tables that they write."""
    g = torch.Generator().manual_seed(9)
    R, H, page = 3, 16, 16
    w = pkg.w4.w4_quantize((torch.randn(H * 576, D, generator=g) * D ** -0.5).half().to(dev), 64)
    cache = torch.randn(16, page, 576, generator=g).half().to(dev)
    x = torch.randn(R, D, generator=g).half().to(dev)
    cs, new = (torch.tensor(v, dtype=I32, device=dev) for v in ([0, 3], [1, 1, 1]))
    mask = torch.ones(R, dtype=torch.int64, device=dev)

    def run(x, bt, seq, free, count):
        slots, pos, cu, granted = pkg.paging.extend_tables(bt, seq, new, free, count, page, 5)
        shared = pkg.paging.shared_lengths(bt, seq, cs, page)
        q = pkg.w4.w4_linear(x, w).view(R, H, 576)
        o, lse = pkg.mla_prefix.shared_prefix_attention(q, cache, bt, seq, cs, shared, 0.05)
        o2, lse2 = pkg.mla_prefix.shared_prefix_attention(q, cache, bt, seq, cs, shared, 0.05, cu, mask)
        rows, lens = pkg.paging.token_tables(bt, seq, cu, 5, 4)
        v = pkg.w4.w4_dequant(w) + 1
        pkg.paging.truncate_tables(bt, seq, seq - 3, free, count, page)
        return slots, pos, cu, granted, shared, o * 2, lse, o2, lse2, rows, lens, v

    got = []
    for f in (run, torch.compile(run, backend=backend, fullgraph=True)):
        bt = torch.tensor([[3, 5, 7, -1, -1], [3, 5, 2, -1, -1], [3, 5, 1, -1, -1]], dtype=I32, device=dev)
        seq = torch.tensor([33, 48, 34], dtype=I32, device=dev)
        free = torch.tensor([8, 9, 10, 11, 0, 0], dtype=I32, device=dev)
        count = torch.tensor([4], dtype=I32, device=dev)
        for _ in range(2):
            out = f(x, bt, seq, free, count)
        got.append([*out, bt, seq, free, count])
    for a, b in zip(*got):
        assert torch.equal(a, b)
    assert got[0][4].tolist() == [32] and bool(got[0][3].all())
