"""GPU tests of DsaLayer.verify_tree: the rotary positions, the cache writes, tree
attention and the projections of a step of drafted trees, run together.

Tolerance of the attention (as for tree attention alone): with A = sum p |v| / sum p,
P is rounded to fp16 (2^-11 A) and so is o (2^-11 |o|); scores are off by ds <= 600
2^-24 scale sum |q k| + 2^-21, twice over with the sum; a subnormal p costs 2^-25 max
|v| a key.  The cache rows (read back as fp16 values) and the latent q are the same
fp16 numbers on both sides."""
import pytest
import torch

pytestmark = pytest.mark.gpu

H16 = 2.0 ** -11
P, V, PAGE = 128, 128, 16
PARENTS = [[-1, 0, 0, 1, 2, 2, 5], [-1], [-1, -1, 0, 1, 3]]


def layer(pkg, dev, H, fp8, idx_fp8=False, blocks=40, seed=3):
    g = torch.Generator().manual_seed(seed)
    m = pkg.dsa_layer
    w = m.DsaLayerWeights((torch.randn(H, P, 512, generator=g) * 0.05).half().to(dev),
                          (torch.randn(H, 512, V, generator=g) * 0.05).half().to(dev), 192 ** -0.5)
    lat = torch.zeros(blocks, PAGE, 656, dtype=torch.uint8, device=dev) if fp8 else \
        torch.zeros(blocks, PAGE, 576, dtype=torch.float16, device=dev)
    ik = torch.zeros(blocks, PAGE, 132, dtype=torch.uint8, device=dev) if idx_fp8 else \
        torch.zeros(blocks, PAGE, 128, dtype=torch.float16, device=dev)
    return m.DsaLayer(w, lat, ik)


def slots(bt, r, pos):
    pos = torch.as_tensor(pos)
    return bt[r].long()[pos // PAGE] * PAGE + pos % PAGE


def step(pkg, dev, ctx, parents, bt, H, dtype, g):
    """Arguments of one verify_tree call after contexts of ctx tokens."""
    mask, posn, slot, cu, seq = [], [], [], [0], []
    for r, (n, par) in enumerate(zip(ctx, parents)):
        m, depth = pkg.mla_tree.tree_masks(par)
        mask += m
        posn += [n + d for d in depth]
        slot += slots(bt, r, range(n, n + len(par))).tolist()
        cu.append(cu[-1] + len(par))
        seq.append(n + len(par))
    T = cu[-1]
    i32 = dict(dtype=torch.int32, device=dev)
    return dict(q=torch.randn(T, H, P + 64, generator=g).half().to(dev),
                kv_c=torch.randn(T, 512, generator=g).to(dtype).to(dev),
                k_pe=torch.randn(T, 64, generator=g).to(dtype).to(dev),
                positions=torch.tensor(posn, device=dev),
                slot_mapping=torch.tensor(slot, device=dev), block_table=bt.to(dev),
                seq_lens=torch.tensor(seq, **i32), cu_seqlens_q=torch.tensor(cu, **i32),
                tree_mask=torch.tensor(mask, device=dev),
                idx_k=torch.randn(T, 128, generator=g).to(dtype).to(dev))


def write_context(pkg, dev, L, tab, ctx, bt, dtype, g):
    for r, n in enumerate(ctx):
        if n:
            pkg._cache_ops.rope_concat_and_cache_mla(
                torch.arange(n, device=dev), tab, torch.randn(n, 512, generator=g).to(dtype).to(dev),
                torch.randn(n, 64, generator=g).to(dtype).to(dev), L.latent_cache,
                slots(bt, r, range(n)).to(dev), L.kv_dtype)


def check_attention(pkg, dev, L, a, ctx, parents, tab):
    """last_o of the layer against every node's context and ancestors, read back."""
    qr = pkg.rope.apply_rotary(a["q"], a["positions"], tab, P)
    ql = pkg.dsa_layer.q_latent(qr, L.w).double().cpu()
    starts = [0]
    for s in a["seq_lens"].tolist():
        starts.append(starts[-1] + s)
    cu = torch.tensor(starts, dtype=torch.int32, device=dev)
    kv = pkg._cache_ops.gather_latent_cache(L.latent_cache, a["block_table"], cu, starts[-1])
    kv, t = kv.double().cpu(), 0
    for r, par in enumerate(parents):
        for j in range(len(par)):
            see, k = list(range(ctx[r])), j
            while k >= 0:
                see.append(ctx[r] + k)
                k = par[k]
            K = kv[starts[r]:][see]
            s = ql[t] @ K.T * L.w.scale
            p = s.softmax(1)
            want, A = p @ K[:, :512], p @ K[:, :512].abs()
            ds = 600 * 2.0 ** -24 * L.w.scale * (ql[t].abs() @ K.abs().T).amax(1) + 2.0 ** -21
            tol = (1.01 * H16 + 2 * ds[:, None]) * A + H16 * want.abs() \
                + len(see) * 2.0 ** -25 * K.abs().max() + 2.0 ** -25
            assert bool(((L.last_o[t].double().cpu() - want).abs() <= tol).all()), (r, j)
            lse = s.logsumexp(1)
            assert bool(((L.last_lse[t].double().cpu() - lse).abs()
                         <= ds + len(see) * 2.0 ** -24 + 2.0 ** -22 * lse.abs().clamp(1, 1e3)).all())
            t += 1


@pytest.mark.parametrize("fp8,idx_fp8,dtype", [(False, False, torch.float16),
                                               (True, True, torch.float16),
                                               (True, False, torch.bfloat16)])
@pytest.mark.parametrize("H", [3, 16, 64])
def test_equals_its_parts(pkg, lib, dev, H, fp8, idx_fp8, dtype):
    g = torch.Generator().manual_seed(H)
    ctx = [100, 0, 37]
    bt = torch.randperm(36, generator=g).int().view(3, 12)
    tab = pkg.rope.rotary_table(64, 256, device=dev)
    A, B = (layer(pkg, dev, H, fp8, idx_fp8) for _ in range(2))
    write_context(pkg, dev, A, tab, ctx, bt, dtype, g)
    B.latent_cache.copy_(A.latent_cache)
    a = step(pkg, dev, ctx, PARENTS, bt, H, dtype, g)
    keep = {k: a[k].clone() for k in ("q", "k_pe", "idx_k", "kv_c")}
    out = A.verify_tree(table=tab, **a)
    for k, v in keep.items():
        assert torch.equal(a[k], v), k
    q, ik = (pkg.rope.apply_rotary(a[k], a["positions"], tab, o, i)
             for k, o, i in (("q", P, True), ("idx_k", 0, False)))
    kpe = pkg.rope.apply_rotary(a["k_pe"], a["positions"], tab)
    B.store(a["kv_c"], kpe, ik, a["slot_mapping"])
    o, lse = pkg.mla_tree.tree_attention(pkg.dsa_layer.q_latent(q, B.w), B.latent_cache,
                                         a["block_table"], a["seq_lens"], a["cu_seqlens_q"],
                                         a["tree_mask"], B.w.scale)
    assert torch.equal(A.latent_cache, B.latent_cache) and torch.equal(A.idx_k_cache, B.idx_k_cache)
    assert torch.equal(A.last_o, o) and torch.equal(A.last_lse, lse)
    assert torch.equal(out, pkg.dsa_layer.v_up(o, B.w))


@pytest.mark.parametrize("fp8", [False, True])
def test_two_steps_of_drafting(pkg, lib, dev, fp8):
    """A step's trees, a path of each accepted and written behind the context, and the
    next step's trees over it."""
    g = torch.Generator().manual_seed(8)
    H, ctx = 16, [100, 15, 37]
    bt = torch.randperm(36, generator=g).int().view(3, 12)
    tab = pkg.rope.rotary_table(64, 256, device=dev)
    L = layer(pkg, dev, H, fp8)
    write_context(pkg, dev, L, tab, ctx, bt, torch.float16, g)
    a = step(pkg, dev, ctx, PARENTS, bt, H, torch.float16, g)
    L.verify_tree(table=tab, **a)
    check_attention(pkg, dev, L, a, ctx, PARENTS, tab)
    cu = a["cu_seqlens_q"].tolist()
    for r, path in enumerate([[0, 2, 5, 6], [0], [1, 3]]):
        t = torch.tensor([cu[r] + j for j in path], device=dev)
        new = range(ctx[r], ctx[r] + len(path))
        assert a["positions"][t].tolist() == list(new)
        pkg._cache_ops.rope_concat_and_cache_mla(a["positions"][t], tab, a["kv_c"][t], a["k_pe"][t],
                                                 L.latent_cache, slots(bt, r, new).to(dev), L.kv_dtype)
    ctx = [104, 16, 39]
    par = [[-1, -1, 1], [-1, 0, 1, 2, 3, 4], [-1] * 5]
    a = step(pkg, dev, ctx, par, bt, H, torch.float16, g)
    L.verify_tree(table=tab, **a)
    check_attention(pkg, dev, L, a, ctx, par, tab)


def test_padded_batch(pkg, lib, dev):
    """Tokens behind the last request: no row is written, their output is zero."""
    g = torch.Generator().manual_seed(9)
    H, ctx = 16, [40]
    bt = torch.randperm(12, generator=g).int().view(1, 12)
    tab = pkg.rope.rotary_table(64, 256, device=dev)
    A, B = layer(pkg, dev, H, True), layer(pkg, dev, H, True)
    write_context(pkg, dev, A, tab, ctx, bt, torch.float16, g)
    B.latent_cache.copy_(A.latent_cache)
    a = step(pkg, dev, ctx, PARENTS[:1], bt, H, torch.float16, g)
    want = A.verify_tree(table=tab, **a)
    pad = {k: torch.cat([v, v[:3]]) for k, v in a.items()
           if k in ("q", "kv_c", "k_pe", "idx_k", "tree_mask")}
    for k in ("positions", "slot_mapping"):
        pad[k] = torch.cat([a[k], torch.full((3,), -1, device=dev)])
    out = B.verify_tree(table=tab, **{**a, **pad})
    assert torch.equal(out[:-3], want) and bool((out[-3:] == 0).all())
    assert torch.equal(A.latent_cache, B.latent_cache) and torch.equal(A.idx_k_cache, B.idx_k_cache)


def test_captured(pkg, lib, dev):
    """Captured once, replayed with new inputs, other work between the replays."""
    g = torch.Generator().manual_seed(10)
    H, ctx = 16, [100, 5, 37]
    bt = torch.randperm(36, generator=g).int().view(3, 12)
    tab = pkg.rope.rotary_table(64, 256, device=dev)
    A, B = layer(pkg, dev, H, True), layer(pkg, dev, H, True)
    write_context(pkg, dev, A, tab, ctx, bt, torch.float16, g)
    B.latent_cache.copy_(A.latent_cache)
    a = step(pkg, dev, ctx, PARENTS, bt, H, torch.float16, g)
    A.verify_tree(table=tab, **a)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = A.verify_tree(table=tab, **a)
    for k in range(4):
        b = step(pkg, dev, [c + k for c in ctx], PARENTS, bt, H, torch.float16, g)
        for n in a:
            a[n].copy_(b[n])
        graph.replay()
        want = B.verify_tree(table=tab, **b)
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(A.latent_cache, B.latent_cache)
        assert torch.equal(A.idx_k_cache, B.idx_k_cache)
