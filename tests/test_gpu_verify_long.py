"""GPU tests of DsaLayer.verify_tree where the block table holds more positions than
topk: drafts are accepted by what decode gives, the attention over the indexer's choice
out of the positions that a token sees.

Indexer inputs are small dyadic numbers and the tokens' positions have no table row (so
nothing is rotated), which makes every score exact and the choice unique; the attention
is held to the sparse attention's definition, scores of fp16(q * fp16(scale)), and its
bounds (2e-3 relative, 1e-3 absolute, lse 1e-4).  Without those two roundings in the
expected scores lse would be off by 2^-11 of a score from the scale alone: 3e-3 at 7."""
import pytest
import torch

from test_gpu_verify_tree import P, PAGE, V, slots

pytestmark = pytest.mark.gpu

TOPK = 128


def exact(rows):
    """Cache rows in fp64; of fp8_ds_mla rows e4m3 * scale, which the sparse attention does
    not round to fp16 (that would move scores by 2^-12 of sum |q k|)."""
    if rows.dtype != torch.uint8:
        return rows.double()
    n = rows.shape[0]
    v = rows[:, :512].contiguous().view(torch.float8_e4m3fn).double().view(n, 4, 128)
    v = v * rows[:, 512:528].contiguous().view(torch.float32).double()[:, :, None]
    return torch.cat([v.view(n, 512), rows[:, 528:].contiguous().view(torch.float16).double()], 1)


def dyadic(g, *shape, num=8, den=8):
    return (torch.randint(-num, num + 1, shape, generator=g) / den).half()


def layer(pkg, dev, H, fp8, blocks=120, seed=3):
    g = torch.Generator().manual_seed(seed)
    m = pkg.dsa_layer
    w = m.DsaLayerWeights((torch.randn(H, P, 512, generator=g) * 0.05).half().to(dev),
                          (torch.randn(H, 512, V, generator=g) * 0.05).half().to(dev), 192 ** -0.5)
    lat = torch.zeros(blocks, PAGE, 656, dtype=torch.uint8, device=dev) if fp8 else \
        torch.zeros(blocks, PAGE, 576, dtype=torch.float16, device=dev)
    return m.DsaLayer(w, lat, torch.zeros(blocks, PAGE, 128, dtype=torch.float16, device=dev), TOPK)


def fill(L, ctx, bt, dev, g):
    for r, n in enumerate(ctx):
        if n:
            L.store(torch.randn(n, 512, generator=g).half().to(dev),
                    torch.randn(n, 64, generator=g).half().to(dev), dyadic(g, n, 128).to(dev),
                    slots(bt, r, range(n)).to(dev))


def step(ctx, counts, bt, H, dev, g):
    T = sum(counts)
    slot = torch.cat([slots(bt, r, range(n, n + k)) for r, (n, k) in enumerate(zip(ctx, counts))])
    return dict(q=torch.randn(T, H, P + 64, generator=g).half().to(dev),
                kv_c=torch.randn(T, 512, generator=g).half().to(dev),
                k_pe=torch.randn(T, 64, generator=g).half().to(dev),
                slot_mapping=slot.to(dev), idx_k=dyadic(g, T, 128).to(dev),
                idx_q=dyadic(g, T, 32, 128).to(dev), idx_w=dyadic(g, T, 32, num=4, den=4).to(dev))


def meta(ctx, counts, bt, dev):
    i32 = dict(dtype=torch.int32, device=dev)
    return dict(block_table=bt.to(dev),
                seq_lens=torch.tensor([a + b for a, b in zip(ctx, counts)], **i32),
                cu_seqlens_q=torch.tensor([sum(counts[:i]) for i in range(len(counts) + 1)], **i32))


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("H", [16, 64])
@pytest.mark.parametrize("n", [1, 2, 4])
def test_chains_as_decode(pkg, lib, dev, n, H, fp8):
    """Chains of drafts: the choice and the outputs of decode, bit for bit."""
    g = torch.Generator().manual_seed(n + H)
    ctx = [300, 60, 411]
    bt = torch.randperm(111, generator=g).int().view(3, 37)
    A, B = layer(pkg, dev, H, fp8), layer(pkg, dev, H, fp8)
    fill(A, ctx, bt, dev, g)
    B.latent_cache.copy_(A.latent_cache)
    B.idx_k_cache.copy_(A.idx_k_cache)
    a, m = step(ctx, [n] * 3, bt, H, dev, g), meta(ctx, [n] * 3, bt, dev)
    tab = pkg.rope.rotary_table(64, 512, device=dev)
    pos = torch.cat([torch.arange(c, c + n) for c in ctx]).to(dev)
    mask = torch.tensor([2 ** (j + 1) - 1 for _ in ctx for j in range(n)], device=dev)
    out = A.verify_tree(positions=pos, table=tab, tree_mask=mask, **a, **m)
    q, pe, ik, iq = pkg.rope.apply_rotary([a["q"], a["k_pe"], a["idx_k"], a["idx_q"]], pos, tab,
                                          [P, 0, 0, 0], [True, True, False, False])
    want = B.decode(q, iq, a["idx_w"], m["block_table"], m["seq_lens"], a["kv_c"], pe, ik,
                    a["slot_mapping"])
    assert torch.equal(A.latent_cache, B.latent_cache) and torch.equal(A.idx_k_cache, B.idx_k_cache)
    # decode lists a row's choice first; hidden drafted tokens leave gaps here
    for x, y in zip(A.last_idx.tolist(), B.last_idx.tolist()):
        assert [i for i in x if i >= 0] == [i for i in y if i >= 0]
    assert torch.equal(A.last_o, B.last_o) and torch.equal(out, want)
    assert torch.equal(A.last_lse, B.last_lse)


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("H,extra", [(16, 0), (16, 30), (64, 3)])
def test_trees(pkg, lib, dev, H, extra, fp8):
    """Trees of several shapes, one with a token that sees nothing, tokens of no request
    behind them (30: the kernel for many tokens of few heads)."""
    g = torch.Generator().manual_seed(H + extra)
    ctx = [300, 0, 470, 150]
    par = [[-1, 0, 0, 1, 2, 2, 5], [-1, 0], [-1, -1, 0, 1, 3], [-1, 0, 1]]
    bt = torch.randperm(120, generator=g).int().view(4, 30)
    L = layer(pkg, dev, H, fp8)
    lens = [len(x) for x in par]
    fill(L, ctx, bt, dev, g)
    a, m = step(ctx, lens, bt, H, dev, g), meta(ctx, lens, bt, dev)
    mask = [x for p in par for x in pkg.mla_tree.tree_masks(p)[0]]
    mask[lens[0]] = 0  # of the request without a context: sees nothing
    T = len(mask)
    if extra:
        for k in ("q", "kv_c", "k_pe", "idx_k", "idx_q", "idx_w"):
            a[k] = torch.cat([a[k], a[k].new_ones((extra, *a[k].shape[1:]))])
        a["slot_mapping"] = torch.cat([a["slot_mapping"], torch.full((extra,), -1, device=dev)])
    pos = torch.full((T + extra,), -1, device=dev)
    tab = pkg.rope.rotary_table(64, 8, device=dev)
    out = L.verify_tree(positions=pos, table=tab, tree_mask=torch.tensor(mask + [-1] * extra, device=dev),
                        **a, **m)
    ql = (pkg.dsa_layer.q_latent(a["q"], L.w).cpu().float() * torch.tensor(L.w.scale).half().float())
    ql = ql.half().double()  # an fp16 product is exact in fp32
    rows, keys = L.latent_cache.flatten(0, 1).cpu(), L.idx_k_cache.flatten(0, 1).double().cpu()
    t = 0
    for r, p in enumerate(par):
        for j in range(len(p)):
            see = list(range(ctx[r])) + [ctx[r] + i for i in range(len(p)) if mask[t] >> i & 1]
            at = slots(bt, r, see) if see else torch.zeros(0, dtype=torch.long)
            s = (a["idx_q"][t].double().cpu() @ keys[at].T).clamp_min(0).T @ a["idx_w"][t].double().cpu()
            order = sorted(range(len(see)), key=lambda i: (-float(s[i]), see[i]))[:TOPK]
            pick = sorted(order)
            assert [i for i in L.last_idx[t].tolist() if i >= 0] == [see[i] for i in pick], (r, j)
            if not see:
                assert bool((L.last_o[t] == 0).all()) and bool((out[t] == 0).all())
                assert bool((L.last_lse[t] == -torch.inf).all())
            else:
                K = exact(rows[at[pick]])
                s = ql[t] @ K.T
                want = s.softmax(1) @ K[:, :512]
                torch.testing.assert_close(L.last_o[t].double().cpu(), want, rtol=2e-3, atol=1e-3)
                assert (L.last_lse[t].double().cpu() - s.logsumexp(1)).abs().max() <= 1e-4
            t += 1
    assert bool((out[T:] == 0).all()) and bool((L.last_o[T:] == 0).all())
    assert bool((L.last_lse[T:] == -torch.inf).all())


def test_lengths_past_the_table_and_below_nothing(pkg, lib, dev):
    """A length past the table: its positions are seen, the drafted tokens have none; a
    negative one: nothing is seen; offsets past the tokens end with them."""
    g = torch.Generator().manual_seed(12)
    H, ctx, counts = 16, [477, 100, 200], [3, 2, 2]
    bt = torch.randperm(90, generator=g).int().view(3, 30)
    L = layer(pkg, dev, H, False)
    fill(L, ctx, bt, dev, g)
    a, m = step(ctx, counts, bt, H, dev, g), meta(ctx, counts, bt, dev)
    m["seq_lens"] = torch.tensor([500, -7, 202], dtype=torch.int32, device=dev)
    m["cu_seqlens_q"] = torch.tensor([0, 3, 5, 9], dtype=torch.int32, device=dev)  # 7 tokens
    a["slot_mapping"][:5] = -1
    mask = torch.tensor([1, 3, 5, 1, 3, 1, 3], device=dev)
    pos = torch.full((7,), -1, device=dev)
    out = L.verify_tree(positions=pos, table=pkg.rope.rotary_table(64, 8, device=dev), tree_mask=mask,
                        **a, **m)
    keys = L.idx_k_cache.flatten(0, 1).double().cpu()
    for t in range(7):
        r = [0, 0, 0, 1, 1, 2, 2][t]
        j = t - [0, 3, 5][r]
        see = [list(range(480)), [], list(range(200)) + [200 + i for i in range(j + 1)]][r]
        at = slots(bt, r, see) if see else torch.zeros(0, dtype=torch.long)
        s = (a["idx_q"][t].double().cpu() @ keys[at].T).clamp_min(0).T @ a["idx_w"][t].double().cpu()
        pick = sorted(sorted(range(len(see)), key=lambda i: (-float(s[i]), see[i]))[:TOPK])
        assert [i for i in L.last_idx[t].tolist() if i >= 0] == [see[i] for i in pick], t
    assert bool((out[3:5] == 0).all()) and bool((L.last_lse[3:5] == -torch.inf).all())
    assert bool((out[:3] != 0).any()) and bool((out[5:] != 0).any())


def test_captured(pkg, lib, dev):
    """Captured once, replayed with other lengths and inputs and eager work between."""
    g = torch.Generator().manual_seed(9)
    H, ctx = 16, [300, 150]
    bt = torch.randperm(100, generator=g).int().view(2, 50)
    A, B = layer(pkg, dev, H, True), layer(pkg, dev, H, True)
    fill(A, ctx, bt, dev, g)
    B.latent_cache.copy_(A.latent_cache)
    B.idx_k_cache.copy_(A.idx_k_cache)
    tab = pkg.rope.rotary_table(64, 512, device=dev)

    def args(c):
        par = [[-1, 0, 0, 2], [-1, 0, 1]]
        depth = [pkg.mla_tree.tree_masks(p) for p in par]
        return dict(positions=torch.tensor([n + d for n, (_, ds) in zip(c, depth) for d in ds], device=dev),
                    tree_mask=torch.tensor([m for ms, _ in depth for m in ms], device=dev),
                    **step(c, [4, 3], bt, H, dev, g), **meta(c, [4, 3], bt, dev))

    a = args(ctx)
    A.verify_tree(table=tab, **a)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = A.verify_tree(table=tab, **a)
    for k in range(4):
        b = args([n + 3 * k for n in ctx])
        for x in a:
            a[x].copy_(b[x])
        graph.replay()
        want = B.verify_tree(table=tab, **b)
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(A.latent_cache, B.latent_cache)
        assert torch.equal(A.idx_k_cache, B.idx_k_cache)
