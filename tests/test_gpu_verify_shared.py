"""DsaLayer.verify_tree told of shared rows, at sizes where they are read once for all requests and
where tree attention is faster: the definition in both (tolerances of test_gpu_verify_tree), and
what it gives without in the latter."""
import pytest
import torch
from test_gpu_verify_tree import PAGE, check_attention, layer, step, write_context

pytestmark = pytest.mark.gpu
I32 = torch.int32


@pytest.mark.parametrize("fp8,dtype", [(False, torch.float16), (True, torch.bfloat16)])
@pytest.mark.parametrize("n_req", [5, 130])
def test_verify_tree_of_shared_rows(pkg, lib, dev, fp8, dtype, n_req, monkeypatch):
    g = torch.Generator().manual_seed(n_req)
    H, shared = 4, 48
    ctx = [shared + 1 + 3 * r % 11 for r in range(n_req)]
    parents = [[[-1], [-1, 0], [-1, -1, 1]][r % 3] for r in range(n_req)]
    pages = torch.randperm(3 + n_req, generator=g).int()
    bt = torch.empty(n_req, 4, dtype=I32)
    bt[:, :3], bt[:, 3] = pages[:3], pages[3:]
    tab = pkg.rope.rotary_table(64, 256, device=dev)
    A, B = (layer(pkg, dev, H, fp8, blocks=3 + n_req) for _ in range(2))
    write_context(pkg, dev, A, tab, ctx, bt, dtype, g)
    B.latent_cache.copy_(A.latent_cache)
    a = step(pkg, dev, ctx, parents, bt, H, dtype, g)
    cs = torch.tensor([0, n_req], dtype=I32, device=dev)
    lens = pkg.paging.shared_lengths(a["block_table"], a["seq_lens"], cs, PAGE)
    assert lens.tolist() == [shared]
    called = []
    for m, name in ((pkg.mla_prefix, "shared_prefix_attention"), (pkg.mla_tree, "tree_attention")):
        f = getattr(m, name)
        monkeypatch.setattr(m, name, lambda *x, f=f, n=name, **kw: (called.append(n), f(*x, **kw))[1])
    out = A.verify_tree(table=tab, cu_shared=cs, shared_lens=lens, **a)
    assert called == ["shared_prefix_attention" if n_req > 128 else "tree_attention"]
    check_attention(pkg, dev, A, a, ctx, parents, tab)
    want = B.verify_tree(table=tab, **a)
    assert torch.equal(A.latent_cache, B.latent_cache) and torch.equal(A.idx_k_cache, B.idx_k_cache)
    if n_req <= 128:
        assert torch.equal(out, want)
    assert torch.equal(out, pkg.dsa_layer.v_up(A.last_o, A.w))
