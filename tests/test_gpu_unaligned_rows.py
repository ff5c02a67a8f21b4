"""Views that do not start on 16 bytes, or whose one row has an odd stride, give what
aligned copies of them give: one token (which torch counts as contiguous wherever it
starts) as several."""
import pytest
import torch

from test_gpu_verify_tree import P, layer

pytestmark = pytest.mark.gpu


def view(x, off, wide=613):
    """x [T, ...] as part of a wider buffer, `off` elements from its start."""
    flat = x.reshape(x.shape[0], -1)
    buf = torch.full((x.shape[0], flat.shape[1] + wide), 7.0, dtype=x.dtype, device=x.device)
    buf[:, off:off + flat.shape[1]] = flat
    st = (buf.stride(0), *x.stride()[1:])
    return buf.as_strided(x.shape, st, off)


@pytest.mark.parametrize("T", [1, 3])
@pytest.mark.parametrize("off,wide", [(3, 613), (3, 616), (8, 613), (1, 64), (0, 1)])
def test_cache_rows(pkg, lib, dev, T, off, wide):
    g = torch.Generator().manual_seed(T)
    kv, pe = (torch.randn(T, d, generator=g).half().to(dev) for d in (512, 64))
    q = torch.randn(T, 5, 192, generator=g).half().to(dev)
    pos, slot = torch.arange(T, device=dev), torch.arange(T, device=dev)
    tab = pkg.rope.rotary_table(64, 8, device=dev)
    one = torch.ones((), device=dev)
    got = []
    for a, b, c in ((kv, pe, q), (view(kv, off, wide), view(pe, off, wide), view(q, off, wide))):
        x, y = (torch.zeros(1, 8, 656, dtype=torch.uint8, device=dev) for _ in range(2))
        pkg._cache_ops.concat_and_cache_mla(a, b, x, slot, "fp8_ds_mla", one)
        r = pkg._cache_ops.rope_concat_and_cache_mla(pos, tab, a, b, y, slot, "fp8_ds_mla", q=c,
                                                     q_offset=128)
        got.append((x, y, r, pkg.rope.apply_rotary(c, pos, tab, 128)))
    for a, b in zip(*got):
        assert torch.equal(a, b)


@pytest.mark.parametrize("T,H", [(1, 1), (1, 5), (3, 5)])
@pytest.mark.parametrize("off", [1, 4, 8])
def test_tree_attention(pkg, lib, dev, T, H, off):
    g = torch.Generator().manual_seed(T + H)
    q = torch.randn(T, H, 576, generator=g).half().to(dev)
    kv = torch.randn(4, 16, 576, generator=g).half().to(dev)
    bt = torch.arange(4, dtype=torch.int32, device=dev).view(1, 4)
    seq, cu = (torch.tensor(x, dtype=torch.int32, device=dev) for x in ([50], [0, T]))
    mask = torch.tensor([1, 3, 5][:T], device=dev)
    a = pkg.mla_tree.tree_attention(q, kv, bt, seq, cu, mask, 0.07)
    b = pkg.mla_tree.tree_attention(view(q, off), kv, bt, seq, cu, mask, 0.07)
    buf = torch.zeros(q.numel() + off, dtype=torch.float16, device=dev)
    buf[off:] = q.flatten()
    c = pkg.mla_tree.tree_attention(buf[off:].view(T, H, 576), kv, bt, seq, cu, mask, 0.07)
    for x in (b, c):
        assert torch.equal(a[0], x[0]) and torch.equal(a[1], x[1])


@pytest.mark.parametrize("T", [1, 2])
@pytest.mark.parametrize("off", [3, 8])
def test_layer_steps(pkg, lib, dev, T, off):
    """decode and verify_tree of views."""
    g = torch.Generator().manual_seed(T)
    H = 16
    t = dict(q=(H, P + 64), kv_c=(512,), k_pe=(64,), idx_k=(128,))
    t = {k: torch.randn(T, *d, generator=g).half().to(dev) for k, d in t.items()}
    iq, iw = (torch.randn(T, *d, generator=g).half().to(dev) for d in ((32, 128), (32,)))
    bt = torch.arange(4, dtype=torch.int32, device=dev).view(1, 4)
    seq, cu = (torch.tensor(x, dtype=torch.int32, device=dev) for x in ([T], [0, T]))
    pos = slot = torch.arange(T, device=dev)
    tab = pkg.rope.rotary_table(64, 8, device=dev)
    mask = torch.tensor([1, 3][:T], device=dev)
    got = []
    for s in (t, {k: view(x, off) for k, x in t.items()}):
        L, M = layer(pkg, dev, H, True), layer(pkg, dev, H, True)
        o = L.verify_tree(s["q"], s["kv_c"], s["k_pe"], pos, tab, slot, bt, seq, cu, mask, s["idx_k"])
        d = M.decode(s["q"], iq, iw, bt, seq, s["kv_c"], s["k_pe"], s["idx_k"].clone(), slot)
        got.append((o, d, L.latent_cache, M.latent_cache, L.idx_k_cache, M.idx_k_cache))
    for a, b in zip(*got):
        assert torch.equal(a, b)
