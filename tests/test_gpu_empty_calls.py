"""Calls with no tokens, no heads, no requests or no rows: an empty result or an untouched
output, no error."""
import pytest
import torch

from test_gpu_verify_tree import P, layer

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T", [0, 1, 5])
def test_rotary_of_no_heads(pkg, lib, dev, T):
    tab = pkg.rope.rotary_table(64, 16, device=dev)
    pos = torch.arange(T, device=dev)
    x, y = torch.empty(T, 0, 192, device=dev).half(), torch.randn(T, 3, 128, device=dev).half()
    assert pkg.rope.apply_rotary(x, pos, tab, 128).shape == (T, 0, 192)
    assert pkg.rope.apply_rotary(x, pos, tab, 128, outs=x) is x
    a, b = pkg.rope.apply_rotary([x, y], pos, tab, [128, 0])
    assert a.shape == x.shape and torch.equal(b, pkg.rope.apply_rotary(y, pos, tab))


@pytest.mark.parametrize("T,H", [(0, 3), (0, 0), (4, 0)])
def test_cache_write(pkg, lib, dev, T, H):
    tab = pkg.rope.rotary_table(64, 16, device=dev)
    pos = torch.arange(T, device=dev)
    kv, pe = torch.randn(T, 512, device=dev).half(), torch.randn(T, 64, device=dev).half()
    q = torch.randn(T, H, 192, device=dev).half()
    a, b = (torch.zeros(1, 16, 656, dtype=torch.uint8, device=dev) for _ in range(2))
    f = pkg._cache_ops.rope_concat_and_cache_mla
    assert f(pos, tab, kv, pe, a, pos, "fp8_ds_mla", q=q, q_offset=128).shape == (T, H, 192)
    f(pos, tab, kv, pe, b, pos, "fp8_ds_mla")
    assert torch.equal(a, b)


def test_read_back(pkg, lib, dev):
    kv = torch.randn(2, 16, 576, device=dev).half()
    i32 = dict(dtype=torch.int32, device=dev)
    f = pkg._cache_ops.gather_latent_cache
    bt = torch.zeros(1, 2, **i32)
    assert f(kv, bt, torch.zeros(2, **i32), 0).shape == (0, 576)
    out = torch.full((3, 576), 7.0, device=dev).half()
    f(kv, bt, torch.zeros(2, **i32), 3, out=out)
    f(kv, bt[:0], torch.zeros(1, **i32), 3, out=out)
    assert bool((out == 7).all())
    f(kv, bt[:, :0], torch.tensor([0, 3], **i32), 3, out=out)  # no pages: zeros
    assert bool((out == 0).all())


@pytest.mark.parametrize("T,R", [(0, 2), (0, 0), (4, 0)])
def test_tree_attention(pkg, lib, dev, T, R):
    i32 = dict(dtype=torch.int32, device=dev)
    q = torch.randn(T, 3, 576, device=dev).half()
    kv = torch.randn(2, 16, 576, device=dev).half()
    out = torch.full((T, 3, 512), 7.0, device=dev).half()
    lse = torch.full((T, 3), 7.0, device=dev)
    pkg.mla_tree.tree_attention(q, kv, torch.zeros(R, 2, **i32), torch.zeros(R, **i32),
                                torch.zeros(R + 1, **i32), torch.ones(T, dtype=torch.int64, device=dev),
                                0.1, out, lse)
    assert bool((out == 7).all()) and bool((lse == 7).all())


@pytest.mark.parametrize("topk", [2048, 16])
@pytest.mark.parametrize("T,R", [(0, 2), (0, 0), (4, 0)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_verify_tree(pkg, lib, dev, T, R, topk, dtype):
    i32 = dict(dtype=torch.int32, device=dev)
    L = layer(pkg, dev, 3, True)
    L.topk = topk  # of the 32 positions of a table
    tab = pkg.rope.rotary_table(64, 16, device=dev)
    slot = torch.full((T,), -1, device=dev)
    before = L.latent_cache.clone(), L.idx_k_cache.clone()
    out = L.verify_tree(torch.randn(T, 3, P + 64, device=dev).half(),
                        torch.randn(T, 512, device=dev).to(dtype), torch.randn(T, 64, device=dev).to(dtype),
                        slot, tab, slot, torch.zeros(R, 2, **i32), torch.zeros(R, **i32),
                        torch.zeros(R + 1, **i32), torch.ones(T, dtype=torch.int64, device=dev),
                        torch.randn(T, 128, device=dev).to(dtype),
                        idx_q=torch.randn(T, 32, 128, device=dev).half(),
                        idx_w=torch.randn(T, 32, device=dev).half())
    assert out.shape == (T, 3 * L.w.v_dim) and bool((out == 0).all())
    assert torch.equal(before[0], L.latent_cache) and torch.equal(before[1], L.idx_k_cache)
