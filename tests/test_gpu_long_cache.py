"""GPU tests of the latent cache's operators with rows past 4 GiB: written, read back and
attended to.  Only the pages in use are ever touched."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fp8", [False, True])
def test_rows_past_4_gib(pkg, lib, dev, fp8):
    page, row = 64, 656 if fp8 else 1152
    blocks = (2 ** 32 + 2 ** 28) // (page * row) + 3
    big = torch.empty(blocks, page, 656, dtype=torch.uint8, device=dev) if fp8 else \
        torch.empty(blocks, page, 576, dtype=torch.float16, device=dev)
    small = torch.zeros(4, page, big.shape[2], dtype=big.dtype, device=dev)
    pages = [blocks - 1, 0, blocks - 2, 2 ** 32 // (page * row)]  # the last one crosses 4 GiB
    g = torch.Generator().manual_seed(5)
    n, H = 4 * page, 16
    kv_c, k_pe = (torch.randn(n, d, generator=g).half().to(dev) for d in (512, 64))
    tab = pkg.rope.rotary_table(64, n, device=dev)
    pos = torch.arange(n, device=dev)
    bt = [torch.tensor([x], dtype=torch.int32, device=dev) for x in (pages, [0, 1, 2, 3])]
    kind = "fp8_ds_mla" if fp8 else "auto"
    q = torch.randn(3, H, 576, generator=g).half().to(dev)
    seq, cu = (torch.tensor(x, dtype=torch.int32, device=dev) for x in ([n - 5], [0, 3]))
    ends = torch.tensor([0, n], dtype=torch.int32, device=dev)
    mask = torch.tensor([1, 3, 5], device=dev)
    got = []
    for cache, t in ((big, bt[0]), (small, bt[1])):
        slot = t[0].long()[pos // page] * page + pos % page
        assert cache is small or int(slot.max()) * row > 2 ** 32
        pkg._cache_ops.rope_concat_and_cache_mla(pos, tab, kv_c, k_pe, cache, slot, kind)
        got.append((cache[t[0].long()], pkg._cache_ops.gather_latent_cache(cache, t, ends, n),
                    *pkg.mla_tree.tree_attention(q, cache, t, seq, cu, mask, 0.07)))
    for a, b in zip(*got):
        assert torch.equal(a, b)
    assert bool(torch.isfinite(got[0][2]).all())
