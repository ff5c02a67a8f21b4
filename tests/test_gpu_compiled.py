"""The rotary, latent cache and tree attention entry points in compiled functions, whole
graphs: the eager results, bit for bit, in-place outputs and written caches included."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("backend", ["eager", "aot_eager"])
@pytest.mark.parametrize("kv", ["fp16", "fp8"])
def test_step(pkg, lib, dev, backend, kv):
    g = torch.Generator().manual_seed(5)
    T, H, page = 6, 16, 16
    fp8 = kv == "fp8"
    tab = pkg.rope.rotary_table(64, 256, device=dev)
    bt = torch.randperm(16, generator=g).int().view(2, 8).to(dev)
    seq, cu = (torch.tensor(x, dtype=torch.int32, device=dev) for x in ([100, 37], [0, 4, 6]))
    pos = torch.tensor([96, 97, 98, 99, 35, 36], device=dev)
    slot = torch.cat([bt[0][pos[:4] // page] * page + pos[:4] % page,
                      bt[1][pos[4:] // page] * page + pos[4:] % page]).long()
    mask = torch.tensor([1, 3, 5, 9, 1, 3], device=dev)
    x = dict(q=torch.randn(T, H, 192, generator=g).half(), kv_c=torch.randn(T, 512, generator=g).half(),
             k_pe=torch.randn(T, 64, generator=g).half(), idx=torch.randn(T, 3, 128, generator=g).half(),
             lat=torch.randn(T, H, 576, generator=g).half())
    kvc = torch.randn(256, 512, generator=g).half().to(dev)
    ends = torch.tensor([0, 100, 137], dtype=torch.int32, device=dev)
    name = "fp8_ds_mla" if fp8 else "auto"

    def step(q, kv_c, k_pe, idx, lat, cache):
        pkg.rope.apply_rotary(idx, pos, tab, 0, False, idx)
        q2 = pkg.rope.apply_rotary([q, k_pe], pos, tab, [128, 0])
        y = pkg._cache_ops.rope_concat_and_cache_mla(pos, tab, kv_c, k_pe, cache, slot, name, q=q,
                                                     q_offset=128)
        pkg._cache_ops.rope_concat_and_cache_mla(pos, tab, kv_c, k_pe, cache, slot, name, q=q,
                                                 q_offset=128, q_out=q)
        rows = pkg._cache_ops.gather_latent_cache(cache, bt, ends, 137)
        o, lse = pkg.mla_tree.tree_attention(lat, cache, bt, seq, cu, mask, 0.07)
        return (*q2, y, rows, o * 2, lse)

    got = []
    for f in (step, torch.compile(step, backend=backend, fullgraph=True)):
        cache = torch.zeros(16, page, 656 if fp8 else 576, dtype=torch.uint8 if fp8 else torch.float16,
                            device=dev)
        pkg._cache_ops.concat_and_cache_mla(kvc, kvc[:, :64].contiguous(), cache,
                                            torch.arange(256, device=dev), name,
                                            torch.ones((), device=dev))
        a = {k: v.clone().to(dev) for k, v in x.items()}
        for _ in range(2):  # the second time on rotated inputs
            out = f(a["q"], a["kv_c"], a["k_pe"], a["idx"], a["lat"], cache)
        got.append([*out, cache, a["q"], a["idx"], a["k_pe"]])
    for a, b in zip(*got):
        assert torch.equal(a, b)
    assert not torch.equal(got[0][-2].cpu(), x["idx"])
