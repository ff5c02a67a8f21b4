"""GPU parity of the latent cache written with the rotation in the same launch
(_cache_ops.rope_concat_and_cache_mla) and read back (gather_latent_cache): the
first equals, bit for bit, the two calls it replaces; the second equals the rows'
values computed with torch on the CPU (one fp32 product, one rounding: exact), and a
chain of both with the dense chunk attention is compared with 64 bits."""
import math

import pytest
import torch

from test_gpu_mla_tree import H16, quantise

pytestmark = pytest.mark.gpu


def read(rows, dtype, pe):
    if rows.dtype != torch.uint8:
        return rows.to(dtype)
    n = rows.shape[0]
    v = rows[:, :512].contiguous().view(torch.float8_e4m3fn).float().view(n, 4, 128)
    v = v * rows[:, 512:528].contiguous().view(torch.float32)[:, :, None]
    return torch.cat([v.view(n, 512).to(dtype), rows[:, 528:].contiguous().view(pe).to(dtype)], 1)


@pytest.mark.parametrize("inter", [True, False])
@pytest.mark.parametrize("kv,dtype", [("fp8", torch.float16), ("fp8", torch.bfloat16),
                                      ("fp16", torch.float16)])
@pytest.mark.parametrize("T,H", [(1, 64), (7, 5), (130, 16), (1025, 2)])
def test_write_equals_the_two_calls(pkg, lib, dev, T, H, kv, dtype, inter):
    g = torch.Generator().manual_seed(T)
    page, blocks = 16, T // 16 + 3
    q = torch.randn(T, H, 192, generator=g).to(dtype).to(dev)
    kvc = torch.randn(T, 600, generator=g).to(dtype).to(dev)[:, 8:520]
    pe = torch.randn(T, 64, generator=g).to(dtype).to(dev)
    pos = torch.randint(0, 3000, (T,), generator=g).to(dev)
    slot = torch.randperm(blocks * page, generator=g)[:T]
    if T > 1:
        slot[T // 2] = -1
        pos[0] = -1
    slot = slot.to(dev)
    tab = pkg.rope.rotary_table(64, 3000, device=dev)
    fp8 = kv == "fp8"
    a = torch.full((blocks, page, 656 if fp8 else 576), 3, dtype=torch.uint8 if fp8 else dtype,
                   device=dev)
    b = a.clone()
    name = "fp8_ds_mla" if fp8 else "auto"
    wq, wpe = pkg.rope.apply_rotary([q, pe], pos, tab, offsets=[128, 0], interleaved=inter)
    pkg._cache_ops.concat_and_cache_mla(kvc, wpe, a, slot, name, torch.ones((), device=dev))
    q0, pe0 = q.clone(), pe.clone()
    got = pkg._cache_ops.rope_concat_and_cache_mla(pos, tab, kvc, pe, b, slot, name,
                                                   interleaved=inter, q=q, q_offset=128)
    assert torch.equal(got, wq) and torch.equal(a, b)
    assert torch.equal(q, q0) and torch.equal(pe, pe0)
    # int32 slots and positions, q in place; without q
    c = torch.full_like(b, 3)
    got = pkg._cache_ops.rope_concat_and_cache_mla(pos.int(), tab, kvc, pe, c, slot.int(), name,
                                                   interleaved=inter, q=q, q_offset=128, q_out=q)
    assert got is q and torch.equal(q, wq) and torch.equal(c, b)
    c.fill_(3)
    assert pkg._cache_ops.rope_concat_and_cache_mla(pos, tab, kvc, pe, c, slot, name,
                                                    interleaved=inter) is None
    assert torch.equal(c, b)


def test_write_of_extreme_values(pkg, lib, dev):
    """Zero tiles, huge and tiny values, infinities: as the writer alone."""
    kvc = torch.randn(6, 512).bfloat16()
    kvc[0] = 0
    kvc[1, :128] = 3e38
    kvc[2, 128:256] = 1e-38
    kvc[3, 5] = math.inf
    kvc[4, 300] = math.nan
    pe = torch.randn(6, 64).bfloat16()
    tab = pkg.rope.rotary_table(64, 10, device=dev)
    pos = torch.arange(6, device=dev)
    a = torch.zeros(1, 8, 656, dtype=torch.uint8, device=dev)
    b = a.clone()
    slot = torch.arange(6, device=dev)
    pkg._cache_ops.concat_and_cache_mla(kvc.to(dev), pkg.rope.apply_rotary(pe.to(dev), pos, tab), a,
                                        slot, "fp8_ds_mla", torch.ones((), device=dev))
    pkg._cache_ops.rope_concat_and_cache_mla(pos, tab, kvc.to(dev), pe.to(dev), b, slot, "fp8_ds_mla")
    assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("kv,pe", [("fp16", torch.float16), ("fp8", torch.float16),
                                   ("fp8", torch.bfloat16)])
@pytest.mark.parametrize("lens,page,first", [
    ([1], 64, 0), ([0], 16, 0), ([5, 0, 3, 64, 0], 16, 0), ([100, 33, 257], 48, 7),
    ([(13 * i) % 41 for i in range(200)], 5, 2), ([2000, 1], 1, 0)])
def test_read_back(pkg, lib, dev, lens, page, first, kv, pe, dtype):
    g = torch.Generator().manual_seed(len(lens) + page)
    R = len(lens)
    need = [max(1, -(-(n + first) // page)) for n in lens]
    perm = torch.randperm(sum(need) + 1, generator=g).int()
    bt = torch.full((R, max(need)), -1, dtype=torch.int32)
    at = 0
    for r, k in enumerate(need):
        bt[r, :k] = perm[at:at + k]
        at += k
    lat = torch.randn((sum(need) + 1) * page, 576, generator=g)
    rows = quantise(lat) if kv == "fp8" else lat.half()
    if pe is torch.bfloat16:
        rows[:, 528:] = lat[:, 512:].bfloat16().view(torch.uint8)
    cu = torch.tensor([sum(lens[:i]) for i in range(R + 1)], dtype=torch.int32)
    idx = [int(bt[r, p // page]) * page + p % page for r in range(R)
           for p in range(first, first + lens[r])]
    want = read(rows[torch.tensor(idx, dtype=torch.long)], dtype, pe)
    total = sum(lens)
    kvd = rows.view(-1, page, rows.shape[1]).to(dev)
    st = torch.full((R,), first, dtype=torch.int32, device=dev) if first else None
    got = pkg._cache_ops.gather_latent_cache(kvd, bt.to(dev), cu.to(dev), total, starts=st,
                                             dtype=dtype, pe_dtype=pe)
    assert torch.equal(got.cpu(), want)
    # more rows than the requests have, and a wider row: the rest stays
    buf = torch.full((total + 9, 640), 5.0, dtype=dtype, device=dev)
    got = pkg._cache_ops.gather_latent_cache(kvd, bt.to(dev), cu.to(dev), total + 9, starts=st,
                                             dtype=dtype, pe_dtype=pe, out=buf[:, :576])
    assert torch.equal(buf[:total, :576].cpu(), want)
    assert bool((buf[total:] == 5).all()) and bool((buf[:, 576:] == 5).all())


def test_unresolved_positions_read_as_zeros(pkg, lib, dev):
    rows = torch.randn(64, 576).half()
    bt = torch.tensor([[0, -1, 2], [1, 99, 3]], dtype=torch.int32)
    cu = torch.tensor([2, 50, 98], dtype=torch.int32)  # two rows before the first request
    starts = torch.tensor([-8, 16], dtype=torch.int32)  # before the sequence, and past the table
    out = torch.full((98, 576), 7.0, dtype=torch.float16, device=dev)
    pkg._cache_ops.gather_latent_cache(rows.view(4, 16, 576).to(dev), bt.to(dev), cu.to(dev), 98,
                                       starts=starts.to(dev), out=out)
    want = torch.zeros(98, 576).half()
    want[:2] = 7
    for r in range(2):
        for i in range(48):
            p = int(starts[r]) + i
            if 0 <= p < 48 and 0 <= int(bt[r, p // 16]) < 4:
                want[int(cu[r]) + i] = rows[int(bt[r, p // 16]) * 16 + p % 16]
    assert torch.equal(out.cpu(), want)


def test_graph_and_other_stream(pkg, lib, dev):
    T = 48
    q = torch.randn(T, 8, 192, device=dev).half()
    kvc, pe = torch.randn(T, 512, device=dev).half(), torch.randn(T, 64, device=dev).half()
    pos, slot = torch.arange(T, device=dev), torch.randperm(64, device=dev)[:T]
    tab = pkg.rope.rotary_table(64, 64, device=dev)
    bt = torch.arange(4, dtype=torch.int32, device=dev).view(1, 4)
    cu = torch.tensor([0, 64], dtype=torch.int32, device=dev)

    def step(cache):
        y = pkg._cache_ops.rope_concat_and_cache_mla(pos, tab, kvc, pe, cache, slot, "fp8_ds_mla",
                                                     q=q, q_offset=128)
        return y, pkg._cache_ops.gather_latent_cache(cache, bt, cu, 64)

    a = torch.zeros(4, 16, 656, dtype=torch.uint8, device=dev)
    b, c = a.clone(), a.clone()
    torch.cuda.synchronize()
    st = torch.cuda.Stream()
    with torch.cuda.stream(st):
        ya, va = step(a)
    st.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        yb, vb = step(b)
    for k in range(3):
        kvc.mul_(1.25)
        g.replay()
        yc, vc = step(c)
        torch.cuda.synchronize()
        assert torch.equal(yb, yc) and torch.equal(vb, vc) and torch.equal(b, c)
    assert torch.equal(ya, yb) and not torch.equal(va, vb)


def test_chunked_prefill_chain(pkg, lib, dev):
    """A chunk rotated and written, its context read back, projected to keys and values
    of heads, and the dense chunk attention over it.

    Bounds: the keys and values are fp16 matrices of the read-back values on both
    sides; the attention rounds P and o to fp16 (2^-11 of sum p |v| and of |o|), scores
    are off by at most 200 2^-24 scale sum |q k| and as much again through the sum."""
    g = torch.Generator().manual_seed(21)
    H, page, lens, chunk = 4, 16, [70, 33], 20
    tab = pkg.rope.rotary_table(64, 128, device=dev)
    bt = torch.randperm(12, generator=g).int().view(2, 6).to(dev)
    cache = torch.zeros(12, page, 656, dtype=torch.uint8, device=dev)
    W = (torch.randn(512, H * 256, generator=g) / 512 ** 0.5).to(dev)

    def rows(r, lo, hi):
        p = torch.arange(lo, hi)
        return bt[r].cpu().long()[p // page] * page + p % page, p

    lat, pes = [], []
    for r, n in enumerate(lens):  # the history, then the chunk, each in one call
        for lo, hi in ((0, n - chunk), (n - chunk, n)):
            kvc, pe = torch.randn(hi - lo, 512, generator=g).half(), torch.randn(hi - lo, 64, generator=g).half()
            slot, pos = rows(r, lo, hi)
            q = torch.randn(hi - lo, H, 192, generator=g).half().to(dev)
            qr = pkg._cache_ops.rope_concat_and_cache_mla(pos.to(dev), tab, kvc.to(dev), pe.to(dev),
                                                          cache, slot.to(dev), "fp8_ds_mla", q=q,
                                                          q_offset=128)
        lat.append(qr)
    qn = torch.cat(lat)
    cu_q = torch.tensor([0, chunk, 2 * chunk], dtype=torch.int32, device=dev)
    ctx = torch.tensor([0, 50, 63], dtype=torch.int32, device=dev)
    kv = pkg._cache_ops.gather_latent_cache(cache, bt, ctx, 63)
    flat = cache.view(-1, 656).cpu()
    idx = torch.cat([rows(0, 0, 50)[0], rows(1, 0, 13)[0]])
    assert torch.equal(kv.cpu(), read(flat[idx], torch.float16, torch.float16))
    up = (kv[:, :512].float() @ W).half().view(63, H, 256)
    k = torch.cat([up[..., :128], kv[:, None, 512:].expand(63, H, 64)], 2)
    v = up[..., 128:].contiguous()
    o, lse = pkg.mla_prefill.SM70MLAPrefill(192 ** -0.5).run_prefill_context_chunk(qn, k, v, cu_q, ctx)
    for r in range(2):
        for t in range(cu_q[r], cu_q[r + 1]):
            ks, vs = k[ctx[r]:ctx[r + 1]].double().cpu(), v[ctx[r]:ctx[r + 1]].double().cpu()
            q = qn[t].double().cpu()
            s = torch.einsum("hd,khd->hk", q, ks) * 192 ** -0.5
            p = s.softmax(1)
            want, A = torch.einsum("hk,khd->hd", p, vs), torch.einsum("hk,khd->hd", p, vs.abs())
            ds = 200 * 2.0 ** -24 * 192 ** -0.5 * torch.einsum("hd,khd->hk", q.abs(), ks.abs()).amax() \
                + 2.0 ** -20
            tol = (1.01 * H16 + 2 * ds) * A + H16 * want.abs() + 2.0 ** -25 * 64
            assert bool(((o[t].double().cpu() - want).abs() <= tol).all())
