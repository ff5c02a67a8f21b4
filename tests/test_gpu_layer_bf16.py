"""GPU tests of DsaLayer steps whose kv_c and k_pe are bf16: the layer's rows hold their
rope values as fp16, which is what everything that attends to them reads.  Expected rows
come from the bf16 inputs themselves (the quantised values from the row format's
definition on the CPU, the rope values as the numbers that k_pe holds), never from the
cache.  Bounds of the tree attention as in test_gpu_verify_tree, of decode the op's own
(2e-3 relative, 1e-3 absolute)."""
import pytest
import torch

from test_gpu_mla_tree import H16, quantise, values
from test_gpu_verify_tree import P, PAGE, PARENTS, layer, slots, step

pytestmark = pytest.mark.gpu

BF = torch.bfloat16


def row_values(kv_c, k_pe):
    """What the rows of these inputs stand for, in fp64 on the CPU."""
    kv = values(quantise(torch.cat([kv_c.float().cpu(), torch.zeros(kv_c.shape[0], 64)], 1)))
    return torch.cat([kv[:, :512], k_pe.double().cpu()], 1)


def context(L, tab, pkg, ctx, bt, dev, g):
    """Contexts written by DsaLayer.store from rotated bf16 tensors; their values."""
    out = []
    for r, n in enumerate(ctx):
        kv, pe, ik = (torch.randn(n, d, generator=g).to(BF).to(dev) for d in (512, 64, 128))
        if n:
            pe = pkg.rope.apply_rotary(pe, torch.arange(n, device=dev), tab)
            L.store(kv, pe, ik, slots(bt, r, range(n)).to(dev))
        out.append(row_values(kv, pe))
    return out


@pytest.mark.parametrize("with_idx", [True, False])
@pytest.mark.parametrize("H", [3, 16, 64])
def test_verify_tree(pkg, lib, dev, H, with_idx):
    g = torch.Generator().manual_seed(40 + H)
    ctx = [100, 0, 37]
    bt = torch.randperm(36, generator=g).int().view(3, 12)
    tab = pkg.rope.rotary_table(64, 256, device=dev)
    L = layer(pkg, dev, H, True)
    hist = context(L, tab, pkg, ctx, bt, dev, g)
    a = step(pkg, dev, ctx, PARENTS, bt, H, BF, g)
    if not with_idx:
        a["idx_k"] = None
    L.verify_tree(table=tab, **a)
    new = row_values(a["kv_c"], pkg.rope.apply_rotary(a["k_pe"], a["positions"], tab))
    qr = pkg.rope.apply_rotary(a["q"], a["positions"], tab, P)
    ql = pkg.dsa_layer.q_latent(qr, L.w).double().cpu()
    t = 0
    for r, par in enumerate(PARENTS):
        first = t
        for j in range(len(par)):
            see, k = [], j
            while k >= 0:
                see.append(first + k)
                k = par[k]
            K = torch.cat([hist[r], new[see]])
            s = ql[t] @ K.T * L.w.scale
            p = s.softmax(1)
            want, A = p @ K[:, :512], p @ K[:, :512].abs()
            ds = 600 * 2.0 ** -24 * L.w.scale * (ql[t].abs() @ K.abs().T).amax(1) + 2.0 ** -21
            tol = (1.01 * H16 + 2 * ds[:, None]) * A + H16 * want.abs() \
                + K.shape[0] * 2.0 ** -25 * K.abs().max() + 2.0 ** -25
            assert bool(((L.last_o[t].double().cpu() - want).abs() <= tol).all()), (r, j)
            lse = s.logsumexp(1)
            assert bool(((L.last_lse[t].double().cpu() - lse).abs()
                         <= ds + K.shape[0] * 2.0 ** -24 + 2.0 ** -22 * lse.abs().clamp(1, 1e3)).all())
            t += 1


@pytest.mark.parametrize("how", ["store", "prologue", "decode", "verify_tree"])
def test_rope_values_of_the_rows(pkg, lib, dev, how):
    """Values at both ends of bf16's exact range in fp16 and far outside it."""
    g = torch.Generator().manual_seed(50)
    H, T = 16, 4
    L = layer(pkg, dev, H, True)
    kv, pe, ik = (torch.randn(T, d, generator=g).to(BF).to(dev) for d in (512, 64, 128))
    pe[0, :6] = torch.tensor([1.0, -0.5, 2.0 ** -14, 65280.0, 2.0 ** -20, -3e38]).to(BF)
    q = torch.randn(T, H, P + 64, generator=g).half().to(dev)
    iq = torch.randn(T, 32, 128, generator=g).half().to(dev)
    iw = torch.randn(T, 32, generator=g).half().to(dev)
    bt = torch.arange(4, dtype=torch.int32, device=dev).view(1, 4)
    slot = torch.tensor([3, 0, 2, 1], device=dev)
    seq = torch.tensor([T], dtype=torch.int32, device=dev)
    if how == "store":
        L.store(kv, pe, ik, slot)
    elif how == "prologue":
        L._prologue(q, kv, pe, ik, slot)
    elif how == "decode":
        L.decode(q, iq, iw, bt, seq, kv, pe, ik, slot)
    else:
        tab = pkg.rope.rotary_table(64, 1, device=dev)  # position 0: not turned
        pos = torch.zeros(T, dtype=torch.int64, device=dev)
        L.verify_tree(q, kv, pe, pos, tab, slot, bt, seq,
                      torch.tensor([0, T], dtype=torch.int32, device=dev),
                      torch.ones(T, dtype=torch.int64, device=dev), ik)
    rows = L.latent_cache.view(-1, 656)[slot]
    assert torch.equal(rows[:, 528:].contiguous().view(torch.float16), pe.half())
    want = quantise(torch.cat([kv.float().cpu(), torch.zeros(T, 64)], 1))
    assert torch.equal(rows[:, :528].cpu(), want[:, :528])


def test_decode(pkg, lib, dev):
    """A step of the layer's sparse attention, every position selected."""
    g = torch.Generator().manual_seed(60)
    H, n = 64, [150, 33]
    bt = torch.randperm(36, generator=g).int().view(2, 18)
    tab = pkg.rope.rotary_table(64, 256, device=dev)
    L = layer(pkg, dev, H, True)
    hist = context(L, tab, pkg, n, bt, dev, g)
    kv, pe, ik = (torch.randn(2, d, generator=g).to(BF).to(dev) for d in (512, 64, 128))
    q = torch.randn(2, H, P + 64, generator=g).half().to(dev)
    iq, iw = (torch.randn(2, *d, generator=g).half().to(dev) for d in ((32, 128), (32,)))
    slot = torch.cat([slots(bt, r, [n[r]]) for r in range(2)]).to(dev)
    seq = torch.tensor([x + 1 for x in n], dtype=torch.int32, device=dev)
    L.decode(q, iq, iw, bt.to(dev), seq, kv, pe, ik, slot)
    new, ql = row_values(kv, pe), pkg.dsa_layer.q_latent(q, L.w).double().cpu()
    for r in range(2):
        K = torch.cat([hist[r], new[r:r + 1]])
        want = (ql[r] @ K.T * L.w.scale).softmax(1) @ K[:, :512]
        torch.testing.assert_close(L.last_o[r].double().cpu(), want, rtol=2e-3, atol=1e-3)
