"""GPU parity of the rotary kernel (rope.apply_rotary) and its table against the
definition in 64 bits on the CPU.

Tolerance: y = a c - b s is computed in fp32 from table values rounded to fp32 and
rounded once to the tensor's type: half a step of the type (eps / 2 |y|), and four
fp32 half-steps (table, two products, sum: 2^-24 each) of |a c| + |b s|."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
TYPES = [torch.float16, torch.bfloat16, torch.float32]


def freqs(rot, base=10000.0):
    return torch.tensor([base ** (-2 * i / rot) for i in range(rot // 2)], dtype=torch.float64)


def rotated(x, pos, rot, offset, inter, n_pos, freq=None, mag=1.0):
    """(definition in fp64, bound on the error) for x of any type on the CPU."""
    freq = freqs(rot) if freq is None else freq
    z = x.double()
    z3 = z[:, None] if z.dim() == 2 else z
    y, slack = z3.clone(), torch.zeros_like(z3)
    ang = pos.double()[:, None] * freq
    c, s = mag * ang.cos()[:, None], mag * ang.sin()[:, None]
    live = ((pos >= 0) & (pos < n_pos))[:, None, None]
    i = torch.arange(rot // 2)
    ia, ib = (offset + 2 * i, offset + 2 * i + 1) if inter else (offset + i, offset + i + rot // 2)
    a, b = z3[..., ia], z3[..., ib]
    y[..., ia] = torch.where(live, a * c - b * s, a)
    y[..., ib] = torch.where(live, b * c + a * s, b)
    m = 4 * 2.0 ** -24 * (a.abs() + b.abs()) * max(mag, 1)
    slack[..., ia] = slack[..., ib] = torch.where(live, m, torch.zeros_like(m))
    tiny = torch.finfo(x.dtype).smallest_normal * torch.finfo(x.dtype).eps
    turned = torch.zeros_like(z3, dtype=torch.bool)
    turned[..., ia] = turned[..., ib] = live.expand_as(a)
    tol = torch.where(turned, torch.finfo(x.dtype).eps / 2 * y.abs() + slack + tiny / 2,
                      torch.zeros_like(y))
    return y.view(x.shape), tol.view(x.shape)


def close(got, want):
    y, tol = want
    d = (got.double().cpu() - y).abs()
    assert bool((d <= tol).all()), float((d - tol).max())


def table(pkg, rot, n, dev, **kw):
    return pkg.rope.rotary_table(rot, n, device=dev, **kw)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("inter", [True, False])
@pytest.mark.parametrize("T,H,D,rot,offset", [
    (1, 64, 192, 64, 128), (5, 3, 64, 64, 0), (300, 16, 128, 64, 0), (2, 1, 2, 2, 0),
    (7, 5, 101, 36, 13), (33, 2, 40, 10, 30), (1, 1, 576, 64, 512), (1030, 2, 24, 16, 8),
    (3, 128, 320, 256, 0), (257, 7, 72, 8, 64)])
def test_matches_definition(pkg, lib, dev, dtype, inter, T, H, D, rot, offset):
    g = torch.Generator().manual_seed(T + D)
    x = torch.randn(T, H, D, generator=g).to(dtype)
    pos = torch.randint(0, 5000, (T,), generator=g)
    tab = table(pkg, rot, 5000, dev)
    want = rotated(x, pos, rot, offset, inter, 5000)
    xd = x.to(dev)
    got = pkg.rope.apply_rotary(xd, pos.to(dev), tab, offsets=offset, interleaved=inter)
    close(got, want)
    assert torch.equal(xd.cpu(), x)
    # int32 positions, in place: the same bits
    ret = pkg.rope.apply_rotary(xd, pos.int().to(dev), tab, offsets=offset, interleaved=inter,
                                outs=xd)
    assert ret is xd and torch.equal(xd, got)


@pytest.mark.parametrize("dtype", TYPES)
def test_a_steps_tensors_in_one_launch(pkg, lib, dev, dtype):
    g = torch.Generator().manual_seed(3)
    T = 9
    xs = [torch.randn(T, 64, 192, generator=g).to(dtype), torch.randn(T, 64, generator=g).to(dtype),
          torch.randn(T, 32, 128, generator=g).to(dtype), torch.randn(T, 128, generator=g).to(dtype)]
    offs, inter = [128, 0, 0, 0], [True, True, False, False]
    pos = torch.randint(0, 184320, (T,), generator=g)
    tab = table(pkg, 64, 184320, dev)
    got = pkg.rope.apply_rotary([x.to(dev) for x in xs], pos.to(dev), tab, offsets=offs,
                                interleaved=inter)
    for x, o, i, y in zip(xs, offs, inter, got):
        close(y, rotated(x, pos, 64, o, i, 184320))


@pytest.mark.parametrize("inter", [True, False])
@pytest.mark.parametrize("D,offset", [(192, 128), (101, 13)])
def test_positions_outside_the_table_are_not_rotated(pkg, lib, dev, inter, D, offset):
    x = torch.randn(6, 3, D).half()
    x[1] = math.inf
    x[3, 0, :] = math.nan
    pos = torch.tensor([0, -1, 99, 100, 1 << 40, -(1 << 40)])
    tab = table(pkg, 64, 100, dev)
    want = rotated(x[[0, 2]], pos[[0, 2]], 64, offset, inter, 100)
    xd = x.to(dev)
    for out in (None, xd):
        got = pkg.rope.apply_rotary(xd, pos.to(dev), tab, offsets=offset, interleaved=inter, outs=out)
        close(got[[0, 2]], want)
        same = got[[1, 3, 4, 5]].cpu().view(torch.int16)
        assert torch.equal(same, x[[1, 3, 4, 5]].view(torch.int16))


def test_strided_views_and_what_surrounds_them(pkg, lib, dev):
    """Heads of a wider projection, a transposed [H, T, D] tensor, unaligned rows; what
    lies around an out view stays."""
    g = torch.Generator().manual_seed(5)
    wide = torch.randn(50, 8, 200, generator=g).half()
    pos = torch.arange(50)
    tab = table(pkg, 64, 64, dev)
    for lo in (0, 8, 3):
        x = wide[:, ::2, lo:lo + 96]
        buf = torch.full((50, 4, 120), 7.0, dtype=torch.float16, device=dev)
        out = buf[:, :, 8:104]
        pkg.rope.apply_rotary(wide.to(dev)[:, ::2, lo:lo + 96], pos.to(dev), tab, offsets=32, outs=out)
        close(out, rotated(x, pos, 64, 32, True, 64))
        assert bool((buf[:, :, :8] == 7).all()) and bool((buf[:, :, 104:] == 7).all())
        v = wide.to(dev).clone()
        pkg.rope.apply_rotary(v[:, ::2, lo:lo + 96], pos.to(dev), tab, offsets=32,
                              outs=v[:, ::2, lo:lo + 96])
        want = wide.clone()
        want[:, ::2, lo:lo + 96] = out.cpu()
        assert torch.equal(v.cpu(), want)
    ht = torch.randn(8, 50, 96, generator=g).half()
    got = pkg.rope.apply_rotary(ht.to(dev).transpose(0, 1), pos.to(dev), tab)
    close(got, rotated(ht.transpose(0, 1), pos, 64, 0, True, 64))
    one = torch.randn(1, 8, 96, generator=g).half()  # the same row for every token
    got = pkg.rope.apply_rotary(one.to(dev).expand(50, 8, 96), pos.to(dev), tab)
    close(got, rotated(one.expand(50, 8, 96), pos, 64, 0, True, 64))


def test_far_positions_and_yarn(pkg, lib, dev):
    """Angles of positions to 180k: the table is built in fp64.  YaRN from its formula."""
    rot, f, n = 64, 40.0, 4096
    x = torch.randn(8, 4, 64)
    pos = torch.tensor([0, 1, 4095, 4096, 65536, 131071, 184318, 184319])
    lo = math.floor(rot * math.log(n / (32 * 2 * math.pi)) / (2 * math.log(10000.0)))
    hi = math.ceil(rot * math.log(n / (1 * 2 * math.pi)) / (2 * math.log(10000.0)))
    fr = []
    for i in range(rot // 2):
        r = min(max((i - lo) / (hi - lo), 0.0), 1.0)
        w = 10000.0 ** (-2 * i / rot)
        fr.append(w / f * r + w * (1 - r))
    tab = table(pkg, rot, 184320, dev, scaling=dict(type="yarn", factor=f, original_max_positions=n))
    got = pkg.rope.apply_rotary(x.to(dev), pos.to(dev), tab)
    close(got, rotated(x, pos, rot, 0, True, 184320, torch.tensor(fr, dtype=torch.float64),
                       0.1 * math.log(f) + 1))


def test_other_stream_and_graph(pkg, lib, dev):
    x = torch.randn(40, 6, 192).half()
    pos = torch.arange(40)
    tab = table(pkg, 64, 64, dev)
    want = rotated(x, pos, 64, 128, True, 64)
    xd, pd = x.to(dev), pos.to(dev)
    torch.cuda.synchronize()
    st = torch.cuda.Stream()
    with torch.cuda.stream(st):
        y = pkg.rope.apply_rotary(xd, pd, tab, offsets=128)
    st.synchronize()
    close(y, want)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = pkg.rope.apply_rotary(xd, pd, tab, offsets=128)
    for k in range(3):
        pd.copy_(pos + k)
        g.replay()
        e = pkg.rope.apply_rotary(xd, pd, tab, offsets=128)
        torch.cuda.synchronize()
        assert torch.equal(e, y)
