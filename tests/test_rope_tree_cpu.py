"""Rotary table, tree masks, and the refusals of the rotary, cache read-back and tree
attention entry points, without a GPU: bad arguments come back as errors before any
launch, and CPU tensors are refused."""
import ctypes
import math

import pytest
import torch


def err(pkg):
    return pkg._lib.last_error()


# ---------------------------------------------------------------------------
# table and masks
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("rot", [2, 36, 64])
@pytest.mark.parametrize("scaling", [None, dict(type="linear", factor=4), dict(type="ntk", factor=8)])
def test_table(pkg, rot, scaling):
    if rot == 2 and scaling and scaling["type"] == "ntk":
        with pytest.raises(RuntimeError, match="rot_dim > 2"):
            pkg.rope.rotary_table(rot, 4, scaling=scaling, device="cpu")
        return
    t = pkg.rope.rotary_table(rot, 300, 5000.0, scaling, device="cpu")
    assert t.shape == (300, rot) and t.dtype == torch.float32
    base, div = 5000.0, 1.0
    if scaling and scaling["type"] == "linear":
        div = 4.0
    elif scaling:
        base = 5000.0 * 8 ** (rot / (rot - 2))
    for p in (0, 1, 7, 299):
        for i in (0, rot // 2 - 1):
            a = p / div * base ** (-2 * i / rot)
            # fp64 angle, one rounding to fp32
            assert abs(float(t[p, i]) - math.cos(a)) <= 2.0 ** -24
            assert abs(float(t[p, rot // 2 + i]) - math.sin(a)) <= 2.0 ** -24


def test_yarn_ends(pkg):
    """Fast dims keep their frequency, slow ones are divided by the factor; magnitudes."""
    f, n, rot = 40.0, 4096, 64
    kw = dict(type="yarn", factor=f, original_max_positions=n)
    t = pkg.rope.rotary_table(rot, 2, scaling=kw, device="cpu").double()
    m = 0.1 * math.log(f) + 1
    assert abs(float(t[1, 0]) - m * math.cos(1.0)) <= 2.0 ** -23
    slow = 10000.0 ** (-62 / 64) / f
    assert abs(float(t[1, 63]) - m * math.sin(slow)) <= 2.0 ** -24
    even = pkg.rope.rotary_table(rot, 2, scaling=dict(kw, mscale=1.0, mscale_all_dim=1.0), device="cpu")
    assert float(even[0, 0]) == 1.0


@pytest.mark.parametrize("kw", [dict(rot_dim=3, max_positions=4), dict(rot_dim=0, max_positions=4),
                                dict(rot_dim=4, max_positions=-1), dict(rot_dim=4, max_positions=4, base=0),
                                dict(rot_dim=4, max_positions=4, scaling=dict(type="other", factor=2)),
                                dict(rot_dim=4, max_positions=4, scaling=dict(type="linear", factor=0.5)),
                                dict(rot_dim=4, max_positions=4, scaling=dict(type="yarn", factor=2))])
def test_table_refusals(pkg, kw):
    with pytest.raises(RuntimeError, match="rotary_table"):
        pkg.rope.rotary_table(device="cpu", **kw)


def test_tree_masks(pkg):
    mask, depth = pkg.mla_tree.tree_masks([-1, 0, 0, 2, -1])
    assert mask == [0b1, 0b11, 0b101, 0b1101, 0b10000] and depth == [0, 1, 1, 2, 0]
    mask, depth = pkg.mla_tree.tree_masks(range(-1, 63))  # a chain of 64
    assert mask[62] == 2 ** 63 - 1 and mask[63] == -1 and depth[63] == 63
    assert pkg.mla_tree.tree_masks([]) == ([], [])
    for bad in ([0], [-1, 1], [-2], [-1] * 65):
        with pytest.raises(RuntimeError, match="tree_masks"):
            pkg.mla_tree.tree_masks(bad)


# ---------------------------------------------------------------------------
# C ABI refusals (addresses are never read: the checks come first)
# ---------------------------------------------------------------------------
def part(pkg, **kw):
    d = dict(out=4096, x=8192, out_tok_stride=192, out_head_stride=192, x_tok_stride=192,
             x_head_stride=192, n_head=1, dim=192, offset=128, dtype=0, interleaved=1)
    d.update(kw)
    return pkg._lib.RotaryPart(**d)


def rotary(pkg, lib, p, n=1, tok=4, rot=64, pos=4096, cs=4096, max_pos=10):
    return lib.mi355_dsa_rotary((pkg._lib.RotaryPart * 1)(p), n, pos, 1, tok, cs, max_pos, rot, None)


@pytest.mark.parametrize("kw,msg", [
    (dict(offset=129), "does not lie"), (dict(offset=-1), "does not lie"), (dict(dim=60), "does not lie"),
    (dict(dtype=3), "dtype"), (dict(n_head=0), "n_head"), (dict(out=None), "null"),
    (dict(x=None), "null"), (dict(x=8193), "misaligned"), (dict(dtype=2, out=4098), "misaligned"),
    (dict(out_tok_stride=100), "out strides"), (dict(n_head=2, out_head_stride=0), "out strides"),
    (dict(x_tok_stride=-192), "strides"), (dict(x=4096, x_tok_stride=200), "in place"),
    (dict(n_head=1 << 30), "too many heads")])
def test_rotary_refuses_parts(pkg, lib, kw, msg):
    if "n_head" in kw and kw["n_head"] > 2:
        kw = dict(kw, out_head_stride=192)
    assert rotary(pkg, lib, part(pkg, **kw)) == 1 and msg in err(pkg)


def test_rotary_refuses(pkg, lib):
    p = part(pkg)
    assert rotary(pkg, lib, p, n=5) == 1 and "0 to 4" in err(pkg)
    assert rotary(pkg, lib, p, rot=63) == 1 and "even" in err(pkg)
    assert rotary(pkg, lib, p, rot=0) == 1 and "even" in err(pkg)
    assert rotary(pkg, lib, p, pos=None) == 1 and "null" in err(pkg)
    assert rotary(pkg, lib, p, cs=None) == 1 and "null" in err(pkg)
    assert rotary(pkg, lib, p, pos=4100) == 1 and "misaligned" in err(pkg)
    assert rotary(pkg, lib, p, tok=-1) == 1 and "n_tok" in err(pkg)
    assert rotary(pkg, lib, p, tok=1 << 40) == 1 and "too many tokens" in err(pkg)
    assert rotary(pkg, lib, p, tok=0) == 0 and rotary(pkg, lib, p, n=0) == 0


def write(lib, **kw):
    d = dict(kv=4096, fp8=1, rows=64, kv_c=4096, cs=512, pe=4096, ps=64, bf16=0, tok=2, slot=4096,
             s64=1, pos=4096, p64=1, tab=4096, mp=10, inter=1, q=None)
    d.update(kw)
    return lib.mi355_dsa_rope_concat_and_cache_mla(*d.values(), None)


def test_write_refuses(pkg, lib):
    assert write(lib, kv=None) == 1 and "null" in err(pkg)
    assert write(lib, slot=None) == 1 and "null" in err(pkg)
    assert write(lib, tab=None) == 1 and "null" in err(pkg)
    assert write(lib, kv_c=4104) == 1 and "aligned" in err(pkg)
    assert write(lib, cs=500) == 1 and "row strides" in err(pkg)
    assert write(lib, ps=60) == 1 and "row strides" in err(pkg)
    assert write(lib, fp8=0, bf16=1) == 1 and "fp16 inputs" in err(pkg)
    q = part(pkg, dtype=1)
    assert write(lib, q=ctypes.byref(q)) == 1 and "type of kv_c" in err(pkg)
    q = part(pkg, offset=150)
    assert write(lib, q=ctypes.byref(q)) == 1 and "does not lie" in err(pkg)
    assert write(lib, tok=0, kv=None) == 0


def gather(lib, **kw):
    d = dict(out=4096, os=576, dt=0, total=5, kv=4096, fp8=1, pe=0, rows=64, page=16, bt=4096, mb=4,
             cu=4096, st=None, r=1)
    d.update(kw)
    return lib.mi355_dsa_gather_latent_cache(*d.values(), None)


def test_gather_refuses(pkg, lib):
    assert gather(lib, out=None) == 1 and "null" in err(pkg)
    assert gather(lib, bt=None) == 1 and "null" in err(pkg)
    assert gather(lib, os=575) == 1 and "576" in err(pkg)
    assert gather(lib, os=577) == 1 and "aligned" in err(pkg)
    assert gather(lib, out=4104) == 1 and "misaligned" in err(pkg)
    assert gather(lib, dt=3) == 1 and "dtype" in err(pkg)
    assert gather(lib, page=0) == 1 and "page size" in err(pkg)
    assert gather(lib, fp8=0, pe=1) == 1 and "fp16 values" in err(pkg)
    assert gather(lib, total=-1) == 1 and gather(lib, r=-1) == 1
    assert gather(lib, total=0, out=None) == 0 and gather(lib, r=0, out=None) == 0


def tree(lib, **kw):
    d = dict(o=4096, lse=4096, q=4096, tok=4, heads=16, kv=4096, fp8=0, rows=64, page=16, bt=4096,
             mb=4, seq=4096, cu=4096, r=1, mask=4096, scale=0.1, ws=4096, wsb=1 << 40)
    d.update(kw)
    return lib.mi355_dsa_mla_tree_attention(*d.values(), None)


def test_tree_refuses(pkg, lib):
    for name in ("o", "lse", "q", "kv", "bt", "seq", "cu", "mask"):
        assert tree(lib, **{name: None}) == 1 and "null" in err(pkg), name
    assert tree(lib, ws=None) == 1 and "workspace too small" in err(pkg)
    need = lib.mi355_dsa_mla_tree_workspace_size(4, 16)
    assert need > 0 and tree(lib, wsb=need - 1) == 1 and f"need {need} bytes" in err(pkg)
    assert tree(lib, ws=4104) == 1 and "16-byte" in err(pkg)
    for name in ("o", "q", "kv"):
        assert tree(lib, **{name: 4104}) == 1 and "misaligned" in err(pkg)
    assert tree(lib, scale=math.nan) == 1 and "finite" in err(pkg)
    assert tree(lib, scale=math.inf) == 1 and "finite" in err(pkg)
    assert tree(lib, heads=0) == 1 and tree(lib, tok=-1) == 1 and tree(lib, page=0) == 1
    assert tree(lib, mb=1 << 26) == 1 and "too wide" in err(pkg)
    assert tree(lib, rows=1 << 31) == 1 and "too many rows" in err(pkg)
    assert tree(lib, tok=1 << 27, wsb=1 << 60) == 1 and "too many rows" in err(pkg)
    assert tree(lib, tok=0, q=None) == 0 and tree(lib, r=0, q=None) == 0


def test_tree_workspace_size(lib):
    assert lib.mi355_dsa_mla_tree_workspace_size(0, 16) == 0
    sizes = [lib.mi355_dsa_mla_tree_workspace_size(t, h) for t, h in ((1, 1), (4, 16), (8, 64), (640, 64))]
    assert sizes == sorted(sizes) and sizes[0] > 0 and sizes[2] == sizes[3] <= 160 << 20


# ---------------------------------------------------------------------------
# torch layer
# ---------------------------------------------------------------------------
def test_cpu_tensors_are_refused(pkg, lib):
    t = pkg.rope.rotary_table(64, 8, device="cpu")
    with pytest.raises(RuntimeError, match="on the GPU"):
        pkg.rope.apply_rotary(torch.zeros(2, 3, 64), torch.arange(2), t)
    kv = torch.zeros(2, 16, 656, dtype=torch.uint8)
    bt, cu = torch.zeros(1, 2, dtype=torch.int32), torch.tensor([0, 3], dtype=torch.int32)
    with pytest.raises(RuntimeError, match="GPU"):
        pkg._cache_ops.gather_latent_cache(kv, bt, cu, 3)
    with pytest.raises(RuntimeError, match="GPU"):
        pkg._cache_ops.rope_concat_and_cache_mla(torch.arange(2), t, torch.zeros(2, 512).half(),
                                                 torch.zeros(2, 64).half(), kv, torch.arange(2),
                                                 "fp8_ds_mla")
    with pytest.raises(RuntimeError, match="GPU"):
        pkg.mla_tree.tree_attention(torch.zeros(3, 2, 576).half(), kv, bt,
                                    torch.tensor([3], dtype=torch.int32), cu,
                                    torch.zeros(3, dtype=torch.int64), 0.1)
