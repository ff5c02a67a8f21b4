"""Refusals of attention over a shared prefix without a GPU, and its call under tracing."""
import math

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.fx.experimental.proxy_tensor import make_fx

F16, I32, I64 = torch.float16, torch.int32, torch.int64


def err(pkg):
    return pkg._lib.last_error()


def call(lib, **kw):
    d = dict(o=4096, lse=4096, q=4096, T=4, H=16, kv=4096, fp8=0, rows=640, page=64, bt=4096, W=4,
             seq=4096, cu=4096, R=3, mask=4096, cs=4096, shared=4096, S=2, scale=0.1, ws=4096,
             n=1 << 62)
    d.update(kw)
    return lib.mi355_dsa_mla_prefix_attention(*d.values(), None)


@pytest.mark.parametrize("kw,msg", [
    (dict(T=-1), "bad sizes"), (dict(R=-1), "bad sizes"), (dict(S=-1), "bad sizes"), (dict(H=0), "bad sizes"),
    (dict(W=-1), "bad sizes"), (dict(rows=-1), "bad sizes"), (dict(fp8=3), "kv_fp8"), (dict(page=0), "page size"),
    (dict(rows=1 << 31), "too many rows"), (dict(W=1 << 17), "too wide"), (dict(page=1 << 21), "too wide"),
    (dict(scale=math.inf), "scale must be finite"), (dict(scale=3e38), "scale must be finite"),
    (dict(cu=None), "go together"), (dict(mask=None), "go together"),
    (dict(cu=None, mask=None), "one token a request"),
    (dict(T=1 << 30), "too many rows"), (dict(T=1 << 26), "too many rows"),
    (dict(T=1 << 22, H=128, S=7), "too many rows"), (dict(T=1 << 27, H=1, S=1 << 27), "too many rows"),
    *[({k: None}, "null pointer") for k in ("o", "lse", "q", "kv", "bt", "seq", "cs", "shared")],
    (dict(q=4104), "misaligned"), (dict(kv=4104), "misaligned"), (dict(o=4104), "misaligned"),
    (dict(ws=None), "workspace too small"), (dict(n=100), "workspace too small"),
    (dict(ws=4104), "16-byte aligned")])
def test_c_refusals(pkg, lib, kw, msg):
    assert call(lib, **kw) == 1 and msg in err(pkg)


def test_nothing_to_do(lib):
    for kw in (dict(T=0), dict(R=0), dict(S=0)):
        assert call(lib, o=None, ws=None, n=0, **kw) == 0
    size = lib.mi355_dsa_mla_prefix_workspace_size
    assert size(0, 16, 3, 1) == size(4, 0, 3, 1) == size(4, 16, 0, 1) == size(4, 16, 3, 0) == 0
    assert size(1, 1, 1, 1) < size(1, 33, 1, 1) < size(1, 128, 1, 1) < size(10, 128, 10, 10)


def tensors(dev, T=4, R=4, fp8=False):
    def e(*shape, dtype=I32):
        return torch.zeros(*shape, dtype=dtype, device=dev)

    return dict(q=e(T, 16, 576, dtype=F16), kv_cache=e(8, 16, 656, dtype=torch.uint8) if fp8
                else e(8, 16, 576, dtype=F16), block_table=e(R, 3), seq_lens=e(R), cu_shared=e(3),
                shared_lens=e(2), scale=0.1)


@pytest.mark.parametrize("kw,msg", [
    ({}, "GPU"), (dict(q=torch.zeros(4, 16 * 576, dtype=F16)), "tokens, heads"),
    (dict(q=torch.zeros(4, 16, 576, dtype=F16, requires_grad=True)), "no backward")])
def test_cpu_tensors(pkg, lib, kw, msg):
    with pytest.raises(RuntimeError, match=msg):
        pkg.mla_prefix.shared_prefix_attention(**{**tensors("cpu"), **kw})


def test_shared_groups(pkg):
    f, i = pkg.mla_prefix._check_shared, torch.zeros(3, dtype=I32)
    f(i, i[:2], i.device)
    for cs, sh, msg in [(i[:0], i[:0], "cu_shared"), (i.long(), i[:2], "cu_shared"), (i.view(1, 3), i[:2], "cu_shared"),
                        (i, i, "shared_lens"), (i, i[:2].long(), "shared_lens")]:
        with pytest.raises(RuntimeError, match=msg):
            f(cs, sh, i.device)


def test_verify_tree_refuses_half_of_it(pkg):
    from test_verify_tree_cpu import args

    m = pkg.dsa_layer
    w = m.DsaLayerWeights(torch.zeros(3, 128, 512).half(), torch.zeros(3, 512, 128).half(), 0.1)
    L = m.DsaLayer(w, torch.zeros(2, 16, 576).half(), torch.zeros(2, 16, 128).half())
    for kw, msg in [(dict(cu_shared=torch.zeros(2, dtype=I32)), "go together"),
                    (dict(shared_lens=torch.zeros(1, dtype=I32)), "go together"),
                    (dict(cu_shared=torch.zeros(2, dtype=I32), shared_lens=torch.zeros(2, dtype=I32)),
                     "shared_lens")]:
        with pytest.raises(RuntimeError, match=msg):
            L.verify_tree(**args(pkg), **kw)


def test_traced(pkg, lib):
    def step(q, kv, bt, seq, cs, sh, cu, mask):
        f = pkg.mla_prefix.shared_prefix_attention
        return *f(q, kv, bt, seq, cs, sh, 0.1), *f(q, kv, bt, seq, cs, sh, 0.1, cu, mask)

    with FakeTensorMode():
        t = list(tensors("cuda").values())[:-1]
        t += [torch.zeros(5, dtype=I32, device="cuda"), torch.zeros(4, dtype=I64, device="cuda")]
        o, lse, o2, lse2 = step(*t)
    assert o.shape == o2.shape == (4, 16, 512) and o.dtype == F16
    assert lse.shape == lse2.shape == (4, 16) and lse.dtype == torch.float32
    g = make_fx(step, tracing_mode="fake")(*t)
    ns = pkg.ops.NAMESPACE
    calls = [str(n.target) for n in g.graph.nodes if n.op == "call_function" and ns in str(n.target)]
    assert calls == [f"{ns}.mla_prefix_attention.default"] * 2
