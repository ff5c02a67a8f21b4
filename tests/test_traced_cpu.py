"""The rotary, latent cache and tree attention entry points under tracing, without a GPU:
they are ops with a fake form, their outputs have the right shapes and types, and tensors
that require grad are refused instead of losing it."""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.fx.experimental.proxy_tensor import make_fx

H16, I32 = torch.float16, torch.int32


def tensors(dev, T=3, H=4, R=2):
    def e(*shape, dtype=H16):
        return torch.empty(*shape, dtype=dtype, device=dev)

    return dict(q=e(T, H, 192), kv_c=e(T, 512), k_pe=e(T, 64), lat=e(T, H, 576),
                cache=e(8, 16, 656, dtype=torch.uint8), table=e(32, 64, dtype=torch.float32),
                pos=e(T, dtype=torch.int64), slot=e(T, dtype=torch.int64), bt=e(R, 4, dtype=I32),
                seq=e(R, dtype=I32), cu=e(R + 1, dtype=I32), mask=e(T, dtype=torch.int64))


def step(pkg, t):
    """A decode step's calls, one after the other."""
    q, pe = pkg.rope.apply_rotary([t["q"], t["k_pe"]], t["pos"], t["table"], [128, 0])
    y = pkg.rope.apply_rotary(t["q"], t["pos"], t["table"], 128, outs=t["q"])
    w = pkg._cache_ops.rope_concat_and_cache_mla(t["pos"], t["table"], t["kv_c"], t["k_pe"], t["cache"],
                                                 t["slot"], "fp8_ds_mla", q=t["q"], q_offset=128)
    kv = pkg._cache_ops.gather_latent_cache(t["cache"], t["bt"], t["cu"], 7, dtype=torch.bfloat16)
    o, lse = pkg.mla_tree.tree_attention(t["lat"], t["cache"], t["bt"], t["seq"], t["cu"], t["mask"], 0.1)
    return q, pe, y, w, kv, o, lse


def test_fake_tensors(pkg, lib):
    with FakeTensorMode():
        t = tensors("cuda")
        q, pe, y, w, kv, o, lse = step(pkg, t)
    assert y is t["q"] and q.shape == w.shape == (3, 4, 192) and pe.shape == (3, 64)
    assert kv.shape == (7, 576) and kv.dtype == torch.bfloat16 and o.shape == (3, 4, 512)
    assert o.dtype == H16 and lse.shape == (3, 4) and lse.dtype == torch.float32


def test_recorded_as_ops(pkg, lib):
    with FakeTensorMode():
        t = tensors("cuda")
    names = list(t)
    g = make_fx(lambda *a: step(pkg, dict(zip(names, a))), tracing_mode="fake")(*t.values())
    ns = pkg.ops.NAMESPACE
    calls = [str(n.target) for n in g.graph.nodes if n.op == "call_function" and ns in str(n.target)]
    assert calls == [f"{ns}.{x}.default" for x in (
        "apply_rotary", "apply_rotary", "rope_concat_and_cache_mla", "gather_latent_cache",
        "mla_tree_attention")]


@pytest.mark.parametrize("which", ["q", "k_pe", "kv_c", "lat"])
def test_tensors_that_require_grad(pkg, lib, which):
    """Refused in grad mode (before the refusal of CPU tensors), not without it."""
    t = {k: torch.zeros_like(v) if v.dtype != torch.uint8 else v for k, v in tensors("cpu").items()}
    t[which].requires_grad_()

    def call():
        if which == "lat":
            pkg.mla_tree.tree_attention(t["lat"], t["cache"], t["bt"], t["seq"], t["cu"], t["mask"], 0.1)
        elif which == "kv_c":
            pkg._cache_ops.rope_concat_and_cache_mla(t["pos"], t["table"], t["kv_c"], t["k_pe"],
                                                     t["cache"], t["slot"], "fp8_ds_mla")
        else:
            pkg.rope.apply_rotary([t["k_pe"], t["q"]], t["pos"], t["table"])

    with pytest.raises(RuntimeError, match="no backward pass"):
        call()
    with torch.no_grad(), pytest.raises(RuntimeError, match="GPU"):
        call()
