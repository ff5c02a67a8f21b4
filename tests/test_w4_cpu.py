"""Refusals of the 4-bit projections without a GPU, and their calls under tracing."""
from dataclasses import replace

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.fx.experimental.proxy_tensor import make_fx

F16 = torch.float16


def err(pkg):
    return pkg._lib.last_error()


def linear(lib, **kw):
    d = dict(y=64, x=64, stride=256, q=64, sz=64, dtype=0, M=2, N=16, K=256, group=128, ws=None, n=0)
    d.update(kw)
    return lib.mi355_dsa_w4_linear(*d.values(), None)


@pytest.mark.parametrize("kw,msg", [
    (dict(M=65), "M must be 0..64, got 65"), (dict(M=-1), "M must be"), (dict(N=-1), "bad sizes"),
    (dict(K=-8), "bad sizes"), (dict(K=252), "multiple of 8"), (dict(group=16), "group must be"),
    (dict(group=256), "group must be"), (dict(dtype=2), "dtype must be"), (dict(stride=252), "stride"),
    (dict(stride=248), "stride"), (dict(x=66), "misaligned"), (dict(q=72), "misaligned"),
    (dict(sz=66), "misaligned"), (dict(N=(1 << 31) - 1, M=1), "too many rows"),
    (dict(K=1 << 24, stride=1 << 24), "too many columns"), (dict(stride=1 << 29), "row stride"),
    (dict(M=64, N=6144, K=24576, stride=24576), "workspace too small"),
    (dict(M=64, N=6144, K=24576, stride=24576, ws=72, n=1 << 40), "16-byte aligned"),
    *[({k: None}, "null pointer") for k in ("y", "x", "q", "sz")]])
def test_linear(pkg, lib, kw, msg):
    assert linear(lib, **kw) == 1 and msg in err(pkg)
    assert linear(lib, M=0, y=None) == 0 and linear(lib, N=0, q=None) == 0


def test_workspace_sizes(lib):
    size = lib.mi355_dsa_w4_linear_workspace_size
    assert size(0, 16, 128) == size(1, 0, 128) == size(1, 16, 0) == size(65, 16, 128) == 0
    assert size(64, 24576, 6144) == 0          # enough workgroups without slices
    n = size(64, 6144, 24576)                  # slices of whole fp32 tiles
    assert n and n % (64 * 6144 * 4) == 0


def quant(lib, **kw):
    d = dict(q=64, sz=64, w=64, dtype=0, N=16, K=256, group=64, symmetric=0)
    d.update(kw)
    return lib.mi355_dsa_w4_quantize(*d.values(), None)


def pack(lib, **kw):
    d = dict(q=64, sz=64, codes=64, s=64, z=64, dtype=1, N=16, K=256, group=64)
    d.update(kw)
    return lib.mi355_dsa_w4_pack(*d.values(), None)


def dequant(lib, **kw):
    d = dict(out=64, q=64, sz=64, dtype=0, N=16, K=256, group=64)
    d.update(kw)
    return lib.mi355_dsa_w4_dequant(*d.values(), None)


@pytest.mark.parametrize("call,ptrs,big", [(quant, ("q", "sz", "w"), "w"), (pack, ("q", "sz", "codes", "s"), "codes"),
                                           (dequant, ("out", "q", "sz"), "out")])
def test_weights(pkg, lib, call, ptrs, big):
    for kw, msg in [(dict(N=-1), "bad sizes"), (dict(K=100), "multiple of 8"), (dict(group=48), "group must"),
                    (dict(dtype=-1), "dtype must"), ({big: 68}, "misaligned"),
                    (dict(N=(1 << 31) - 1, K=1 << 20), "too many weights"),
                    *[({k: None}, "null pointer") for k in ptrs]]:
        assert call(lib, **kw) == 1 and msg in err(pkg), kw
    assert call(lib, N=0, q=None) == 0 and call(lib, K=0, q=None) == 0


def test_python_refusals(pkg, lib):
    W = pkg.w4
    with pytest.raises(RuntimeError, match="GPU"):
        W.w4_quantize(torch.zeros(4, 64, dtype=F16))
    for call, msg in [
            (lambda: W.w4_quantize(torch.zeros(4, 64)), "fp16 or bf16"),
            (lambda: W.w4_quantize(torch.zeros(4, 60, dtype=F16)), "multiple of 8"),
            (lambda: W.w4_quantize(torch.zeros(64, dtype=F16)), "2-D"),
            (lambda: W.w4_quantize(torch.zeros(4, 64, dtype=F16), 100), "group"),
            (lambda: W.w4_quantize(torch.zeros(4, 64, dtype=F16, requires_grad=True)), "no backward"),
            (lambda: W.w4_pack(torch.zeros(4, 64), torch.zeros(4, 1, dtype=F16)), "uint8"),
            (lambda: W.w4_pack(torch.zeros(4, 64, dtype=torch.uint8), torch.zeros(4, 2, dtype=F16)), "scales"),
            (lambda: W.w4_pack(torch.zeros(4, 64, dtype=torch.uint8), torch.zeros(4, 1, dtype=F16),
                               torch.zeros(4, 1)), "zeros")]:
        with pytest.raises(RuntimeError, match=msg):
            call()
    w = W._empty(20, 64, 32, F16, "cpu")
    assert w.q.shape == (2, 1, 64, 4) and w.sz.shape == (2, 4, 16)
    for x, msg in [(torch.zeros(2, 72, dtype=F16), r"\[M, K\]"), (torch.zeros(2, 64), "type"),
                   (torch.zeros(65, 64, dtype=F16), "at most 64"), (torch.zeros(2, 64, dtype=F16), "GPU"),
                   (torch.zeros(2, 64, dtype=F16, requires_grad=True), "no backward")]:
        with pytest.raises(RuntimeError, match=msg):
            W.w4_linear(x, w)
    with pytest.raises(RuntimeError, match="out must"):
        W.w4_linear(torch.zeros(2, 64, dtype=F16), w, torch.zeros(2, 21, dtype=F16))
    for kw in (dict(group=64), dict(n=33), dict(k=136), dict(q=w.q.float()), dict(sz=w.sz[:, ::2])):
        with pytest.raises(RuntimeError, match="not of weights"):
            replace(w, **kw)


def test_traced(pkg, lib):
    def step(weight, codes, s, x):
        W = pkg.w4
        a, b = W.w4_quantize(weight, 64), W.w4_pack(codes, s)
        return W.w4_linear(x, a), W.w4_linear(x, b), W.w4_dequant(a)

    with FakeTensorMode():
        args = (torch.empty(20, 128, dtype=F16, device="cuda"),
                torch.empty(9, 128, dtype=torch.uint8, device="cuda"),
                torch.empty(9, 1, dtype=F16, device="cuda"), torch.empty(3, 128, dtype=F16, device="cuda"))
        y, y2, v = step(*args)
    assert y.shape == (3, 20) and y2.shape == (3, 9) and v.shape == (20, 128) and v.dtype == F16
    g = make_fx(step, tracing_mode="fake")(*args)
    ns = pkg.ops.NAMESPACE
    calls = [str(n.target) for n in g.graph.nodes if n.op == "call_function" and ns in str(n.target)]
    assert calls == [f"{ns}.{x}.default" for x in ("w4_quantize", "w4_pack", "w4_linear", "w4_linear",
                                                  "w4_dequant")]


def test_ops_check_what_they_are_given(pkg, lib):
    """A call of the registered op itself, with tensors that no function of w4 has made."""
    op, w = pkg.ops.IMPLS, pkg.w4._empty(20, 64, 32, F16, "cpu")
    e = lambda *s, dtype=F16: torch.zeros(*s, dtype=dtype)
    codes, scales = e(20, 64, dtype=torch.uint8), e(20, 2)
    for name, args, msg in [
            ("w4_linear", (e(2, 20), e(2, 136), w.q, w.sz, 32), "not of weights"),
            ("w4_linear", (e(2, 40), e(2, 64), w.q, w.sz, 32), "not of weights"),
            ("w4_linear", (e(3, 20), e(2, 64), w.q, w.sz, 32), "out must"),
            ("w4_linear", (e(2, 20).float(), e(2, 64).float(), w.q, w.sz, 32), "fp16 or bf16"),
            ("w4_linear", (e(2, 20), e(2, 64), w.q, w.sz, 0), "group"),
            ("w4_quantize", (w.q, w.sz, e(20, 136), 32, False), "not of weights"),
            ("w4_quantize", (w.q, w.sz[:1], e(20, 64), 32, False), "not of weights"),
            ("w4_quantize", (w.q, w.sz, e(40, 64), 32, False), "not of weights"),
            ("w4_pack", (w.q, w.sz, codes, e(20, 1), None, 32), "scales"),
            ("w4_pack", (w.q, w.sz, codes, scales, e(20, 2), 32), "zeros"),
            ("w4_pack", (w.q, w.sz, codes[:16], scales[:16], None, 32), "not of weights"),
            ("w4_dequant", (e(20, 136), w.q, w.sz, 32), "not of weights"),
            ("w4_dequant", (e(64, 20).t(), w.q, w.sz, 32), "contiguous"),
            ("w4_dequant", (e(20, 64), w.q, w.sz, 32), "GPU")]:
        with pytest.raises(RuntimeError, match=msg):
            op[name](*args)
