"""Refusals of the paging entry points without a GPU, and their calls under tracing."""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.fx.experimental.proxy_tensor import make_fx

I32 = torch.int32


def err(pkg):
    return pkg._lib.last_error()


def ext(lib, **kw):
    d = dict(bt=64, seq=64, new=64, R=3, W=4, free=64, count=64, P=9, page=16, slots=64, pos=64, T=9,
             cu=64, granted=64)
    d.update(kw)
    return lib.mi355_dsa_extend_tables(*d.values(), None)


@pytest.mark.parametrize("kw,msg", [
    (dict(R=-1), "bad sizes"), (dict(W=-1), "bad sizes"), (dict(P=-1), "bad sizes"),
    (dict(T=-1), "bad sizes"), (dict(page=0), "page size"), (dict(T=1 << 31), "too many tokens"),
    *[({k: None}, "null pointer") for k in ("bt", "seq", "new", "free", "count", "slots", "pos", "cu",
                                            "granted")]])
def test_extend(pkg, lib, kw, msg):
    assert ext(lib, **kw) == 1 and msg in err(pkg)


def cut(lib, **kw):
    d = dict(bt=64, seq=64, new=64, R=3, W=4, free=64, count=64, P=9, page=16, ws=64, n=16)
    d.update(kw)
    return lib.mi355_dsa_truncate_tables(*d.values(), None)


@pytest.mark.parametrize("kw,msg", [
    (dict(R=-1), "bad sizes"), (dict(W=-1), "bad sizes"), (dict(P=-1), "bad sizes"),
    (dict(page=-2), "page size"), (dict(n=15), "workspace too small"), (dict(ws=None), "workspace"),
    (dict(ws=66), "4-byte aligned"),
    *[({k: None}, "null pointer") for k in ("bt", "seq", "new", "free", "count")]])
def test_truncate(pkg, lib, kw, msg):
    assert cut(lib, **kw) == 1 and msg in err(pkg)
    assert cut(lib, R=0, bt=None, ws=None, n=0) == 0


def rows(lib, **kw):
    d = dict(out=64, lens=64, T=5, cols=4, bt=64, stride=4, seq=64, cu=64, R=2)
    d.update(kw)
    return lib.mi355_dsa_token_tables(*d.values(), None)


@pytest.mark.parametrize("kw,msg", [
    (dict(T=-1), "bad sizes"), (dict(cols=-1), "bad sizes"), (dict(R=-1), "bad sizes"),
    (dict(stride=3), "bad sizes"), (dict(T=1 << 31), "too many tokens"),
    (dict(cols=1 << 27, stride=1 << 27), "too many entries"),
    *[({k: None}, "null pointer") for k in ("out", "lens", "bt", "seq", "cu")]])
def test_token_tables(pkg, lib, kw, msg):
    assert rows(lib, **kw) == 1 and msg in err(pkg)
    assert rows(lib, T=0, out=None) == 0


def shared(lib, **kw):
    d = dict(out=64, cu=64, G=2, bt=64, seq=64, R=3, W=4, page=16, ws=64, n=12)
    d.update(kw)
    return lib.mi355_dsa_shared_lengths(*d.values(), None)


@pytest.mark.parametrize("kw,msg", [
    (dict(G=-1), "bad sizes"), (dict(R=-1), "bad sizes"), (dict(W=-1), "bad sizes"),
    (dict(page=0), "page size"), (dict(n=11), "workspace too small"), (dict(ws=62), "aligned"),
    (dict(R=1 << 24, n=1 << 30), "too many requests"), (dict(W=1 << 27), "too wide"),
    *[({k: None}, "null pointer") for k in ("out", "cu", "bt", "seq")]])
def test_shared_lengths(pkg, lib, kw, msg):
    assert shared(lib, **kw) == 1 and msg in err(pkg)
    assert shared(lib, G=0, out=None, cu=None) == 0


def tensors(dev):
    def e(*shape, dtype=I32):
        return torch.zeros(*shape, dtype=dtype, device=dev)

    return dict(bt=e(3, 4), seq=e(3), new=e(3), free=e(9), count=e(1), cu=e(4), cs=e(3))


def test_cpu_tensors_are_refused(pkg, lib):
    t = tensors("cpu")
    P = pkg.paging
    for call in (lambda: P.extend_tables(t["bt"], t["seq"], t["new"], t["free"], t["count"], 16, 5),
                 lambda: P.truncate_tables(t["bt"], t["seq"], t["new"], t["free"], t["count"], 16),
                 lambda: P.token_tables(t["bt"], t["seq"], t["cu"], 5),
                 lambda: P.shared_lengths(t["bt"], t["seq"], t["cs"], 16)):
        with pytest.raises(RuntimeError, match="GPU"):
            call()


def test_traced(pkg, lib):
    def step(bt, seq, new, free, count, cu, cs):
        P = pkg.paging
        out = P.extend_tables(bt, seq, new, free, count, 16, 5)
        rows = P.token_tables(bt, seq, cu, 5, 2)
        sh = P.shared_lengths(bt, seq, cs, 16)
        P.truncate_tables(bt, seq, new, free, count, 16)
        return *out, *rows, sh

    with FakeTensorMode():
        t = tensors("cuda")
        slots, pos, cu, granted, rows, lens, sh = step(*t.values())
    assert slots.shape == pos.shape == lens.shape == (5,) and cu.shape == (4,)
    assert granted.shape == (3,) and granted.dtype == torch.bool
    assert rows.shape == (5, 2) and sh.shape == (2,) and sh.dtype == I32
    g = make_fx(step, tracing_mode="fake")(*t.values())
    ns = pkg.ops.NAMESPACE
    calls = [str(n.target) for n in g.graph.nodes if n.op == "call_function" and ns in str(n.target)]
    assert calls == [f"{ns}.{x}.default" for x in ("extend_tables", "token_tables", "shared_lengths",
                                                  "truncate_tables")]


def test_ops_check_what_they_are_given(pkg, lib):
    """A call of the registered op itself, with outputs that no function of paging has made."""
    t, op = tensors("cpu"), pkg.ops.IMPLS
    e = lambda *s, dtype=I32: torch.zeros(*s, dtype=dtype)
    ins = (t["bt"], t["seq"], t["new"], t["free"], t["count"], 16)
    outs = [e(5), e(5), e(4), e(3, dtype=torch.bool)]
    names = ("slot_mapping", "positions", "cu_seqlens_q", "granted")
    for i, bad in enumerate((e(5, dtype=torch.int64), e(4), e(3), e(3))):
        with pytest.raises(RuntimeError, match=names[i]):
            op["extend_tables"](*outs[:i], bad, *outs[i + 1:], *ins)
    for out, lens in ((e(5, 5), e(5)), (e(5, 2), e(4)), (e(2, 5).t(), e(5)), (e(5), e(5)),
                      (e(5, 2), e(5, dtype=torch.int64))):
        with pytest.raises(RuntimeError, match="must be"):
            op["token_tables"](out, lens, t["bt"], t["seq"], t["cu"])
    for out in (e(3), e(2, dtype=torch.int64), e(4)[::2]):
        with pytest.raises(RuntimeError, match="out must"):
            op["shared_lengths"](out, t["bt"], t["seq"], t["cs"], 16)
    with pytest.raises(RuntimeError, match="GPU"):
        op["extend_tables"](*outs, *ins)
