"""Calls too large for a grid, of tree attention, rotation and the cache, are refused before any launch, without a GPU."""
import pytest
from test_rope_tree_cpu import err, gather, part, rotary, tree, write


@pytest.mark.parametrize("kw", [dict(tok=1 << 29, heads=1, r=1 << 29),   # a merge unit a request
                                dict(tok=1 << 62, heads=4), dict(tok=(1 << 60) + 1, heads=16),
                                dict(tok=1 << 20, heads=1 << 10)])
def test_too_many_rows(pkg, lib, kw):
    assert tree(lib, wsb=1 << 62, **kw) == 1 and "too many rows" in err(pkg)


@pytest.mark.parametrize("n", [1 << 41, 1 << 62, (1 << 63) - 1])
def test_too_many_tokens(pkg, lib, n):
    assert rotary(pkg, lib, part(pkg), tok=n) == 1 and "too many tokens" in err(pkg)
    assert write(lib, tok=n) == 1 and "too many tokens" in err(pkg)
    assert gather(lib, total=n) == 1 and "too many rows" in err(pkg)
