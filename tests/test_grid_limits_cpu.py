"""Calls whose grids have 2^32 threads or more, which no launch takes, are refused before
any launch: rotation, the cache written and read back, tree attention (whose second
launch is the one that would fail, after the first has written o).  Without a GPU."""
import ctypes

import pytest
from test_rope_tree_cpu import err, gather, part, rotary, tree, write

BLOCKS = 1 << 24  # of 256 threads: one more than a grid may have


# a workgroup takes 10 tokens of 24 pieces; a token of 64 x 24 pieces takes 2 workgroups
@pytest.mark.parametrize("heads,tok", [(1, 10 * BLOCKS), (1, 1 << 40), (64, BLOCKS // 2), (64, 1 << 36)])
def test_rotary(pkg, lib, heads, tok):
    p = part(pkg, n_head=heads, x_tok_stride=192 * heads, out_tok_stride=192 * heads)
    assert rotary(pkg, lib, p, tok=tok) == 1 and "rotary: too many tokens" in err(pkg)


def test_rotary_of_several_tensors(pkg, lib):
    p = (pkg._lib.RotaryPart * 4)(*[part(pkg, out=16384 * (i + 1)) for i in range(4)])
    assert lib.mi355_dsa_rotary(p, 4, 4096, 1, 10 * BLOCKS // 4, 4096, 10, 64, None) == 1
    assert "rotary: too many tokens" in err(pkg)


@pytest.mark.parametrize("q,tok", [(False, 4 * BLOCKS), (False, 1 << 40), (True, 3 * BLOCKS)])
def test_write(pkg, lib, q, tok):
    assert write(lib, tok=tok, q=ctypes.byref(part(pkg)) if q else None) == 1
    assert "too many tokens" in err(pkg)


@pytest.mark.parametrize("total", [8 * BLOCKS, 1 << 40])
def test_gather(pkg, lib, total):
    assert gather(lib, total=total) == 1 and "too many rows" in err(pkg)


@pytest.mark.parametrize("tok,heads,req", [(1 << 20, 1, 1 << 20), (1 << 27, 1, 1), (1 << 22, 32, 7)])
def test_tree(pkg, lib, tok, heads, req):
    assert tree(lib, tok=tok, heads=heads, r=req, wsb=1 << 62) == 1 and "too many rows" in err(pkg)
