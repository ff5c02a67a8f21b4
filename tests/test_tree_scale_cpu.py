"""Scales whose product with log2 e is not finite, and kinds of rows that there are not, are
refused by tree attention."""
import math

import pytest
from test_rope_tree_cpu import err, tree


@pytest.mark.parametrize("scale", [2.4e38, -3e38, math.inf, math.nan])
def test_refused(pkg, lib, scale):
    assert tree(lib, scale=scale) == 1 and "finite" in err(pkg)


@pytest.mark.parametrize("kind", [-1, 3])
def test_kind_of_rows(pkg, lib, kind):
    assert tree(lib, fp8=kind) == 1 and "kv_fp8" in err(pkg)
