"""Scales whose product with log2 e is not finite are refused by tree attention."""
import math

import pytest
from test_rope_tree_cpu import err, tree


@pytest.mark.parametrize("scale", [2.4e38, -3e38, math.inf, math.nan])
def test_refused(pkg, lib, scale):
    assert tree(lib, scale=scale) == 1 and "finite" in err(pkg)
