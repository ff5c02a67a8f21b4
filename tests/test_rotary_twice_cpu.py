"""A rotary call that would write the same elements from two of its tensors, which no
order of the launch's workgroups makes right, is refused."""
import pytest
from test_rope_tree_cpu import err, part


def call(pkg, lib, *parts):
    return lib.mi355_dsa_rotary((pkg._lib.RotaryPart * len(parts))(*parts), len(parts), 4096, 1, 4,
                                4096, 10, 64, None)


@pytest.mark.parametrize("a,b", [
    (dict(x=4096), dict(x=4096)),                          # in place, twice
    (dict(x=4096, offset=64), dict(x=4096, offset=100)),   # parts that overlap
    (dict(x=4096, offset=0), dict(x=8192, offset=128)),    # in place, and from elsewhere
    (dict(), dict(x=16384))])                              # two tensors into one
@pytest.mark.parametrize("between", [0, 1])
def test_refused(pkg, lib, a, b, between):
    mid = [part(pkg, out=1 << 20, x=1 << 21)] * between
    assert call(pkg, lib, part(pkg, **a), *mid, part(pkg, **b)) == 1
    assert "same place" in err(pkg)
