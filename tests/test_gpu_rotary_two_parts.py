"""Two parts of one tensor's heads rotated in place by one call, as by two."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("offs", [(0, 64), (128, 3), (64, 0)])
def test_in_place(pkg, lib, dev, dtype, offs):
    x = torch.randn(37, 5, 192, device=dev).to(dtype)
    pos = torch.arange(37, device=dev)
    tab = pkg.rope.rotary_table(64, 64, device=dev)
    want = x.clone()
    for o, inter in zip(offs, (True, False)):
        pkg.rope.apply_rotary(want, pos, tab, o, inter, want)
    pkg.rope.apply_rotary([x, x], pos, tab, list(offs), [True, False], [x, x])
    assert torch.equal(x, want)
    with pytest.raises(RuntimeError, match="same place"):
        pkg.rope.apply_rotary([x, x], pos, tab, [0, 0], True, [x, x])
    assert torch.equal(x, want)
