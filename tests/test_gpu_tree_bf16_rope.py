"""Tree attention over fp8_ds_mla rows whose rope values were written as bf16 (pe_dtype):
against the definition with those values, and bit for bit the result over rows that hold
the same values as fp16.  Bounds as in test_gpu_mla_tree."""
import math

import pytest
import torch
from test_gpu_mla_tree import SCALE, cache, call, check, make, oracle

pytestmark = pytest.mark.gpu

BF = torch.bfloat16


def both(lens, counts, H, page, seed):
    """A case whose rope values are bf16 numbers, and the same with rows that hold them as
    bf16."""
    c = make(lens, counts, H, page, "fp8", seed=seed)
    pe = c["rows"][:, 528:].contiguous().view(torch.float16).to(BF)
    c["rows"][:, 528:] = pe.half().view(torch.uint8)
    b = dict(c, rows=c["rows"].clone())
    b["rows"][:, 528:] = pe.view(torch.uint8)
    return c, b


@pytest.mark.parametrize("lens,counts,H,page", [
    ([1], [1], 1, 64), ([31, 32, 33], [1, 2, 3], 8, 16), ([64, 65, 97], [5, 1, 33], 20, 48),
    ([130, 3, 0, 700], [7, 3, 1, 2], 64, 64), ([300, 200], [64, 17], 3, 1), ([2500], [9], 64, 128),
    ([(53 * i) % 310 + 9 for i in range(300)], [1 + (7 * i) % 9 for i in range(300)], 16, 16)])
def test_matches_definition(pkg, lib, dev, lens, counts, H, page):
    c, b = both(lens, counts, H, page, sum(lens) + H)
    got = call(pkg, b, dev, pe_dtype=BF)
    check(got, oracle(c))
    same = call(pkg, c, dev)
    assert torch.equal(got[0], same[0]) and torch.equal(got[1], same[1])


def test_block_table_longer_than_a_segment(pkg, lib, dev):
    c, b = both([9000], [3], 2, 1, 81)
    got, same = call(pkg, b, dev, pe_dtype=BF), call(pkg, c, dev)
    assert torch.equal(got[0], same[0]) and torch.equal(got[1], same[1])
    check(got, oracle(c))


@pytest.mark.parametrize("bad", [math.nan, math.inf, 3e38])
def test_values_that_fp16_does_not_hold(pkg, lib, dev, bad):
    """In masked places they touch nothing; rows that see them are NaN (3e38 as fp16 is
    infinite)."""
    c, b = both([70, 40], [6, 4], 16, 16, 82)
    for x in (c, b):
        x["mask"][:6] = torch.tensor([1, 3, 4, 12, 16, 33])  # token 2 is seen by 2 and 3 only
    want = oracle(c)
    p = 70 - 6 + 2
    b["rows"][int(b["bt"][0, p // 16]) * 16 + p % 16, 528:].view(BF)[5] = bad
    got = call(pkg, b, dev, pe_dtype=BF)
    live = torch.ones(10, dtype=torch.bool)
    live[2] = live[3] = False
    check(got, want, live)
    assert bool(torch.isnan(got[0][2:4]).all())


def test_rows_written_from_bf16(pkg, lib, dev):
    """Rotated and written by one call, read back and attended to: one type throughout."""
    g = torch.Generator().manual_seed(83)
    c = make([200, 77], [4, 3], 16, 16, "fp8", seed=83)
    kv = torch.zeros(c["rows"].shape[0] // 16, 16, 656, dtype=torch.uint8, device=dev)
    tab = pkg.rope.rotary_table(64, 256, device=dev)
    bt = c["bt"].to(dev)
    for r, n in enumerate([200, 77]):
        p = torch.arange(n, device=dev)
        pkg._cache_ops.rope_concat_and_cache_mla(
            p, tab, torch.randn(n, 512, generator=g).to(BF).to(dev),
            torch.randn(n, 64, generator=g).to(BF).to(dev), kv, bt[r][p // 16].long() * 16 + p % 16,
            "fp8_ds_mla")
    cu = torch.tensor([0, 200, 277], dtype=torch.int32, device=dev)
    rows = pkg._cache_ops.gather_latent_cache(kv, bt, cu, 277, pe_dtype=BF).cpu()
    want = dict(c, rows=torch.zeros(c["rows"].shape[0], 576).half())
    for r, (a, n) in enumerate([(0, 200), (200, 77)]):
        p = torch.arange(n)
        want["rows"][c["bt"][r].long()[p // 16] * 16 + p % 16] = rows[a:a + n]
    got = pkg.mla_tree.tree_attention(c["q"].to(dev), kv, bt, c["seq"].to(dev), c["cu"].to(dev),
                                      c["mask"].to(dev), SCALE, pe_dtype=BF)
    check(got, oracle(want))


def test_refused_types(pkg, lib, dev):
    c = make([20], [2], 4, 16, "fp16", seed=84)
    with pytest.raises(RuntimeError, match="pe_dtype"):
        call(pkg, c, dev, pe_dtype=BF)
    c = make([20], [2], 4, 16, "fp8", seed=84)
    with pytest.raises(RuntimeError, match="pe_dtype"):
        call(pkg, c, dev, pe_dtype=torch.float32)
    assert cache(c, dev).dtype == torch.uint8
