"""The division of tree attention's work (csrc/mla_tree_plan.h) against whole numbers on the
CPU: the pieces of some workgroups, of calls up to the largest that the entry point takes.
Nothing but the division runs, from the lengths alone."""
import ctypes
import os

import pytest
import torch

pytestmark = pytest.mark.gpu

LIB = os.path.join(os.path.dirname(os.path.abspath(__file__)), "hip", "libdsa_testkit.so")
WGS, ROWS, TILE, MIN_TILES = 256, 128, 32, 3
PIECES = 6


def divide(dev, counts, lens, H, blocks, page, runs):
    kit = ctypes.CDLL(LIB)
    p, i = ctypes.c_void_p, ctypes.c_int
    kit.dsa_test_tree_division.argtypes = [p, p, i, i, i, i, i, p, i, i, p]
    cu = [0]
    for n in counts:
        cu.append(cu[-1] + n)
    t = [torch.tensor(x, dtype=torch.int32, device=dev) for x in (cu, lens, runs)]
    out = torch.full((len(runs), 2 + 5 * PIECES), -7, dtype=torch.int64, device=dev)
    torch.cuda.synchronize()
    assert kit.dsa_test_tree_division(t[0].data_ptr(), t[1].data_ptr(), len(counts), cu[-1], H,
                                      blocks, page, t[2].data_ptr(), len(runs), PIECES,
                                      out.data_ptr()) == 0
    return out.tolist()


def groups_of(counts, lens, H, width):
    g = [(-(-n * H // ROWS), max(1, -(-min(max(x, 0), width) // TILE))) for n, x in zip(counts, lens)]
    return g, sum(a * b for a, b in g)


def line_pieces(groups, per, run):
    """The first PIECES pieces of a run of the line of all groups' tiles."""
    out, at, end, base = [], run * per, (run + 1) * per, 0
    for r, (n, tiles) in enumerate(groups):
        while at < base + n * tiles and at < end and len(out) < PIECES:
            g = (at - base) // tiles
            start = base + g * tiles
            hi = min(tiles, at - start + end - at)
            out.append([r, g, at - start, hi, start])
            at = start + hi
        base += n * tiles
    return out + [[-1, -1, -1, -1, -1]] * (PIECES - len(out))


RUNS = [0, 1, 2, 31, 100, 127, 128, 129, 200, 254, 255]


@pytest.mark.parametrize("counts,lens,H,blocks,page", [
    ([40] * 16, [32768] * 16, 64, 1024, 64),              # all groups whole
    ([1] * 300, [31 * i for i in range(300)], 16, 200, 64),
    ([2056], [1 << 28], 16, 1 << 22, 64),                 # 257 groups x 2^23 tiles: 2^31 and more
    ([1 << 21], [1 << 23], 16, 1 << 17, 64),              # 2^18 groups x 2^18 tiles
    ([5, 1 << 20, 3], [100, (1 << 30) - 64, 77], 64, 1 << 24, 64 - 1),
    ([7, 1 << 26, 1, 9], [1 << 29, (1 << 30) - 1, 0, 5], 1, 1 << 29, 1),  # runs of 2^36 tiles
    ([0, 0, 1 << 23, 0] * 3, [5, 0, 1 << 25, 9] * 3, 2, 1 << 20, 48)])
def test_runs_of_the_line(dev, counts, lens, H, blocks, page):
    groups, line = groups_of(counts, lens, H, blocks * page)
    per = max(MIN_TILES, -(-line // WGS))
    for run, got in zip(RUNS, divide(dev, counts, lens, H, blocks, page, RUNS)):
        assert got[:2] == [0, per]
        pieces = [got[2 + 5 * i:7 + 5 * i] for i in range(PIECES)]
        assert pieces == line_pieces(groups, per, run), run


@pytest.mark.parametrize("counts,lens,H,blocks,page", [
    ([4], [500], 16, 8, 64), ([64], [184320], 16, 2880, 64), ([8] * 8, [16384] * 8, 64, 256, 64),
    ([1], [(1 << 30) - 1], 1, 1 << 29, 1),                # 2^25 tiles of one group
    ([64, 1, 0, 3], [1 << 29, 3, 10, 0], 4, 1 << 23, 64)])
def test_cells(dev, counts, lens, H, blocks, page):
    """Every tile of every group once, by one workgroup each, in cells of at most kt."""
    groups, _ = groups_of(counts, lens, H, blocks * page)
    seen = {}
    for got in divide(dev, counts, lens, H, blocks, page, list(range(WGS))):
        kt, per = got[:2]
        assert kt > 0 and per == 1 and got[7:] == [-1] * (5 * (PIECES - 1))
        r, g, lo, hi, _ = got[2:7]
        if r >= 0:
            assert lo < hi <= lo + max(kt, 1)
            seen.setdefault((r, g), []).append((lo, hi))
    assert sorted(seen) == [(r, g) for r, (n, _) in enumerate(groups) for g in range(n)]
    for (r, _), parts in seen.items():
        parts.sort()
        assert parts[0][0] == 0 and parts[-1][1] == groups[r][1]
        assert all(a[1] == b[0] for a, b in zip(parts, parts[1:]))
