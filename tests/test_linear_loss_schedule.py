"""The order of work of linear_cross_entropy's backward, on the CPU: every unit of every product comes exactly once, and whatever a
unit waits for stands before it in the order in which units are claimed (that is what keeps the kernel from waiting forever)."""
import itertools

import pytest

from streamep_b200 import _ext

DZ, DX, DW = 1, 2, 3


def up(a, b):
    return -(-a // b)


@pytest.mark.parametrize("want_dx,want_dw", [(True, True), (True, False), (False, True)])
@pytest.mark.parametrize("T,H,V", [(1, 8, 1), (1, 64, 300), (64, 256, 1000), (128, 2048, 100003), (129, 520, 4097), (1777, 1000, 50257),
                                   (8192, 2048, 65536), (16384, 72, 131072), (300, 7168, 9000), (5003, 4096, 257)])
def test_units_and_order(T, H, V, want_dx, want_dw):
    (pieces, piece, splits, ahead, buffers, row_units, split2, group), *units = _ext.load().linear_loss_schedule(T, H, V, 148, want_dx, want_dw)
    assert piece % 256 == 0 and (pieces - 1) * piece < V <= pieces * piece
    assert row_units == up(T, 256) and (not split2 or T <= 64) and pieces >= buffers >= min(ahead + 1, pieces)
    cols = [min(piece, V - j * piece) for j in range(pieces)]
    want = set()
    for j in range(pieces):
        tiles = up(cols[j], 256)
        want |= {(DZ, j, m, n, 0) for m, n in itertools.product(range(row_units), range(tiles))}
        if want_dx:
            want |= {(DX, j, m, n, s) for m, n, s in itertools.product(range(row_units), range(up(H, 256)), range(splits))}
        if want_dw:
            want |= {(DW, j, m, n, 0) for m, n in itertools.product(range(tiles), range(0, up(H, 256), group))}
    assert len(units) == len(want) and {tuple(u[:5]) for u in units} == want
    place = {}
    for i, u in enumerate(units):
        place.setdefault((u[0], u[1]), []).append(i)
    blocks = {}
    for i, (kind, j, m, n, s, k0, k) in enumerate(units):
        if kind == DZ:
            assert (k0, k) == (0, up(H, 64))
            if j >= buffers:        # the buffer it writes is no longer read
                assert all(max(place.get((other, j - buffers), [-1])) < i for other in (DX, DW))
        else:
            assert max(place[DZ, j]) < i
            if kind == DX:
                assert j == 0 or max(place[DX, j - 1]) < i
                blocks.setdefault((j, m, n), []).append((k0, k))
            else:
                assert (k0, k) == (0, up(T, 32 if T <= 32 else 64) * (2 if split2 else 1))
    for (j, m, n), got in blocks.items():      # the splits of a dx tile cover its piece once
        covered = [b for k0, k in got for b in range(k0, k0 + k)]
        assert sorted(covered) == list(range(up(cols[j], 64)))
