"""The experts' products are dealt out to workgroups so that every tile is taken once: whole, in halves or in quarters."""
import ctypes
import random

import numpy as np
import pytest

from rocknpu_amd import _lib, moe
from tests.moe_places import forms, places, tiles_of


def covered(tokens, experts, top_k, hidden, ffn, row_tiles, cus):
    for gated, n in ((1, ffn), (0, hidden)):
        tile, p = places(tokens, experts, top_k, hidden, ffn, gated, row_tiles, cus)
        columns = -(-n // tile[1])
        used = p[p[:, 0] >= 0]
        assert (used[:, 0] < row_tiles).all() and (used[:, 1] >= 0).all() and (used[:, 1] < columns).all()
        assert set(used[:, 3].tolist()) <= ({1, 2, 4} if tile[0] == 256 else {1}) and (used[:, 2] >= 0).all() and (used[:, 2] < used[:, 3]).all()
        quarters = np.zeros((row_tiles, columns, 4), np.int64)  # [row, column] halves of a tile
        for row, column, part, parts in used.tolist():
            taken = {1: (0, 1, 2, 3), 2: (part, part + 2), 4: (part,)}[parts]
            quarters[row, column, list(taken)] += 1
        assert (quarters == 1).all(), (gated, tile, row_tiles, columns, cus)


@pytest.mark.parametrize("cus", [1, 7, 8, 80, 104, 228, 256, 304])
def test_every_tile_once(cus):
    rng = random.Random(cus)
    for _ in range(60):
        experts = rng.choice([1, 2, 5, 8, 24, 64, 256])
        top_k = min(experts, rng.choice([1, 2, 3, 8]))
        tokens = int(2 ** rng.uniform(2, 14)) + 8
        hidden, ffn = int(2 ** rng.uniform(0, 12)), int(2 ** rng.uniform(0, 12))
        rows = tokens * top_k
        tile_rows = places(tokens, experts, top_k, hidden, ffn, 1, 0, cus)[0][0]
        if not tile_rows:
            continue
        most = rows // tile_rows + min(rows, experts)
        for row_tiles in {0, 1, most, rng.randint(0, most), min(most, 63), min(most, 64)}:
            covered(tokens, experts, top_k, hidden, ffn, row_tiles, cus)


def test_ways_to_share_a_last_round():
    """On 256 CUs, 32 an XCD: 25 row tiles by 8 and 4 columns, 40 by 8, 70 by 4."""
    t25, t40 = tiles_of((600, 833, 1100, 300, 900, 64, 1000, 323), 256), tiles_of((2560, 2560, 2560, 2560), 256)
    p = places(2560, 8, 2, 1024, 1024, 1, 25, 256)[1]
    assert forms(p, t25, 1024) == {(1, 64), (1, 128), (1, 192), (1, 256)}
    assert forms(p, t25, 1088) == {(1, 64), (1, 128), (1, 256)}
    assert forms(places(2560, 8, 2, 1024, 1024, 0, 25, 256)[1], t25, 1024) == {(2, 128), (2, 256)}
    assert forms(places(5120, 4, 2, 1024, 1024, 1, 40, 256)[1], t40, 1024) == {(1, 256), (4, 128)}
    p = places(9000, 8, 2, 1024, 256, 0, 70, 256)[1]
    for xcd in range(8):
        used = p[xcd::8][p[xcd::8, 0] >= 0]
        assert [int((used[:, 3] == parts).sum()) for parts in (1, 2, 4)] == [32, 0, 12]


def test_calls_without_tiles_and_refusals():
    assert places(1, 64, 8, 256, 256, 1, 1)[0] == (0, 0)
    assert places(0, 64, 8, 256, 256, 1, 0)[0] == (0, 0)
    lib, n, tile, out = _lib.load(), ctypes.c_size_t(), (ctypes.c_int32 * 2)(), (ctypes.c_int32 * 4)()
    f, args = lib.rocknpu_hip_moe_product_places, moe._ExpertsStruct(tokens=100, experts=4, top_k=2, hidden=64, hidden_pad=64, ffn=64, ffn_pad=64)
    a = ctypes.byref(args)
    assert f(a, 1, 1, 256, tile, None, 0, ctypes.byref(n)) == 0 and n.value > 4
    for bad in ((None, 1, 1, 256, tile, None, 0, ctypes.byref(n)), (a, 1, -1, 256, tile, None, 0, ctypes.byref(n)), (a, 1, 1 << 20, 256, tile, None, 0, ctypes.byref(n)),
                (a, 1, 1, 256, None, None, 0, ctypes.byref(n)), (a, 1, 1, 256, tile, None, 0, None), (a, 1, 1, 256, tile, out, 1, ctypes.byref(n))):
        assert f(*bad) == -1
    args.hidden_pad = 63
    assert f(a, 1, 1, 256, tile, None, 0, ctypes.byref(n)) == -1
