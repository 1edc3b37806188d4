"""Which workgroup takes which part of the experts' products (rocknpu_hip_moe_product_places)."""
import ctypes

import numpy as np

from rocknpu_amd import _lib, moe


def pad(k):
    return (k + 63) // 64 * 64


def places(tokens, experts, top_k, hidden, ffn, gated, row_tiles, cus=0):
    """((a tile's rows, its columns), [workgroups, 4]: row tile, column tile, part, parts)."""
    lib, n, tile = _lib.load(), ctypes.c_size_t(), (ctypes.c_int32 * 2)()
    args = moe._ExpertsStruct(tokens=tokens, experts=experts, top_k=top_k, hidden=hidden, hidden_pad=pad(hidden), ffn=ffn, ffn_pad=pad(ffn))
    assert lib.rocknpu_hip_moe_product_places(ctypes.byref(args), gated, row_tiles, cus, tile, None, 0, ctypes.byref(n)) == 0
    out = np.empty((n.value, 4), np.int32)
    if n.value:
        assert lib.rocknpu_hip_moe_product_places(ctypes.byref(args), gated, row_tiles, cus, tile, out.ctypes.data, n.value, ctypes.byref(n)) == 0
    return tuple(tile), out


def tiles_of(counts, tile_rows):
    """Rows of the row tiles of experts with that many rows each."""
    return [min(tile_rows, c - at) for c in counts for at in range(0, c, tile_rows)]


def forms(places, tiles, k):
    """What of 256 x 256 tiles runs: pairs of the parts (1: whole, 2: halves, 4: quarters) and the rows of the form that
    takes them. 192 rows are a form of 128-byte stages, which K has to be a multiple of."""
    got = set()
    for row, _, part, parts in places[places[:, 0] >= 0].tolist():
        n = min(tiles[row] - part // 2 * 128, 128) if parts == 4 else tiles[row]
        steps = (128, 256) if parts > 1 else (64, 128, 192, 256) if k % 128 == 0 else (64, 128, 256)
        if n > 0:
            got.add((parts, next(s for s in steps if n <= s)))
    return got
