"""How an attention call's blocks are shared out over workgroups: every sequence gets its parts, and all of them fit the
launch, whatever the lengths are. The host asks the function that the kernels ask."""
import ctypes

import numpy as np
import pytest

from rocknpu_amd import _lib
from tests.test_kv import attention_struct, cache_struct

BATCHES = [1, 2, 3, 17, 48, 63, 64, 65, 66, 80, 96, 100, 128, 200, 333, 512, 1023, 1024, 1025, 4000]


def parts_of(c, a, blocks, cus=256):
    blocks = np.ascontiguousarray(blocks, np.int32)
    parts, slots = np.full(len(blocks), -1, np.int32), ctypes.c_int64(-1)
    at = blocks.ctypes.data, parts.ctypes.data
    assert _lib.load().rocknpu_hip_kv_attention_parts(ctypes.byref(c), ctypes.byref(a), cus, *at, ctypes.byref(slots)) == 0
    return parts, slots.value


def lengths(g, batch, most):
    """Equal, ragged, one long among short ones, and some sequences without rows."""
    yield np.full(batch, most)
    yield g.integers(1, most + 1, batch)
    yield np.minimum(most, np.maximum(1, (most * g.random(batch) ** 6).astype(int)))
    yield np.where(np.arange(batch) == batch // 2, most, 1)
    yield g.integers(1, most + 1, batch) * (g.random(batch) < 0.8)


@pytest.mark.parametrize("batch", BATCHES)
@pytest.mark.parametrize("d", [64, 128, 192, 256])
def test_every_sequence_gets_its_parts(batch, d):
    g = np.random.default_rng(batch + d)
    shared = 0
    for kv_heads in (1, 2, 3, 4, 8, 32):
        for group, new, kind in ((1, 1, 0), (4, 1, 2), (8, 5, 1), (4, 12, 2), (4, 64, 0)):
            for most, cus in ((33, 256), (127, 256), (500, 256), (5000, 256), (127, 304), (127, 64)):
                c = cache_struct(batch=batch, kv_heads=kv_heads, head_dim=d, max_blocks=most)
                a = attention_struct(heads=kv_heads * group, max_new=new, rows=batch * new, type=kind, out_head=d,
                                     out_row=kv_heads * group * d)
                for blocks in lengths(g, batch, most):
                    parts, slots = parts_of(c, a, blocks, cus)
                    what = (kv_heads, group, new, most, cus)
                    assert parts.sum() <= slots, what
                    assert np.all(parts[blocks > 0] >= 1) and np.all(parts <= np.maximum(blocks, 1)), what
                    assert parts.max() <= 256, what
                    shared += parts.max() > 1
    assert shared or batch > 256


def test_refusals():
    lib, at = _lib.load(), 1 << 20
    blocks, parts, slots = (ctypes.c_int32 * 2)(), (ctypes.c_int32 * 2)(), ctypes.c_int64()
    good = [ctypes.byref(cache_struct()), ctypes.byref(attention_struct()), 256, ctypes.byref(blocks), ctypes.byref(parts),
            ctypes.byref(slots)]
    assert lib.rocknpu_hip_kv_attention_parts(*good) == 0
    for i, v in ((0, None), (0, ctypes.byref(cache_struct(batch=0))), (1, None), (1, ctypes.byref(attention_struct(q=at + 1))),
                 (3, None), (4, None), (5, None)):
        assert lib.rocknpu_hip_kv_attention_parts(*good[:i], v, *good[i + 1:]) == -1, i
