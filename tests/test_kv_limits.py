"""The key/value cache's entry points at the ends of their arguments' ranges, on the CPU."""
import ctypes

import pytest

from rocknpu_amd import _lib
from tests.test_kv import attention_struct, cache_struct


def workspace(c, a, cus=256):
    n = ctypes.c_size_t(1 << 63)
    status = _lib.load().rocknpu_hip_kv_attention_workspace(ctypes.byref(c), ctypes.byref(a), cus, ctypes.byref(n))
    return status, n.value


@pytest.mark.parametrize("kv_heads,heads,max_new", [(256, 256, 2 ** 31 - 1), (32768, 32768, 2 ** 24), (65535, 65535, 2 ** 31 - 1),
                                                    (1, 1, 2 ** 31 - 1), (4, 65532, 1000)])
@pytest.mark.parametrize("batch", [1, 300])
@pytest.mark.parametrize("kind", [0, 2])
def test_the_workspace_of_calls_of_any_size(kv_heads, heads, max_new, batch, kind):
    """Kv heads times tiles of rows may pass 32 bits."""
    c = cache_struct(kv_heads=kv_heads, batch=batch, max_blocks=4000)
    a = attention_struct(heads=heads, max_new=max_new, rows=2 ** 31 - 1, type=kind)
    status, n = workspace(c, a)
    # far more tiles than the GPU holds workgroups: nothing is shared out, so nothing is joined
    assert (status, n) == (0, 0)


@pytest.mark.parametrize("max_new", [3, 4, 1000, 10 ** 6, 2 ** 31 - 1])
@pytest.mark.parametrize("weights", [False, True])
def test_no_sequence_has_more_rows_than_the_step(max_new, weights):
    """A bound above the step's rows, as a caller gives that keeps one for all its steps, is the step's rows."""
    lib = _lib.load()
    if weights and max_new * 2 > 256:
        return  # over the limit of such calls
    c = cache_struct(batch=7, max_blocks=500)
    kw = dict(rows=3, weights_out=1 << 20 if weights else 0, heads=4)
    exact, loose = attention_struct(max_new=3, **kw), attention_struct(max_new=max_new, **kw)
    assert workspace(c, loose) == workspace(c, exact)
    blocks, parts, slots = (ctypes.c_int32 * 7)(*[400] * 7), (ctypes.c_int32 * 7)(), ctypes.c_int64()
    got = []
    for a in (exact, loose):
        assert lib.rocknpu_hip_kv_attention_parts(ctypes.byref(c), ctypes.byref(a), 256, blocks, parts, ctypes.byref(slots)) == 0
        got.append((list(parts), slots.value))
    assert got[0] == got[1]


@pytest.mark.parametrize("max_tokens", [2 ** 31 - 1, 2 ** 40, 2 ** 63 - 32, 2 ** 63 - 1])
def test_expecting_more_tokens_than_the_table_holds(max_tokens):
    """An expectation without limit plans for the table's width, as none does."""
    c = cache_struct(batch=2, max_blocks=4000)
    assert workspace(c, attention_struct(max_tokens=max_tokens)) == workspace(c, attention_struct(max_tokens=0))


@pytest.mark.parametrize("bad", [dict(out_row=0), dict(out_row=63), dict(out_head=0), dict(out_head=63)], ids=str)
def test_outputs_that_overlap(bad):
    """Rows or heads that share elements would be written in no order, as an expanded tensor's."""
    c = cache_struct()
    assert workspace(c, attention_struct(**bad))[0] == -1
    # a single row's or head's stride does not matter; another order of the two is one
    assert workspace(cache_struct(kv_heads=1), attention_struct(rows=1, heads=1, **bad))[0] == 0
    assert workspace(c, attention_struct(out_row=64, out_head=128))[0] == 0
