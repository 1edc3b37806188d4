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
