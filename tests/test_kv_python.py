"""The Python entry points of the key/value cache on the CPU: what they refuse, and what they make."""
import pytest
import torch

from rocknpu_amd import kv
from tests.test_kv import small_cache


def lengths(n):
    return torch.zeros(n, dtype=torch.int32)


@pytest.mark.parametrize("what,bad", [("window", 2 ** 31), ("window", 2 ** 32 + 5), ("window", -1), ("max_new", 2 ** 64 + 1),
                                      ("max_new", -1), ("max_tokens", 2 ** 64 + 9), ("max_tokens", -5)])
def test_sizes_that_an_attention_call_does_not_hold(what, bad):
    """They are refused by name: none is cut to its low bits."""
    c, q = small_cache(), torch.zeros((2, 1, 64))
    kw = {"max_new": 1, what: bad}
    with pytest.raises(ValueError, match=what):
        kv.attention(c, q, lengths(2), lengths(3), kw.pop("max_new"), **kw)


def test_sizes_that_an_append_or_a_read_does_not_hold():
    c, k = small_cache(), torch.zeros((2, 1, 64))
    for bad in (2 ** 64 + 1, -1):
        with pytest.raises(ValueError, match="max_new"):
            kv.append(c, k, k, lengths(2), lengths(3), bad)
    for bad in (2 ** 31, -1):
        with pytest.raises(ValueError, match="count"):
            kv.read(c, lengths(2), lengths(2), bad)


@pytest.mark.parametrize("what,bad", [("budget", 2 ** 32 + 2), ("sinks", 2 ** 32), ("recent", 2 ** 32 + 1), ("budget", -1)])
def test_sizes_that_an_eviction_does_not_hold(what, bad):
    t = torch.zeros((2, 1, 5), dtype=torch.int32)
    kw = {"budget": 2, "sinks": 0, "recent": 1, what: bad}
    with pytest.raises(ValueError, match=what):
        kv.evict(t, t, torch.zeros(t.shape), lengths(2), lengths(2), kw.pop("budget"), **kw)


@pytest.mark.parametrize("bad", ["elsewhere", "strided"])
def test_a_workspace_that_the_kernels_cannot_write(bad):
    """Its address goes to the kernels: it has to be the cache's device's memory, all of it."""
    c = small_cache(weights=torch.zeros((2, 1, 3)))
    ws = torch.empty(1 << 21, dtype=torch.uint8, device="meta") if bad == "elsewhere" else torch.zeros(1 << 21, dtype=torch.uint8)[::2]
    with pytest.raises(ValueError, match="workspace"):
        kv.attention(c, torch.zeros((2, 1, 64)), lengths(2), lengths(3), 1, weights_out=c.weights, workspace=ws)


@pytest.mark.parametrize("dtype", [torch.float64, torch.bfloat16])
def test_an_empty_cache_is_f32_whatever_torch_makes_by_default(dtype):
    before = torch.get_default_dtype()
    torch.set_default_dtype(dtype)
    try:
        c = kv.Cache.empty(2, 1, 64, 3, device="cpu")
    finally:
        torch.set_default_dtype(before)
    assert c.scales.dtype is torch.float32 and c.weights.dtype is torch.float32


@pytest.mark.parametrize("name", ["pages", "scales", "table", "starts", "dropped", "weights", "head_dim", "max_blocks"])
def test_a_cache_does_not_take_other_tensors(name):
    """The kernels use the buffers that it was made with: an assignment would change what Python shows alone."""
    c = small_cache()
    value = getattr(c, name)
    with pytest.raises(AttributeError, match="new Cache"):
        setattr(c, name, value)
    c.table[:] = 1  # its contents are the caller's
    assert getattr(c, name) is value and int(c.table.sum()) == 6
