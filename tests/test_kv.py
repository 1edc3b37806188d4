"""The 8-bit key/value cache on the CPU: what its entry points refuse, the
ctypes structures against the header's, and the plain forms that the GPU tests
check against."""
import ctypes
import math
import shutil
import subprocess
from pathlib import Path

import numpy as np
import pytest
import torch

from rocknpu_amd import _lib, kv
from tests import kv_ref

ROOT = Path(__file__).resolve().parents[1]
INVALID = -1


@pytest.fixture
def lib():
    return _lib.load()


def cache_struct(**kw):
    at = 1 << 20  # never read: a refused call touches nothing
    base = dict(pages=at, scales=at, table=at, starts=at, dropped=at, weights=at, n_pages=8, batch=2, kv_heads=2,
                head_dim=64, max_blocks=4)
    return kv._CacheStruct(**{**base, **kw})


def attention_struct(**kw):
    at = 1 << 20
    base = dict(q=at, out=at, past=at, cu=at, prefix=0, slopes=0, weights_out=0, q_row=256, q_head=64, out_row=256,
                out_head=64, rows=2, max_new=1, max_tokens=0, type=0, heads=4, causal=1, window=0, scale=0.125, softcap=0.0)
    return kv._AttentionStruct(**{**base, **kw})


def evict_struct(**kw):
    at = 1 << 20
    base = dict(table=at, starts=at, weights=at, tokens=at, dropped=at, table_out=at, starts_out=at, weights_out=at,
                dropped_out=at + 64, batch=1, kv_heads=1, max_blocks=8, budget=4, sinks=1, recent=1)
    return kv._EvictStruct(**{**base, **kw})


BAD_CACHES = [dict(pages=0), dict(scales=0), dict(table=0), dict(starts=0), dict(dropped=0), dict(pages=(1 << 20) + 8),
              dict(scales=(1 << 20) + 4), dict(head_dim=0), dict(head_dim=80), dict(head_dim=320), dict(n_pages=0),
              dict(n_pages=1 << 31), dict(batch=0), dict(batch=65536), dict(kv_heads=0), dict(kv_heads=65536), dict(max_blocks=0),
              dict(max_blocks=1 << 26)]


@pytest.mark.parametrize("bad", BAD_CACHES, ids=str)
def test_refused_caches(lib, bad):
    c, a, at = cache_struct(**bad), attention_struct(), 1 << 20
    n = ctypes.c_size_t()
    assert lib.rocknpu_hip_kv_append(ctypes.byref(c), 0, at, 128, 64, at, 128, 64, 1, at, at, 1, None) == INVALID
    assert lib.rocknpu_hip_kv_read(ctypes.byref(c), at, at, 1, 0, at, at, None) == INVALID
    assert lib.rocknpu_hip_kv_attention(ctypes.byref(c), ctypes.byref(a), None, 0, None) == INVALID
    assert lib.rocknpu_hip_kv_attention_workspace(ctypes.byref(c), ctypes.byref(a), 256, ctypes.byref(n)) == INVALID


def test_refused_appends_and_reads(lib):
    c, at = cache_struct(), 1 << 20
    good = [ctypes.byref(c), 0, at, 128, 64, at, 128, 64, 1, at, at, 1, None]
    for i, v in ((0, None), (1, 3), (2, None), (2, at + 2), (3, -1), (4, -64), (5, None), (6, -1), (7, -1), (8, 1 << 31),
                 (9, None), (10, None), (11, 1 << 31)):
        assert lib.rocknpu_hip_kv_append(*good[:i], v, *good[i + 1:]) == INVALID, (i, v)
    # nothing to do needs no rows
    assert lib.rocknpu_hip_kv_append(*good[:2], None, 0, 0, None, 0, 0, 0, at, at, 1, None) == 0
    good = [ctypes.byref(c), at, at, 1, 0, at, at, None]
    for i, v in ((0, None), (1, None), (2, None), (3, 1 << 31), (4, 3), (5, None), (5, at + 8), (6, None), (6, at + 4)):
        assert lib.rocknpu_hip_kv_read(*good[:i], v, *good[i + 1:]) == INVALID, (i, v)
    assert lib.rocknpu_hip_kv_read(ctypes.byref(c), at, at, 0, 0, None, None, None) == 0


@pytest.mark.parametrize("bad", [
    dict(q=0), dict(out=0), dict(past=0), dict(cu=0), dict(q=(1 << 20) + 2), dict(q_row=-1), dict(q_head=-1), dict(out_row=-1),
    dict(out_head=-1), dict(rows=-1), dict(rows=1 << 31), dict(max_new=-1), dict(max_new=1 << 31), dict(max_tokens=-1),
    dict(type=3), dict(heads=0), dict(heads=3), dict(heads=-2), dict(window=-1), dict(causal=0, window=5),
    dict(causal=0, prefix=1 << 20), dict(scale=math.inf), dict(scale=math.nan), dict(softcap=-1.0), dict(softcap=math.inf),
    dict(softcap=math.nan), dict(weights_out=1 << 20, heads=32, max_new=17)], ids=str)
def test_refused_attention(lib, bad):
    c, a, n = cache_struct(), attention_struct(**bad), ctypes.c_size_t()
    assert lib.rocknpu_hip_kv_attention(ctypes.byref(c), ctypes.byref(a), None, 0, None) == INVALID
    assert lib.rocknpu_hip_kv_attention_workspace(ctypes.byref(c), ctypes.byref(a), 256, ctypes.byref(n)) == INVALID


def test_refused_workspaces(lib):
    c, n = cache_struct(), ctypes.c_size_t()
    # block weights without a cache that accumulates them
    bare, a = cache_struct(weights=0), attention_struct(weights_out=1 << 20)
    assert lib.rocknpu_hip_kv_attention(ctypes.byref(bare), ctypes.byref(a), None, 0, None) == INVALID
    assert lib.rocknpu_hip_kv_attention_workspace(ctypes.byref(c), ctypes.byref(a), 256, ctypes.byref(n)) == 0
    assert n.value > 0
    at = 1 << 20
    for ws, size in ((None, 0), (at, n.value - 1), (at + 128, n.value)):
        assert lib.rocknpu_hip_kv_attention(ctypes.byref(c), ctypes.byref(a), ws, size, None) == INVALID
    assert lib.rocknpu_hip_kv_attention_workspace(ctypes.byref(c), ctypes.byref(a), 256, None) == INVALID


@pytest.mark.parametrize("bad", [
    dict(table=0), dict(starts=0), dict(weights=0), dict(tokens=0), dict(dropped=0), dict(table_out=0), dict(starts_out=0),
    dict(weights_out=0), dict(dropped_out=0), dict(dropped_out=1 << 20), dict(batch=0), dict(kv_heads=0), dict(max_blocks=0),
    dict(max_blocks=16385), dict(budget=0), dict(sinks=-1), dict(recent=0), dict(sinks=4), dict(recent=2 ** 31 - 1),
    dict(batch=1 << 16, kv_heads=1 << 16)], ids=str)
def test_refused_evictions(lib, bad):
    a = evict_struct(**bad)
    assert lib.rocknpu_hip_kv_evict(ctypes.byref(a), None) == INVALID
    assert lib.rocknpu_hip_kv_evict(None, None) == INVALID


def small_cache(**kw):
    t = torch.zeros((2, 1, 3), dtype=torch.int32)
    base = dict(pages=torch.zeros((6, 4096), dtype=torch.int8), scales=torch.ones((6, 2)), table=t, starts=t.clone(),
                dropped=torch.zeros(2, dtype=torch.int32), weights=None, head_dim=64)
    return kv.Cache(**{**base, **kw})


def test_python_refusals():
    for kw in (dict(head_dim=72), dict(pages=torch.zeros((6, 4096))), dict(pages=torch.zeros((6, 8192), dtype=torch.int8)),
               dict(pages=torch.zeros((0, 4096), dtype=torch.int8)), dict(scales=torch.ones((6, 1))),
               dict(scales=torch.ones((2, 6)).T), dict(starts=torch.zeros((2, 1, 4), dtype=torch.int32)),
               dict(dropped=torch.zeros(2)), dict(weights=torch.zeros((2, 1, 2))), dict(table=torch.zeros(6, dtype=torch.int32))):
        with pytest.raises(ValueError):
            small_cache(**kw)
    c = small_cache()
    k, past, cu = torch.zeros((2, 1, 64)), torch.zeros(2, dtype=torch.int32), torch.zeros(3, dtype=torch.int32)
    for args in ((k.double(), k.double(), past, cu), (k, k.half(), past, cu), (k, k[:1], past, cu), (k[..., :32], k, past, cu),
                 (k.expand(2, 2, 64), k, past, cu), (torch.zeros((2, 1, 128))[..., ::2], k, past, cu), (k, k, past[:1], cu),
                 (k, k, past, past), (k, k, past.long(), cu)):
        with pytest.raises(ValueError):
            kv.append(c, *args, 1)
    for kw in (dict(q=k.double()), dict(q=torch.zeros((2, 64))), dict(out=k.half()), dict(out=torch.zeros((1, 1, 64))),
               dict(prefix=cu), dict(slopes=torch.zeros(2)), dict(weights_out=torch.zeros((2, 1, 2)))):
        with pytest.raises(ValueError):
            kv.attention(c, kw.pop("q", k), past, cu, 1, **kw)
    with pytest.raises(ValueError):
        kv.read(c, past, past, 1, dtype=torch.int8)
    with pytest.raises(ValueError):
        kv.evict(c.table, c.starts, c.table, past, past, 2)


@pytest.mark.skipif(shutil.which("gcc") is None, reason="gcc not installed")
@pytest.mark.parametrize("c,py", [("rocknpu_kv_cache", kv._CacheStruct), ("rocknpu_kv_attention_args", kv._AttentionStruct),
                                  ("rocknpu_kv_evict_args", kv._EvictStruct)], ids=lambda x: x if isinstance(x, str) else "")
def test_structures_match_the_header(c, py, tmp_path):
    src = tmp_path / "layout.c"
    body = "".join(f'    printf("%zu\\n", offsetof({c}, {f}));\n' for f, _ in py._fields_)
    src.write_text('#include <stddef.h>\n#include <stdio.h>\n#include "rocknpu_kv.h"\nint main(void) {\n'
                   f'    printf("%zu\\n", sizeof({c}));\n' + body + "    return 0;\n}\n")
    exe = tmp_path / "layout"
    r = subprocess.run(["gcc", "-std=c99", "-Wall", "-Werror", f"-I{ROOT / 'include'}", str(src), "-o", str(exe)],
                       capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    got = [int(v) for v in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    assert got == [ctypes.sizeof(py)] + [getattr(py, f).offset for f, _ in py._fields_]


@pytest.mark.parametrize("d", kv.HEAD_DIMS)
def test_a_page_holds_every_code_once(d):
    at = np.concatenate((kv_ref.key_index(d).ravel(), kv_ref.value_index(d).ravel()))
    assert np.array_equal(np.sort(at), np.arange(64 * d))
    assert kv_ref.key_index(d).max() < 32 * d <= kv_ref.value_index(d).min()


def test_plain_append_holds_values_to_half_a_step():
    """The plain form itself: what it stores is within half a step of the value, older tokens within a step and a half."""
    c = kv.Cache.empty(1, 2, 64, 3, device="cpu")
    r = kv_ref.Ref(c)
    g = np.random.default_rng(1)
    rows = [g.standard_normal((n, 2, 64)).astype(np.float32) * s for n, s in ((20, 1.0), (30, 3.0))]
    r.append(rows[0], rows[0], [0], [0, 20])
    r.append(rows[1], rows[1], [20], [0, 30])
    x = np.concatenate(rows)
    for h in range(2):
        for at in range(2):
            page = r.table[0, h, at]
            live = min(50 - 32 * at, 32)
            for i, v in enumerate(r.values(page)):
                off = np.abs(v[:live] - x[32 * at:32 * at + live, h]) / r.scales[page, i]
                assert off.max() <= 1.001 and np.all(off[(20 if at == 0 else 0):] <= 0.5001)


def test_plain_attention_against_a_softmax_by_hand():
    c = kv.Cache.empty(1, 1, 64, 2, device="cpu")
    r = kv_ref.Ref(c)
    g = np.random.default_rng(2)
    x = g.standard_normal((40, 1, 64)).astype(np.float32)
    r.append(x, x[::-1].copy(), [0], [0, 40])
    q = g.standard_normal((40, 2, 64))
    keys, values = (np.concatenate([r.values(p)[i] for p in r.table[0, 0]])[:40] for i in (0, 1))
    s = torch.from_numpy(q).transpose(0, 1) @ torch.from_numpy(keys).T / 8
    s = s.masked_fill(~torch.ones(40, 40).tril().bool(), -math.inf).softmax(-1) @ torch.from_numpy(values)
    out, mag, _, weights = r.attention(q, [0], [0, 40])
    assert np.allclose(out, s.transpose(0, 1).numpy(), atol=1e-12) and np.all(np.abs(out) <= mag + 1e-12)
    assert np.isclose(weights.sum(), 80)
