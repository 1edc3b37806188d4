"""Blocks whose scales are zero or far from the other blocks', against the 64-bit definition: a value is code times scale
whatever the scale, and its key takes its share of the softmax. Bounds are test_gpu_kv's and test_gpu_kv_prompt's."""
import numpy as np
import pytest
import torch

from rocknpu_amd import kv
from tests import kv_ref, test_gpu_kv, test_gpu_kv_prompt
from tests.test_gpu_kv import DEV, TYPES, ints, offsets, random_cache
from tests.test_gpu_kv_prompt import BATCH, GROUP, KV_HEADS, check_attention, lengths, many_tiles

pytestmark = pytest.mark.gpu

SCALES = {"zero": 0.0, "minus-zero": -0.0, "least": 2.0 ** -100, "below": 2.0 ** -130, "large": 2.0 ** 40, "edge": 2.0 ** -40,
          "under-edge": 2.0 ** -41}


def set_scales(c, which, value):
    """Every third block's scale of the keys (0) or values (1)."""
    pages = c.table[:, :, ::3].flatten().long()
    c.scales[pages, which] = value
    return c


@pytest.mark.parametrize("name", list(SCALES))
@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_value_scales(name, kind):
    for new in (1, 3):
        c = set_scales(random_cache(80, 3, 2, 64, 30), 1, SCALES[name])
        test_gpu_kv.run_attention(81, kind, 64, 2, 4, [800, 90, 3], [new] * 3, cache=c, weights=True, window=700)
    past, new = lengths(6)
    assert many_tiles(new)
    c = set_scales(random_cache(82, BATCH, KV_HEADS, 64, 12), 1, SCALES[name])
    test_gpu_kv_prompt.run_attention(83, kind, 64, KV_HEADS, GROUP, past, new, cache=c)
    test_gpu_kv_prompt.run_attention(84, kind, 64, KV_HEADS, GROUP, past, new, cache=c, slopes=0.1 * torch.ones(16))


@pytest.mark.parametrize("name", ["zero", "minus-zero", "least"])
@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_key_scales(name, kind):
    for new in (1, 3):
        c = set_scales(random_cache(85, 3, 2, 64, 30), 0, SCALES[name])
        test_gpu_kv.run_attention(86, kind, 64, 2, 4, [800, 90, 3], [new] * 3, cache=c, weights=True)
    past, new = lengths(7)
    c = set_scales(random_cache(87, BATCH, KV_HEADS, 64, 12), 0, SCALES[name])
    test_gpu_kv_prompt.run_attention(88, kind, 64, KV_HEADS, GROUP, past, new, cache=c)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("new", [1, 41])
def test_heavy_blocks_of_zero_values(kind, new):
    """Scores that rise by 122 and 140 powers of two, the first rise to a block of zero values as append leaves one."""
    past, news = [100] * BATCH, [new] * BATCH
    c = random_cache(91, BATCH, KV_HEADS, 64, 6)
    for at, score in ((0, 0.0), (1, 122.0), (2, 140.0), (3, 100.0)):
        pages = c.table[:, :, at].flatten().long()
        c.pages[pages, :32 * 64] = 127
        c.scales[pages, 0] = score * float(np.log(2)) / (0.125 * 64 * 127)
        if at == 1:
            c.pages[pages, 32 * 64:] = 0
            c.scales[pages, 1] = 2.0 ** -100
    cu = offsets(news)
    q = torch.ones((cu[-1], KV_HEADS * GROUP, 64)).to(TYPES[kind])
    o = kv.attention(c, q.to(DEV), ints(past), ints(cu), new)
    check_attention(o, kv_ref.Ref(c).attention(q.double().numpy(), past, cu), kind, 64, 141)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("new", [1, 41])
def test_blocks_of_zeros_beside_large_values(kind, new):
    """The zeros' keys keep their share of the denominator, however far the scales lie apart."""
    past, news = [100] * BATCH, [new] * BATCH
    c = set_scales(random_cache(94, BATCH, KV_HEADS, 64, 6), 1, 2.0 ** 40)
    pages = c.table[:, :, 1::3].flatten().long()
    c.pages[pages, 32 * 64:] = 0
    c.scales[pages, 1] = 2.0 ** -100
    test_gpu_kv_prompt.run_attention(95, kind, 64, KV_HEADS, GROUP, past, news, cache=c)


@pytest.mark.parametrize("which", [0, 1])
@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_negative_scales_count_as_not_finite(kind, which):
    """NaN in the rows that see the block and in no other, through both kernels."""
    for past, new, kv_heads, group in (([800, 90, 3], [2] * 3, 2, 4), (*lengths(9), KV_HEADS, GROUP)):
        outs, q = [], None
        for value in (-0.02, float("nan")):
            c = set_scales(random_cache(96, len(past), kv_heads, 64, 30), which, value)
            cu = offsets(new)
            q = torch.randn((cu[-1], kv_heads * group, 64), generator=torch.Generator().manual_seed(97)).to(TYPES[kind])
            outs.append(kv.attention(c, q.to(DEV), ints(past), ints(cu), max(new), window=40).cpu())
        torch.testing.assert_close(outs[0], outs[1], rtol=0, atol=0, equal_nan=True)
        assert torch.isnan(outs[0]).any() and not torch.isnan(outs[0]).all()


@pytest.mark.parametrize("old", [0.0, -0.0, 2.0 ** -130, 3.0, -0.03, float("-inf"), float("inf"), float("nan")])
def test_appending_to_blocks_of_any_scale(old):
    """A block's older values are kept to half a step of its new scale; a scale that is negative or not finite leaves NaN."""
    c = random_cache(92, 1, 2, 64, 3)
    page = c.table[0, :, 0].long()
    c.scales[page] = old
    r = kv_ref.Ref(c)
    k = torch.randn((5, 2, 64), generator=torch.Generator().manual_seed(93))
    kv.append(c, k.to(DEV), k.to(DEV), ints([20]), ints([0, 5]), 5)
    got = kv_ref.Ref(c)
    for h in range(2):
        scale = got.scales[got.table[0, h, 0]]
        if not (np.isfinite(old) and old >= 0):
            assert np.isnan(scale).all()
            continue
        top = k[:, h].abs().max().numpy() / np.float32(127)
        assert np.all(scale == max(top, np.float32(old)))
        for x, y in zip(got.values(got.table[0, h, 0]), r.values(r.table[0, h, 0])):
            assert np.all(np.abs(x[:20] - y[:20]) <= 0.5001 * scale[0])
            assert np.all(np.abs(x[20:25] - k[:, h].numpy()) <= 0.5001 * scale[0])
