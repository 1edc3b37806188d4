"""Attention over more sequences than a wave has lanes, against the 64-bit definition: every sequence is computed, with
outputs that held NaN and a workspace that held anything. Bounds are test_gpu_kv's."""
import numpy as np
import pytest
import torch

from rocknpu_amd import kv
from tests import kv_ref
from tests.test_gpu_kv import DEV, TYPES, check_attention, ints, offsets, random_cache

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("batch,kv_heads,d,group,new,equal", [
    (65, 8, 64, 2, 1, False), (80, 4, 128, 4, 1, False), (100, 1, 128, 3, 1, True), (128, 4, 64, 8, 1, False),
    (200, 2, 64, 4, 1, False), (100, 2, 192, 2, 3, False), (300, 1, 64, 1, 1, False), (65, 1, 256, 2, 1, True),
    (100, 2, 128, 4, 12, False), (70, 1, 64, 4, 40, True)])
@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_more_sequences_than_lanes(batch, kv_heads, d, group, new, equal, kind):
    print(batch, kv_heads, d, group, new, equal, kind, flush=True)
    g = np.random.default_rng(batch)
    past = [1500] * batch if equal else g.integers(1030, 1700, batch).tolist()
    news = [new] * batch if equal else g.integers(0, new + 1, batch).tolist()
    news[-1] = new
    if not equal:
        past[7], past[batch - 3] = 0, 3
    c = random_cache(60, batch, kv_heads, d, 55)
    cu = offsets(news)
    q = torch.randn((cu[-1], kv_heads * group, d), generator=torch.Generator().manual_seed(61)).to(TYPES[kind])
    weigh = new == 1
    out = torch.full(q.shape, float("nan"), dtype=q.dtype, device=DEV)
    wo = torch.full_like(c.weights, float("nan")) if weigh else None
    ws = torch.full((1 << 28,), 0xff, dtype=torch.uint8, device=DEV)
    kv.attention(c, q.to(DEV), ints(past), ints(cu), new, max_tokens=1720, out=out, weights_out=wo, workspace=ws)
    torch.cuda.synchronize()
    ref = kv_ref.Ref(c)
    want = ref.attention(q.double().numpy(), past, cu)
    check_attention(out, want, kind, d, 1720)
    if weigh:
        weights = ref.weights.astype(np.float64) + want[3]
        rel = 2 * (2.0 ** -22 + (np.sqrt(d) + 8) * 2.0 ** -24) * want[2].max() + 2.0 ** -20
        assert np.all(np.abs(wo.cpu().double().numpy() - weights) <= rel * want[3] + 2.0 ** -22 * weights + 1e-30)
