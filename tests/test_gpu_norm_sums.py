"""The bits of hip.norm_a8's mean: squares are added up in 64 bits.

f is then right to about k 2^-53, so a scale is off by its one rounding to f32, 2^-24 of it, and `out` by that of
u * f to f32 and its own to a type of fewer bits. 2^-36 stands for f's error: k is at most 2^16."""
import numpy as np
import pytest
import torch

from rocknpu_amd import hip

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
OFF = 2.0 ** -24 + 2.0 ** -36


def rows_with_strong_channels(seed, m, k, kind, how):
    """Rows of which one channel (or some, or none) is about 1000 times the others."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((m, k), generator=g)
    if how == "one":
        x[torch.arange(m), torch.randint(0, k, (m,), generator=g)] *= 1000.0
    elif how == "some":
        x *= 1.0 + 999.0 * (torch.rand((1, k), generator=g) < 0.003)
    return x.to(TYPES[kind])


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("k", [64, 2047, 4096, 8200, 16384, 33001, 65536])
@pytest.mark.parametrize("how", ["one", "some", "none"])
def test_scales_are_rounded_once(kind, k, how):
    print("norm sums", kind, k, how, flush=True)
    m = 64 if k <= 4096 else 24
    x, r = rows_with_strong_channels(k, m, k, kind, how), rows_with_strong_channels(k + 1, m, k, kind, how)
    w = 1 + 0.3 * torch.randn(k, generator=torch.Generator().manual_seed(k + 2))
    out = torch.zeros((m, k), dtype=TYPES[kind], device=DEV)
    a8, scales, _ = hip.norm_a8(x.to(DEV), w.to(DEV), residual=r.to(DEV), out=out)
    torch.cuda.synchronize()
    h = x.float().numpy() + r.float().numpy()
    u = h * w.numpy()
    f = 1.0 / np.sqrt((h.astype(np.float64) ** 2).mean(1) + np.float64(np.float32(1e-5)))
    want = (np.abs(u).max(1) / np.float32(127)).astype(np.float64) * f
    got = scales.cpu().double().numpy()
    assert (np.abs(got - want) <= OFF * want).all(), np.abs(got / want - 1).max() * 2 ** 24
    normed = u.astype(np.float64) * f[:, None]
    info = torch.finfo(TYPES[kind])
    own = info.eps / 2 if kind != "f32" else 0.0
    off = np.abs(out.cpu().double().numpy() - normed) - (OFF + own) * (1 + OFF) * np.abs(normed) - info.smallest_normal * info.eps
    assert (off <= 0).all(), off.max()
