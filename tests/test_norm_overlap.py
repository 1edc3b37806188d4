"""hip.norm_a8's outputs may be x or the residual in place, and overlap nothing else."""
import ctypes

import pytest
import torch

from rocknpu_amd import _lib, hip

AT = {n: (i + 1) << 20 for i, n in enumerate(("x", "residual", "weight", "hidden", "out", "a8", "scales"))}  # never read: a refused call touches nothing
PLACES = dict(rows=5, k=100, k_pad=128, x_row=300, residual_row=300, hidden_row=300, out_row=300, type=0, weight_type=0, eps=1e-5)


def call(**kw):
    return _lib.load().rocknpu_hip_norm_a8(ctypes.byref(hip._NormStruct(**{**AT, **PLACES, **kw})), None)


X, R, W, H = AT["x"], AT["residual"], AT["weight"], AT["hidden"]
REFUSED = [
    dict(out=H), dict(out=H + 4), dict(out=H - 4), dict(out=H + 396), dict(out=H - 396), dict(out=H + 1200 * 2), dict(out=H + 1200 - 396), dict(out=H - 1200 + 396),
    dict(out=H, residual=H), dict(out=H + 400, out_row=301), dict(out=H + 400, out_row=100), dict(out=H + 5196), dict(hidden=X + 4), dict(hidden=X - 4), dict(hidden=X + 1200),
    dict(hidden=X - 1200), dict(hidden=R + 1200 * 4), dict(hidden=R + 4), dict(out=R + 4), dict(out=X + 8), dict(hidden=X, hidden_row=301), dict(hidden=X, hidden_row=100),
    dict(hidden=X, x_row=0), dict(out=X, out_row=200), dict(hidden=X, out=X), dict(hidden=X, out=X, residual=X), dict(hidden=X, residual=X + 4), dict(hidden=W), dict(out=W + 396),
    dict(hidden=W - 1200), dict(a8=X), dict(a8=R + 5196), dict(a8=W + 399), dict(a8=H + 5199), dict(a8=H - 639), dict(a8=AT["out"]), dict(scales=X), dict(scales=W), dict(scales=R + 5196),
    dict(scales=H - 16), dict(scales=AT["a8"] + 636), dict(scales=AT["a8"] - 16), dict(rows=1, out=H + 396), dict(rows=1, hidden=X + 4), dict(rows=1, scales=W + 396),
    dict(type=2, weight_type=2, out=H + 198), dict(type=2, weight_type=2, out=H - 198)]


@pytest.mark.parametrize("kw", REFUSED, ids=str)
def test_refused(kw):
    assert call(**kw) == -1


ALLOWED = [
    {}, dict(hidden=X), dict(hidden=R), dict(out=X), dict(out=R), dict(hidden=X, out=R), dict(hidden=R, out=X), dict(residual=X, hidden=X), dict(residual=X, out=X),
    dict(out=H + 400), dict(out=H + 800), dict(out=H - 400), dict(out=H - 800), dict(out=H + 1200 + 400), dict(out=H - 2 * 1200 - 400), dict(hidden=X + 400), dict(hidden=X + 400, out=X + 800),
    dict(x=H, residual=H + 400, out=H + 800), dict(out=H + 5200), dict(out=H + 5200, out_row=100), dict(a8=H + 5200), dict(a8=H - 640), dict(scales=AT["a8"] + 640), dict(scales=H - 20),
    dict(rows=1, out=H + 400), dict(rows=1, out=H - 400, out_row=7), dict(rows=1, hidden=X, hidden_row=100), dict(x_row=0), dict(x_row=0, residual_row=0, residual=X), dict(x_row=1, residual_row=2),
    dict(type=2, weight_type=2, out=H + 200), dict(type=2, weight_type=2, out=H + 400), dict(hidden=0), dict(hidden=0, residual=0, out=X)]


@pytest.mark.skipif(torch.cuda.is_available(), reason="such a call would run on the GPU")
@pytest.mark.parametrize("kw", ALLOWED, ids=str)
def test_allowed(kw):
    """Without a GPU what the checks let through fails at its launch."""
    assert call(**kw) == -3


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_in_one_buffer(dtype):
    """Columns of one wide buffer as inputs and outputs; the same with outputs that reach into each other are refused, and nothing is written."""
    m, k = 40, 96
    g = torch.Generator().manual_seed(1)
    wide = torch.randn((m, 4 * k), generator=g).to(dtype).cuda()
    x, r, h, o = (wide[:, i * k:(i + 1) * k] for i in range(4))
    w = torch.randn(k, generator=g).cuda()
    want_out = torch.empty((m, k), dtype=dtype, device="cuda")
    a8, s, want = hip.norm_a8(x.contiguous(), w, residual=r.contiguous(), out=want_out)
    got = hip.norm_a8(x, w, residual=r, hidden=h, out=o)
    torch.cuda.synchronize()
    assert torch.equal(got[0], a8) and torch.equal(got[1], s) and torch.equal(h, want) and torch.equal(o, want_out)
    before = wide.clone()
    for kw in (dict(hidden=h, out=wide[:, 3 * k - 1:4 * k - 1]), dict(hidden=wide[:, k + 1:2 * k + 1]), dict(hidden=x, out=wide[:, 1:k + 1]), dict(hidden=wide.view(-1)[:m * k].view(m, k))):
        with pytest.raises(hip.LaunchError):
            hip.norm_a8(x, w, residual=r, **kw)
    torch.cuda.synchronize()
    assert torch.equal(wide, before)
