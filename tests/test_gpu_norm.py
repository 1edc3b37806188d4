"""hip.norm_a8 on the GPU against its definition.

The definition fixes every f32 operation behind the codes and `hidden`: those are
exact. The mean's f32 partial sums hold at most 64 squares a thread: relative
error at most 65 2^-24 of the mean, half of it in 1 / sqrt, and one rounding more in
the scale: 34 2^-24. `out` has that and its own rounding."""
import numpy as np
import pytest
import torch

from rocknpu_amd import hip

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
OFF = 34 * 2.0 ** -24


def reference(x, w, eps, r=None):
    """Codes, scales and normed rows (64 bits), and x + r in x's type."""
    h = x.float().cpu().numpy()
    if r is not None:
        h = h + r.float().cpu().numpy()
    with np.errstate(all="ignore"):
        u = h * w.float().cpu().numpy()
        fine = np.isfinite(u).all(1)
        peak = np.where(fine, np.abs(u).max(1), np.float32(0)).astype(np.float32)
        step = np.where(peak == 0, np.float32(1), peak / np.float32(127)).astype(np.float32)
        q = np.where(fine[:, None], u, np.float32(0)) / step[:, None]
        assert q.dtype == np.float32
        q = q.astype(np.float64)
        codes = np.clip(np.copysign(np.floor(np.abs(q) + 0.5), q), -127, 127)
        f = 1.0 / np.sqrt((h.astype(np.float64) ** 2).mean(1) + np.float64(np.float32(eps)))
        f = np.where(fine, f, np.nan)
        return codes.astype(np.int8), step * f, u.astype(np.float64) * f[:, None], torch.from_numpy(h).to(x.dtype)


def check(x, w, eps=1e-5, r=None, what="", **kw):
    print("norm", what, tuple(x.shape), x.dtype, w.dtype, x.stride(), "r" if r is not None else "", sorted(kw), flush=True)
    m, k = x.shape
    xc, rc = x.clone(), None if r is None else r.clone()
    a8, scales, hidden = hip.norm_a8(x, w, eps, residual=r, **kw)
    torch.cuda.synchronize()
    codes, want, normed, h = reference(xc, w, eps, rc)
    got = a8.cpu().numpy()
    assert np.array_equal(got[:, :k], codes)
    assert not got[:, k:].any()
    s = scales.cpu().double().numpy()
    assert np.array_equal(np.isnan(s), np.isnan(want))
    assert (np.nan_to_num(np.abs(s - want) - OFF * np.abs(want)) <= 2.0 ** -149).all(), np.nanmax(np.abs(s / want - 1))
    if r is None:
        assert hidden is None
    else:
        bits = torch.int32 if x.dtype is torch.float32 else torch.int16
        a, b = hidden.cpu(), h
        assert torch.equal(a.isnan(), b.isnan())
        assert torch.equal(a.nan_to_num(0, None, None).contiguous().view(bits), b.nan_to_num(0, None, None).contiguous().view(bits))
    if "out" in kw:
        y = kw["out"].cpu().double().numpy()
        info = torch.finfo(x.dtype)
        assert np.array_equal(np.isnan(y), np.isnan(normed))
        off = np.abs(y - normed) - (OFF + info.eps / 2) * np.abs(normed) - info.smallest_normal * info.eps
        big = np.abs(normed) > info.max
        assert (np.nan_to_num(np.where(big, 0, off)) <= 0).all()
    return a8, scales, hidden


def rows(seed, m, k, kind, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    return (spread * torch.randn((m, k), generator=g)).to(TYPES[kind]).to(DEV)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("k", [1, 2, 3, 63, 64, 65, 100, 256, 1000, 1024, 2047, 2048, 4096, 5632, 8200, 14336, 16384, 16392, 33000, 65535, 65536])
def test_widths(kind, k):
    m = 3 if k > 8192 else 5
    x, r = rows(k, m, k, kind), rows(k + 1, m, k, kind, 2.0)
    w = 1 + 0.3 * torch.randn(k, generator=torch.Generator().manual_seed(k + 2))
    check(x, w.to(DEV), r=r, out=torch.full_like(x, 7.0))
    check(x, w.to(TYPES[kind]).to(DEV))


@pytest.mark.parametrize("m,k", [(1, 2048), (600, 2048), (513, 4096), (2000, 72), (4097, 64)])
@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
def test_many_rows(kind, m, k):
    check(rows(m, m, k, kind), rows(1, 1, k, "f32")[0], r=rows(m + 1, m, k, kind))


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_strides_and_places(kind):
    """Slices of wider rows, odd bases, k_pad beyond a multiple of 64, and outputs in place."""
    wide = rows(3, 6, 700, kind)
    w = rows(4, 1, 513, "f32")[0]
    for at, k in ((0, 512), (8, 512), (1, 512), (3, 513)):
        x, r = wide[:, at:at + k], rows(5, 6, 640, kind)[:, 16:16 + k]
        check(x, w[:k], r=r, out=torch.zeros((6, 600), dtype=TYPES[kind], device=DEV)[:, 8:8 + k], k_pad=777)
        before = wide.clone()
        check(x, w[:k], r=r, hidden=r, out=x, what="in place")
        assert torch.equal(wide[:, :at], before[:, :at]) and torch.equal(wide[:, at + k:], before[:, at + k:])
        check(x, w[:k], r=r, hidden=x, out=r, what="in place, crossed")
    one = rows(6, 1, 512, kind)
    check(one.expand(4, 512), w[:512], r=one.expand(4, 512), what="rows 0 apart")
    check(one[0][None], w[:512])
    check(wide[::2, :512], w[:512])


def test_no_rows():
    a8, scales, hidden = hip.norm_a8(torch.zeros((0, 64), device=DEV), torch.ones(64, device=DEV), residual=torch.zeros((0, 64), device=DEV))
    assert a8.shape == (0, 64) and scales.shape == (0,) and hidden.shape == (0, 64)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("k", [257, 512])
def test_values_at_the_ends(kind, k):
    info = torch.finfo(TYPES[kind])
    x = rows(9, 16, k, kind)
    w = torch.ones(k, device=DEV)
    x[0] = 0.0                              # a row of zeros
    x[1, 5], x[2, 6], x[3, 7] = torch.inf, -torch.inf, torch.nan
    x[4] = info.max                         # f32: squares beyond its range
    x[5] = info.smallest_normal
    x[6] = info.smallest_normal * info.eps  # the least value there is
    x[7, ::2], x[7, 1::2] = info.max, -info.max
    x[8] *= info.smallest_normal
    x[9] = 0.0
    x[9, 3] = 1.0
    x[10] = torch.arange(k) - k // 2        # ties of the rounding
    x[10, 0] = 127.0
    x[11] = 0.5 * (torch.arange(k) % 255 - 127)
    x[11, 1] = 127.0
    for eps in (1e-5, 1e-30):
        check(x, w, eps, out=torch.zeros_like(x))
        check(x, w, eps, r=torch.zeros_like(x), out=torch.zeros_like(x))
    check(x[4:8], w, r=x[4:8], what="sums beyond the type")
    w[3], w[4] = torch.inf, torch.nan
    check(x, w, out=torch.zeros_like(x), what="a weight that is not finite")


def test_as_quantize_a8():
    """Behind a norm whose factor is 1 the codes and scales are quantize_a8's."""
    x = rows(11, 64, 1024, "f32")
    a8, s, _ = hip.norm_a8(x, torch.ones(1024, device=DEV))
    q8, qs = hip.quantize_a8(x)
    assert torch.equal(a8, q8)
    f = 1.0 / (x.double().square().mean(1) + 1e-5).sqrt()
    assert torch.allclose(s.double(), qs.double() * f, rtol=OFF + 2.0 ** -23, atol=0)


def test_product_of_normed_rows():
    """The rows feed gemm_w8a8 as they are."""
    x, w = rows(12, 33, 1000, "bf16"), rows(13, 1, 1000, "f32")[0]
    w8, ws = hip.quantize_a8(rows(14, 70, 1000, "f32"))
    a8, s, _ = hip.norm_a8(x, w)
    got = hip.gemm_w8a8(a8, s, w8, ws).double()
    want = (a8.double() * s.double()[:, None]) @ (w8.double() * ws.double()[:, None]).T.contiguous()
    assert ((got - want).abs() <= 3 * 2.0 ** -24 * want.abs() + 1e-12).all()


def test_streams_and_graphs():
    """On another stream, and captured: every replay sees the buffers as they are then."""
    x, r, w = rows(15, 40, 2048, "bf16"), rows(16, 40, 2048, "bf16"), rows(17, 1, 2048, "f32")[0]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        check(x, w, r=r)
        out = [torch.empty((40, 2048), dtype=torch.int8, device=DEV), torch.empty(40, device=DEV), torch.empty_like(x)]
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            hip.norm_a8(x, w, residual=r, a8=out[0], scales=out[1], hidden=out[2])
    for seed in range(4):
        x.copy_(rows(20 + seed, 40, 2048, "bf16"))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        a8, s, h = hip.norm_a8(x, w, residual=r)
        torch.cuda.synchronize()
        assert torch.equal(out[0], a8) and torch.equal(out[1], s) and torch.equal(out[2], h)


def test_more_rows_than_a_launch_has_threads():
    """2^26 rows of a wave each are 2^32 threads."""
    rows, k = (1 << 26) + 5, 60
    x, w = torch.randn((1, k), generator=torch.Generator().manual_seed(1)).to(DEV), torch.ones(k, device=DEV)
    one, s = hip.norm_a8(x, w)[:2]
    a8, scales, _ = hip.norm_a8(x.expand(rows, k), w)
    assert bool((scales == s).all())
    for part in a8.split(1 << 22):
        assert bool((part == one).all())
