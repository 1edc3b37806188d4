"""moe.experts on the GPU against its definition. Products, SwiGLU's values, codes and scales are fixed to the bit by
it; the weighted sum of top_k f32 terms has one rounding a product and one an addition, (top_k + 1) 2^-24 of the
terms' magnitudes at most, and its own rounding to the output's type."""
import math

import numpy as np
import pytest
import torch

from rocknpu_amd import hip, moe, synth
from tests import moe_ref

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def pad(k):
    return (k + 63) // 64 * 64


def stack(g, experts, n, k):
    """Codes behind k are zeros, scales of the size that keeps products near 1."""
    w = torch.zeros((experts, n, pad(k)), dtype=torch.int8)
    w[:, :, :k] = (torch.randn((experts, n, k), generator=g) * 40).round().clamp(-127, 127).to(torch.int8)
    return w.to(DEV), ((0.5 + torch.rand((experts, n), generator=g)) / (40 * math.sqrt(k))).to(DEV)


def layer(seed, experts, hidden, ffn):
    g = torch.Generator().manual_seed(seed)
    return moe.Experts(stack(g, experts, ffn, hidden), stack(g, experts, ffn, hidden), stack(g, experts, hidden, ffn), hidden=hidden, ffn=ffn)


def tokens_of(seed, tokens, hidden):
    g = torch.Generator().manual_seed(seed)
    a = torch.zeros((tokens, pad(hidden)), dtype=torch.int8)
    a[:, :hidden] = (torch.randn((tokens, hidden), generator=g) * 40).round().clamp(-127, 127).to(torch.int8)
    return a.to(DEV), ((0.5 + torch.rand(tokens, generator=g)) / 40).to(DEV)


def verify(w, a8, scales, r, out):
    want, size = moe_ref.experts(a8, scales, r.ids.cpu().numpy(), r.weights.cpu().numpy(), w.gate, w.up, w.down, w.hidden, w.ffn)
    got = out.cpu().double().numpy()
    assert got.shape == want.shape
    assert np.array_equal(np.isnan(got), np.isnan(want))
    info = torch.finfo(out.dtype)
    off = np.abs(got - want) - (r.ids.shape[1] + 1) * 2.0 ** -24 * size - info.eps / 2 * np.abs(want) - info.smallest_normal * info.eps
    worst = np.nanmax(off) if off.size else 0.0
    assert not worst > 0, f"{(off > 0).sum()} of {off.size} outside, worst by {worst:.3g}"


def check(seed, tokens, experts, top_k, hidden, ffn, dtype="f32", masked=0.0, w=None, x=None, what="", **kw):
    print("experts", what, tokens, experts, top_k, hidden, ffn, dtype, masked, flush=True)
    w = w or layer(seed, experts, hidden, ffn)
    a8, scales = tokens_of(seed + 1, tokens, hidden)
    g = torch.Generator().manual_seed(seed + 2)
    if x is None:
        x = torch.randn((tokens, experts), generator=g)
        x[torch.rand(tokens, generator=g) < masked] = -math.inf
        x = x.to(DEV)
    r = moe.route(x, top_k, **kw)
    out = moe.experts(w, a8, scales, r, dtype=TYPES[dtype])
    torch.cuda.synchronize()
    verify(w, a8, scales, r, out)
    return w, a8, scales, r, out


@pytest.mark.parametrize("tokens", [1, 2, 3, 7, 15, 16, 17, 31, 33, 64, 65, 127, 129, 200, 300])
def test_token_counts(tokens):
    check(tokens, tokens, 8, 2, 256, 192)
    check(tokens, tokens, 5, 3, 128, 64, "bf16")


@pytest.mark.parametrize("hidden,ffn", [(1, 1), (3, 5), (63, 65), (64, 64), (65, 63), (100, 100), (128, 320), (200, 33), (1000, 77), (31, 1000),
                                        (512, 704), (2048, 128), (96, 2112)])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_widths(hidden, ffn, dtype):
    for tokens in (1, 37, 150):
        check(hidden + ffn, tokens, 4, 2, hidden, ffn, dtype)


@pytest.mark.parametrize("experts,top_k", [(1, 1), (2, 2), (3, 1), (16, 8), (24, 3), (64, 8), (64, 64), (129, 4), (1024, 2)])
def test_experts(experts, top_k):
    for tokens in (1, 5, 70):
        check(experts, tokens, experts, top_k, 128, 64)
    check(experts, 40, experts, top_k, 64, 128, masked=0.4, score="sigmoid", bias=torch.linspace(-0.1, 0.1, experts, device=DEV))


@pytest.mark.parametrize("tokens,experts,top_k,hidden,ffn", [(1500, 4, 2, 256, 320), (700, 3, 1, 640, 192), (2100, 8, 2, 192, 256), (600, 16, 4, 320, 130),
                                                             (1025, 2, 2, 130, 260), (4000, 2, 1, 128, 128)])
def test_long(tokens, experts, top_k, hidden, ffn):
    check(tokens, tokens, experts, top_k, hidden, ffn, "bf16", masked=0.1)


def test_all_rows_on_one_expert_and_none():
    for tokens in (1, 40, 400):
        x = torch.full((tokens, 12), -math.inf, device=DEV)
        *_, out = check(1, tokens, 12, 2, 192, 128, x=x, what="no choices")
        assert not out.any()
        x[:, 7] = 0.0
        check(2, tokens, 12, 2, 192, 128, x=x, what="one expert")
        x[tokens // 2:] = -math.inf
        check(3, tokens, 12, 2, 192, 128, x=x, what="half of the rows")


def test_sums_at_the_ends_of_int32():
    """The largest codes over a long K: sums beyond 2^24, and the largest there are."""
    for k in (2112, 8192):
        w = layer(1, 2, k, 64)
        w.gate[0].fill_(127)
        w.up[0].fill_(-127)
        a8, scales = torch.full((9, k), 127, dtype=torch.int8, device=DEV), torch.full((9,), 1e-6, device=DEV)
        a8[4], a8[5, ::2] = -127, -127
        r = moe.route(torch.randn((9, 2), generator=torch.Generator().manual_seed(1)).to(DEV), 2)
        verify(w, a8, scales, r, moe.experts(w, a8, scales, r))


def test_nan_rows_stay_alone():
    w = layer(3, 6, 256, 128)
    for tokens in (3, 90):
        a8, scales = tokens_of(4, tokens, 256)
        x = torch.randn((tokens, 6), generator=torch.Generator().manual_seed(5)).to(DEV)
        scales[1] = math.nan
        x[2, 3] = math.nan
        r = moe.route(x, 3)
        out = moe.experts(w, a8, scales, r)
        torch.cuda.synchronize()
        bad = out.isnan().any(1)
        assert bad[1] and bad[2] and bad.sum() == 2
        verify(w, a8, scales, r, out)


def test_values_that_overflow():
    """A product beyond f32 makes its token NaN, large and tiny ones do not."""
    w = layer(6, 3, 128, 64)
    a8, scales = tokens_of(7, 50, 128)
    scales[0], scales[1], scales[2], scales[3] = 1e30, 1e18, 1e-30, 0.0
    r = moe.route(torch.randn((50, 3), generator=torch.Generator().manual_seed(8)).to(DEV), 2)
    verify(w, a8, scales, r, moe.experts(w, a8, scales, r))
    for kind in ("f16", "bf16"):
        verify(w, a8[3:], scales[3:], *(lambda q: (q, moe.experts(w, a8[3:].contiguous(), scales[3:].contiguous(), q, dtype=TYPES[kind])))(
            moe.route(torch.randn((47, 3), generator=torch.Generator().manual_seed(9)).to(DEV), 2)))


def test_outputs_in_wider_rows():
    w = layer(9, 4, 200, 96)
    for tokens in (1, 60):
        a8, scales = tokens_of(10, tokens, 200)
        r = moe.route(torch.randn((tokens, 4), generator=torch.Generator().manual_seed(11)).to(DEV), 2)
        for kind in TYPES.values():
            wide = torch.full((tokens, 333), 7.0, dtype=kind, device=DEV)
            out = wide[:, 5:205]
            assert moe.experts(w, a8, scales, r, out=out) is out
            torch.cuda.synchronize()
            assert (wide[:, :5] == 7).all() and (wide[:, 205:] == 7).all()
            assert torch.equal(out, moe.experts(w, a8, scales, r, dtype=kind))


def test_no_tokens():
    w = layer(12, 4, 64, 64)
    r = moe.route(torch.zeros((0, 4), device=DEV), 2)
    assert moe.experts(w, torch.zeros((0, 64), dtype=torch.int8, device=DEV), torch.zeros(0, device=DEV), r).shape == (0, 64)


def test_same_bits_twice_and_in_any_company():
    """A token's output does not depend on the others in its call."""
    w, a8, scales, r, out = check(13, 300, 16, 4, 384, 256)
    assert torch.equal(out, moe.experts(w, a8, scales, r))
    x = torch.randn((300, 16), generator=torch.Generator().manual_seed(15)).to(DEV)
    r = moe.route(x, 4)
    out = moe.experts(w, a8, scales, r)
    for n in (1, 9, 60, 150):
        few = moe.experts(w, a8[:n].contiguous(), scales[:n].contiguous(), moe.route(x[:n], 4))
        assert torch.equal(out[:n], few), n


def test_workspace():
    w = layer(16, 4, 128, 64)
    a8, scales = tokens_of(17, 20, 128)
    r = moe.route(torch.randn((20, 4), generator=torch.Generator().manual_seed(18)).to(DEV), 2)
    out = moe.experts(w, a8, scales, r)
    need = w._needs[20, 2]
    ws = torch.full((need,), 255, dtype=torch.uint8, device=DEV)
    assert torch.equal(out, moe.experts(w, a8, scales, r, workspace=ws))
    with pytest.raises(moe.LaunchError):
        moe.experts(w, a8, scales, r, workspace=ws[:need - 1])
    with pytest.raises(ValueError):
        moe.experts(w, a8, scales, r, workspace=torch.zeros(2 * need, dtype=torch.uint8, device=DEV)[::2])


@pytest.mark.parametrize("tokens", [1, 4, 120])
def test_streams_and_graphs(tokens):
    """Captured with the routing that feeds it: every replay goes by that replay's logits and rows."""
    w = layer(19, 8, 256, 192)
    a8, scales = tokens_of(20, tokens, 256)
    x = torch.randn((tokens, 8), generator=torch.Generator().manual_seed(21)).to(DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        r = moe.route(x, 2)
        out = moe.experts(w, a8, scales, r)
        torch.cuda.synchronize()
        verify(w, a8, scales, r, out)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            r = moe.route(x, 2)
            out = moe.experts(w, a8, scales, r)
    for seed in range(4):
        new, s = tokens_of(30 + seed, tokens, 256)
        a8.copy_(new)
        scales.copy_(s)
        x.copy_(torch.randn((tokens, 8), generator=torch.Generator().manual_seed(40 + seed)))
        if seed == 2:
            x[:, 1:] = -math.inf
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        verify(w, a8, scales, r, out)
        assert torch.equal(out, moe.experts(w, a8, scales, moe.route(x, 2)))


def test_a_layer_of_quantised_weights():
    """The run of calls a model makes: Q4_K, Q5_K and Q6_K stacks repacked once, then norm, router, choice, experts."""
    experts, hidden, ffn, tokens, top_k = 6, 512, 256, 37, 2

    def repacked(kind, n, k, index):
        blocks = synth.kquant(kind, experts * n, k, index=index)
        w8, s = hip.repack_w8(kind, torch.from_numpy(blocks).to(DEV), k, experts * n)
        return w8.view(experts, n, -1), s.view(experts, n)

    w = moe.Experts(repacked(4, ffn, hidden, 1), repacked(5, ffn, hidden, 2), repacked(6, hidden, ffn, 3), hidden=hidden, ffn=ffn)
    g = torch.Generator().manual_seed(22)
    x, h = torch.randn((tokens, hidden), generator=g).to(DEV), torch.randn((tokens, hidden), generator=g).to(DEV)
    norm = (1 + 0.1 * torch.randn(hidden, generator=g)).to(DEV)
    router = hip.quantize_a8(torch.randn((experts, hidden), generator=g).to(DEV) / math.sqrt(hidden))
    a8, scales, h = hip.norm_a8(x, norm, residual=h, hidden=h)
    logits = hip.gemm_w8a8(a8, scales, *router)
    r = moe.route(logits, top_k)
    out = moe.experts(w, a8, scales, r)
    torch.cuda.synchronize()
    ids, weights, *_ = moe_ref.route(logits, top_k)
    assert np.array_equal(r.ids.cpu().numpy(), ids)
    verify(w, a8, scales, r, out)


def whole_layer(dtype=torch.float32, tokens=37, experts=6, hidden=512, ffn=256):
    g = torch.Generator().manual_seed(23)
    w = layer(24, experts, hidden, ffn)
    x, h = (torch.randn((tokens, hidden), generator=g).to(dtype).to(DEV) for _ in range(2))
    norm = (1 + 0.1 * torch.randn(hidden, generator=g)).to(DEV)
    return x, h, norm, hip.quantize_a8(torch.randn((experts, hidden), generator=g).to(DEV) / math.sqrt(hidden)), w


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_feed_forward_is_its_parts(dtype):
    for tokens in (1, 3, 37, 700):
        x, h, norm, router, w = whole_layer(dtype, tokens)
        out, hidden = moe.feed_forward(x, norm, router, w, 2, residual=h, score="sigmoid", normalise=False)
        a8, s, want_h = hip.norm_a8(x, norm, residual=h)
        r = moe.route(hip.gemm_w8a8(a8, s, *router), 2, score="sigmoid", normalise=False)
        assert torch.equal(hidden, want_h) and torch.equal(out, moe.experts(w, a8, s, r, dtype=dtype)) and out.dtype is dtype
        alone, none = moe.feed_forward(x, norm, router, w, 2)
        assert none is None and alone.shape == x.shape
    x = x[:0]
    assert moe.feed_forward(x, norm, router, w, 2, residual=x)[0].shape == (0, 512)
    with pytest.raises(ValueError):
        moe.feed_forward(h, norm, (router[0][:5], router[1][:5]), w, 2)


def test_layers_in_a_graph():
    """Two layers of norm, router, choice and experts as one graph, replayed on new rows."""
    for tokens in (1, 60):
        x, h, norm, router, w = whole_layer(torch.bfloat16, tokens)
        second = layer(25, 6, 512, 256)

        def step():
            o, r = moe.feed_forward(x, norm, router, w, 2, residual=h)
            return moe.feed_forward(o, norm, router, second, 2, residual=r)

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                got = step()
        for seed in range(4):
            x.copy_(torch.randn(x.shape, generator=torch.Generator().manual_seed(50 + seed)))
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            for a, b in zip(got, step()):
                assert torch.equal(a, b)


def test_two_streams_at_once():
    """Calls on different streams have workspaces of their own."""
    w = layer(26, 8, 256, 192)
    jobs = []
    for i, tokens in enumerate((300, 290)):
        a8, s = tokens_of(60 + i, tokens, 256)
        x = torch.randn((tokens, 8), generator=torch.Generator().manual_seed(70 + i)).to(DEV)
        jobs.append((a8, s, x, moe.experts(w, a8, s, moe.route(x, 2)), torch.cuda.Stream()))
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(8):
        for i, (a8, s, x, _, stream) in enumerate(jobs):
            with torch.cuda.stream(stream):
                outs[i].append(moe.experts(w, a8, s, moe.route(x, 2)))
    torch.cuda.synchronize()
    for i, job in enumerate(jobs):
        assert all(torch.equal(o, job[3]) for o in outs[i])


def test_more_rows_than_a_launch_quantises():
    """2^26 rows and more: over 2^32 threads of one launch, values at offsets past 32 bits."""
    tokens, n, top_k = (1 << 25) + 3, 64, 2
    w = layer(5, 3, n, n)
    g = torch.Generator(DEV).manual_seed(6)
    a8 = torch.randint(-127, 128, (tokens, n), dtype=torch.int8, device=DEV, generator=g)
    scales = torch.rand(tokens, device=DEV, generator=g) / 40
    r = moe.route(torch.randn((tokens, 3), dtype=torch.float16, device=DEV, generator=g), top_k)
    space = torch.empty(tokens * top_k * (5 * n + 4) + 1024, dtype=torch.uint8, device=DEV)
    out = moe.experts(w, a8, scales, r, dtype=torch.float16, workspace=space)
    some = torch.cat([torch.arange(20), torch.randint(0, tokens, (400,), generator=torch.Generator().manual_seed(7)), torch.arange(tokens - 20, tokens)]).to(DEV)
    part = moe.Routing(r.ids[some], r.weights[some], r.plan, 3)
    verify(w, a8[some], scales[some], part, out[some])


def test_other_weights():
    w, a8, scales, r, _ = check(9, 50, 6, 3, 128, 64)
    r.weights = r.weights * 0.25 - 1
    verify(w, a8, scales, r, moe.experts(w, a8, scales, r))
    for bad in (r.weights.half(), r.weights[:, :2], r.weights.t().contiguous().t(), r.weights.cpu()):
        with pytest.raises(ValueError):
            moe.experts(w, a8, scales, moe.Routing(r.ids, bad, r.plan, 6))
    for ids, plan in ((r.ids.long(), r.plan), (r.ids, r.plan[:-1]), (r.ids, r.plan.long()), (r.ids[:40], r.plan)):
        with pytest.raises(ValueError):
            moe.experts(w, a8, scales, moe.Routing(ids, r.weights, plan, 6))


@pytest.mark.parametrize("experts,top_k,ffn", [(8, 8, 14336), (2, 2, 61440), (2, 2, 70000), (64, 64, 1984), (64, 64, 2048)])
def test_one_token_of_long_rows(experts, top_k, ffn):
    """The rows' codes fill most of LDS, or do not fit it."""
    check(ffn, 1, experts, top_k, 64, ffn)
