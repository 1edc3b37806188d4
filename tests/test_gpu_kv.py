"""The 8-bit key/value cache on the GPU (include/rocknpu_kv.h) against its
definitions in plain form (tests/kv_ref.py).

Codes, scales, tables and eviction are exact: the definitions fix every f32
operation. Attention is held to a bound derived per row from the 64-bit result:
with T = the largest sum of |terms| of a seen score, A = sum p |v| and N keys,
  - a score's error is at most T times (2^-22 for q as a pair of f16, or 0 for
    f16 and bf16 rows, whose values the pair or single f16 holds to 2^-11 of the
    row's rounding, + (sqrt(D) + 8) 2^-24 for the f32 sum and the operations
    behind it);
  - a weight p has that error twice (its own and its sum's), plus 2^-21 for the
    exponential and, where weights enter as one f16, 2^-10;
  - the output's f32 sum adds (sqrt(N) + 8) 2^-24, and its rounding half an ulp.
"""
import numpy as np
import pytest
import torch

from rocknpu_amd import kv
from tests import kv_ref

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
ULP = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}


def ints(v):
    return torch.tensor(list(v), dtype=torch.int32, device=DEV)


def offsets(new):
    return np.concatenate(([0], np.cumsum(new))).astype(int).tolist()


def random_cache(seed, batch, kv_heads, d, max_blocks, lost=None, past=None, weights=True, spare=3):
    """Random codes and scales, pages in scattered order, `lost` blocks of each sequence evicted."""
    g = torch.Generator().manual_seed(seed)
    n = batch * kv_heads * max_blocks
    pages = torch.randint(-127, 128, (n + spare, 64 * d), generator=g, dtype=torch.int8)
    scales = 0.01 * torch.exp(0.7 * torch.randn((n + spare, 2), generator=g))
    table = torch.randperm(n + spare, generator=g)[:n].to(torch.int32).view(batch, kv_heads, max_blocks)
    starts = (32 * torch.arange(max_blocks, dtype=torch.int32)).expand(batch, kv_heads, -1).contiguous()
    dropped = torch.zeros(batch, dtype=torch.int32)
    for b in range(batch):
        gone = lost[b] if lost else 0
        dropped[b] = gone
        for h in range(kv_heads if gone else 0):
            full = past[b] // 32
            kept = torch.randperm(full, generator=g)[:full - gone].sort().values
            starts[b, h] = 32 * torch.cat((kept, torch.arange(full, full + max_blocks)))[:max_blocks]
    w = torch.rand((batch, kv_heads, max_blocks), generator=g) if weights else None
    return kv.Cache(*(None if t is None else t.to(DEV) for t in (pages, scales, table, starts, dropped, w)), head_dim=d)


def check_attention(got, ref, kind, d, keys, what=""):
    out, mag, big, _ = ref
    got = got.cpu().double().numpy()
    assert np.array_equal(np.isnan(got), np.isnan(out)), what
    score = big[..., None] * ((2.0 ** -22 if kind == "f32" else 0.0) + (np.sqrt(d) + 8) * 2.0 ** -24)
    weight = 2 * score + 2.0 ** -21 + (0.0 if kind == "f32" else 2.0 ** -10)
    bound = mag * (weight + (np.sqrt(keys) + 8) * 2.0 ** -24) + ULP[kind] * np.abs(out) + 1e-30
    bad = np.nan_to_num(np.abs(got - out) - bound) > 0
    assert not bad.any(), f"{what}: {bad.sum()} of {bad.size} outside, worst {np.nanmax(np.abs(got - out) / bound):.3g} of the bound"


def run_attention(seed, kind, d, kv_heads, group, past, new, lost=None, what="", weights=False, cache=None, spread=1.0, **kw):
    lost = lost or [0] * len(past)
    print(what or "attention", kind, d, kv_heads, group, past, new, lost, {k: v for k, v in kw.items() if k != "slopes"}, flush=True)
    blocks = max(-(-(p + n) // 32) - e for p, n, e in zip(past, new, lost)) + 2
    c = cache or random_cache(seed, len(past), kv_heads, d, max(blocks, 1), lost, past)
    cu = offsets(new)
    g = torch.Generator().manual_seed(seed + 1)
    q = (spread * torch.randn((cu[-1], kv_heads * group, d), generator=g)).to(TYPES[kind])
    dev = {k: ints(v) if k == "prefix" else v.to(DEV) if k == "slopes" else v for k, v in kw.items()}
    wo = torch.full_like(c.weights, -7.0) if weights else None
    o = kv.attention(c, q.to(DEV), ints(past), ints(cu), max(new), weights_out=wo, **dev)
    torch.cuda.synchronize()
    r = kv_ref.Ref(c)
    kw.pop("max_tokens", None)
    ref = r.attention(q.double().numpy(), past, cu, **{k: v.numpy() if k == "slopes" else v for k, v in kw.items()})
    check_attention(o, ref, kind, d, max(p + n for p, n in zip(past, new)), what)
    if weights:
        want = r.weights.astype(np.float64) + ref[3]
        # a weight's relative error is the probabilities', and the sum's rounding is of the result
        rel = 2 * (2.0 ** -22 + (np.sqrt(d) + 8) * 2.0 ** -24) * (ref[2].max() if ref[2].size else 0) + 2.0 ** -20
        assert np.all(np.abs(wo.cpu().double().numpy() - want) <= rel * ref[3] + 2.0 ** -22 * np.abs(want) + 1e-30), what
    return o, ref


# ------------------------------------------------------------------- append
@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("d", kv.HEAD_DIMS)
@pytest.mark.parametrize("past,new", [([0], [1]), ([31, 32, 33], [1, 1, 1]), ([0, 5, 64], [32, 27, 33]),
                                      ([7, 0, 100, 31], [0, 1, 95, 2]), ([0], [257])])
def test_append(kind, d, past, new):
    print("append", kind, d, past, new, flush=True)
    heads = 3
    c = random_cache(5, len(past), heads, d, max(-(-(p + n) // 32) for p, n in zip(past, new)) + 1)
    r = kv_ref.Ref(c)
    cu = offsets(new)
    g = torch.Generator().manual_seed(9)
    k, v = (torch.randn((cu[-1], heads, d), generator=g).to(TYPES[kind]) for _ in range(2))
    r.append(k.float().numpy(), v.float().numpy(), past, cu)
    kv.append(c, k.to(DEV), v.to(DEV), ints(past), ints(cu), max(new))
    torch.cuda.synchronize()
    same_cache(c, r, [p + n for p, n in zip(past, new)])
    # reading back gives code * scale in the type asked for
    tokens = [p + n for p, n in zip(past, new)]
    first = [max(p - 3, 0) for p in past]
    got = kv.read(c, ints(first), ints(tokens), max(new) + 5, dtype=TYPES[kind])
    check_read(c, r, got, first, tokens, max(new) + 5, kind)


def same_cache(c, r, tokens):
    got = kv_ref.Ref(c)
    assert np.array_equal(got.scales.view(np.uint32)[~np.isnan(r.scales)], r.scales.view(np.uint32)[~np.isnan(r.scales)])
    assert np.array_equal(np.isnan(got.scales), np.isnan(r.scales))
    assert np.array_equal(got.starts, r.starts)
    assert r.weights is None or np.array_equal(got.weights, r.weights)
    for b, total in enumerate(tokens):
        for h in range(r.table.shape[1]):
            held = r.held(b, total)
            for at in range(held):
                live = min(total - r.starts[b, h, at], 32)
                for x, y in zip(got.codes(r.table[b, h, at]), r.codes(r.table[b, h, at])):
                    assert np.array_equal(x[:live], y[:live]), (b, h, at)


def check_read(c, r, got, first, tokens, count, kind):
    for i, x in enumerate(got):
        want = np.zeros(x.shape, np.float32)
        for b in range(len(tokens)):
            for h in range(c.kv_heads):
                for at in range(r.held(b, tokens[b])):
                    page, start = r.table[b, h, at], r.starts[b, h, at]
                    values = r.codes(page)[i].astype(np.float32) * r.scales[page, i]
                    for t in range(32):
                        if 0 <= start + t - first[b] < count and start + t < tokens[b]:
                            want[b, start + t - first[b], h] = values[t]
        assert torch.equal(x.cpu(), torch.from_numpy(want).to(TYPES[kind]))


def test_append_step_by_step_requantises_as_scales_grow():
    d, heads = 128, 2
    c = kv.Cache.empty(2, heads, d, 4)
    r = kv_ref.Ref(c)
    g = torch.Generator().manual_seed(3)
    past = [0, 17]
    for step in range(70):
        gain = 1.5 ** (step % 9)
        k, v = (gain * torch.randn((2, heads, d), generator=g) for _ in range(2))
        r.append(k.numpy(), v.numpy(), past, [0, 1, 2])
        kv.append(c, k.to(DEV), v.to(DEV), ints(past), ints([0, 1, 2]), 1)
        past = [p + 1 for p in past]
    torch.cuda.synchronize()
    # the tokens that sequence 1 claims to hold before its first row were never written: the scale floor's codes
    same_cache(c, r, past)


def test_append_strided_rows():
    """k and v as slices of one projection's output, offset so that no 16-byte alignment is left."""
    d, heads = 64, 2
    for pad in (0, 3):
        fused = torch.randn((40, 5 * heads * d + pad), device=DEV)
        k = fused[:, heads * d + pad:2 * heads * d + pad].unflatten(1, (heads, d))
        v = fused[:, 3 * heads * d + pad:4 * heads * d + pad].unflatten(1, (heads, d))
        c = kv.Cache.empty(1, heads, d, 3)
        r = kv_ref.Ref(c)
        r.append(k.cpu().numpy(), v.cpu().numpy(), [20], [0, 40])
        kv.append(c, k, v, ints([20]), ints([0, 40]), 40)
        torch.cuda.synchronize()
        same_cache(c, r, [60])


@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
def test_append_poisons_the_block_of_a_value_that_is_not_finite(value):
    d, heads = 64, 2
    c = kv.Cache.empty(1, heads, d, 4)
    r = kv_ref.Ref(c)
    k, v = torch.randn((70, heads, d)), torch.randn((70, heads, d))
    k[40, 1, 13] = value
    r.append(k.numpy(), v.numpy(), [0], [0, 70])
    kv.append(c, k.to(DEV), v.to(DEV), ints([0]), ints([0, 70]), 70)
    # it stays so when tokens join it, and is gone when the block is started anew
    assert np.isnan(c.scales.cpu().numpy()[r.table[0, 1, 1], 0]) and not np.isnan(c.scales.cpu().numpy()[r.table[0, 0, 1]]).any()
    same_cache(c, r, [70])
    again = torch.randn((32, heads, d))
    r.append(again.numpy(), again.numpy(), [50], [0, 32])
    kv.append(c, again.to(DEV), again.to(DEV), ints([50]), ints([0, 32]), 32)
    same_cache(c, r, [82])
    r.append(again.numpy(), again.numpy(), [32], [0, 32])
    kv.append(c, again.to(DEV), again.to(DEV), ints([32]), ints([0, 32]), 32)
    same_cache(c, r, [64])
    assert not np.isnan(c.scales.cpu().numpy()).any()


def test_append_zeros_and_tiny_values():
    d = 64
    c = kv.Cache.empty(1, 1, d, 2)
    r = kv_ref.Ref(c)
    k, v = torch.zeros((40, 1, d)), torch.zeros((40, 1, d))
    v[3, 0, 5] = 1e-38
    k[35, 0, 7] = 2.0 ** -101
    r.append(k.numpy(), v.numpy(), [0], [0, 40])
    kv.append(c, k.to(DEV), v.to(DEV), ints([0]), ints([0, 40]), 40)
    same_cache(c, r, [40])
    o = kv.attention(c, torch.randn((1, 2, d), device=DEV), ints([39]), ints([0, 1]), 1)
    assert torch.equal(o, torch.zeros_like(o))


def test_append_and_attention_skip_what_lies_outside():
    """Lengths and pages that only the device sees: nothing outside the buffers is touched."""
    d = 64
    c = kv.Cache.empty(2, 1, d, 2, weights=False)
    before = c.pages.clone()
    k = torch.randn((4, 1, d), device=DEV)
    kv.append(c, k, k, ints([64, 1000]), ints([0, 2, 4]), 2)       # past the table
    c.table[:] = ints([-1, 99, 7, -5]).view(2, 1, 2)
    kv.append(c, k, k, ints([0, 0]), ints([0, 2, 4]), 2)           # no such page
    torch.cuda.synchronize()
    assert torch.equal(c.pages, before)
    o = kv.attention(c, k, ints([0, 0]), ints([0, 2, 4]), 2)
    assert torch.isnan(o).all()
    o = kv.attention(c, k, ints([0, 0]), ints([0, 50, 3]), 2, out=torch.zeros_like(k))  # rows that are not there
    torch.cuda.synchronize()
    for x in kv.read(c, ints([0, 0]), ints([2, 2]), 2):
        assert not x.any()


# --------------------------------------------------------------------- read
def test_read_after_eviction_and_at_any_offset():
    past, lost = [200, 64, 31], [3, 1, 0]
    c = random_cache(7, 3, 2, 128, 8, lost, past)
    r = kv_ref.Ref(c)
    for first, count in (([0, 0, 0], 230), ([5, 63, 31], 40), ([190, 70, 0], 1)):
        got = kv.read(c, ints(first), ints(past), count)
        check_read(c, r, got, first, past, count, "f32")


# ---------------------------------------------------------------- attention
@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("d", kv.HEAD_DIMS)
@pytest.mark.parametrize("group", [1, 4, 8, 16])
def test_single_tokens(kind, d, group):
    run_attention(11, kind, d, 2, group, [0, 31, 32, 450, 1000], [1, 1, 1, 1, 1], weights=True)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("group,new", [(1, 16), (1, 17), (3, 5), (4, 7), (5, 3), (7, 2), (8, 2), (24, 1), (40, 1)])
def test_few_tokens(kind, group, new):
    run_attention(12, kind, 64, 3, group, [0, 300, 77, 31], [new, new, 1, 0], weights=True)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("d", kv.HEAD_DIMS)
@pytest.mark.parametrize("past,new", [([0], [130]), ([64, 0, 5], [65, 33, 200])])
def test_prompts(kind, d, past, new):
    run_attention(13, kind, d, 2, 3, past, new)


@pytest.mark.parametrize("kind", list(TYPES))
def test_long_prompt(kind):
    run_attention(14, kind, 128, 1, 4, [3], [700], spread=2.0)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("past", [[5000], [4095, 1, 2050]])
def test_long_contexts_split_over_workgroups(kind, past):
    run_attention(15, kind, 128, 2, 4, past, [1] * len(past), weights=True, spread=2.0)
    run_attention(16, kind, 64, 1, 2, past, [40] * len(past))


@pytest.mark.parametrize("max_tokens", [0, 1, 200, 100000])
def test_the_expected_length_sizes_the_split_only(max_tokens):
    run_attention(17, "f32", 64, 2, 4, [3000, 10], [1, 1], weights=True, max_tokens=max_tokens)
    run_attention(18, "f16", 64, 2, 4, [700, 10], [60, 30], max_tokens=max_tokens)


@pytest.mark.parametrize("new", [1, 3, 50])
@pytest.mark.parametrize("kw", [dict(window=1), dict(window=33), dict(window=100, prefix=[7, 40, 0]), dict(prefix=[300, 90, 1]),
                                dict(softcap=30.0), dict(softcap=5.0, window=64, prefix=[4, 4, 4])],
                         ids=lambda k: "-".join(k))
@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_masks_and_caps(kind, new, kw):
    run_attention(19, kind, 64, 2, 4, [500, 64, 3], [new, new, new], weights=new < 50, **kw)


@pytest.mark.parametrize("new", [1, 5, 60])
@pytest.mark.parametrize("kind", ["f32", "f16"])
def test_distance_bias(kind, new):
    slopes = 2.0 ** (-8.0 * torch.arange(1, 13) / 12)
    run_attention(20, kind, 64, 3, 4, [0, 400], [new, new], slopes=slopes, weights=new < 60)
    run_attention(21, kind, 128, 3, 4, [900, 40], [new, new], slopes=-0.01 * slopes, softcap=20.0, scale=0.05)


@pytest.mark.parametrize("new", [1, 4, 80])
def test_evicted_blocks(new):
    run_attention(22, "f32", 64, 2, 4, [700, 320, 64], [new, new, new], lost=[9, 4, 2], weights=new < 80)
    run_attention(23, "f16", 128, 2, 4, [700, 320, 64], [new, new, new], lost=[9, 4, 2], window=200, prefix=[50, 0, 64])


@pytest.mark.parametrize("new", [1, 40])
def test_not_causal(new):
    run_attention(24, "f32", 64, 2, 2, [300, 0], [new, new], causal=False, weights=new == 1)


def test_rows_that_see_nothing_are_zero():
    d = 64
    for new in (1, 3, 70):
        # the only blocks are gone: every key that a row could see was evicted
        c = random_cache(25, 2, 1, d, 8)
        c.dropped[:] = ints([99, 8])
        q = torch.randn((2 * new, 4, d), device=DEV)
        wo = torch.full_like(c.weights, -7.0) if new < 70 else None
        o = kv.attention(c, q, ints([100, 64]), ints([0, new, 2 * new]), new, weights_out=wo)
        assert torch.equal(o, torch.zeros_like(o))
        assert wo is None or torch.equal(wo, c.weights)
        # a window over a place where blocks are missing, some rows see keys and some none
        run_attention(26, "f32", d, 1, 2, [320], [new], lost=[9], window=40, prefix=[3])


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("new", [1, 50])
def test_values_not_finite_in_masked_places(kind, new):
    """A poisoned block reaches the rows that see it and no other; unused slots may hold anything."""
    past = [400, 90]
    for w in (0, 1):
        c = random_cache(27, 2, 2, 64, 18)
        table = c.table.cpu().numpy()
        c.scales[table[0, 0, 2], w] = float("nan")   # positions 64..95
        c.scales[table[1, 1, 0], w] = float("inf")   # positions 0..31
        run_attention(27, kind, 64, 2, 4, past, [new, new], cache=c, window=64)
        c.scales[table[1, 1, 0], w] = float("nan")
        run_attention(27, kind, 64, 2, 4, past, [new, new], cache=c)


def test_large_and_equal_scores():
    """Scores far beyond exp's range, and all equal ones."""
    for spread in (0.0, 1e-30, 60.0):
        run_attention(28, "f32", 64, 1, 4, [600], [2], spread=spread, weights=True)
        run_attention(29, "bf16", 128, 1, 4, [90], [100], spread=spread)


def test_strided_queries_and_outputs():
    d, heads = 64, 4
    c = random_cache(30, 2, 2, d, 6)
    past, cu = [60, 100], [0, 3, 40]
    for pad in (0, 8, 3):
        fused = torch.randn((40, 2 * heads * d + pad), device=DEV)
        q = fused[:, pad:pad + heads * d].unflatten(1, (heads, d))
        want = kv.attention(c, q.contiguous(), ints(past), ints(cu), 37)
        o = torch.zeros((40, heads, 2 * d + pad), device=DEV)
        kv.attention(c, q, ints(past), ints(cu), 37, out=o[:, :, :d])
        assert torch.equal(o[:, :, :d], want) and not o[:, :, d:].any()
        check_attention(want, kv_ref.Ref(c).attention(q.cpu().double().numpy(), past, cu), "f32", d, 137)


def test_pages_beyond_two_gigabytes():
    d = 256
    n = (2 ** 31) // (64 * d) + 300
    pages = torch.empty((n, 64 * d), dtype=torch.int8, device=DEV)
    pages[-300:].random_(-127, 128)
    scales = torch.full((n, 2), 0.02, device=DEV)
    table = torch.arange(n - 12, n, dtype=torch.int32, device=DEV).view(1, 2, 6)
    c = kv.Cache(pages, scales, table, (32 * torch.arange(6, dtype=torch.int32, device=DEV)).expand(1, 2, 6).contiguous(),
                 ints([0]), torch.zeros((1, 2, 6), device=DEV), head_dim=d)
    small = kv.Cache(pages[-300:].clone(), scales[-300:].clone(), table - (n - 300), c.starts, c.dropped, c.weights, head_dim=d)
    for new in (1, 70):
        q = torch.randn((new, 4, d), device=DEV)
        args = (q, ints([100]), ints([0, new]), new)
        assert torch.equal(kv.attention(c, *args), kv.attention(small, *args))
    k = torch.randn((20, 2, d), device=DEV)
    kv.append(c, k, k, ints([100]), ints([0, 20]), 20)
    kv.append(small, k, k, ints([100]), ints([0, 20]), 20)
    assert torch.equal(pages[-300:], small.pages)


def test_other_stream_and_graph():
    """A decode step captured once and replayed over growing lengths, on a stream of its own."""
    d, kv_heads, group = 64, 2, 4
    stream = torch.cuda.Stream()
    c, eager = (kv.Cache.empty(2, kv_heads, d, 40) for _ in range(2))
    x = torch.zeros((2, kv_heads * (group + 2), d), device=DEV)
    past, cu = ints([0, 900]), ints([0, 1, 2])
    q, k, v = x[:, :kv_heads * group], x[:, kv_heads * group:kv_heads * (group + 1)], x[:, kv_heads * (group + 1):]

    def step(cache, out):
        kv.append(cache, k, v, past, cu, 1)
        kv.attention(cache, q, past, cu, 1, weights_out=cache.weights, out=out)

    o, want = torch.zeros_like(q.contiguous()), torch.zeros_like(q.contiguous())
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        kv.attention(c, q, past, cu, 1, weights_out=c.weights.clone(), out=o)  # the stream's workspace
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            step(c, o)
        for _ in range(50):
            x.normal_()
            step(eager, want)
            graph.replay()
            past += 1
            stream.synchronize()
            assert torch.equal(o, want) and torch.equal(c.weights, eager.weights)
    assert torch.equal(c.pages, eager.pages) and torch.equal(c.scales, eager.scales)


# -------------------------------------------------------------------- evict
@pytest.mark.parametrize("width,blocks,budget,sinks,recent", [
    (1, [1, 0], 1, 0, 1), (5, [5, 2], 2, 1, 1), (40, [40, 33, 12], 12, 2, 4), (256, [255, 256], 100, 0, 1),
    (257, [257, 100], 100, 4, 8), (1024, [1024, 1000], 1023, 1, 1), (1500, [1499], 64, 32, 32),
    (4099, [4099, 4096, 5], 1000, 2, 4), (16384, [16384], 9001, 4, 16)])
@pytest.mark.parametrize("how", ["tail", "ties", "odd"])
def test_evict(width, blocks, budget, sinks, recent, how):
    print("evict", width, blocks, budget, sinks, recent, how, flush=True)
    g = np.random.default_rng(width + budget)
    heads, batch = 2, len(blocks)
    dropped = g.integers(0, 9, batch).astype(np.int32)
    tokens = np.array([max(0, 32 * (n + d) - g.integers(0, 32)) for n, d in zip(blocks, dropped)], np.int32)
    table = g.permutation(batch * heads * width).astype(np.int32).reshape(batch, heads, width)
    starts = np.sort(g.integers(0, 10 ** 6, table.shape).astype(np.int32), -1) * 32
    weights = (1 / (1.001 - g.random(table.shape))).astype(np.float32)
    if how == "ties":
        weights = g.integers(0, 3, table.shape).astype(np.float32) * np.float32(0.5)
    elif how == "odd":
        weights = g.choice(np.array([np.nan, np.inf, -np.inf, 0.0, -0.0, 1e-45, -3.0, 3.4e38], np.float32), table.shape)
    want = kv_ref.evict(table, starts, weights, tokens, dropped, budget, sinks, recent)
    dev = [torch.from_numpy(x).to(DEV) for x in (table, starts, weights, tokens, dropped)]
    got = kv.evict(*dev, budget, sinks=sinks, recent=recent)
    inputs = [x.clone() for x in dev]
    same = kv.evict(*dev, budget, sinks=sinks, recent=recent, out=(*dev[:3], torch.empty_like(dev[4])))
    torch.cuda.synchronize()
    for x, y, z in zip(got, same, want):
        assert np.array_equal(x.cpu().numpy(), z, equal_nan=z.dtype.kind == "f")
        assert np.array_equal(y.cpu().numpy(), z, equal_nan=z.dtype.kind == "f")
    assert torch.equal(inputs[4], dev[4])


def test_a_budgeted_sequence_over_many_steps():
    """Append, attend with weights, evict, swap: pages are reused and no key that is held is lost."""
    d, heads, budget, room = 64, 2, 5, 3
    c = kv.Cache.empty(1, heads, d, budget + room)
    g = torch.Generator().manual_seed(31)
    past = 0
    for step, n in enumerate([50, 1, 1, 40, 64, 1, 90, 1, 33]):
        k, v = (torch.randn((n, heads, d), generator=g).to(DEV) for _ in range(2))
        q = torch.randn((n, heads * 2, d), generator=g).to(DEV)
        p, cu = ints([past]), ints([0, n])
        kv.append(c, k, v, p, cu, n)
        before = kv_ref.Ref(c)
        o = kv.attention(c, q, p, cu, n, weights_out=c.weights)
        ref = before.attention(q.cpu().double().numpy(), [past], [0, n])
        check_attention(o, ref, "f32", d, past + n, f"step {step}")
        past += n
        table, starts, weights, dropped = kv.evict(c.table, c.starts, c.weights, ints([past]), c.dropped, budget, sinks=1,
                                                   recent=2)
        c = kv.Cache(c.pages, c.scales, table, starts, dropped, weights, head_dim=d)
        held = -(-past // 32) - int(dropped[0])
        assert held <= budget
        for h in range(heads):
            s = starts[0, h, :held].cpu().numpy()
            assert s[0] == 0 and s[-1] == (past - 1) // 32 * 32 and np.all(np.diff(s) > 0)
            assert sorted(table[0, h].tolist()) == list(range(h * (budget + room), (h + 1) * (budget + room)))
