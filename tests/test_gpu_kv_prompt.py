"""Attention launches of many rows (more than four 16-row tiles a compute unit, or long contexts under many rows),
which the kernel for prompts serves, against the 64-bit definition. Bounds are test_gpu_kv's: per row, twice a score's
error, 2^-21 for the exponential and 2^-10 for weights of 16-bit calls, then the f32 sum and the output's rounding: half
an ulp, which for f16 results below 2^-14 is 2^-25 (the exact result rounded to f16 is that far off)."""
import numpy as np
import pytest
import torch

from rocknpu_amd import kv
from tests import kv_ref
from tests.test_gpu_kv import DEV, TYPES, ULP, ints, offsets, random_cache

pytestmark = pytest.mark.gpu

BATCH, KV_HEADS, GROUP = 33, 4, 4


def lengths(seed, lo=0, hi=260, most=41):
    """Ragged sequences: some without new rows, some without old ones, one with `most` new."""
    g = np.random.default_rng(seed)
    past, new = g.integers(lo, hi, BATCH).tolist(), g.integers(0, most + 1, BATCH).tolist()
    past[3], new[5], new[6], new[7] = 0, most, 0, 1
    return past, new


def check_attention(got, ref, kind, d, keys):
    out, mag, big, _ = ref
    got = got.cpu().double().numpy()
    assert np.array_equal(np.isnan(got), np.isnan(out))
    score = big[..., None] * ((2.0 ** -22 if kind == "f32" else 0.0) + (np.sqrt(d) + 8) * 2.0 ** -24)
    weight = 2 * score + 2.0 ** -21 + (0.0 if kind == "f32" else 2.0 ** -10)
    rounding = np.maximum(ULP[kind] * np.abs(out), 2.0 ** -25 if kind == "f16" else 1e-30)
    bound = mag * (weight + (np.sqrt(keys) + 8) * 2.0 ** -24) + rounding
    bad = np.nan_to_num(np.abs(got - out) - bound) > 0
    assert not bad.any(), f"{bad.sum()} of {bad.size} outside, worst {np.nanmax(np.abs(got - out) / bound):.3g} of the bound"


def run_attention(seed, kind, d, kv_heads, group, past, new, lost=None, cache=None, **kw):
    lost = lost or [0] * len(past)
    print(kind, d, kv_heads, group, past, new, lost, {k: v for k, v in kw.items() if k != "slopes"}, flush=True)
    blocks = max(-(-(p + n) // 32) - e for p, n, e in zip(past, new, lost)) + 2
    c = cache or random_cache(seed, len(past), kv_heads, d, max(blocks, 1), lost, past)
    cu = offsets(new)
    g = torch.Generator().manual_seed(seed + 1)
    q = torch.randn((cu[-1], kv_heads * group, d), generator=g).to(TYPES[kind])
    dev = {k: ints(v) if k == "prefix" else v.to(DEV) if k == "slopes" else v for k, v in kw.items()}
    o = kv.attention(c, q.to(DEV), ints(past), ints(cu), max(new), **dev)
    torch.cuda.synchronize()
    plain = {k: v.numpy() if k == "slopes" else v for k, v in kw.items()}
    ref = kv_ref.Ref(c).attention(q.double().numpy(), past, cu, **plain)
    check_attention(o, ref, kind, d, max(p + n for p, n in zip(past, new)))


def many_tiles(new, group=GROUP):
    """Past four 16-row tiles a compute unit."""
    cus = torch.cuda.get_device_properties(0).multi_processor_count
    return -(-max(new) * group // 16) * BATCH * KV_HEADS > 4 * cus


OPTIONS = {
    "plain": {},
    "window": dict(window=33),
    "narrow": dict(window=1),
    "prefix": dict(window=70, prefix=[(37 * b) % 200 for b in range(BATCH)]),
    "ahead": dict(prefix=[(53 * b) % 320 for b in range(BATCH)]),
    "capped": dict(softcap=5.0),
    "capped-window": dict(softcap=30.0, window=64),
    "bias": dict(slopes=2.0 ** (-8.0 * torch.arange(1, KV_HEADS * GROUP + 1) / 16)),
    "bias-window": dict(slopes=-0.01 * torch.arange(KV_HEADS * GROUP, dtype=torch.float32), window=90),
    "bias-capped": dict(slopes=2.0 ** (-8.0 * torch.arange(1, KV_HEADS * GROUP + 1) / 16), softcap=20.0),
    "negative": dict(scale=-0.1),
    "whole": dict(causal=False),
}


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("d", kv.HEAD_DIMS)
@pytest.mark.parametrize("option", list(OPTIONS))
def test_ragged_pieces(kind, d, option):
    past, new = lengths(1)
    assert many_tiles(new)
    run_attention(41, kind, d, KV_HEADS, GROUP, past, new, **OPTIONS[option])


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("option", ["plain", "prefix", "bias", "bias-window", "whole"])
def test_evicted_blocks(kind, option):
    past, new = lengths(2, 64)
    lost = [min(p // 32, b % 6) for b, p in enumerate(past)]
    lost[9] = past[9] // 32
    run_attention(42, kind, 64, KV_HEADS, GROUP, past, new, lost=lost, **OPTIONS[option])


@pytest.mark.parametrize("group", [1, 3, 7])
def test_heads_that_do_not_divide_a_tile(group):
    past, new = lengths(3, most=180 // group)
    run_attention(43, "f32", 64, KV_HEADS, group, past, new, window=100)


def test_heavy_tokens_with_zero_codes():
    """A row whose greatest weight meets zero codes gets the others' result to its full bits, however light they are."""
    for kind in ("f16", "bf16", "f32"):
        past, new = [100] * BATCH, [41] * BATCH
        assert many_tiles(new)
        c = random_cache(50, BATCH, KV_HEADS, 64, 6)
        pages = c.table[:, :, 1].flatten().long()  # positions 32..63: heavy keys, and values of zero
        c.pages[pages, :32 * 64] = 127
        c.pages[pages, 32 * 64:] = 0
        c.scales[pages, 0] = 0.05
        cu = offsets(new)
        q = torch.rand((cu[-1], KV_HEADS * GROUP, 64), generator=torch.Generator().manual_seed(51)).to(TYPES[kind]) * 0.8
        scale = 0.125
        o = kv.attention(c, q.to(DEV), ints(past), ints(cu), 41, scale=scale)
        check_attention(o, kv_ref.Ref(c).attention(q.double().numpy(), past, cu, scale=scale), kind, 64, 141)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("option", [{}, dict(window=3000), dict(softcap=20.0), dict(slopes=2.0 ** (-torch.arange(1, 33) / 4))],
                         ids=["plain", "window", "capped", "bias"])
def test_long_contexts_are_shared_out(kind, option):
    """64 rows of 32 heads over 16000 tokens: parts of a context on several workgroups, joined."""
    run_attention(44, kind, 128, 8, 4, [16000], [64], **option)
    run_attention(45, kind, 128, 8, 4, [6000, 31, 4500], [33, 64, 0], lost=[100, 0, 7], **option)


@pytest.mark.parametrize("kind", list(TYPES))
def test_values_not_finite_and_pages_out_of_range(kind):
    past, new = lengths(4)
    for what in ("scale", "page"):
        c = random_cache(46, BATCH, KV_HEADS, 64, 12)
        table = c.table.cpu().numpy()
        for b, h, i, w in ((0, 0, 2, 0), (5, 3, 0, 1), (8, 1, 3, 0), (11, 2, 1, 1)):
            if what == "scale":
                c.scales[table[b, h, i], w] = float("nan") if b % 2 else float("inf")
            else:
                c.table[b, h, i] = -1 if b % 2 else 2 ** 31 - 1
        if what == "scale":
            run_attention(47, kind, 64, KV_HEADS, GROUP, past, new, cache=c, window=64)
            run_attention(47, kind, 64, KV_HEADS, GROUP, past, new, cache=c)
            continue
        cu = offsets(new)
        q = torch.randn((cu[-1], KV_HEADS * GROUP, 64), device=DEV).to(TYPES[kind])
        o = kv.attention(c, q, ints(past), ints(cu), max(new)).cpu()
        for b in range(BATCH):
            for head in range(KV_HEADS * GROUP):
                for i in range(cu[b], cu[b + 1]):
                    last = (past[b] + i - cu[b]) // 32
                    sees = any(b == x and head // GROUP == h and last >= at
                               for x, h, at in ((0, 0, 2), (5, 3, 0), (8, 1, 3), (11, 2, 1)))
                    assert bool(torch.isnan(o[i, head]).any()) == sees


def test_strides_and_repeated_calls():
    past, new = lengths(5)
    cu, heads, d = offsets(new), KV_HEADS * GROUP, 64
    c = random_cache(48, BATCH, KV_HEADS, d, 12)
    for kind, pad in (("f32", 8), ("f32", 3), ("bf16", 8), ("bf16", 5)):
        fused = torch.randn((cu[-1], 2 * heads * d + pad), device=DEV).to(TYPES[kind])
        q = fused[:, pad:pad + heads * d].unflatten(1, (heads, d))
        want = kv.attention(c, q.contiguous(), ints(past), ints(cu), max(new))
        out = torch.zeros((cu[-1], heads, 2 * d + pad), device=DEV, dtype=TYPES[kind])
        for _ in range(2):
            kv.attention(c, q, ints(past), ints(cu), max(new), out=out[:, :, :d])
            assert torch.equal(out[:, :, :d], want) and not out[:, :, d:].any()
        ref = kv_ref.Ref(c).attention(q.double().cpu().numpy(), past, cu)
        check_attention(want, ref, kind, d, max(p + n for p, n in zip(past, new)))


def test_a_workspace_may_hold_anything():
    """Splits, their states and the sequences' parts are written before they are read, also where some have no rows."""
    for new, heads in (([1, 0, 1, 1], 8), ([64, 0, 3, 33], 32)):
        c = random_cache(52, 4, 8, 128, 130)
        past, cu = [4000, 4000, 70, 2050], offsets(new)
        q = torch.randn((cu[-1], heads, 128), device=DEV)
        weigh = max(new) == 1
        results = []
        for fill in (0, 0x7f, 0xff):
            ws = torch.full((1 << 28,), fill, dtype=torch.uint8, device=DEV)
            wo = torch.empty_like(c.weights) if weigh else None
            results.append((kv.attention(c, q, ints(past), ints(cu), max(new), max_tokens=4100, workspace=ws, weights_out=wo), wo))
        for o, wo in results[1:]:
            assert torch.equal(o, results[0][0]) and (wo is None or torch.equal(wo, results[0][1]))
        assert torch.isfinite(results[0][0]).all()
