"""How many bits attention keeps, against the 64-bit definition, through both kernels (one new token: streaming; 41 of
each of 33 sequences: prompts). With T the largest sum of |terms| of a seen score, D dims and N keys:
  - a score's error is at most T (sqrt(D) + 8) 2^-24 for the f32 sum and the operations behind it, and T 2^-22 more in f32
    calls for q as two f16 (f16 and bf16 rows are held exactly);
  - a weight has that error twice, 2^-21 for the exponential, and 2^-16 in 16-bit calls, whose weights have 16 bits;
  - the output's f32 sum adds (sqrt(N) + 8) 2^-24, and its rounding half an ulp (f16 below 2^-14: 2^-25)."""
import numpy as np
import pytest
import torch

from rocknpu_amd import kv
from tests import kv_ref
from tests.test_gpu_kv import DEV, TYPES, ULP, ints, offsets, random_cache
from tests.test_gpu_kv_prompt import BATCH, GROUP, KV_HEADS, many_tiles

pytestmark = pytest.mark.gpu
HEADS = KV_HEADS * GROUP


def check(c, q, past, new, kind, d, more=0.0, **kw):
    """`more`: what a score's error may be beyond its sum's, as the test says."""
    cu, keys = offsets(new), max(p + n for p, n in zip(past, new))
    dev = {k: v.to(DEV) if k == "slopes" else v for k, v in kw.items()}
    got = kv.attention(c, q.to(DEV), ints(past), ints(cu), max(new), **dev).cpu().double().numpy()
    plain = {k: v.numpy() if k == "slopes" else v for k, v in kw.items()}
    out, mag, big, _ = kv_ref.Ref(c).attention(q.double().numpy(), past, cu, **plain)
    score = big[..., None] * ((2.0 ** -22 if kind == "f32" else 0.0) + (np.sqrt(d) + 8) * 2.0 ** -24) + more
    weight = 2 * score + 2.0 ** -21 + (0.0 if kind == "f32" else 2.0 ** -16)
    rounding = np.maximum(ULP[kind] * np.abs(out), 2.0 ** -25 if kind == "f16" else 1e-30)
    bound = mag * (weight + (np.sqrt(keys) + 8) * 2.0 ** -24) + rounding
    off = np.abs(got - out) / bound
    assert np.isfinite(got).all()
    print(f"worst {off.max():.3g} of the bound", flush=True)
    assert off.max() <= 1, f"{(off > 1).sum()} of {off.size} outside, worst {off.max():.3g} of the bound"


def case(seed, d, new):
    past, news = [100] * BATCH, [new] * BATCH
    assert new <= 8 or many_tiles(news)
    c = random_cache(seed, BATCH, KV_HEADS, d, 6)
    g = torch.Generator().manual_seed(seed + 1)
    return c, torch.randn((BATCH * new, HEADS, d), generator=g), past, news


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("new", [1, 41])
@pytest.mark.parametrize("d", [64, 128])
def test_biased_queries_and_a_strong_key_channel(kind, new, d):
    """One channel takes the codes' range and the queries do not look at it: the others' codes are small beside it."""
    c, q, past, news = case(100, d, new)
    g = torch.Generator().manual_seed(102)
    for t in range(32):
        small = torch.randint(-3, 4, (c.pages.shape[0], d), generator=g, dtype=torch.int8)
        small[:, 5] = 127
        for j in range(d // 64):
            at = (j * 32 + t) * 64
            c.pages[:, at:at + 64] = small[:, 64 * j:64 * j + 64].to(DEV)
    q = q + 10
    q[..., 5] = 0
    c.scales[:, 0] = 0.05
    check(c, q.to(TYPES[kind]), past, news, kind, d)


@pytest.mark.parametrize("new", [8, 41])
def test_outputs_do_not_lean(new):
    """The outputs' mean relative error: rounding to f16 leaves 2^-12 over the square root of their number at most, six of
    that are allowed, and 2^-20 for what the weights' 16 bits may leave in the mean when they are rounded, not cut off
    (cut off they leave 2^-17)."""
    c, q, past, news = case(104, 64, new)
    c.pages[:, 32 * 64:] = torch.randint(60, 128, (c.pages.shape[0], 32 * 64), dtype=torch.int8, device=DEV)
    q = q.to(torch.float16)
    cu = offsets(news)
    got = kv.attention(c, q.to(DEV), ints(past), ints(cu), new).cpu().double().numpy()
    out = kv_ref.Ref(c).attention(q.double().numpy(), past, cu)[0]
    mean = float(((got - out) / out).mean())
    print(f"mean {mean:.3g}", flush=True)
    assert abs(mean) <= 2.0 ** -20 + 6 * 2.0 ** -12 / np.sqrt(out.size)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("new", [1, 41])
@pytest.mark.parametrize("cap", [0.02, 1.0, 50.0, 1e4, 1e6, 1e20, 3e38])
def test_caps_of_any_size(cap, new, kind):
    """A capped score has the bits that it has without a cap, however large the cap."""
    c, q, past, news = case(106, 64, new)
    check(c, q.to(TYPES[kind]), past, news, kind, 64, softcap=cap)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("new", [1, 41])
def test_capped_scores_from_zero_to_far_beyond_the_cap(new, kind):
    c, q, past, news = case(108, 64, new)
    q = q * 2.0 ** torch.arange(-8, 8).view(1, HEADS, 1)
    check(c, q.to(TYPES[kind]), past, news, kind, 64, softcap=2.0)
