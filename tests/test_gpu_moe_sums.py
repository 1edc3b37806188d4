"""The bits of moe.experts' weighted sum: terms are multiplied (exactly) and added up in 64 bits.

An output is then off by its one rounding to f32, 2^-24 of it, and by that to a type of fewer bits; the additions' own
errors are below 2^-46 of the terms' magnitudes for the 64 choices that there are at most."""
import numpy as np
import pytest
import torch

from rocknpu_amd import moe
from tests import moe_ref
from tests.test_gpu_moe_experts import DEV, TYPES, layer, tokens_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("tokens", [1, 2, 100])
@pytest.mark.parametrize("experts,top_k", [(8, 2), (64, 8), (5, 5), (64, 64)])
@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("signs", [False, True])
def test_outputs_are_rounded_once(tokens, experts, top_k, kind, signs):
    print("experts' sums", tokens, experts, top_k, kind, signs, flush=True)
    w = layer(experts, experts, 320, 192)
    a8, scales = tokens_of(experts + 1, tokens, 320)
    g = torch.Generator().manual_seed(experts + tokens)
    r = moe.route(torch.randn((tokens, experts), generator=g).to(DEV), top_k)
    if signs:  # terms of either sign that cancel
        r.weights = torch.randn((tokens, top_k), generator=g).to(DEV)
    out = moe.experts(w, a8, scales, r, dtype=TYPES[kind])
    torch.cuda.synchronize()
    want, size = moe_ref.experts(a8, scales, r.ids.cpu().numpy(), r.weights.cpu().numpy(), w.gate, w.up, w.down, 320, 192)
    info = torch.finfo(TYPES[kind])
    own = info.eps / 2 * (1 + 2.0 ** -24) if kind != "f32" else 0.0
    off = np.abs(out.cpu().double().numpy() - want) - (2.0 ** -24 + own) * np.abs(want) - 2.0 ** -46 * size - info.smallest_normal * info.eps
    assert (off <= 0).all(), f"{(off > 0).sum()} of {off.size} outside, worst by {off.max():.3g}"
