"""moe.experts' 256 x 256 tiles in the forms that long prompts use, against the definition: whole tiles of every height,
last rounds in halves and in quarters, few row tiles and many, both stage lengths. Which forms a call runs follows
from its plan and the GPU's compute units: each test asserts that it runs those that it is there for."""
import pytest
import torch

from rocknpu_amd import moe
from tests.moe_places import forms, pad, places, tiles_of
from tests.test_gpu_moe_experts import DEV, TYPES, layer, tokens_of, verify

pytestmark = pytest.mark.gpu

# experts' rows with last tiles of 1 to 64, 65 to 128, 129 to 192 and 193 to 255 rows: 25, 40, 74 and 8 row tiles
MIXED25 = (600, 833, 1100, 300, 900, 64, 1000, 323)
MIXED40 = (1300, 1430, 1000, 1279, 1500, 1100, 1444, 299)
MIXED74 = (2561, 3100, 2000, 1390, 2203, 1836, 1950, 2600)
MIXED8 = (300, 450, 700, 180)


def routed(seed, counts, top_k):
    """Logits that send counts[e] choices to expert e, to a token's top_k different ones each, in any order of the tokens."""
    experts, rows = len(counts), sum(counts)
    tokens = rows // top_k
    assert tokens * top_k == rows and max(counts) <= tokens
    g = torch.Generator().manual_seed(seed)
    flat = torch.repeat_interleave(torch.arange(experts), torch.tensor(counts))
    chosen = flat.view(top_k, tokens)[:, torch.randperm(tokens, generator=g)]
    x = torch.randn((tokens, experts), generator=g) - 20.0
    x.scatter_(1, chosen.T.contiguous(), 2.0 * torch.rand((tokens, top_k), generator=g))
    return x.to(DEV)


# counts, top_k, hidden, ffn, and what gate and up, and down, have to run as: (parts, rows of the form)
CASES = {
    # each XCD has its own column of gate's; down is halves throughout
    "whole and halves": (MIXED25, 2, 1024, 1024, {(1, 64), (1, 128), (1, 192), (1, 256)}, {(2, 128), (2, 256)}),
    # a full round, then one in quarters; own and shared columns, a full round, then one in halves
    "rounds and their rest": (MIXED40, 2, 2304, 1024, {(1, 64), (1, 128), (1, 192), (1, 256), (4, 128)}, {(1, 256), (2, 128), (2, 256)}),
    # many row tiles over three columns and over four
    "many row tiles": (MIXED74, 2, 1024, 384, {(1, 64), (1, 128), (1, 192), (1, 256)}, {(1, 64), (1, 128), (1, 192), (1, 256), (4, 128)}),
    "quarters": (MIXED8, 1, 768, 640, {(4, 128)}, {(4, 128)}),
    # 64-byte stages, widths that end inside a tile
    "short stages, whole and halves": (MIXED25, 2, 1088, 1088, {(1, 64), (1, 128), (1, 256)}, {(2, 128), (2, 256)}),
    "short stages, many row tiles": (MIXED74, 2, 960, 320, {(1, 64), (1, 128), (1, 256)}, {(1, 64), (1, 128), (1, 256), (4, 128)}),
    "short stages, quarters": (MIXED8, 1, 320, 192, {(4, 128)}, {(4, 128)}),
    "odd widths": (MIXED25, 2, 1000, 1003, {(1, 64), (1, 128), (1, 192), (1, 256)}, {(2, 128), (2, 256)}),
    "odd widths, rounds and their rest": (MIXED40, 2, 250, 1001, {(1, 64), (1, 128), (1, 192), (1, 256), (4, 128)}, {(4, 128)}),
    "one expert": ((6000,), 1, 640, 1024, {(1, 128), (1, 256)}, {(2, 128), (2, 256)}),
    "very uneven": ((5, 4700, 0, 1, 130, 200, 64, 4700), 2, 768, 1024, {(1, 64), (1, 128), (1, 192), (1, 256), (2, 256)}, {(1, 64), (1, 256), (2, 128), (2, 256)}),
}


@pytest.mark.parametrize("name", CASES)
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_forms(name, dtype):
    counts, top_k, hidden, ffn, gate, down = CASES[name]
    print("experts' tiles", name, dtype, sum(counts), hidden, ffn, flush=True)
    x = routed(1, counts, top_k)
    tokens, experts = x.shape
    w = layer(2, experts, hidden, ffn)
    a8, scales = tokens_of(3, tokens, hidden)
    r = moe.route(x, top_k)
    assert torch.equal(r.offsets.cpu().diff(), torch.tensor(counts, dtype=torch.int32))
    row_tiles = int(r.plan[0])
    tiles = tiles_of(counts, 256)
    assert row_tiles == len(tiles)
    for gated, k, want in ((1, pad(hidden), gate), (0, pad(ffn), down)):
        tile, at = places(tokens, experts, top_k, hidden, ffn, gated, row_tiles)
        assert tile[0] == 256 and want <= forms(at, tiles, k), (gated, forms(at, tiles, k))
    out = moe.experts(w, a8, scales, r, dtype=TYPES[dtype])
    torch.cuda.synchronize()
    verify(w, a8, scales, r, out)
