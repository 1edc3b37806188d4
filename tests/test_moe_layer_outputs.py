"""feed_forward's out and hidden may not overlap; out may be x or the residual."""
import itertools
import random

import pytest
import torch

from rocknpu_amd import hip, moe
from tests.test_moe_refused_layers import layer


def test_what_overlaps():
    """Against the sets of bytes themselves."""
    buffer, rng = torch.zeros(400, dtype=torch.uint8), random.Random(1)
    seen = set()
    for _ in range(4000):
        def rows(count, step):
            wide = rng.randint(1, 12)
            return buffer[rng.randint(0, 150):].as_strided((count, wide), (step, 1))
        count, step = rng.randint(1, 8), rng.randint(12, 24)
        a, b = rows(count, step), rows(count, step)
        sets = [{t.data_ptr() + i * t.stride(0) + j for i, j in itertools.product(range(t.shape[0]), range(t.shape[1]))} for t in (a, b)]
        assert moe._apart(a, b) == moe._apart(b, a) == (not sets[0] & sets[1]), (a.shape, b.shape, step)
        seen.add(moe._apart(a, b))
    assert seen == {True, False}
    assert not moe._apart(buffer.as_strided((3, 10), (20, 1)), buffer[10:].as_strided((3, 10), (21, 1)))  # reach into each other
    assert moe._apart(buffer[:0].view(0, 5), buffer.view(-1, 5))


@pytest.mark.parametrize("shift", [0, 1, -1, 99, 100 * 3 - 1])
def test_refused(shift, monkeypatch):
    launched = []
    monkeypatch.setattr(hip, "stream_of", lambda device: (0, 0))
    monkeypatch.setattr(hip, "call_on", lambda index, function, *args: launched.append(function) or 0)
    monkeypatch.setattr(moe, "workspace_for", lambda device, nbytes: torch.zeros(nbytes, dtype=torch.uint8))
    good, buffer = layer(), torch.zeros(1000)
    hidden, out = buffer[300:600].view(3, 100), buffer[300 + shift:600 + shift].view(3, 100)
    with pytest.raises(ValueError, match="overlap"):
        moe.feed_forward(**good, residual=hidden, hidden=hidden, out=out)
    assert not launched
    moe.feed_forward(**good, residual=hidden, hidden=hidden, out=buffer[600:900].view(3, 100))
    assert len(launched) == 4


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [1, 50])
def test_in_place(tokens):
    good = layer("cuda", tokens)
    good["x"] = torch.randn((tokens, 100), generator=torch.Generator().manual_seed(1)).cuda()
    h = torch.randn((tokens, 100), generator=torch.Generator().manual_seed(2)).cuda()
    want, want_h = moe.feed_forward(**good, residual=h)
    x, r = good.pop("x").clone(), h.clone()
    out, hidden = moe.feed_forward(x, **good, residual=r, hidden=r, out=x)  # the sum in the residual, the output in x
    torch.cuda.synchronize()
    assert out is x and hidden is r and torch.equal(x, want) and torch.equal(r, want_h)
    wide = torch.zeros((tokens, 200), device="cuda")
    out, hidden = moe.feed_forward(h, **good, residual=h, hidden=wide[:, :100], out=wide[:, 100:])
    torch.cuda.synchronize()
    want, want_h = moe.feed_forward(h, **good, residual=h)
    assert torch.equal(wide[:, :100], want_h) and torch.equal(wide[:, 100:], want)
