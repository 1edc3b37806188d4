"""A feed_forward that is refused has launched nothing: hidden may be the residual itself, and a second try adds x once."""
import math

import pytest
import torch

from rocknpu_amd import hip, moe

BAD = [
    dict(top_k=0), dict(top_k=5), dict(top_k=2.0), dict(score="tanh"), dict(groups=3), dict(groups=2, top_groups=3), dict(groups=2, top_groups=1, top_k=3), dict(group_top=3),
    dict(bias=3), dict(bias="half"), dict(factor=math.nan), dict(factor=math.inf), dict(factor=1e39), dict(normalise="yes"), dict(out="narrow"), dict(out="double"), dict(out="overlapping"),
    dict(unknown=1), dict(hidden="narrow"), dict(eps="?"), dict(router="unaligned")]


def layer(device="cpu", tokens=3):
    i8, f = (lambda *s: torch.ones(s, dtype=torch.int8, device=device)), (lambda *s: torch.ones(s, device=device) / 64)
    w = moe.Experts((i8(4, 60, 128), f(4, 60)), (i8(4, 60, 128), f(4, 60)), (i8(4, 100, 64), f(4, 100)), hidden=100, ffn=60)
    return dict(x=torch.ones((tokens, 100), device=device), norm_weight=torch.ones(100, device=device), router=(i8(4, 128), f(4)), weights=w, top_k=2)


def spoiled(good, kw):
    device = good["x"].device
    bad = {**good, **kw}
    tokens = good["x"].shape[0]
    if "bias" in kw:
        bad["bias"] = torch.zeros(3 if kw["bias"] == 3 else 4, device=device, dtype=torch.float16 if kw["bias"] == "half" else torch.float32)
    if "out" in kw:
        bad["out"] = {"narrow": torch.zeros((tokens, 99), device=device), "double": torch.zeros((tokens, 100), device=device, dtype=torch.float64),
                      "overlapping": torch.zeros(4096, device=device).as_strided((tokens, 100), (99, 1))}[kw["out"]]
    if "router" in kw:
        bad["router"] = (torch.ones(520, dtype=torch.int8, device=device)[8:].view(4, 128), good["router"][1])
    if kw.get("hidden") == "narrow":
        bad["hidden"] = torch.zeros((tokens, 99), device=device)
    return bad


@pytest.mark.parametrize("kw", BAD, ids=str)
@pytest.mark.parametrize("tokens", [0, 3])
def test_checks_come_first(kw, tokens, monkeypatch):
    if tokens == 0 and kw.get("out") == "overlapping":
        pytest.skip("no rows overlap")
    good, launched = layer(tokens=tokens), []
    monkeypatch.setattr(hip, "stream_of", lambda device: (0, 0))
    monkeypatch.setattr(hip, "call_on", lambda index, function, *args: launched.append(function) or 0)
    monkeypatch.setattr(moe, "workspace_for", lambda device, nbytes: torch.zeros(nbytes, dtype=torch.uint8))
    moe.feed_forward(**good, residual=good["x"].clone())
    assert len(launched) == (4 if tokens else 1)
    launched.clear()
    with pytest.raises(Exception) as refused:
        moe.feed_forward(**spoiled(good, kw), residual=good["x"].clone())
    assert not isinstance(refused.value, AssertionError) and not launched


def test_a_missing_workspace_comes_first(monkeypatch):
    def none(device, nbytes):
        raise moe.LaunchError("under capture")

    good, launched = layer(), []
    monkeypatch.setattr(hip, "stream_of", lambda device: (0, 1 << 40))
    monkeypatch.setattr(hip, "call_on", lambda index, function, *args: launched.append(function) or 0)
    monkeypatch.setattr(moe, "workspace_for", none)
    with pytest.raises(moe.LaunchError):
        moe.feed_forward(**good, residual=good["x"].clone())
    assert not launched
    good = layer(tokens=0)
    moe.feed_forward(**good, residual=good["x"].clone())  # which needs none


def test_unaligned_weights():
    i8, f = (lambda *s: torch.zeros(s, dtype=torch.int8)), torch.zeros
    good = dict(gate=(i8(4, 60, 128), f(4, 60)), up=(i8(4, 60, 128), f(4, 60)), down=(i8(4, 100, 64), f(4, 100)))
    for name, (w8, scales) in good.items():
        moved = torch.zeros(w8.numel() + 8, dtype=torch.int8)[8:].view(w8.shape)
        with pytest.raises(ValueError, match=f"{name} has to begin"):
            moe.Experts(**{**good, name: (moved, scales)}, hidden=100, ffn=60)


def test_rows_that_overlap_are_refused_by_name():
    i8, f = (lambda *s: torch.zeros(s, dtype=torch.int8)), torch.zeros
    w = moe.Experts((i8(4, 60, 128), f(4, 60)), (i8(4, 60, 128), f(4, 60)), (i8(4, 100, 64), f(4, 100)), hidden=100, ffn=60)
    r = moe.Routing(torch.zeros((3, 2), dtype=torch.int32), f(3, 2), torch.zeros(moe.plan_words(3, 4, 2), dtype=torch.int32), 4)
    for step in (0, 99):
        with pytest.raises(ValueError, match="overlap"):
            moe.experts(w, i8(3, 128), f(3), r, out=f(400).as_strided((3, 100), (step, 1)))


@pytest.mark.gpu
@pytest.mark.parametrize("kw", BAD, ids=str)
def test_the_residual_keeps_its_bits(kw):
    good = layer("cuda")
    h = torch.randn((3, 100), generator=torch.Generator().manual_seed(1)).cuda()
    before = h.clone()
    bad = spoiled(good, kw)
    bad.setdefault("hidden", h)
    with pytest.raises(Exception):
        moe.feed_forward(**bad, residual=h)
    torch.cuda.synchronize()
    assert torch.equal(h, before)
    out, hidden = moe.feed_forward(**good, residual=h, hidden=h)
    torch.cuda.synchronize()
    assert hidden is h and torch.equal(h, before + good["x"]) and bool(out.isfinite().all())
