"""Expert feed-forwards on the CPU: what moe.route refuses, the plan's size, and the structures against the header's."""
import ctypes
import math
import shutil
import subprocess
from pathlib import Path

import numpy as np
import pytest
import torch

from rocknpu_amd import _lib, moe
from tests import moe_ref

ROOT = Path(__file__).resolve().parents[1]
AT = 1 << 20  # never read: a refused call touches nothing


def route_struct(**kw):
    base = dict(logits=AT, bias=AT, ids=AT, weights=AT, plan=AT, tokens=5, logits_row=16, type=0, experts=16, top_k=4,
                groups=4, top_groups=2, group_top=2, score=0, normalise=1, factor=1.0)
    return moe._RouteStruct(**{**base, **kw})


@pytest.mark.parametrize("bad", [
    dict(logits=0), dict(ids=0), dict(weights=0), dict(plan=0), dict(logits=AT + 2), dict(bias=AT + 2), dict(ids=AT + 2),
    dict(weights=AT + 2), dict(plan=AT + 2), dict(type=1, logits=AT + 1), dict(type=3), dict(tokens=-1), dict(tokens=1 << 28),
    dict(tokens=1 << 62), dict(logits_row=-1), dict(experts=0), dict(experts=1025, groups=1, top_groups=1), dict(top_k=0),
    dict(top_k=17, groups=1, top_groups=1), dict(top_k=65, experts=128), dict(groups=0), dict(groups=3), dict(groups=-4),
    dict(experts=130, groups=65, top_groups=65), dict(top_groups=0), dict(top_groups=5), dict(top_k=9), dict(group_top=0),
    dict(group_top=3), dict(groups=16, top_groups=16), dict(score=2), dict(score=-1), dict(factor=math.nan), dict(factor=math.inf)], ids=str)
def test_refused_routes(bad):
    assert _lib.load().rocknpu_hip_moe_route(ctypes.byref(route_struct(**bad)), None) == -1


def test_no_arguments():
    lib, n = _lib.load(), ctypes.c_size_t()
    assert lib.rocknpu_hip_moe_route(None, None) == -1
    assert lib.rocknpu_hip_moe_plan_words(4, 8, 2, None) == -1
    for tokens, experts, top_k in ((-1, 8, 2), (1, 0, 1), (1, 1025, 1), (1, 8, 0), (1, 8, 9), (1, 128, 65), ((1 << 27) + 1, 8, 2)):
        assert lib.rocknpu_hip_moe_plan_words(tokens, experts, top_k, ctypes.byref(n)) == -1


@pytest.mark.parametrize("tokens,experts,top_k", [(0, 1, 1), (1, 1, 1), (1, 1024, 64), (7, 60, 4), (4096, 64, 8), (16384, 256, 8), (1 << 22, 64, 64)])
def test_plan_words_hold_the_public_part(tokens, experts, top_k):
    assert moe.plan_words(tokens, experts, top_k) >= moe.PLAN_HEADER + experts + 1 + tokens * top_k


def test_refused_in_python():
    x = torch.zeros((4, 16))
    for kw in (dict(logits=x.double()), dict(logits=x[0]), dict(logits=torch.zeros((16, 4)).T), dict(bias=torch.zeros(15)),
               dict(bias=torch.zeros(16).half()), dict(bias=torch.zeros(32)[::2]), dict(score="tanh"), dict(top_k=0), dict(top_k=17),
               dict(groups=3), dict(groups=0), dict(groups=4, top_groups=0), dict(groups=4, top_groups=5), dict(groups=4, top_groups=1, top_k=5),
               dict(group_top=0), dict(group_top=3), dict(groups=16, group_top=2), dict(logits=torch.zeros((4, 1025))), {}):
        a = {"logits": x, "top_k": 2, **kw}
        with pytest.raises(ValueError):
            moe.route(a.pop("logits"), a.pop("top_k"), **a)


def test_the_plain_form():
    """Cases that can be worked out by hand."""
    x = torch.tensor([[0.0, 2.0, 2.0, 1.0], [-math.inf, 0.0, -math.inf, -math.inf], [-math.inf] * 4, [0.0, math.nan, 5.0, 1.0]])
    ids, w, offsets, order = moe_ref.route(x, 2)
    assert ids.tolist() == [[1, 2], [1, -1], [-1, -1], [0, 1]]
    assert w[0].tolist() == [0.5, 0.5] and w[1].tolist() == [1.0, 0.0] and not w[2].any() and np.isnan(w[3]).all()
    assert offsets.tolist() == [0, 1, 4, 5, 5] and order.tolist() == [6, 0, 2, 7, 1, -1, -1, -1]
    # the bias turns the choice, not the weight; two groups, one open
    x = torch.log(torch.tensor([[1.0, 2.0, 3.0, 4.0]]))
    ids, w, *_ = moe_ref.route(x, 1, bias=torch.tensor([1.0, 0, 0, 0]), normalise=False)
    assert ids.tolist() == [[0]] and abs(w[0, 0] - 0.1) < 1e-7
    ids, *_ = moe_ref.route(x, 2, bias=torch.tensor([0.0, 0.5, 0, 0]), groups=2, top_groups=1, group_top=2)
    assert ids.tolist() == [[1, 0]]  # 0.1 + 0.7 against 0.3 + 0.4
    ids, w, *_ = moe_ref.route(torch.zeros((1, 2)), 1, score="sigmoid", normalise=False, factor=3.0)
    assert ids.tolist() == [[0]] and w[0, 0] == 1.5


@pytest.mark.skipif(shutil.which("gcc") is None, reason="gcc not installed")
@pytest.mark.parametrize("name,struct", [("rocknpu_moe_route_args", moe._RouteStruct), ("rocknpu_moe_experts_args", moe._ExpertsStruct)], ids=str)
def test_struct_layouts(name, struct, tmp_path):
    fields = [f for f, _ in struct._fields_]
    src = tmp_path / "layout.c"
    src.write_text('#include <stddef.h>\n#include <stdio.h>\n#include "rocknpu_moe.h"\nint main(void) {\n'
                   + f'    printf("%zu\\n", sizeof({name}));\n'
                   + "".join(f'    printf("%zu\\n", offsetof({name}, {f}));\n' for f in fields) + "    return 0;\n}\n")
    subprocess.run(["gcc", "-std=c99", f"-I{ROOT / 'include'}", str(src), "-o", str(tmp_path / "layout")], check=True)
    got = [int(v) for v in subprocess.run([str(tmp_path / "layout")], capture_output=True, text=True, check=True).stdout.split()]
    assert got == [ctypes.sizeof(struct)] + [getattr(struct, f).offset for f in fields]


def experts_struct(**kw):
    names = ("a8", "a_scales", "gate", "up", "down", "gate_scales", "up_scales", "down_scales", "ids", "weights", "plan", "out")
    base = dict.fromkeys(names, AT) | dict(tokens=5, out_row=100, experts=8, top_k=2, hidden=100, hidden_pad=128, ffn=60, ffn_pad=64, out_type=0)
    return moe._ExpertsStruct(**{**base, **kw})


@pytest.mark.parametrize("bad", [
    *(dict([(n, 0)]) for n, _ in moe._ExpertsStruct._fields_[:12]), *(dict([(n, AT + 8)]) for n in ("a8", "gate", "up", "down")),
    *(dict([(n, AT + 2)]) for n in ("a_scales", "gate_scales", "up_scales", "down_scales", "ids", "weights", "plan", "out")), dict(out_type=2, out=AT + 1),
    dict(out_type=3), dict(tokens=-1), dict(tokens=1 << 28), dict(out_row=-1), dict(out_row=99), dict(experts=0), dict(experts=1025), dict(top_k=0),
    dict(top_k=9), dict(hidden=0), dict(hidden=129), dict(hidden_pad=120), dict(hidden_pad=0), dict(hidden_pad=133184), dict(ffn=0), dict(ffn=65),
    dict(ffn_pad=100), dict(ffn_pad=133184), dict(workspace=0), dict(workspace=AT + 16), dict(short=1)], ids=str)
def test_refused_experts(bad):
    lib, need = _lib.load(), ctypes.c_size_t()
    assert lib.rocknpu_hip_moe_experts_workspace(ctypes.byref(experts_struct()), ctypes.byref(need)) == 0
    bad = dict(bad)
    ws, short = bad.pop("workspace", AT), bad.pop("short", 0)
    assert lib.rocknpu_hip_moe_experts(ctypes.byref(experts_struct(**bad)), ws, need.value - short, None) == -1


def test_experts_without_tokens_or_arguments():
    lib, need = _lib.load(), ctypes.c_size_t()
    assert lib.rocknpu_hip_moe_experts(None, None, 0, None) == -1
    assert lib.rocknpu_hip_moe_experts_workspace(None, ctypes.byref(need)) == -1
    assert lib.rocknpu_hip_moe_experts_workspace(ctypes.byref(experts_struct()), None) == -1
    assert lib.rocknpu_hip_moe_experts(ctypes.byref(experts_struct(tokens=0, a8=0, a_scales=0, out=0)), None, 0, None) == 0


def test_refused_experts_in_python():
    i8 = lambda *s: torch.zeros(s, dtype=torch.int8)  # noqa: E731
    f = torch.zeros
    good = dict(gate=(i8(4, 60, 128), f(4, 60)), up=(i8(4, 60, 128), f(4, 60)), down=(i8(4, 100, 64), f(4, 100)), hidden=100, ffn=60)
    w = moe.Experts(**good)
    for kw in (dict(gate=(i8(60, 128), f(60))), dict(gate=(i8(4, 60, 120), f(4, 60))), dict(up=(i8(4, 61, 128), f(4, 61))), dict(up=(i8(4, 60, 192), f(4, 60))),
               dict(up=(f(4, 60, 128), f(4, 60))), dict(up=(i8(4, 60, 128), f(4, 60).double())), dict(up=(i8(4, 60, 128), f(240))), dict(down=(i8(4, 100, 50), f(4, 100))),
               dict(down=(i8(4, 101, 64), f(4, 101))), dict(hidden=0), dict(hidden=129), dict(ffn=0), dict(ffn=59), dict(gate=(i8(1025, 1, 64), f(1025, 1)), ffn=1, hidden=1),
               dict(gate=(i8(4, 128, 60).transpose(1, 2), f(4, 60)))):
        with pytest.raises(ValueError):
            moe.Experts(**{**good, **kw})
    r = moe.Routing(torch.zeros((3, 2), dtype=torch.int32), f(3, 2), torch.zeros(100, dtype=torch.int32), 4)
    args = dict(weights=w, a8=i8(3, 128), a_scales=f(3), routing=r)
    for kw in (dict(a8=i8(2, 128)), dict(a8=i8(3, 64)), dict(a8=f(3, 128)), dict(a8=i8(128, 3).T), dict(a_scales=f(2)), dict(a_scales=f(3).double()),
               dict(routing=moe.Routing(r.ids, r.weights, r.plan, 5)), dict(dtype=torch.float64), dict(out=f(3, 99)), dict(out=f(3, 100).double()),
               dict(out=f(100, 3).T), {}):
        a = {**args, **kw}
        with pytest.raises(ValueError):
            moe.experts(a.pop("weights"), a.pop("a8"), a.pop("a_scales"), a.pop("routing"), **a)


def test_experts_keep_their_tensors():
    i8, f = (lambda *s: torch.zeros(s, dtype=torch.int8)), torch.zeros
    w = moe.Experts((i8(2, 3, 64), f(2, 3)), (i8(2, 3, 64), f(2, 3)), (i8(2, 5, 64), f(2, 5)), hidden=5, ffn=3)
    for name in ("gate", "up", "down", "experts", "hidden", "ffn", "device", "pointers"):
        with pytest.raises(AttributeError):
            setattr(w, name, None)


def test_refused_layers():
    i8, f = (lambda *s: torch.zeros(s, dtype=torch.int8)), torch.zeros
    w = moe.Experts((i8(4, 60, 128), f(4, 60)), (i8(4, 60, 128), f(4, 60)), (i8(4, 100, 64), f(4, 100)), hidden=100, ffn=60)
    good = dict(x=f(3, 100), norm_weight=f(100), router=(i8(4, 128), f(4)), weights=w, top_k=2)
    for kw, what in ((dict(router=(f(4, 128), f(4))), "router"), (dict(router=(i8(4, 128), f(4).double())), "router's scales"), (dict(router=(i8(3, 128), f(3))), "router"),
                     (dict(router=(i8(128, 4).T, f(4))), "router"), (dict(router=(i8(4, 128), f(3))), "router's scales"), (dict(x=f(3, 128)), "x has"), (dict(x=f(100)), "x has")):
        with pytest.raises(ValueError, match=what):
            moe.feed_forward(**{**good, **kw})


@pytest.mark.parametrize("kw,what", [(dict(ids=torch.zeros((3, 2), dtype=torch.int64)), "ids"), (dict(weights=torch.zeros((3, 2)).half()), "weights"),
                                     (dict(weights=torch.zeros((2, 3)).T), "weights"), (dict(plan=torch.zeros(10, dtype=torch.int32)), "plan"), (dict(weights=torch.zeros(3)), "weights")])
def test_refused_routings(kw, what):
    i8, f = (lambda *s: torch.zeros(s, dtype=torch.int8)), torch.zeros
    w = moe.Experts((i8(4, 60, 128), f(4, 60)), (i8(4, 60, 128), f(4, 60)), (i8(4, 100, 64), f(4, 100)), hidden=100, ffn=60)
    good = dict(ids=torch.zeros((3, 2), dtype=torch.int32), weights=f(3, 2), plan=torch.zeros(moe.plan_words(3, 4, 2), dtype=torch.int32))
    with pytest.raises(ValueError, match=what):
        moe.experts(w, i8(3, 128), f(3), moe.Routing(**{**good, **kw}, experts=4))
    with pytest.raises(ValueError, match="a GPU's are wanted"):
        moe.experts(w, i8(3, 128), f(3), moe.Routing(**good, experts=4))
