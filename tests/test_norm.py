"""hip.norm_a8 on the CPU: what it refuses, and its structure against the header's."""
import ctypes
import math
import shutil
import subprocess
from pathlib import Path

import pytest
import torch

from rocknpu_amd import _lib, hip

ROOT = Path(__file__).resolve().parents[1]
AT = 1 << 20  # never read: a refused call touches nothing


def struct(**kw):
    base = dict(x=AT, residual=AT, weight=AT, hidden=AT, out=AT, a8=AT, scales=AT, rows=2, k=100, k_pad=128, x_row=100,
                residual_row=100, hidden_row=100, out_row=100, type=0, weight_type=0, eps=1e-5)
    return hip._NormStruct(**{**base, **kw})


@pytest.mark.parametrize("bad", [
    dict(x=0), dict(weight=0), dict(a8=0), dict(scales=0), dict(residual=0), dict(x=AT + 2), dict(residual=AT + 2),
    dict(hidden=AT + 2), dict(out=AT + 2), dict(weight=AT + 2), dict(scales=AT + 2), dict(type=1, weight_type=1, x=AT + 1),
    dict(rows=-1), dict(rows=1 << 31), dict(k=0), dict(k=-1), dict(k=65537, k_pad=65600), dict(k_pad=99), dict(k_pad=1 << 31),
    dict(x_row=-1), dict(residual_row=-1), dict(hidden_row=-1), dict(out_row=-1), dict(hidden_row=99), dict(out_row=99),
    dict(type=3), dict(weight_type=1), dict(type=1, weight_type=2), dict(type=2, weight_type=1), dict(eps=0.0), dict(eps=-1.0),
    dict(eps=1e-31), dict(eps=math.nan), dict(eps=math.inf)], ids=str)
def test_refused(bad):
    assert _lib.load().rocknpu_hip_norm_a8(ctypes.byref(struct(**bad)), None) == -1


def test_no_rows_and_no_arguments():
    lib = _lib.load()
    assert lib.rocknpu_hip_norm_a8(None, None) == -1
    assert lib.rocknpu_hip_norm_a8(ctypes.byref(struct(rows=0, x=0, a8=0, scales=0)), None) == 0


def test_refused_in_python():
    x, w = torch.zeros((2, 8)), torch.ones(8)
    bad = [
        dict(x=x.double()), dict(x=x[0]), dict(weight=w.half()), dict(weight=w[:7]), dict(weight=torch.ones(16)[::2]),
        dict(hidden=torch.empty_like(x)), dict(residual=x.half()), dict(residual=x[:1]), dict(residual=torch.zeros((8, 2)).T),
        dict(out=x.half()), dict(out=x[:, :7]), dict(k_pad=7), dict(k_pad=1 << 31), dict(a8=torch.zeros((2, 8), dtype=torch.int8)),
        dict(a8=torch.zeros((2, 64))), dict(scales=torch.zeros(3)), dict(scales=torch.zeros(2).double()),
        dict(residual=x, hidden=x, out=x), dict(x=torch.zeros((8, 2)).T), {}]
    for kw in bad:
        a = {"x": x, "weight": w, **kw}
        with pytest.raises(ValueError):
            hip.norm_a8(a.pop("x"), a.pop("weight"), **a)


@pytest.mark.skipif(shutil.which("gcc") is None, reason="gcc not installed")
def test_struct_layout(tmp_path):
    fields = [f for f, _ in hip._NormStruct._fields_]
    src = tmp_path / "layout.c"
    src.write_text('#include <stddef.h>\n#include <stdio.h>\n#include "rocknpu_hip.h"\nint main(void) {\n'
                   + '    printf("%zu\\n", sizeof(rocknpu_norm_args));\n'
                   + "".join(f'    printf("%zu\\n", offsetof(rocknpu_norm_args, {f}));\n' for f in fields) + "    return 0;\n}\n")
    subprocess.run(["gcc", "-std=c99", f"-I{ROOT / 'include'}", str(src), "-o", str(tmp_path / "layout")], check=True)
    got = [int(v) for v in subprocess.run([str(tmp_path / "layout")], capture_output=True, text=True, check=True).stdout.split()]
    assert got == [ctypes.sizeof(hip._NormStruct)] + [getattr(hip._NormStruct, f).offset for f in fields]
