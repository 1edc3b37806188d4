"""The sizes that moe.experts refuses, by name."""
import ctypes

import pytest
import torch

from rocknpu_amd import _lib, moe


def on_meta(tokens, hidden, experts=2, ffn=64):
    i8 = lambda *s: torch.empty(s, dtype=torch.int8, device="meta")  # noqa: E731
    f = lambda *s: torch.empty(s, device="meta")  # noqa: E731
    pad = (hidden + 63) // 64 * 64
    w = moe.Experts((i8(experts, ffn, pad), f(experts, ffn)), (i8(experts, ffn, pad), f(experts, ffn)), (i8(experts, hidden, 64), f(experts, hidden)), hidden=hidden, ffn=ffn)
    plan = torch.empty(moe.plan_words(tokens, experts, 1), dtype=torch.int32, device="meta")
    return w, i8(tokens, pad), f(tokens), moe.Routing(torch.empty((tokens, 1), dtype=torch.int32, device="meta"), f(tokens, 1), plan, experts)


@pytest.mark.parametrize("tokens,hidden", [(1 << 26, 64), (1 << 20, 4096), ((1 << 32) // 133120 + 1, 133120)])
def test_rows_beyond_32_bits_of_bytes(tokens, hidden):
    with pytest.raises(ValueError, match="2\\^32 bytes"):
        moe.experts(*on_meta(tokens, hidden))
    for n, status in ((tokens, -1), ((1 << 32) // hidden - 1, 0)):
        a, need = moe._ExpertsStruct(tokens=n, experts=2, top_k=1, hidden=hidden, hidden_pad=hidden, ffn=64, ffn_pad=64), ctypes.c_size_t()
        assert _lib.load().rocknpu_hip_moe_experts_workspace(ctypes.byref(a), ctypes.byref(need)) == status


def test_rows_within():
    """The next smaller number of rows passes the checks of sizes: what is missing is a GPU."""
    with pytest.raises(ValueError, match="a GPU's are wanted"):
        moe.experts(*on_meta((1 << 26) - 1, 64))
