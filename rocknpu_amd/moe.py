"""A feed-forward made of experts (include/rocknpu_moe.h) on device tensors.

    a8, a_scales, hidden = hip.norm_a8(x, norm_weight, residual=hidden)
    routing = moe.route(logits, top_k)                  # which experts a token goes to
    out = moe.experts(weights, a8, a_scales, routing)   # the chosen experts' products, weighted and summed

Calls enqueue on the tensors' device's current torch stream and return
immediately; they read nothing on the host, so a step can be captured in a HIP
graph.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib, hip
from .hip import TYPES, LaunchError  # noqa: F401

SCORES = {"softmax": 0, "sigmoid": 1}
MAX_EXPERTS = 1024
MAX_TOP_K = 64
MAX_GROUPS = 64
MAX_ROWS = 1 << 28
PLAN_HEADER = 16

_vp = ctypes.c_void_p
_i32 = ctypes.c_int32
_i64 = ctypes.c_int64


class _RouteStruct(ctypes.Structure):
    """rocknpu_moe_route_args (include/rocknpu_moe.h)."""

    _fields_ = [("logits", _vp), ("bias", _vp), ("ids", _vp), ("weights", _vp), ("plan", _vp), ("tokens", _i64),
                ("logits_row", _i64), ("type", ctypes.c_uint32), ("experts", _i32), ("top_k", _i32), ("groups", _i32),
                ("top_groups", _i32), ("group_top", _i32), ("score", _i32), ("normalise", _i32), ("factor", ctypes.c_float)]


class Routing:
    """What route returns: `ids` int32 and `weights` f32 [tokens, top_k], and the
    plan of the experts' products, of which `offsets` int32 [experts + 1] and
    `order` int32 [tokens * top_k] are views: order[offsets[e]:offsets[e + 1]]
    are the numbers token * top_k + place of the choices that fell on expert e,
    ascending; behind offsets[experts] it is -1."""

    __slots__ = ("ids", "weights", "plan", "experts")

    def __init__(self, ids: torch.Tensor, weights: torch.Tensor, plan: torch.Tensor, experts: int):
        self.ids, self.weights, self.plan, self.experts = ids, weights, plan, experts

    @property
    def offsets(self) -> torch.Tensor:
        return self.plan[PLAN_HEADER:PLAN_HEADER + self.experts + 1]

    @property
    def order(self) -> torch.Tensor:
        at = PLAN_HEADER + self.experts + 1
        return self.plan[at:at + self.ids.numel()]


_plan_words: dict[tuple[int, int, int], int] = {}


def plan_words(tokens: int, experts: int, top_k: int) -> int:
    """Words of a routing's plan; refuses sizes that the kernels do not take."""
    key = (tokens, experts, top_k)
    n = _plan_words.get(key)
    if n is None:
        if not (1 <= experts <= MAX_EXPERTS and 1 <= top_k <= min(experts, MAX_TOP_K) and 0 <= tokens * top_k <= MAX_ROWS):
            raise ValueError(f"{top_k} of {experts} experts for {tokens} tokens: at most {MAX_TOP_K} of at most "
                             f"{MAX_EXPERTS}, and at most {MAX_ROWS} choices")
        got = ctypes.c_size_t()
        hip._check(_lib.load().rocknpu_hip_moe_plan_words(tokens, experts, top_k, ctypes.addressof(got)), "moe_plan_words")
        if len(_plan_words) >= 4096:
            _plan_words.clear()
        n = _plan_words[key] = got.value
    return n


def route(logits: torch.Tensor, top_k: int, *, score: str = "softmax", bias: torch.Tensor | None = None, groups: int = 1,
          top_groups: int | None = None, group_top: int = 1, normalise: bool = True, factor: float = 1.0) -> Routing:
    """Chooses top_k experts for every row of logits [tokens, experts] (f32, f16
    or bf16). Experts are ranked by score ("softmax" of the row, or "sigmoid" of
    each) plus `bias` (f32 [experts]), equal ones by index. With `groups` only
    the experts of the `top_groups` groups of highest rank can be chosen, by the
    group's best (group_top=1) or the sum of its two best (group_top=2). Weights
    are the scores without the bias, divided by their sum with `normalise`,
    times `factor`. A logit of -inf is an expert that cannot be chosen: where
    less than top_k can, the last ids are -1 and their weights 0."""
    if logits.dim() != 2 or logits.dtype not in TYPES:
        raise ValueError(f"logits have to be float32, float16 or bfloat16 [tokens, experts], not {logits.dtype} {tuple(logits.shape)}")
    tokens, experts = logits.shape
    at = logits.device
    if logits.stride(1) != 1 and experts > 1:
        raise ValueError("logits have to be contiguous in their last dimension")
    if bias is not None and (bias.shape != (experts,) or bias.dtype is not torch.float32 or bias.device != at or not bias.is_contiguous()):
        raise ValueError(f"bias has to be contiguous float32 [{experts}] on {at}")
    if score not in SCORES:
        raise ValueError(f"score {score!r} is not one of {tuple(SCORES)}")
    words = plan_words(tokens, experts, top_k)
    top_groups = groups if top_groups is None else top_groups
    if not (1 <= groups <= min(MAX_GROUPS, experts) and experts % groups == 0 and 1 <= top_groups <= groups
            and top_groups * (experts // groups) >= top_k):
        raise ValueError(f"{top_groups} of {groups} groups of {experts} experts, top_k {top_k}: groups have to be equal, at "
                         f"most {MAX_GROUPS}, and the chosen ones have to hold top_k experts")
    if not 1 <= group_top <= min(2, experts // groups):
        raise ValueError(f"group_top {group_top} is neither 1 nor 2, or more than a group's experts")
    ids = torch.empty((tokens, top_k), dtype=torch.int32, device=at)
    weights = torch.empty((tokens, top_k), dtype=torch.float32, device=at)
    plan = torch.empty(words, dtype=torch.int32, device=at)
    args = _RouteStruct(logits.data_ptr(), None if bias is None else bias.data_ptr(), ids.data_ptr(), weights.data_ptr(),
                        plan.data_ptr(), tokens, hip._ld(logits), TYPES[logits.dtype], experts, top_k, groups, top_groups,
                        group_top, SCORES[score], normalise, factor)
    with hip.on_device(at) as stream:
        hip._check(_lib.load().rocknpu_hip_moe_route(ctypes.addressof(args), stream), "moe_route")
    return Routing(ids, weights, plan, experts)
