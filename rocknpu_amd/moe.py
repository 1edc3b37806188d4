"""A feed-forward made of experts (include/rocknpu_moe.h) on device tensors.

    a8, a_scales, hidden = hip.norm_a8(x, norm_weight, residual=hidden)
    logits = hip.gemm_w8a8(a8, a_scales, *router)
    routing = moe.route(logits, top_k)                  # which experts a token goes to
    out = moe.experts(weights, a8, a_scales, routing)   # the chosen experts' products, weighted and summed

or, the four together, feed_forward.

Calls enqueue on the tensors' device's current torch stream and return
immediately; they read nothing on the host, so a step can be captured in a HIP
graph.
"""
from __future__ import annotations

import ctypes
import struct

import torch

from . import _lib, hip
from .hip import TYPES, LaunchError  # noqa: F401

SCORES = {"softmax": 0, "sigmoid": 1}
MAX_EXPERTS = 1024
MAX_TOP_K = 64
MAX_GROUPS = 64
MAX_ROWS = 1 << 28
PLAN_HEADER = 16
_F32_MAX = torch.finfo(torch.float32).max

_vp = ctypes.c_void_p
_i32 = ctypes.c_int32
_i64 = ctypes.c_int64


class _RouteStruct(ctypes.Structure):
    """rocknpu_moe_route_args (include/rocknpu_moe.h)."""

    _fields_ = [("logits", _vp), ("bias", _vp), ("ids", _vp), ("weights", _vp), ("plan", _vp), ("tokens", _i64),
                ("logits_row", _i64), ("type", ctypes.c_uint32), ("experts", _i32), ("top_k", _i32), ("groups", _i32),
                ("top_groups", _i32), ("group_top", _i32), ("score", _i32), ("normalise", _i32), ("factor", ctypes.c_float)]


class _ExpertsStruct(ctypes.Structure):
    """rocknpu_moe_experts_args (include/rocknpu_moe.h)."""

    _fields_ = ([(n, _vp) for n in ("a8", "a_scales", "gate", "up", "down", "gate_scales", "up_scales", "down_scales",
                                    "ids", "weights", "plan", "out")]
                + [("tokens", _i64), ("out_row", _i64)]
                + [(n, _i32) for n in ("experts", "top_k", "hidden", "hidden_pad", "ffn", "ffn_pad")]
                + [("out_type", ctypes.c_uint32)])


# The same bytes without an object, as hip's.
_pack_route = struct.Struct("@5P2qI7if0q").pack
_pack_experts = struct.Struct("@12P2q6iI0q").pack


class Routing:
    """What route returns: `ids` int32 and `weights` f32 [tokens, top_k], and the
    plan of the experts' products, of which `offsets` int32 [experts + 1] and
    `order` int32 [tokens * top_k] are views: order[offsets[e]:offsets[e + 1]]
    are the numbers token * top_k + place of the choices that fell on expert e,
    ascending; behind offsets[experts] it is -1. The plan belongs to its ids; other
    weights may be put in place of these."""

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
    routing, index, stream, args = _route_call(logits, top_k, score, bias, groups, top_groups, group_top, normalise, factor)
    hip._check(hip.call_on(index, _lib.load().rocknpu_hip_moe_route, args, stream), "moe_route")
    return routing


# What a call checks, allocates and packs, apart from its launches: feed_forward does
# all of that for its calls before the first one writes anything.
def _route_call(logits, top_k, score="softmax", bias=None, groups=1, top_groups=None, group_top=1, normalise=True, factor=1.0):
    """route's result, still to be filled, and what the library's call for it takes: device, stream, arguments."""
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
    words = _plan_words.get((tokens, experts, top_k)) or plan_words(tokens, experts, top_k)
    top_groups = groups if top_groups is None else top_groups
    if not (1 <= groups <= min(MAX_GROUPS, experts) and experts % groups == 0 and 1 <= top_groups <= groups
            and top_groups * (experts // groups) >= top_k):
        raise ValueError(f"{top_groups} of {groups} groups of {experts} experts, top_k {top_k}: groups have to be equal, at "
                         f"most {MAX_GROUPS}, and the chosen ones have to hold top_k experts")
    if not 1 <= group_top <= min(2, experts // groups):
        raise ValueError(f"group_top {group_top} is neither 1 nor 2, or more than a group's experts")
    if not abs(factor) <= _F32_MAX:
        raise ValueError(f"factor {factor} is not a finite float32")
    ids = logits.new_empty((tokens, top_k), dtype=torch.int32)
    weights = logits.new_empty((tokens, top_k), dtype=torch.float32)
    plan = logits.new_empty((words,), dtype=torch.int32)
    args = _pack_route(logits.data_ptr(), 0 if bias is None else bias.data_ptr(), ids.data_ptr(), weights.data_ptr(),
                       plan.data_ptr(), tokens, logits.stride(0) if tokens > 1 else experts, TYPES[logits.dtype], experts, top_k,
                       groups, top_groups, group_top, SCORES[score], normalise, factor)
    return Routing(ids, weights, plan, experts), *hip.stream_of(at), args


def _pair(pair, shape, what, device):
    """A W8 stack and its scales, as hip.repack_w8 gives them for a stack of matrices."""
    w8, scales = pair
    if w8.dtype is not torch.int8 or tuple(w8.shape) != shape or not w8.is_contiguous() or w8.device != device:
        raise ValueError(f"{what} has to be contiguous int8 {shape} on {device}, not {w8.dtype} {tuple(w8.shape)} on {w8.device}")
    if scales.dtype is not torch.float32 or tuple(scales.shape) != shape[:-1] or not scales.is_contiguous() or scales.device != device:
        raise ValueError(f"{what}'s scales have to be contiguous float32 {shape[:-1]} on {device}")
    if w8.data_ptr() % 16:
        raise ValueError(f"{what} has to begin on 16 bytes")
    return w8, scales


class Experts:
    """A layer's experts: `gate`, `up` and `down`, each a pair of W8 int8 and
    scales f32: gate and up [experts, ffn, hidden_pad] and [experts, ffn], down
    [experts, hidden, ffn_pad] and [experts, hidden], the pads zeros up to a
    multiple of 64. hip.repack_w8 makes them of a stack of GGUF matrices, taken as
    one matrix of experts * ffn (or hidden) rows. The tensors are used in place
    and kept alive by the object."""

    def __setattr__(self, name, value):
        if name in self.__dict__:
            raise AttributeError(f"the kernels use the {name} that the object was made with: make a new Experts")
        object.__setattr__(self, name, value)

    def __init__(self, gate, up, down, *, hidden: int, ffn: int):
        experts = gate[0].shape[0] if gate[0].dim() == 3 else 0
        if not 1 <= experts <= MAX_EXPERTS or hidden < 1 or ffn < 1:
            raise ValueError(f"{experts} experts of {hidden} x {ffn}: gate has to be [experts, ffn, hidden_pad], of 1 to {MAX_EXPERTS} experts")
        self.hidden_pad, self.ffn_pad = gate[0].shape[2], down[0].shape[-1]
        for what, n, pad in (("hidden", hidden, self.hidden_pad), ("ffn", ffn, self.ffn_pad)):
            if pad < n or pad % 64 or pad > hip.MAX_K:
                raise ValueError(f"{what} {n} in rows of {pad}: a multiple of 64 from {n} to {hip.MAX_K} is wanted")
        self.device = gate[0].device
        self.gate = _pair(gate, (experts, ffn, self.hidden_pad), "gate", self.device)
        self.up = _pair(up, (experts, ffn, self.hidden_pad), "up", self.device)
        self.down = _pair(down, (experts, hidden, self.ffn_pad), "down", self.device)
        self.experts, self.hidden, self.ffn = experts, hidden, ffn
        self.pointers = tuple(pair[i].data_ptr() for i in (0, 1) for pair in (self.gate, self.up, self.down))
        self._needs: dict[tuple[int, int], int] = {}  # workspace bytes by tokens and top_k


# Workspaces of the products, one per (device, stream); a call needs nothing of
# what an earlier one left there. A replaced one is kept for the graphs that hold
# its address, as the K-split workspaces are.
_workspaces: dict[tuple[int, int], torch.Tensor] = {}


def workspace_for(device: torch.device, nbytes: int) -> torch.Tensor:
    ws = hip._stream_workspace(_workspaces, device, nbytes, 1 << 20)
    if ws is None:
        raise LaunchError("experts under graph capture need this stream's workspace: make one eager call of the same "
                          "size on the capturing stream first")
    return ws


def experts(weights: Experts, a8: torch.Tensor, a_scales: torch.Tensor, routing: Routing, *,
            dtype: torch.dtype = torch.float32, out: torch.Tensor | None = None,
            workspace: torch.Tensor | None = None) -> torch.Tensor:
    """The chosen experts' feed-forward of every row of a8 [tokens, hidden_pad]
    (int8, with a_scales f32 [tokens]: hip.norm_a8 or hip.quantize_a8), weighted
    by the routing and summed: [tokens, hidden] of `dtype` (f32, f16 or bf16), or
    into `out`. Products are W8A8 as hip.gemm_w8a8's, between them SwiGLU and
    the quantisation of its rows. a8 has to stay below 2^32 bytes."""
    out, key, args, space, nbytes = _experts_call(weights, a8, a_scales, routing, dtype, out, workspace)
    with hip.enqueuing.get(key) or hip.enqueuing_on(key):
        status = hip.call_on(key[0], _lib.load().rocknpu_hip_moe_experts, args, space, nbytes, key[1])
    hip._check(status, "moe_experts")
    return out


def _experts_call(weights, a8, a_scales, routing, dtype, out, workspace=None):
    """experts' result, still to be filled, and what the library's call for it takes: device and stream, arguments, workspace."""
    at = weights.device
    tokens, top_k = routing.ids.shape
    if tokens * weights.hidden_pad >> 32:
        raise ValueError(f"{tokens} rows of {weights.hidden_pad} bytes: a8 has to stay below 2^32 bytes, split the tokens")
    if a8.dtype is not torch.int8 or a8.shape != (tokens, weights.hidden_pad) or not a8.is_contiguous() or a8.device != at:
        raise ValueError(f"a8 has to be contiguous int8 [{tokens}, {weights.hidden_pad}] on {at}")
    if a_scales.dtype is not torch.float32 or a_scales.shape != (tokens,) or not a_scales.is_contiguous() or a_scales.device != at:
        raise ValueError(f"a_scales have to be contiguous float32 [{tokens}] on {at}")
    if routing.experts != weights.experts or routing.plan.device != at:
        raise ValueError(f"the routing is of {routing.experts} experts on {routing.plan.device}, not {weights.experts} on {at}")
    ids, factors, plan = routing.ids, routing.weights, routing.plan
    if (ids.dtype is not torch.int32 or not ids.is_contiguous() or ids.device != at or factors.dtype is not torch.float32
            or factors.shape != ids.shape or not factors.is_contiguous() or factors.device != at or plan.dtype is not torch.int32
            or not plan.is_contiguous() or plan.numel() != (_plan_words.get((tokens, weights.experts, top_k)) or plan_words(tokens, weights.experts, top_k))):
        raise ValueError(f"the routing's ids and plan have to be route's own, and its weights contiguous float32 {tuple(ids.shape)} on {at}")
    if out is None:
        if dtype not in TYPES:
            raise ValueError(f"{dtype}: float32, float16 or bfloat16 is wanted")
        out = torch.empty((tokens, weights.hidden), dtype=dtype, device=at)
    elif out.dtype not in TYPES or out.shape != (tokens, weights.hidden) or out.device != at or (out.stride(1) != 1 and weights.hidden > 1):
        raise ValueError(f"out has to be float32, float16 or bfloat16 [{tokens}, {weights.hidden}] on {at} with contiguous rows")
    elif tokens > 1 and out.stride(0) < weights.hidden:
        raise ValueError(f"out's rows overlap: they are {weights.hidden} wide and {out.stride(0)} apart")
    key = hip.stream_of(at)
    args = _pack_experts(
        a8.data_ptr(), a_scales.data_ptr(), *weights.pointers, ids.data_ptr(), factors.data_ptr(),
        plan.data_ptr(), out.data_ptr(), tokens, out.stride(0) if tokens > 1 else weights.hidden, weights.experts, top_k,
        weights.hidden, weights.hidden_pad, weights.ffn, weights.ffn_pad, TYPES[out.dtype])
    need = weights._needs.get((tokens, top_k))
    if need is None:
        got = ctypes.c_size_t()
        hip._check(_lib.load().rocknpu_hip_moe_experts_workspace(args, ctypes.addressof(got)), "moe_experts_workspace")
        if len(weights._needs) >= 1024:
            weights._needs.clear()
        need = weights._needs[tokens, top_k] = got.value
    if workspace is None and need == 0:  # no tokens
        space, nbytes = 0, 0
    elif workspace is None:
        workspace = _workspaces.get(key)  # the stream's own
        if workspace is None or workspace.numel() < need:
            workspace = workspace_for(at, need)
        space, nbytes = workspace.data_ptr(), workspace.numel()
    elif workspace.device != at or not workspace.is_contiguous():
        raise ValueError(f"workspace has to be a contiguous tensor on {at}")
    else:
        space, nbytes = workspace.data_ptr(), workspace.numel() * workspace.element_size()
    return out, key, args, space, nbytes


def _apart(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether no byte is in both of two matrices of contiguous rows. Rows as far apart as the
    other's may lie between them; otherwise what counts is from where to where they reach."""
    if a.data_ptr() > b.data_ptr():
        a, b = b, a
    if not a.numel() or not b.numel():
        return True
    rows, wide, step = a.shape[0], a.shape[1] * a.element_size(), a.stride(0) * a.element_size()
    d = b.data_ptr() - a.data_ptr()
    if d >= (rows - 1) * step + wide:
        return True
    if rows == 1 or step != b.stride(0) * b.element_size() or step < wide:
        return False
    return d % step >= wide and (d // step + 1 >= rows or d % step + b.shape[1] * b.element_size() <= step)


def feed_forward(x: torch.Tensor, norm_weight: torch.Tensor, router, weights: Experts, top_k: int, *, eps: float = 1e-5,
                 residual: torch.Tensor | None = None, hidden: torch.Tensor | None = None, out: torch.Tensor | None = None, **routing):
    """A layer's second half: hip.norm_a8 of x + residual, the router's product
    (`router`: a W8 pair [experts, hidden_pad] and [experts], for an f32 router
    hip.quantize_a8 of its rows), route with `routing`'s arguments, and experts.
    Returns (out [tokens, hidden] in x's type, x + residual or None); the former
    is the next norm's x, the latter its residual. `out` may be x or the residual,
    but not what x + residual goes to. A call that is refused has written nothing."""
    _pair(router, (weights.experts, weights.hidden_pad), "router", weights.device)
    if x.dim() != 2 or x.shape[1] != weights.hidden or x.device != weights.device:
        raise ValueError(f"x has to be [tokens, {weights.hidden}] on {weights.device}, not {tuple(x.shape)} on {x.device}")
    if hidden is not None and out is not None and out.dim() == 2 == hidden.dim() and not _apart(hidden, out):
        raise ValueError("out and hidden overlap: the layer's output would overwrite x + residual")
    tokens = x.shape[0]
    a8, a_scales = x.new_empty((tokens, weights.hidden_pad), dtype=torch.int8), x.new_empty((tokens,), dtype=torch.float32)
    logits = x.new_empty((tokens, weights.experts), dtype=torch.float32)
    chosen, index, stream, choose = _route_call(logits, top_k, **routing)
    out, key, run, space, nbytes = _experts_call(weights, a8, a_scales, chosen, x.dtype, out)
    hidden = hip.norm_a8(x, norm_weight, eps, residual, hidden=hidden, k_pad=weights.hidden_pad, a8=a8, scales=a_scales)[2]
    if tokens:
        hip.call_on(index, hip.gemm_w8a8, a8, a_scales, *router, logits)
        hip._check(hip.call_on(index, _lib.load().rocknpu_hip_moe_route, choose, stream), "moe_route")
        with hip.enqueuing.get(key) or hip.enqueuing_on(key):
            status = hip.call_on(index, _lib.load().rocknpu_hip_moe_experts, run, space, nbytes, stream)
        hip._check(status, "moe_experts")
    return out, hidden
