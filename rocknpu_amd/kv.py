"""The 8-bit key/value cache and the attention that reads it
(include/rocknpu_kv.h) on device tensors.

A `Cache` is a set of pages, each one block of 32 tokens of one kv head in int8
with an f32 scale for its keys and one for its values, and the table that names
every sequence's pages. A step of a model's layer is

    kv.append(cache, k, v, past, cu, max_new)          # the step's new rows
    out = kv.attention(cache, q, past, cu, max_new)    # its queries over all rows

with past [batch] the tokens that each sequence had before the step and
cu [batch + 1] the row offsets of its new ones, both int32 on the device and
shared by all layers. Calls enqueue on the current torch stream and return
immediately; they read no lengths on the host, so a step can be captured in a
HIP graph.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib, hip
from .hip import LaunchError

BLOCK = 32
HEAD_DIMS = (64, 128, 192, 256)
MAX_WEIGHT_ROWS = 256
MAX_EVICT_BLOCKS = 16384

_TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}

_vp = ctypes.c_void_p
_i32 = ctypes.c_int32
_i64 = ctypes.c_int64


class _CacheStruct(ctypes.Structure):
    """rocknpu_kv_cache (include/rocknpu_kv.h)."""

    _fields_ = [("pages", _vp), ("scales", _vp), ("table", _vp), ("starts", _vp), ("dropped", _vp), ("weights", _vp),
                ("n_pages", _i64), ("batch", _i32), ("kv_heads", _i32), ("head_dim", _i32), ("max_blocks", _i32)]


class _AttentionStruct(ctypes.Structure):
    """rocknpu_kv_attention_args (include/rocknpu_kv.h)."""

    _fields_ = [("q", _vp), ("out", _vp), ("past", _vp), ("cu", _vp), ("prefix", _vp), ("slopes", _vp),
                ("weights_out", _vp), ("q_row", _i64), ("q_head", _i64), ("out_row", _i64), ("out_head", _i64),
                ("rows", _i64), ("max_new", _i64), ("max_tokens", _i64), ("type", ctypes.c_uint32), ("heads", _i32),
                ("causal", _i32), ("window", _i32), ("scale", ctypes.c_float), ("softcap", ctypes.c_float)]


class _EvictStruct(ctypes.Structure):
    """rocknpu_kv_evict_args (include/rocknpu_kv.h)."""

    _fields_ = [("table", _vp), ("starts", _vp), ("weights", _vp), ("tokens", _vp), ("dropped", _vp),
                ("table_out", _vp), ("starts_out", _vp), ("weights_out", _vp), ("dropped_out", _vp), ("batch", _i32),
                ("kv_heads", _i32), ("max_blocks", _i32), ("budget", _i32), ("sinks", _i32), ("recent", _i32)]


# A serving step makes these calls per layer and token: their checks are kept to a
# few comparisons.
def _is(t, shape, dtype, what, device):
    """`t` is a contiguous tensor of that shape and type, on that device."""
    if (not isinstance(t, torch.Tensor) or t.dtype is not dtype or t.shape != shape or t.device != device
            or not t.is_contiguous()):
        raise ValueError(f"{what} has to be a contiguous {dtype} tensor of shape {tuple(shape)} on {device}")
    return t


def _rows(t, heads, head_dim, what, device):
    """`t` is [rows, heads, head_dim] of a known type with a contiguous last dimension: its shape and strides."""
    shape = t.shape
    if t.dtype not in _TYPES or len(shape) != 3 or shape[2] != head_dim or (heads is not None and shape[1] != heads):
        raise ValueError(f"{what} has to be float32, float16 or bfloat16 [rows, {'heads' if heads is None else heads}, "
                         f"{head_dim}], not {t.dtype} {tuple(shape)}")
    row, head, one = t.stride()
    if one != 1 and t.numel():
        raise ValueError(f"{what} has to be contiguous in its last dimension")
    if t.device != device:
        raise ValueError(f"{what} is on {t.device}, the cache on {device}")
    return shape[0], shape[1], row, head


def _sizes(below: int = 1 << 31, **sizes: int) -> None:
    """Refuses by name what a C field does not hold: ctypes cuts it to its low bits. (Callers ask (a | b) >> 31 first.)"""
    for what, n in sizes.items():
        if not 0 <= n < below:
            raise ValueError(f"{what} {n} is not in [0, {below})")


def _stream(device: torch.device) -> int:
    """The device's current stream, as hip._stream gives it, without its object where torch offers that."""
    raw = getattr(torch._C, "_cuda_getCurrentRawStream", None)
    if raw is None or device.index is None:
        return torch.cuda.current_stream(device).cuda_stream
    return raw(device.index)


class Cache:
    """One layer's pages and tables (rocknpu_kv_cache): `pages` int8 or uint8
    [n_pages, 64 * head_dim], `scales` f32 [n_pages, 2], `table` and `starts`
    int32 [batch, kv_heads, max_blocks], `dropped` int32 [batch], `weights` f32
    [batch, kv_heads, max_blocks] or None. The tensors are used in place and
    kept alive by the object; write into them, or make a new Cache of others (an
    assignment is refused)."""

    _FIXED = frozenset(("pages", "scales", "table", "starts", "dropped", "weights", "shape", "batch", "kv_heads",
                        "max_blocks", "head_dim", "device"))

    def __setattr__(self, name, value):
        if name in self._FIXED and name in self.__dict__:
            raise AttributeError(f"the kernels use the {name} that the cache was made with: write into it, or make a new Cache")
        object.__setattr__(self, name, value)

    def __init__(self, pages, scales, table, starts, dropped, weights=None, *, head_dim: int):
        if head_dim not in HEAD_DIMS:
            raise ValueError(f"head_dim {head_dim} is not one of {HEAD_DIMS}")
        if table.dim() != 3 or 0 in table.shape:
            raise ValueError("table has to be [batch, kv_heads, max_blocks]")
        if pages.dtype not in (torch.int8, torch.uint8):
            raise ValueError("pages have to be int8 or uint8")
        at = table.device
        n = pages.shape[0]
        if n == 0:
            raise ValueError("a cache needs at least one page")
        self.shape = table.shape
        self.batch, self.kv_heads, self.max_blocks = table.shape
        self.head_dim, self.device = head_dim, at
        self._lengths, self._offsets = torch.Size((self.batch,)), torch.Size((self.batch + 1,))
        self.pages = _is(pages, torch.Size((n, 2 * BLOCK * head_dim)), pages.dtype, "pages", at)
        self.scales = _is(scales, torch.Size((n, 2)), torch.float32, "scales", at)
        self.table = _is(table, table.shape, torch.int32, "table", at)
        self.starts = _is(starts, table.shape, torch.int32, "starts", at)
        self.dropped = _is(dropped, self._lengths, torch.int32, "dropped", at)
        self.weights = None if weights is None else _is(weights, table.shape, torch.float32, "weights", at)
        self._struct = _CacheStruct(
            pages.data_ptr(), scales.data_ptr(), table.data_ptr(), starts.data_ptr(), dropped.data_ptr(),
            None if weights is None else weights.data_ptr(), n, self.batch, self.kv_heads, head_dim, self.max_blocks)
        self._ref = ctypes.addressof(self._struct)
        self._needs: dict[tuple, int] = {}  # workspace bytes by the sizes that they depend on

    @classmethod
    def empty(cls, batch: int, kv_heads: int, head_dim: int, max_blocks: int, device="cuda", weights: bool = True):
        """A cache with max_blocks pages of its own for every sequence and head."""
        n = batch * kv_heads * max_blocks
        table = torch.arange(n, dtype=torch.int32, device=device).view(batch, kv_heads, max_blocks)
        return cls(torch.zeros((n, 2 * BLOCK * head_dim), dtype=torch.int8, device=device),
                   torch.full((n, 2), 2.0 ** -100, dtype=torch.float32, device=device), table, torch.zeros_like(table),
                   torch.zeros(batch, dtype=torch.int32, device=device),
                   torch.zeros(table.shape, dtype=torch.float32, device=device) if weights else None, head_dim=head_dim)

    def lengths(self, t, what) -> int:
        return _is(t, self._lengths, torch.int32, what, self.device).data_ptr()

    def offsets(self, t) -> int:
        return _is(t, self._offsets, torch.int32, "cu", self.device).data_ptr()


def append(cache: Cache, k: torch.Tensor, v: torch.Tensor, past: torch.Tensor, cu: torch.Tensor, max_new: int) -> None:
    """Quantises rows k and v [rows, kv_heads, head_dim] (f32, f16 or bf16; any
    row and head strides) into the blocks of their sequences. max_new bounds
    the rows of any one sequence. A partly filled block's scale only grows, and
    its older codes are rounded anew when it does; a value that is not finite
    makes its block NaN."""
    rows, _, k_row, k_head = _rows(k, cache.kv_heads, cache.head_dim, "k", cache.device)
    v_rows, _, v_row, v_head = _rows(v, cache.kv_heads, cache.head_dim, "v", cache.device)
    if k.dtype is not v.dtype or rows != v_rows:
        raise ValueError("k and v differ in type or rows")
    if max_new >> 31:
        _sizes(max_new=max_new)
    hip._check(_lib.load().rocknpu_hip_kv_append(
        cache._ref, _TYPES[k.dtype], k.data_ptr(), k_row, k_head, v.data_ptr(), v_row, v_head, rows,
        cache.lengths(past, "past"), cache.offsets(cu), max_new, _stream(cache.device)), "kv_append")


def read(cache: Cache, first: torch.Tensor, tokens: torch.Tensor, count: int, dtype: torch.dtype = torch.float32):
    """(keys, values), each [batch, count, kv_heads, head_dim]: what the cache
    stands for at positions first[b] .. first[b] + count - 1, zero at or past
    tokens[b] and in evicted blocks."""
    if dtype not in _TYPES:
        raise ValueError(f"{dtype}: float32, float16 or bfloat16 is wanted")
    if count >> 31:
        _sizes(count=count)
    k, v = cache.scales.new_empty((2, cache.batch, count, cache.kv_heads, cache.head_dim), dtype=dtype).unbind(0)
    hip._check(_lib.load().rocknpu_hip_kv_read(
        cache._ref, cache.lengths(first, "first"), cache.lengths(tokens, "tokens"), count, _TYPES[dtype],
        k.data_ptr(), v.data_ptr(), _stream(cache.device)), "kv_read")
    return k, v


# Workspaces of the attention, one per (device, stream); a call needs nothing
# of what an earlier one left there. A replaced one is kept for the graphs that
# hold its address, as the K-split workspaces are.
_workspaces: dict[tuple[int, int], torch.Tensor] = {}


def workspace_for(device: torch.device, nbytes: int) -> torch.Tensor:
    ws = hip._stream_workspace(_workspaces, device, nbytes, 1 << 20)
    if ws is None:
        raise LaunchError("attention under graph capture needs this stream's workspace: make one eager call of the "
                          "same shape on the capturing stream first")
    return ws


def attention(cache: Cache, q: torch.Tensor, past: torch.Tensor, cu: torch.Tensor, max_new: int, *,
              max_tokens: int = 0, scale: float | None = None, causal: bool = True, window: int = 0,
              prefix: torch.Tensor | None = None, softcap: float = 0.0, slopes: torch.Tensor | None = None,
              weights_out: torch.Tensor | None = None, out: torch.Tensor | None = None,
              workspace: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of query rows q [rows, heads, head_dim] over the cache, whose
    last rows are theirs (append them first). out has q's shape and type.

    scale defaults to 1 / sqrt(head_dim). A row at position p sees the keys at
    positions s <= p, with `window` only those with s > p - window, and with
    `prefix` (int32 [batch]) all with s < prefix as well; causal=False sees all.
    `softcap` caps scores by softcap * tanh(x / softcap), `slopes` (f32 [heads])
    adds slopes * (s - p). A row that sees nothing is 0. `weights_out` takes
    cache.weights plus what each block got of this step's attention (it may be
    cache.weights; at most 256 rows times heads per kv head). max_tokens, the
    most tokens a sequence is expected to hold, sizes the work split only;
    without it the table's width does."""
    device, dtype = cache.device, q.dtype
    rows, heads, row, head = _rows(q, None, cache.head_dim, "q", device)
    if heads == 0 or heads % cache.kv_heads:
        raise ValueError(f"{heads} query heads over {cache.kv_heads} kv heads")
    if (max_new | window) >> 31 or max_tokens >> 63:
        _sizes(max_new=max_new, window=window)
        _sizes(1 << 63, max_tokens=max_tokens)
    if out is None:
        out = torch.empty_like(q) if q.is_contiguous() else q.new_empty(q.shape)
        o_row, o_head = heads * cache.head_dim, cache.head_dim
    else:
        o_rows, _, o_row, o_head = _rows(out, heads, cache.head_dim, "out", device)
        if out.dtype is not dtype or o_rows != rows:
            raise ValueError("out has to have q's type and shape")
    args = _AttentionStruct(
        q.data_ptr(), out.data_ptr(), cache.lengths(past, "past"), cache.offsets(cu),
        None if prefix is None else cache.lengths(prefix, "prefix"),
        None if slopes is None else _is(slopes, torch.Size((heads,)), torch.float32, "slopes", device).data_ptr(),
        None if weights_out is None else _is(weights_out, cache.shape, torch.float32, "weights_out", device).data_ptr(),
        row, head, o_row, o_head, rows, max_new, max_tokens, _TYPES[dtype], heads, causal, window,
        cache.head_dim ** -0.5 if scale is None else scale, softcap)
    lib = _lib.load()
    ref = ctypes.addressof(args)
    sizes = (dtype, heads, min(max_new, rows), max_tokens, window, weights_out is None)
    need = cache._needs.get(sizes)
    if need is None:
        got = ctypes.c_size_t()
        hip._check(lib.rocknpu_hip_kv_attention_workspace(cache._ref, ref, 0, ctypes.addressof(got)), "kv_attention")
        if len(cache._needs) >= 1024:  # max_tokens may grow from step to step
            cache._needs.clear()
        need = cache._needs[sizes] = got.value
    ws, nbytes = None, 0
    if need:
        if workspace is None:
            workspace = workspace_for(device, need)
        elif workspace.device != device or not workspace.is_contiguous():
            raise ValueError(f"workspace has to be a contiguous tensor on {device}")
        ws, nbytes = workspace.data_ptr(), workspace.numel() * workspace.element_size()
    hip._check(lib.rocknpu_hip_kv_attention(cache._ref, ref, ws, nbytes, _stream(device)), "kv_attention")
    return out


def evict(table: torch.Tensor, starts: torch.Tensor, weights: torch.Tensor, tokens: torch.Tensor, dropped: torch.Tensor,
          budget: int, *, sinks: int = 0, recent: int = 1, out=None):
    """Cuts every sequence's blocks to `budget` by accumulated weight, per kv
    head: the first `sinks`, the last `recent` and the heaviest others stay
    (equal weights: the lowest place). Returns new (table, starts, weights,
    dropped), or fills `out`; each row holds the kept entries in order, then the
    evicted, whose pages the sequence's next blocks take, then the rest. out[:3]
    may be the inputs themselves, out[3] must not be `dropped`. A Cache keeps the
    tensors that it was made with: give its own as out[:3] and copy out[3] into
    its `dropped`, or make a new Cache of what is returned."""
    if table.dim() != 3 or 0 in table.shape:
        raise ValueError("table has to be [batch, kv_heads, max_blocks]")
    at = table.device
    batch, kv_heads, max_blocks = table.shape
    if out is None:
        out = (torch.empty_like(table), torch.empty_like(starts), torch.empty_like(weights), torch.empty_like(dropped))
    table_out, starts_out, weights_out, dropped_out = out
    shape, size = table.shape, torch.Size((batch,))
    for t, what in ((table, "table"), (table_out, "table_out"), (starts, "starts"), (starts_out, "starts_out")):
        _is(t, shape, torch.int32, what, at)
    for t, what in ((weights, "weights"), (weights_out, "weights_out")):
        _is(t, shape, torch.float32, what, at)
    for t, what in ((tokens, "tokens"), (dropped, "dropped"), (dropped_out, "dropped_out")):
        _is(t, size, torch.int32, what, at)
    if (budget | sinks | recent) >> 31:
        _sizes(budget=budget, sinks=sinks, recent=recent)
    args = _EvictStruct(table.data_ptr(), starts.data_ptr(), weights.data_ptr(), tokens.data_ptr(), dropped.data_ptr(),
                        table_out.data_ptr(), starts_out.data_ptr(), weights_out.data_ptr(), dropped_out.data_ptr(),
                        batch, kv_heads, max_blocks, budget, sinks, recent)
    hip._check(_lib.load().rocknpu_hip_kv_evict(ctypes.addressof(args), _stream(at)), "kv_evict")
    return out
