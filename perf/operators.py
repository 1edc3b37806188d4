"""Measured operators: the 8-bit key/value cache and the attention that reads it, as a serving loop calls them between
the q/k/v projections and the output projection.

Three kinds of cases:

- "append": a step's new key and value rows are quantised into the paged cache, and the blocks that they touched are
  read back as the values they now stand for (kv.append, kv.read).
- "attend": attention of a step's query rows over the cache (kv.attention): single tokens, a few tokens, prompts.
- "evict": the blocks of least accumulated attention weight leave a cache that is over its budget (kv.evict).

The cache: a page holds one block of 32 tokens of one key/value head as int8 codes, with an f32 scale for its keys and
one for its values. `table` [batch, kv_heads, max_blocks] names the pages of a sequence and head in order of position,
`starts` the position of each block's first token, `dropped` [batch] how many blocks a sequence has lost to eviction.
A page of 64 * head_dim bytes is the keys, then the values:
  keys    [head_dim / 64][32 tokens][64 dims]
  values  [head_dim / 32][16 dims low][4: token bits 3-2][2: dim bit 4][2: token bit 4][4: token bits 1-0]
Sequence b has past[b] tokens before the step and rows cu[b] .. cu[b + 1] of the step's tensors.
"""
from __future__ import annotations

import math

import torch

own = False

BLOCK = 32
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
SCALE_FLOOR = 2.0 ** -100
EVICT_SINKS, EVICT_RECENT = 2, 4


def listed():
    tiny = {"heads": 32, "kv_heads": 4, "head_dim": 64}    # TinyLlama-1.1B
    small = {"heads": 32, "kv_heads": 8, "head_dim": 64}   # Llama-3.2-1B
    large = {"heads": 32, "kv_heads": 8, "head_dim": 128}  # Llama-3-8B
    plain = {"window": 0, "prefix": 0, "softcap": 0.0, "alibi": False, "weights": False, "evicted": 0}
    return [
        # one user's token on a small model: the smallest call there is
        {"name": "append-tiny-1", "op": "append", **tiny, "type": "f32", "batch": 1, "past_lo": 77, "past_hi": 77, "new_lo": 1, "new_hi": 1},
        # forty-eight users' tokens in one step
        {"name": "append-large-48", "op": "append", **large, "type": "f32", "batch": 48, "past_lo": 100, "past_hi": 8000, "new_lo": 1, "new_hi": 1},
        # a long prompt's keys and values
        {"name": "append-prompt-8192", "op": "append", **large, "type": "bf16", "batch": 1, "past_lo": 0, "past_hi": 0, "new_lo": 8192, "new_hi": 8192},
        # ragged pieces of prompts that start and end inside blocks
        {"name": "append-ragged", "op": "append", **small, "type": "f16", "batch": 11, "past_lo": 0, "past_hi": 1000, "new_lo": 1, "new_hi": 513},
        # one user's token over a short context: latency
        {"name": "decode-tiny-1", "op": "attend", **tiny, **plain, "type": "f32", "batch": 1, "past_lo": 511, "past_hi": 511, "new_lo": 1, "new_hi": 1},
        # thirty-two users' tokens, ragged contexts, with the weights that eviction goes by
        {"name": "decode-large-32", "op": "attend", **large, **plain, "type": "f32", "batch": 32, "past_lo": 500, "past_hi": 4100,
         "new_lo": 1, "new_hi": 1, "weights": True, "evicted": 4},
        # two users' tokens over long documents: the cache streams from memory
        {"name": "decode-long-2", "op": "attend", **large, **plain, "type": "bf16", "batch": 2, "past_lo": 90001, "past_hi": 131000,
         "new_lo": 1, "new_hi": 1},
        # four drafted tokens a user under a window, a kept prefix and capped scores
        {"name": "decode-draft-8", "op": "attend", **large, **plain, "type": "f16", "batch": 8, "past_lo": 200, "past_hi": 20000,
         "new_lo": 4, "new_hi": 4, "window": 4096, "prefix": 64, "softcap": 50.0},
        # a long prompt at once
        {"name": "prompt-large-4096", "op": "attend", **large, **plain, "type": "bf16", "batch": 1, "past_lo": 0, "past_hi": 0,
         "new_lo": 4096, "new_hi": 4096},
        # pieces of several prompts behind what is cached, f32 as the projections give it, distance bias
        {"name": "prompt-ragged-5", "op": "attend", **tiny, **plain, "type": "f32", "batch": 5, "past_lo": 0, "past_hi": 1500,
         "new_lo": 17, "new_hi": 700, "alibi": True},
        # one user over a small budget
        {"name": "evict-tiny-1", "op": "evict", **tiny, "batch": 1, "blocks_lo": 40, "blocks_hi": 40, "budget": 32},
        # sixty-four long sequences cut to a quarter
        {"name": "evict-large-64", "op": "evict", **large, "batch": 64, "blocks_lo": 2000, "blocks_hi": 4096, "budget": 1024},
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def _between(rng, name, hi):
    lo, hi = sorted((_log(rng, 1, hi), _log(rng, 1, hi)))
    return {name + "_lo": lo, name + "_hi": hi}


def draw(rng):
    op = rng.choice(["append", "attend", "attend", "attend", "evict"])
    head_dim = rng.choice([64, 64, 128, 128, 128, 192, 256])
    kv_heads = rng.choice([1, 2, 4, 5, 8])
    heads = kv_heads * rng.choice([1, 2, 3, 4, 4, 7, 8])
    shape = {"heads": heads, "kv_heads": kv_heads, "head_dim": head_dim}
    if op == "evict":
        blocks = _between(rng, "blocks", 4096)
        return {"op": op, **shape, "batch": _log(rng, 1, 64), **blocks,
                "budget": max(EVICT_SINKS + EVICT_RECENT, int(blocks["blocks_hi"] * rng.uniform(0.1, 1.1)))}
    kind = rng.choice(["f32", "f16", "bf16"])
    if op == "append":
        batch = _log(rng, 1, 64)
        most = 8192 * 8 * 128 // (kv_heads * head_dim * batch)
        past = {"past_lo": 0, "past_hi": 0} if rng.random() < 0.2 else _between(rng, "past", 8000)
        new = {"new_lo": 1, "new_hi": 1} if rng.random() < 0.4 else _between(rng, "new", max(2, min(8192, most)))
        return {"op": op, **shape, "type": kind, "batch": batch, **past, **new}
    more = {"window": _log(rng, 1, 8192) if rng.random() < 0.3 else 0, "prefix": _log(rng, 1, 512) if rng.random() < 0.3 else 0,
            "softcap": rng.choice([20.0, 30.0, 50.0]) if rng.random() < 0.3 else 0.0, "alibi": rng.random() < 0.3,
            "weights": False, "evicted": 0}
    if rng.random() < 0.6:  # single tokens, or a few
        batch = _log(rng, 1, 48)
        new = rng.choice([1, 1, 1, 2, 3, 5])
        most = max(64, min(131072, 2 * 110000 * 8 * 128 // (batch * kv_heads * head_dim)))
        case = {"batch": batch, **_between(rng, "past", most), "new_lo": new, "new_hi": new, **more}
        case["weights"] = rng.random() < 0.4
        if not more["window"] and not more["prefix"]:
            case["evicted"] = rng.choice([0, 0, 3, 17])
    else:
        batch = _log(rng, 1, 8)
        # pairs of queries and keys within the longest prompt's, all heads and dims
        most = int(math.sqrt(4096 * 4096 * 32 * 128 / (heads * head_dim * batch * 4)))
        past = {"past_lo": 0, "past_hi": 0} if rng.random() < 0.4 else _between(rng, "past", max(2, most))
        case = {"batch": batch, **past, **_between(rng, "new", max(2, most)), **more}
    return {"op": op, **shape, "type": kind, **case}


def _spread(case, name):
    """The batch's lengths: spread between the case's bounds, the same for every seed."""
    lo, hi, batch = case[name + "_lo"], case[name + "_hi"], case["batch"]
    if batch == 1:
        return [hi]
    return [lo + int(round((hi - lo) * ((b * 0.6180339887 + 0.5) % 1.0))) for b in range(batch)]


def _lengths(case):
    past, new = _spread(case, "past"), _spread(case, "new")
    lost = [min(case.get("evicted", 0), p // BLOCK) for p in past]
    return past, new, lost


def _blocks(tokens):
    return (tokens + BLOCK - 1) // BLOCK


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _pack(k, v):
    """Codes [P, 32, D] of keys and of values (whole numbers) -> pages [P, 64 D] int8."""
    p, _, d = k.shape
    keys = k.to(torch.int8).view(p, BLOCK, d // 64, 64).permute(0, 2, 1, 3).reshape(p, -1)
    values = v.to(torch.int8).view(p, 2, 4, 4, d // 32, 2, 16).permute(0, 4, 6, 2, 5, 1, 3).reshape(p, -1)
    return torch.cat((keys, values), 1)


def _unpack(pages, d):
    """Pages [P, 64 D] -> codes [P, 32, D] of keys and of values, f32."""
    p = pages.shape[0]
    k = pages[:, :BLOCK * d].view(p, d // 64, BLOCK, 64).permute(0, 2, 1, 3).reshape(p, BLOCK, d)
    v = pages[:, BLOCK * d:].view(p, d // 32, 16, 4, 2, 2, 4).permute(0, 5, 3, 6, 1, 4, 2).reshape(p, BLOCK, d)
    return k.float(), v.float()


def _cache(g, batch, kv_heads, head_dim, max_blocks, filled=True):
    """Pages in scattered order, keys with a few strong channels, values that vary from block to block."""
    n = batch * kv_heads * max_blocks
    pages = torch.empty((n, 2 * BLOCK * head_dim), dtype=torch.int8, device="cuda")
    scales = torch.empty((n, 2), device="cuda")
    if filled:
        gain = 1.0 + 3.0 * (torch.rand(head_dim, device="cuda", generator=g) < 0.06)
        for at in range(0, n, 8192):
            p = min(8192, n - at)
            k = torch.randn((p, BLOCK, head_dim), device="cuda", generator=g) * gain
            v = torch.randn((p, BLOCK, head_dim), device="cuda", generator=g)
            v = v * torch.exp(0.5 * torch.randn((p, 1, 1), device="cuda", generator=g))
            sk, sv = k.abs().amax((1, 2)) / 127.0, v.abs().amax((1, 2)) / 127.0
            pages[at:at + p] = _pack(torch.round(k / sk[:, None, None]), torch.round(v / sv[:, None, None]))
            scales[at:at + p, 0], scales[at:at + p, 1] = sk, sv
    else:
        pages.random_(-127, 128, generator=g)
        scales.fill_(1.0)
    table = torch.randperm(n, device="cuda", generator=g).to(torch.int32).view(batch, kv_heads, max_blocks)
    return pages, scales, table


def _starts(g, past, lost, kv_heads, max_blocks):
    """Positions of the blocks' first tokens: what is lost is drawn from the full blocks before the step."""
    starts = torch.empty((len(past), kv_heads, max_blocks), dtype=torch.int32, device="cuda")
    starts[:] = BLOCK * torch.arange(max_blocks, dtype=torch.int32, device="cuda")
    for b, gone in enumerate(lost):
        if not gone:
            continue
        full = past[b] // BLOCK
        order = torch.rand((kv_heads, full), device="cuda", generator=g).argsort(1)
        kept = order[:, :full - gone].sort(1).values.to(torch.int32)
        tail = torch.arange(full, full + max_blocks, dtype=torch.int32, device="cuda").expand(kv_heads, -1)
        starts[b] = BLOCK * torch.cat((kept, tail), 1)[:, :max_blocks]
    return starts


def _prepare_append(case, seed):
    g = _generator(seed)
    past, new, _ = _lengths(case)
    d, h, kind = case["head_dim"], case["kv_heads"], TYPES[case["type"]]
    width = max(_blocks(p + n) for p, n in zip(past, new))
    pages, scales, table = _cache(g, case["batch"], h, d, width)
    n = sum(new)
    k = (torch.randn((n, h, d), device="cuda", generator=g) * 1.2).to(kind)
    v = torch.randn((n, h, d), device="cuda", generator=g).to(kind)
    cu = [0]
    for x in new:
        cu.append(cu[-1] + x)
    # the blocks that the step touches, as a scheduler has them at hand
    touched = [(b, j) for b in range(case["batch"]) for j in range(past[b] // BLOCK, _blocks(past[b] + new[b]))]
    return {"case": case, "k": k, "v": v, "pages": pages, "scales": scales, "table": table,
            "starts": torch.zeros_like(table), "weights": torch.ones(table.shape, device="cuda"), "past": _ints(past),
            "cu": _ints(cu), "dropped": _ints([0] * case["batch"]), "first": _ints([p // BLOCK * BLOCK for p in past]),
            "tokens": _ints([p + x for p, x in zip(past, new)]), "max_new": max(new),
            "count": BLOCK * max(_blocks(p + x) - p // BLOCK for p, x in zip(past, new)),
            "touched": torch.tensor(touched, device="cuda")}


def _prepare_attend(case, seed):
    g = _generator(seed)
    past, new, lost = _lengths(case)
    d, h, heads = case["head_dim"], case["kv_heads"], case["heads"]
    width = max(_blocks(p + n) - e for p, n, e in zip(past, new, lost)) + 1
    pages, scales, table = _cache(g, case["batch"], h, d, width)
    starts = _starts(g, past, lost, h, width)
    n, cu = sum(new), [0]
    for x in new:
        cu.append(cu[-1] + x)
    q = (1.5 * torch.randn((n, heads, d), device="cuda", generator=g)).to(TYPES[case["type"]])
    row = torch.arange(n, device="cuda")
    of = torch.repeat_interleave(torch.arange(len(new), device="cuda"), torch.tensor(new, device="cuda"), output_size=n)
    s = {"case": case, "q": q, "pages": pages, "scales": scales, "table": table, "starts": starts, "past": _ints(past),
         "cu": _ints(cu), "dropped": _ints(lost), "max_new": max(new), "max_tokens": max(p + x for p, x in zip(past, new)),
         "seq": of, "row": row - torch.tensor(cu, device="cuda")[of], "prefix": None, "slopes": None, "weights": None}
    if case["prefix"]:
        s["prefix"] = _ints([min(case["prefix"], p + x) for p, x in zip(past, new)])
    if case["alibi"]:
        s["slopes"] = torch.exp2(-8.0 * torch.arange(1, heads + 1, device="cuda") / heads).float()
    if case["weights"]:
        s["weights"] = torch.rand(table.shape, device="cuda", generator=g)
        s["weights_out"] = torch.empty_like(s["weights"])
    return s


def _prepare_evict(case, seed):
    g = _generator(seed)
    batch, h = case["batch"], case["kv_heads"]
    blocks = _spread(case, "blocks")
    width = max(blocks) + 2
    table = torch.randperm(batch * h * width, device="cuda", generator=g).to(torch.int32).view(batch, h, width)
    starts = (BLOCK * torch.arange(width, dtype=torch.int32, device="cuda")).expand(batch, h, -1).contiguous()
    # heavy-tailed, and equal where nothing was attended to
    u = torch.rand(table.shape, device="cuda", generator=g)
    weights = torch.where(u < 0.2, torch.zeros_like(u), 0.01 / (1.0001 - u))
    return {"case": case, "table": table, "starts": starts, "weights": weights, "tokens": _ints([BLOCK * b - 7 for b in blocks]),
            "dropped": _ints([0] * batch), "out": [torch.empty_like(t) for t in (table, starts, weights)]
            + [torch.empty(batch, dtype=torch.int32, device="cuda")], "pages": None, "scales": None}


def prepare(case, seed):
    return {"append": _prepare_append, "attend": _prepare_attend, "evict": _prepare_evict}[case["op"]](case, seed)


def _handle(s):
    """The framework's cache object over the state's buffers, kept with them."""
    from rocknpu_amd import kv
    if "handle" not in s:
        s["handle"] = kv.Cache(s["pages"], s["scales"], s["table"], s["starts"], s["dropped"], s["weights"],
                               head_dim=s["case"]["head_dim"])
    return kv, s["handle"]


def _stored(s):
    """Keys and values [B, count, kv_heads, D] that the cache holds from s["first"] on, zero where it holds none."""
    c, d, h = s["case"], s["case"]["head_dim"], s["case"]["kv_heads"]
    blocks = s["count"] // BLOCK
    j = (s["first"] // BLOCK)[:, None] + torch.arange(blocks, device="cuda")
    inside = (j * BLOCK < s["tokens"][:, None]) & (j < s["table"].shape[2])
    j = j.clamp(max=s["table"].shape[2] - 1).long()
    page = s["table"].long().gather(2, j[:, None, :].expand(-1, h, -1))
    at = s["first"][:, None] + torch.arange(s["count"], device="cuda")
    seen = (at < s["tokens"][:, None])[:, :, None, None] & inside.repeat_interleave(BLOCK, 1)[:, :, None, None]
    out = []
    for codes, scale in zip(_unpack(s["pages"][page.view(-1)], d), s["scales"][page].unbind(-1)):
        x = codes.view(c["batch"], h, blocks, BLOCK, d) * scale[..., None, None]
        x = x.permute(0, 2, 3, 1, 4).reshape(c["batch"], s["count"], h, d)
        out.append(torch.where(seen, x, torch.zeros_like(x)).to(TYPES[c["type"]]))
    return out


def _quantised(x, fresh, old, old_scale, was):
    """New values x (where fresh) joined to old codes (where was): codes and scales of the blocks."""
    top = torch.where(fresh, x, torch.zeros_like(x)).abs().amax((-2, -1))
    before = torch.where(was.any((-2, -1)), old_scale, torch.zeros_like(old_scale))
    scale = torch.maximum(top / torch.full_like(top, 127.0), before).clamp_min(SCALE_FLOOR)
    code = torch.round(x * (1.0 / scale)[..., None, None]).clamp(-127, 127)
    again = torch.round(old * (before / scale)[..., None, None])
    return torch.where(fresh, code, torch.where(was, again, torch.zeros_like(code))), scale


def _plain_append(s):
    d, h = s["case"]["head_dim"], s["case"]["kv_heads"]
    b, j = s["touched"].unbind(1)
    page = s["table"][b, :, j].long()                                    # [N, H]
    at = j[:, None] * BLOCK + torch.arange(BLOCK, device="cuda")         # [N, 32] positions
    row = at - s["past"][b, None] + s["cu"][b, None]
    was, fresh = at < s["past"][b, None], (at >= s["past"][b, None]) & (at < s["tokens"][b, None])
    row = torch.where(fresh, row, torch.zeros_like(row))
    fresh, was = fresh[:, None, :, None], was[:, None, :, None]
    old = _unpack(s["pages"][page.view(-1)], d)
    codes, scales = [], []
    for x, o, sc in zip((s["k"], s["v"]), old, s["scales"][page].unbind(-1)):
        x = x[row].float().permute(0, 2, 1, 3)                           # [N, H, 32, D]
        c, new = _quantised(x, fresh, o.view(-1, h, BLOCK, d), sc, was)
        codes.append(c.reshape(-1, BLOCK, d))
        scales.append(new)
    s["pages"][page.view(-1)] = _pack(*codes)
    s["scales"][page.view(-1)] = torch.stack(scales, -1).view(-1, 2)
    started = (j * BLOCK >= s["past"][b])[:, None].expand(-1, h)
    s["starts"][b, :, j] = torch.where(started, (j * BLOCK)[:, None], s["starts"][b, :, j]).to(torch.int32)
    s["weights"][b, :, j] = torch.where(started, torch.zeros_like(s["weights"][b, :, j]), s["weights"][b, :, j])


def _visible(s, qpos, kpos, held):
    """[B, 1, rows, H?, keys] truth: what a row at qpos may look at."""
    c = s["case"]
    seen = kpos <= qpos
    if c["window"]:
        seen = seen & (kpos > qpos - c["window"])
    if s["prefix"] is not None:
        seen = seen | (kpos < s["prefix"].view(-1, 1, 1, 1))
    return seen & held


def _plain_attend(s):
    c = s["case"]
    d, h, g, batch, width = c["head_dim"], c["kv_heads"], c["heads"] // c["kv_heads"], c["batch"], s["table"].shape[2]
    page = s["table"].long().view(-1)
    k, v = _unpack(s["pages"][page], d)
    scale = s["scales"][page].view(-1, 2, 1, 1)
    k = (k * scale[:, 0]).view(batch, h, width * BLOCK, d)
    v = (v * scale[:, 1]).view(batch, h, width * BLOCK, d)
    most = s["max_new"]
    q = torch.zeros((batch, most, c["heads"], d), device="cuda")
    q[s["seq"], s["row"]] = s["q"].float()
    q = q.view(batch, most, h, g, d).permute(0, 2, 1, 3, 4).reshape(batch, h, most * g, d)
    t = torch.matmul(q, k.transpose(2, 3).contiguous()) * (1.0 / math.sqrt(d))
    kpos = (s["starts"][..., None] + torch.arange(BLOCK, device="cuda")).view(batch, h, 1, width * BLOCK)
    qpos = (s["past"][:, None] + torch.arange(most, device="cuda").repeat_interleave(g)).view(batch, 1, most * g, 1)
    tokens = (s["past"] + s["cu"][1:] - s["cu"][:-1]).view(batch, 1, 1, 1)
    held = (torch.arange(width * BLOCK, device="cuda") // BLOCK < (tokens + BLOCK - 1) // BLOCK - s["dropped"].view(-1, 1, 1, 1)) \
        & (kpos < tokens)
    if c["softcap"]:
        t = c["softcap"] * torch.tanh(t / c["softcap"])
    if s["slopes"] is not None:
        t = t + s["slopes"].view(1, h, 1, g).expand(1, h, most, g).reshape(1, h, most * g, 1) * (kpos - qpos)
    t = t.masked_fill(~(_visible(s, qpos, kpos, held) & (qpos < tokens)), -math.inf)
    top = t.amax(-1, keepdim=True)
    e = torch.exp(t - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = e.sum(-1, keepdim=True)
    e = e / torch.where(total == 0, torch.ones_like(total), total)
    o = torch.matmul(e, v).view(batch, h, most, g, d).permute(0, 2, 1, 3, 4).reshape(batch, most, c["heads"], d)
    out = {"out": o[s["seq"], s["row"]].to(s["q"].dtype)}
    if c["weights"]:
        torch.add(s["weights"], e.sum(2).view(batch, h, width, BLOCK).sum(-1), out=s["weights_out"])
        out["weights"] = s["weights_out"]
    return out


def _plain_evict(s):
    c, width = s["case"], s["table"].shape[2]
    j = torch.arange(width, device="cuda")
    n = ((s["tokens"] + BLOCK - 1) // BLOCK - s["dropped"]).view(-1, 1, 1)
    safe = (j < EVICT_SINKS) | (j >= n - EVICT_RECENT)
    worth = torch.where(safe, torch.full_like(s["weights"], math.inf), s["weights"]).masked_fill(j >= n, -math.inf)
    order = worth.sort(dim=-1, descending=True, stable=True).indices
    rank = torch.empty_like(order).scatter_(2, order, j.expand_as(order))
    left = torch.where(j >= n, 2, torch.where((rank < c["budget"]) | (n <= c["budget"]), 0, 1))
    order = left.sort(dim=-1, stable=True).indices
    return [t.gather(2, order) for t in (s["table"], s["starts"], s["weights"])] \
        + [(s["dropped"] + (n.view(-1) - c["budget"]).clamp_min(0)).to(torch.int32)]


def run(s):
    c = s["case"]
    if c["op"] == "append":
        if own:
            kv, cache = _handle(s)
            kv.append(cache, s["k"], s["v"], s["past"], s["cu"], s["max_new"])
            k, v = kv.read(cache, s["first"], s["tokens"], s["count"], dtype=s["k"].dtype)
        else:
            _plain_append(s)
            k, v = _stored(s)
        return {"k": k, "v": v, "scales": s["scales"], "starts": s["starts"], "weights": s["weights"]}
    if c["op"] == "evict":
        if own:
            from rocknpu_amd import kv
            return list(kv.evict(s["table"], s["starts"], s["weights"], s["tokens"], s["dropped"], c["budget"],
                                 sinks=EVICT_SINKS, recent=EVICT_RECENT, out=s["out"]))
        return _plain_evict(s)
    if own:
        kv, cache = _handle(s)
        o = kv.attention(cache, s["q"], s["past"], s["cu"], s["max_new"], max_tokens=s["max_tokens"], window=c["window"],
                         prefix=s["prefix"], softcap=c["softcap"], slopes=s["slopes"], weights_out=s.get("weights_out"))
        return {"out": o, "weights": s["weights_out"]} if c["weights"] else {"out": o}
    return _plain_attend(s)


def _seen(case, p, gone):
    """Keys that a row at position p looks at (blocks lost to eviction lie before it)."""
    if not case["window"] or p + 1 <= case["window"]:
        return max(1, p + 1 - BLOCK * gone)
    return case["window"] + min(case["prefix"], max(0, p + 1 - case["window"]))


def work(case):
    d, h = case["head_dim"], case["kv_heads"]
    if case["op"] == "evict":
        n = case["batch"] * h * (max(_spread(case, "blocks")) + 2)
        return {"bytes": 2 * 12 * n, "flops": n}
    past, new, lost = _lengths(case)
    size, rows = SIZE[case["type"]], sum(new)
    if case["op"] == "append":
        count = BLOCK * max(_blocks(p + x) - p // BLOCK for p, x in zip(past, new))
        held = sum(p + x - p // BLOCK * BLOCK for p, x in zip(past, new))
        # rows in and codes out, then the touched blocks' codes in and values out
        return {"bytes": 2 * h * d * (rows * (size + 1) + held + case["batch"] * count * size), "flops": 4 * h * d * rows}
    pairs = keys = 0
    for p, x, e in zip(past, new, lost):
        pairs += sum(_seen(case, p + i, e) for i in range(x))
        span = p + x - BLOCK * e
        keys += min(span, case["window"] + x - 1 + case["prefix"]) if case["window"] else span
    more = 8 * case["batch"] * h * keys // BLOCK if case["weights"] else 0
    return {"bytes": 2 * h * d * keys + 2 * rows * case["heads"] * d * size + more, "flops": 4 * d * case["heads"] * pairs}


def _exact_append(s):
    c = s["case"]
    d, h, batch = c["head_dim"], c["kv_heads"], c["batch"]
    past, new, _ = _lengths(c)
    scales = s["scales"].double()
    shown = [torch.zeros((batch, s["count"], h, d), dtype=torch.float64, device="cuda") for _ in range(2)]
    t = torch.arange(BLOCK, device="cuda")
    lay = torch.arange(d, device="cuda")
    at_k = (lay // 64 * BLOCK)[None, :] * 64 + t[:, None] * 64 + lay % 64
    at_v = ((lay // 32 * 16 + lay % 16)[None, :] * 4 + (t // 4 % 4)[:, None]) * 16 + ((lay // 16 % 2)[None, :] * 2 + (t // 16)[:, None]) * 4 \
        + (t % 4)[:, None] + BLOCK * d
    begin = 0
    for b in range(batch):
        lead = past[b] % BLOCK
        n = _blocks(past[b] + new[b]) - past[b] // BLOCK
        page = s["table"][b, :, past[b] // BLOCK:past[b] // BLOCK + n].long()
        for i, (x, at) in enumerate(((s["k"], at_k), (s["v"], at_v))):
            full = torch.zeros((n * BLOCK, h, d), dtype=torch.float64, device="cuda")
            full[lead:lead + new[b]] = x[begin:begin + new[b]].double()
            blocks = full.view(n, BLOCK, h, d).permute(2, 0, 1, 3)
            scale = (blocks.abs().amax((2, 3)) / 127).clamp_min(SCALE_FLOOR)
            old = s["pages"][page[:, 0]][:, at].double()
            if lead:
                scale[:, 0] = torch.maximum(scale[:, 0], scales[page[:, 0], i])
            value = torch.round(blocks / scale[:, :, None, None]).clamp(-127, 127) * scale[:, :, None, None]
            if lead:
                ratio = (scales[page[:, 0], i] / scale[:, 0])[:, None, None]
                value[:, 0, :lead] = torch.round(old[:, :lead] * ratio) * scale[:, 0, None, None]
            shown[i][b, :n * BLOCK] = value.permute(1, 2, 0, 3).reshape(n * BLOCK, h, d)
            shown[i][b, lead + new[b]:] = 0
            scales[page, i] = scale
        begin += new[b]
    return {"k": shown[0], "v": shown[1], "scales": scales, "starts": None, "weights": None}


def _exact_attend(s):
    c = s["case"]
    d, h, g = c["head_dim"], c["kv_heads"], c["heads"] // c["kv_heads"]
    past, new, lost = _lengths(c)
    if sum(x * (p + x) for p, x in zip(past, new)) * c["heads"] * d > 1.2e11:
        return None
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    weights = s["weights"].double().clone() if c["weights"] else None
    lay, t = torch.arange(d, device="cuda"), torch.arange(BLOCK, device="cuda")
    at_k = (lay // 64 * BLOCK)[None, :] * 64 + t[:, None] * 64 + lay % 64
    at_v = ((lay // 32 * 16 + lay % 16)[None, :] * 4 + (t // 4 % 4)[:, None]) * 16 + ((lay // 16 % 2)[None, :] * 2 + (t // 16)[:, None]) * 4 \
        + (t % 4)[:, None] + BLOCK * d
    begin = 0
    for b in range(c["batch"]):
        total = past[b] + new[b]
        n = _blocks(total) - lost[b]
        qpos = torch.arange(past[b], total, device="cuda")
        for head in range(h):
            page = s["table"][b, head, :n].long()
            keys = s["pages"][page][:, at_k].double() * s["scales"][page, 0].double()[:, None, None]
            values = s["pages"][page][:, at_v].double() * s["scales"][page, 1].double()[:, None, None]
            kpos = (s["starts"][b, head, :n, None] + t).reshape(-1)
            seen = kpos[None, :] <= qpos[:, None]
            if c["window"]:
                seen &= kpos[None, :] > qpos[:, None] - c["window"]
            if c["prefix"]:
                seen |= (kpos < min(c["prefix"], total))[None, :]
            seen &= (kpos < total)[None, :]
            for i in range(head * g, head * g + g):
                x = s["q"][begin:begin + new[b], i].double() @ keys.view(-1, d).T / math.sqrt(d)
                if c["softcap"]:
                    x = c["softcap"] * torch.tanh(x / c["softcap"])
                if s["slopes"] is not None:
                    x = x + s["slopes"][i].double() * (kpos[None, :] - qpos[:, None])
                p = torch.softmax(x.masked_fill(~seen, -math.inf), -1)
                out[begin:begin + new[b], i] = p @ values.view(-1, d)
                if weights is not None:
                    weights[b, head, :n] += p.sum(0).view(n, BLOCK).sum(1)
        begin += new[b]
    return {"out": out, "weights": weights} if c["weights"] else {"out": out}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "append":
        return _exact_append(s)
    if case["op"] == "attend":
        return _exact_attend(s)
    # rows by rows from the rule: what is kept, what leaves, what was never in use
    c, blocks = case, _spread(case, "blocks")
    if c["batch"] * c["kv_heads"] * max(blocks) > 4e6:
        return None
    w = s["weights"].cpu().double().tolist()
    for b, n in enumerate(blocks):
        for row in w[b] if n > c["budget"] else []:
            middle = sorted(range(EVICT_SINKS, n - EVICT_RECENT), key=lambda j: (-row[j], j))[:c["budget"] - EVICT_SINKS - EVICT_RECENT]
            keep = set(middle) | set(range(EVICT_SINKS)) | set(range(n - EVICT_RECENT, n))
            row[:n] = [row[j] for j in range(n) if j in keep] + [row[j] for j in range(n) if j not in keep]
    return [None, None, torch.tensor(w, dtype=torch.float64), None]
