"""Routing and the experts' products by their definitions (include/rocknpu_moe.h), in 64 bits on the host."""
import numpy as np


def route(logits, top_k, *, score="softmax", bias=None, groups=1, top_groups=None, group_top=1, normalise=True, factor=1.0):
    """ids, weights (64 bits), offsets, order; token by token, choice by choice."""
    x = logits.double().cpu().numpy()
    b = None if bias is None else bias.double().cpu().numpy()
    tokens, experts = x.shape
    size = experts // groups
    top_groups = groups if top_groups is None else top_groups
    ids, weights = np.full((tokens, top_k), -1, np.int32), np.zeros((tokens, top_k))
    for t in range(tokens):
        l = x[t]
        bad = bool((np.isnan(l) | (l == np.inf)).any())
        if bad:
            l = np.zeros(experts)
        with np.errstate(all="ignore"):
            if score == "softmax":
                p = np.exp(l - l.max()) if l.max() > -np.inf else np.zeros(experts)
                s = p / p.sum() if p.sum() > 0 else p
            else:
                s = 1.0 / (1.0 + np.exp(-l))
        choice = s if b is None or bad else s + b
        rank = l.copy() if b is None or bad else choice.copy()
        shut = np.isneginf(l) | np.isnan(choice)
        rank[shut] = -np.inf
        if groups > 1:
            v = rank if group_top == 1 else np.where(shut, -np.inf, l if bad else choice)
            of = []
            for g in range(groups):
                best = sorted(v[g * size:(g + 1) * size], reverse=True)[:group_top]
                of.append(-np.inf if best[-1] == -np.inf else sum(best))
            open_ = sorted(range(groups), key=lambda g: (-of[g], g))[:top_groups]
            for g in set(range(groups)) - set(open_):
                rank[g * size:(g + 1) * size] = -np.inf
        chosen = [e for e in sorted(range(experts), key=lambda e: (-rank[e], e)) if rank[e] > -np.inf][:top_k]
        w = s[chosen]
        if normalise:
            w = w / (w.sum() + 1e-20)
        ids[t, :len(chosen)] = chosen
        weights[t, :len(chosen)] = np.nan if bad else w * np.float64(np.float32(factor))
    flat = ids.reshape(-1)
    order = np.full(flat.size, -1, np.int32)
    offsets = np.zeros(experts + 1, np.int32)
    at = 0
    for e in range(experts):
        mine = np.nonzero(flat == e)[0]
        order[at:at + len(mine)] = mine
        at += len(mine)
        offsets[e + 1] = at
    return ids, weights, offsets, order


def a8(v):
    """Codes and scales of the rows of v (f32) by rocknpu_hip_quantize_a8's definition."""
    v = v.astype(np.float32)
    fine = np.isfinite(v).all(1) if v.shape[1] else np.ones(len(v), bool)
    v = np.where(fine[:, None], v, np.float32(0))
    peak = np.abs(v).max(1)
    step = np.where(peak == 0, np.float32(1), peak / np.float32(127)).astype(np.float32)
    q = (v / step[:, None]).astype(np.float64)
    codes = np.clip(np.copysign(np.floor(np.abs(q) + 0.5), q), -127, 127)
    return codes, np.where(fine, step, np.float32(np.nan))


def product(a, sa, w, sw):
    """(f32(sum) * row's scale) * column's scale, each in f32."""
    with np.errstate(all="ignore"):
        return ((a @ w.T).astype(np.float32) * sa[:, None].astype(np.float32)) * sw[None].astype(np.float32)


def experts(codes, scales, ids, weights, gate, up, down, hidden, ffn):
    """(out, the sum of its terms' magnitudes), 64 bits [tokens, hidden]; codes, scales and the pairs as moe.experts takes them."""
    c, sc = codes.cpu().numpy().astype(np.float64), scales.cpu().numpy()
    g, sg, u, su, d, sd = (x.cpu().numpy() for pair in (gate, up, down) for x in pair)
    out, size = np.zeros((c.shape[0], hidden)), np.zeros((c.shape[0], hidden))
    with np.errstate(all="ignore"):
        for e in range(g.shape[0]):
            t, s = np.nonzero(ids == e)
            if not len(t):
                continue
            x = product(c[t], sc[t], g[e].astype(np.float64), sg[e]).astype(np.float64)
            y = product(c[t], sc[t], u[e].astype(np.float64), su[e]).astype(np.float64)
            v, sv = a8((x * y / (1.0 + np.exp(-x))).astype(np.float32))
            r = product(v, sv, d[e][:, :ffn].astype(np.float64), sd[e]).astype(np.float64) * weights[t, s][:, None].astype(np.float64)
            np.add.at(out, t, r)
            np.add.at(size, t, np.abs(r))
    return out, size
