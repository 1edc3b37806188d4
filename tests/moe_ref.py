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
