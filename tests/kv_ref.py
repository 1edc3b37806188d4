"""Plain forms of the 8-bit key/value cache's operators for the tests: the
definitions of include/rocknpu_kv.h written out token by token on the CPU, in
64 bits where numbers are computed."""
import math

import numpy as np
import torch

BLOCK = 32
FLOOR = np.float32(2.0 ** -100)


def key_index(d):
    """Byte offsets [32, d] of a page's keys, from the header's layout."""
    t, e = np.arange(BLOCK)[:, None], np.arange(d)[None, :]
    return (e // 64) * (BLOCK * 64) + t * 64 + e % 64


def value_index(d):
    """Byte offsets [32, d] of a page's values, behind its keys."""
    t, e = np.arange(BLOCK)[:, None], np.arange(d)[None, :]
    at = e // 32
    for bits, n in ((e % 16, 16), (t // 4 % 4, 4), (e // 16 % 2, 2), (t // 16, 2), (t % 4, 4)):
        at = at * n + bits
    return BLOCK * d + at


class Ref:
    """A cache's contents on the CPU."""

    def __init__(self, cache):
        self.d = cache.head_dim
        self.pages = cache.pages.view(torch.int8).cpu().numpy().copy()
        self.scales = cache.scales.cpu().numpy().copy()
        self.table = cache.table.cpu().numpy().copy()
        self.starts = cache.starts.cpu().numpy().copy()
        self.dropped = cache.dropped.cpu().numpy().copy()
        self.weights = None if cache.weights is None else cache.weights.cpu().numpy().copy()

    def held(self, b, tokens):
        return -(-tokens // BLOCK) - int(self.dropped[b])

    def codes(self, page):
        return self.pages[page][key_index(self.d)], self.pages[page][value_index(self.d)]

    def values(self, page):
        """Keys and values of a page; a scale that is not finite makes them NaN."""
        k, v = self.codes(page)
        sk, sv = (float(x) if np.isfinite(x) else np.nan for x in self.scales[page])
        return k.astype(np.float64) * sk, v.astype(np.float64) * sv

    def append(self, k, v, past, cu):
        """k, v: float32 [rows, heads, d] (f16 and bf16 are exact in it)."""
        for b in (b for b in range(len(past)) if cu[b + 1] > cu[b]):
            for h in range(self.table.shape[1]):
                for j in range(past[b] // BLOCK, -(-(past[b] + cu[b + 1] - cu[b]) // BLOCK)):
                    self._append(k, v, past[b], cu[b], cu[b + 1] - cu[b], b, h, j)

    def _append(self, k, v, past, row0, n, b, h, j):
        lead, end = max(past - BLOCK * j, 0), min(past + n - BLOCK * j, BLOCK)
        at = j - int(self.dropped[b])
        page = self.table[b, h, at]
        rows = slice(row0 + BLOCK * j + lead - past, row0 + BLOCK * j + end - past)
        for i, (x, index) in enumerate(((k, key_index(self.d)), (v, value_index(self.d)))):
            new = x[rows, h].astype(np.float32)
            before = self.scales[page, i] if lead else np.float32(0)
            code = np.zeros((BLOCK, self.d), np.int8)
            if np.isfinite(new).all() and np.isfinite(before):
                scale = max(np.float32(np.abs(new).max() / np.float32(127)), before, FLOOR)
                inv, again = np.float32(1) / scale, before / scale
                code[lead:end] = np.clip(np.rint(new * inv), -127, 127)
                code[:lead] = np.rint(self.pages[page][index][:lead].astype(np.float32) * again)
            else:
                scale = np.float32(np.nan)
            self.pages[page][index[:end]] = code[:end]
            self.scales[page, i] = scale
        if lead == 0:
            self.starts[b, h, at] = BLOCK * j
            if self.weights is not None:
                self.weights[b, h, at] = 0

    def attention(self, q, past, cu, scale=None, causal=True, window=0, prefix=None, softcap=0.0, slopes=None):
        """out, its magnitude sum(p |v|), the scores' magnitude and the blocks' weights, all f64.
        q: float64 [rows, heads, d]."""
        rows, heads, d = q.shape
        scale = 1 / math.sqrt(d) if scale is None else scale
        group = heads // self.table.shape[1]
        out, mag, big = np.zeros(q.shape), np.zeros(q.shape), np.zeros((rows, heads))
        weights = np.zeros(self.table.shape)
        for b in range(len(past)):
            n = cu[b + 1] - cu[b]
            total = past[b] + n
            held = self.held(b, total)
            if n == 0 or held <= 0:
                continue
            qpos = (past[b] + np.arange(n))[:, None]
            for h in range(self.table.shape[1]):
                pages = self.table[b, h, :held]
                kv = [self.values(p) for p in pages]
                keys, values = (np.concatenate([x[i] for x in kv]) for i in (0, 1))
                kpos = (self.starts[b, h, :held, None] + np.arange(BLOCK)).reshape(1, -1)
                seen = kpos <= qpos if causal else np.ones((n, kpos.size), bool)
                if window:
                    seen = seen & (kpos > qpos - window)
                if prefix is not None:
                    seen = seen | (kpos < prefix[b])
                seen = seen & (kpos < total)
                for head in range(h * group, (h + 1) * group):
                    qh = q[cu[b]:cu[b + 1], head]
                    x = scale * (qh @ keys.T)
                    if softcap:
                        x = softcap * np.tanh(x / softcap)
                    if slopes is not None:
                        x = x + float(slopes[head]) * (kpos - qpos)
                    x = np.where(seen, x, -np.inf)
                    top = np.fmax.reduce(x, 1, keepdims=True)
                    e = np.where(seen, np.exp(x - np.where(top == -np.inf, 0, top)), 0.0)
                    total_e = e.sum(1, keepdims=True)
                    p = e / np.where(total_e == 0, 1, total_e)
                    r = slice(cu[b], cu[b + 1])
                    # a NaN or infinite value counts only where it is seen
                    masked = np.where(np.isfinite(values), values, 0)
                    out[r, head] = p @ masked + np.where((seen.astype(float) @ ~np.isfinite(values)) > 0, np.nan, 0)
                    mag[r, head] = p @ np.abs(masked)
                    terms = abs(scale) * (np.abs(qh) @ np.abs(np.where(np.isfinite(keys), keys, 0)).T)
                    if slopes is not None:
                        terms = terms + abs(float(slopes[head])) * np.abs(kpos - qpos)
                    big[r, head] = np.where(seen, terms, 0).max(1)
                    weights[b, h, :held] += p.sum(0).reshape(held, BLOCK).sum(1)
        return out, mag, big, weights


def evict(table, starts, weights, tokens, dropped, budget, sinks, recent):
    table, starts, weights = (t.copy() for t in (table, starts, weights))
    gone = dropped.copy()
    for b in range(table.shape[0]):
        n = -(-int(tokens[b]) // BLOCK) - int(dropped[b])
        if n <= budget:
            continue
        gone[b] += n - budget
        for h in range(table.shape[1]):
            w = [-math.inf if math.isnan(x) else float(x) for x in weights[b, h, :n]]
            nan = [math.isnan(x) for x in weights[b, h, :n]]
            middle = sorted(range(sinks, n - recent), key=lambda j: (nan[j], -w[j], j))[:budget - sinks - recent]
            keep = sorted(set(middle) | set(range(sinks)) | set(range(n - recent, n)))
            order = keep + [j for j in range(n) if j not in set(keep)] + list(range(n, table.shape[2]))
            for x in (table, starts, weights):
                x[b, h] = x[b, h, order]
    return table, starts, weights, gone
