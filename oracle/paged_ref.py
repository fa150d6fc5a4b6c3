"""Oracle for the paged-cache serving calls -- TEST INFRASTRUCTURE ONLY.

numpy restatements of what tbh_paged_plan_device, tbh_paged_append_device,
tbh_paged_attention_device and tbh_sample* are defined to compute, one request
(or row) after the other in float64.  Nothing in the product imports it.

Follows (vivekptnk/tinybrain):
  * rotate     Sources/TinyBrainRuntime/ModelRunner.swift:470-494 (interleaved
               pairs), with the angle of real arithmetic
  * attention  ModelRunner.swift:519-579 (scores over the cached positions up
               to the query's own, softmax, weighted values)
  * sample     Sources/TinyBrainRuntime/Sampler.swift (temperature, top-k,
               top-p), with the random number given
Pins against closed forms are in tests/test_paged_oracle.py.
"""
from __future__ import annotations

import numpy as np


def ceil_div(a: int, b: int) -> int:
    return -(-a // b)


def plan(new, context, table, free, count, block, max_tokens):
    """Returns a dict of the outputs; table and free are copies, updated."""
    table, stack, height = table.copy(), free.copy(), int(count)
    for b, n in enumerate(new):
        if n < 0:
            for j in range(ceil_div(int(context[b]), block)):
                stack[height] = table[b, j]
                height += 1
    start, granted, out = [0], [], []
    slots, positions = np.full(max_tokens, -1, np.int32), np.full(max_tokens, -1, np.int32)
    asked = taken = 0
    for b, n in enumerate(new):
        more, c = max(int(n), 0), int(context[b])
        fits = more > 0 and c + more <= table.shape[1] * block and start[-1] + more <= max_tokens
        need = ceil_div(c + more, block) - ceil_div(c, block) if fits else 0
        ok = fits and (need == 0 or asked + need <= height)
        if ok:
            for j in range(need):
                table[b, ceil_div(c, block) + j] = stack[height - 1 - asked - j]
            taken += need
            for i in range(more):
                t, p = start[-1] + i, c + i
                slots[t] = table[b, p // block] * block + p % block
                positions[t] = p
        asked += need
        granted.append(more if ok else 0)
        out.append(0 if n < 0 else c + granted[-1])
        start.append(start[-1] + more)
    return {"start": np.array(start, np.int32), "granted": np.array(granted, np.int32),
            "context": np.array(out, np.int32), "slots": slots, "positions": positions, "count": height - taken,
            "table": table, "free": stack}


def rotate(x, positions, heads, base):
    """x [tokens, heads * hd] -> float64, interleaved pairs."""
    x = np.asarray(x, np.float64)
    t, hd = x.shape[0], x.shape[1] // heads
    angle = np.maximum(np.asarray(positions, np.float64), 0)[:, None] * float(base) ** (-2.0 * np.arange(hd // 2) / hd)
    c, s = np.cos(angle)[:, None], np.sin(angle)[:, None]
    p = x.reshape(t, heads, hd // 2, 2)
    return np.stack([p[..., 0] * c - p[..., 1] * s, p[..., 0] * s + p[..., 1] * c], -1).reshape(x.shape)


def append(cache, rows, slots):
    """cache [blocks, kv heads, block, hd] float64 with rows [tokens, kv heads * hd] at their slots."""
    out = cache.copy()
    blocks, nkv, bs, hd = cache.shape
    for t, slot in enumerate(slots):
        if 0 <= slot < blocks * bs:
            out[slot // bs, :, slot % bs] = rows[t].reshape(nkv, hd)
    return out


def attention(q, keys, values, table, start, context, heads, scale=None):
    """q [tokens, heads * hd] float64; returns (out, bound), both [tokens,
    heads * hd] float64: the result (NaN in rows behind the last request) and,
    per element, an error that fp32 arithmetic of this formula stays below
    (see _bound)."""
    q = np.asarray(q, np.float64)
    blocks, nkv, bs, hd = keys.shape
    rep, scale = heads // nkv, 1.0 / np.sqrt(hd) if scale is None else scale
    out, bound = np.full((q.shape[0], heads, hd), np.nan), np.zeros((q.shape[0], heads, hd))
    x = q.reshape(-1, heads, hd)
    for b in range(len(context)):
        n = start[b + 1] - start[b]
        pages = table[b, :ceil_div(int(context[b]), bs)]
        ok = np.repeat((pages >= 0) & (pages < blocks), bs)[:context[b]]
        where = np.clip(pages, 0, blocks - 1)
        k = np.moveaxis(keys[where], 1, 0).reshape(nkv, -1, hd)[:, :context[b]]
        v = np.moveaxis(values[where], 1, 0).reshape(nkv, -1, hd)[:, :context[b]]
        for i in range(n):
            last = context[b] - n + i
            seen = np.flatnonzero(ok[:max(last + 1, 0)])
            t = start[b] + i
            if t >= q.shape[0]:
                break
            if not len(seen):
                out[t] = 0.0
                continue
            for h in range(heads):
                kk, vv = k[h // rep, seen], v[h // rep, seen]
                with np.errstate(invalid="ignore", over="ignore"):
                    s = kk @ x[t, h] * scale
                    e = np.exp(s - s.max())
                    p = e / e.sum()
                    out[t, h] = p @ vv
                    bound[t, h] = _bound(kk, vv, x[t, h], scale, s, p)
    return out.reshape(q.shape), bound.reshape(q.shape)


U = 2.0 ** -24   # half a step of fp32, relative


def _bound(k, v, q, scale, s, p):
    """A score is a sum of hd products, each and each sum rounded once, then
    scaled: off by at most (hd + 2) U of sum |q k| scale.  exp takes the
    difference to the maximum (one rounding, U of it) and is good to 2 U
    itself.  So p's relative error is at most 2 e + 4 U with e the largest of
    these (the other half is the maximum's and the sum's), and sums over n
    positions add n U of sum p |v|, as does the division's U."""
    e = np.max((len(q) + 2) * U * (np.abs(k) @ np.abs(q)) * abs(scale) + U * np.abs(s - s.max()))
    return (2 * e + (len(s) + 8) * U) * (p @ np.abs(v))


def sample(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """One row: (token, probability).  Weights that are summed count in whole
    steps of 2^-43 of the largest."""
    x = np.asarray(logits, np.float64)
    x = np.where(np.isnan(x), -np.inf, x)
    if not len(x) or x.max() == -np.inf:
        return -1, 0.0
    if not temperature > 0:
        return int(np.argmax(x)), 1.0
    order = np.lexsort((np.arange(len(x)), -x))
    order = order[x[order] > -np.inf]
    if top_k > 0:
        order = order[:top_k]
    top = x[order[0]]

    def weight(i):
        if top == np.inf:
            return np.where(x[i] == np.inf, 1.0, 0.0)
        return np.exp((x[i] - top) * (1.0 / np.float64(temperature)))

    def running(w):
        return np.cumsum(np.floor(w * 2.0 ** 43 + 0.5) * 2.0 ** -43)

    if top_p < 1:
        c = running(weight(order))
        order = order[:max(1, 1 + int(np.sum(c[:-1] < np.float64(top_p) * c[-1])))]
    if min_p > 0:
        keep = weight(order) >= min_p
        keep[0] = True
        order = order[keep]
    kept = np.sort(order)
    c = running(weight(kept))
    at = min(max(float(u), 0.0), 1 - 2.0 ** -24) * c[-1]
    j = int(np.searchsorted(c, at, side="right"))
    return int(kept[j]), weight(kept[j:j + 1])[0] / c[-1]
