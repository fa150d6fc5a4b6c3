"""Float64 restatements of the FP8 product, the mixture-of-experts layer, beam
selection and cache reordering (tbh_fp8_matmul_device, tbh_moe_device,
tbh_beam_select_device, tbh_paged_reorder_device), written from their
definitions in include/tinybrain_hip.h.  numpy only; nothing of the package."""
import math

import numpy as np

BLOCK, MOST = 128, 448.0


def e4m3_value(code):
    """Values of e4m3 bytes."""
    c = np.asarray(code).astype(np.int64)
    e, m = (c >> 3) & 15, c & 7
    v = np.where(e == 0, m * 2.0 ** -9, (1 + m / 8.0) * 2.0 ** (e - 7.0))
    v = np.where((c & 127) == 127, np.nan, v)
    return np.where(c >= 128, -v, v)


def round_e4m3(v):
    """The nearest e4m3 value, ties to even, of finite |v| <= 448."""
    a = np.abs(v)
    power = np.floor(np.log2(np.where(a < 2.0 ** -6, 2.0 ** -6, a)))
    step = 2.0 ** (power - 3)
    return np.copysign(np.rint(a / step) * step, v)


def quantize_rows(x):
    """(q, s) of rows x [M, K]: q [M, K] the e4m3 values, s [M, blocks] their scales."""
    x = np.asarray(x, np.float64)
    m, k = x.shape
    blocks = -(-k // BLOCK)
    q, s = np.empty_like(x), np.empty((m, blocks))
    for b in range(blocks):
        part = x[:, b * BLOCK:(b + 1) * BLOCK]
        most = np.where(np.isfinite(part), np.abs(part), 0.0).max(1)
        for r in range(m):
            e = -126
            while most[r] > MOST * 2.0 ** e:
                e += 1
            s[r, b] = 2.0 ** e
        with np.errstate(invalid="ignore"):
            v = np.where(np.isfinite(part), part / s[:, b:b + 1], np.nan)
            q[:, b * BLOCK:(b + 1) * BLOCK] = np.where(np.isnan(v), np.nan, round_e4m3(np.where(np.isnan(v), 1.0, v)))
    return q, s


def widen(data, scales):
    """The float64 matrix [N, K] of e4m3 bytes and block scales."""
    n, k = data.shape
    rows, cols = np.arange(n) // BLOCK, np.arange(k) // BLOCK
    return e4m3_value(data) * np.asarray(scales, np.float64)[rows[:, None], cols]


def fp8_matmul(x, data, scales):
    """(y, the sum of the magnitudes of its products, and the sum over the blocks
    of at least the largest of them)."""
    q, s = quantize_rows(x)
    xd = q * np.repeat(s, BLOCK, 1)[:, :q.shape[1]]
    w = widen(data, scales)
    largest = sum(np.abs(xd[:, b:b + BLOCK]).max(1)[:, None] * np.abs(w[:, b:b + BLOCK]).max(1)[None]
                  for b in range(0, w.shape[1], BLOCK))
    return xd @ w.T, np.abs(xd) @ np.abs(w.T), largest


def route(x, router, top_k, normalize):
    """(experts, weights) of rows x."""
    z = np.asarray(x, np.float64) @ np.asarray(router, np.float64).T
    experts = np.array([sorted(range(z.shape[1]), key=lambda e: (-row[e], e))[:top_k] for row in z]).reshape(-1, top_k)
    w = np.exp(z - z.max(1, keepdims=True))
    w /= w.sum(1, keepdims=True)
    w = np.take_along_axis(w, experts, 1)
    return experts, w / w.sum(1, keepdims=True) if normalize else w


def moe(x, router, gate, up, down, top_k, normalize, half_step):
    """(y, experts, weights, bound): gate, up, down are lists of (data, scales)
    per expert; bound: how far fp32 sums with exact products, and an h rounded by
    half_step relative, may be from y (before y's own rounding)."""
    x = np.asarray(x, np.float64)
    experts, weights = route(x, router, top_k, normalize)
    y, bound = np.zeros_like(x), np.zeros_like(x)
    unit = 2.0 ** -23                      # a fp32 addition, rounded or cut
    for t in range(len(x)):
        for j, e in enumerate(experts[t]):
            g, u, d = (widen(*m[e]) for m in (gate, up, down))
            c = (x.shape[1] * 3 + 16) * unit       # three pieces of fp32 each
            gv, uv = g @ x[t], u @ x[t]
            ge, ue = c * (np.abs(g) @ np.abs(x[t])), c * (np.abs(u) @ np.abs(x[t]))
            silu = gv / (1 + np.exp(-gv))
            h = silu * uv
            # |silu'| < 1.1; exp, division and products: a few steps
            he = 1.1 * ge * (np.abs(uv) + ue) + np.abs(silu) * ue + np.abs(h) * (16 * unit + half_step)
            p = weights[t, j]
            y[t] += p * (d @ h)
            ad = np.abs(d)
            bound[t] += p * (ad @ he + ((d.shape[1] * 3 + 32 * top_k) * unit) * (ad @ (np.abs(h) + he)))
    return y, experts, weights, bound


def beam_select(logits, scores, beams, k, done=None, eos=-1):
    """(tokens, parents, scores, done), each [requests, k]."""
    x = np.asarray(logits, np.float64)
    rows, vocab = x.shape
    out = [[], [], [], []]
    for r in range(0, rows, beams):
        found = []
        for b in range(r, r + beams):
            score = float(scores[b])
            if not math.isfinite(score):
                continue
            if done is not None and done[b]:
                found.append((-score, b, eos))
                continue
            v = np.where(np.isnan(x[b]), -np.inf, x[b])
            top = v.max()
            if top == -np.inf:
                continue
            if top == np.inf:
                v = np.where(v == np.inf, 0.0, -np.inf)
                total = math.log(np.count_nonzero(v == 0.0))
            else:
                total = top + math.log(np.exp(v - top).sum())
            key = score + (v - total)
            best = np.lexsort((np.arange(vocab), -key))[:k]
            found += [(-key[j], b, int(j)) for j in best if v[j] > -np.inf]
        found = sorted(found)[:k]
        ended = [j == eos or bool(done is not None and done[b]) for _, b, j in found]
        rest = k - len(found)
        out[0].append([j for _, _, j in found] + [-1] * rest)
        out[1].append([b for _, b, _ in found] + [-1] * rest)
        out[2].append([-f for f, _, _ in found] + [-math.inf] * rest)
        out[3].append([int(e) for e in ended] + [0] * rest)
    return tuple(np.array(o).reshape(-1, k) for o in out)


def reorder(table, parents, context, beams, block, blocks, shared=None):
    """(new table, moves, reordered): moves (from block, to block, rows)."""
    table, new = np.asarray(table), np.array(table)
    moves, fine = [], []
    for g in range(0, len(parents), beams):
        group = range(g, g + beams)
        ok = all(p < 0 or p in group for p in parents[g:g + beams]) and len(set(context[g:g + beams])) == 1
        fine.append(int(ok))
        if not ok:
            continue
        holder = {}
        for p in group:
            children = [c for c in group if parents[c] == p]
            if children:
                holder[p if p in children else children[0]] = p
        spare = [p for p in group if p not in holder.values()]
        for c in group:
            if c in holder:
                new[c] = table[holder[c]]
                continue
            new[c] = table[spare.pop(0)]
            if parents[c] < 0:
                continue
            length = min(max(int(context[c]), 0), table.shape[1] * block)
            for at in range((max(int(shared[g // beams]), 0) if shared is not None else 0) // block, -(-length // block)):
                a, b = int(table[parents[c], at]), int(new[c, at])
                if 0 <= a < blocks and 0 <= b < blocks:
                    moves.append((a, b, min(block, length - at * block)))
    return new, moves, np.array(fine)
