"""The operators that serve many requests from one paged key/value cache, with
their plain forms: planning a step (block tables, slots and positions on the
GPU), appending rows to the cache, attention of new tokens over it, and drawing
tokens from logits.

``listed()`` names fixed cases, ``draw(rng)`` gives another of the same ranges;
``prepare`` builds what a serving program holds before the call, ``run`` is one
pass through one operator, ``exact`` the same from its definition in float64,
``work`` the bytes and operations one pass cannot do without.

A cache of one layer is two arrays [blocks][kv heads][block size][head dim].
Request b's position p is in block ``table[b][p // block]`` at row ``p % block``;
its slot is ``table[b][p // block] * block + p % block``.
"""
import math
import random

import numpy as np
import torch

own = False

_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
_BASE = 10000.0       # of the rotary angles

_backend = None


def backend():
    """The one HIPBackend of the process, as a program keeps it."""
    global _backend
    if _backend is None:
        import tinybrain_amd as tb
        _backend = tb.HIPBackend(0)
    return _backend


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def _step(op, single, chunks, new, past, spread, block, heads, kv_heads, head_dim, x, cache):
    """A step's requests: `single` with one new token each, `chunks` with about
    `new` (their lengths vary down to half of it), cached lengths between the two of `past`."""
    return {"op": op, "single": single, "chunks": chunks, "new": new, "past_lo": past[0], "past_hi": past[1],
            "spread": spread, "block": block, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim,
            "x": x, "cache": cache}


def _sample(rows, vocab, mix):
    return {"op": "sample", "rows": rows, "vocab": vocab, "mix": mix}


def listed():
    return [
        # one more token for each of 64 requests: the plan of a decode step
        dict(_step("plan", 64, 0, 0, (16, 4096), 1, 16, 32, 4, 64, "f32", "f32"), name="plan_decode_64"),
        # a step that takes in prompts beside many running requests
        dict(_step("plan", 960, 40, 700, (0, 8192), 2, 16, 32, 4, 64, "f32", "f32"), name="plan_mixed_1000"),
        # eight running requests' rows of q, k, v into an fp32 cache
        dict(_step("append", 8, 0, 0, (16, 512), 3, 16, 32, 4, 64, "f32", "f32"), name="append_decode_8"),
        # a long prompt's rows into a bf16 cache, q kept in bf16 for the attention
        dict(_step("append", 0, 1, 4096, (0, 0), 4, 16, 32, 8, 128, "bf16", "bf16"), name="append_prompt_4096"),
        # one new token over a long fp32 cache, the decode step's own types
        dict(_step("attention", 1, 0, 0, (4095, 4095), 5, 16, 32, 4, 64, "f32", "f32"), name="attn_decode_1"),
        # a decode step of 64 requests of very different lengths, bf16 cache
        dict(_step("attention", 64, 0, 0, (100, 8192), 6, 16, 32, 8, 128, "f32", "bf16"), name="attn_decode_64"),
        # a step of 31 single tokens and a prompt chunk, fp32 throughout
        dict(_step("attention", 31, 1, 333, (50, 2000), 7, 16, 32, 4, 64, "f32", "f32"), name="attn_mixed_f32"),
        # the second half of a long prompt over the first, bf16 throughout
        dict(_step("attention", 0, 1, 2048, (2048, 2048), 8, 16, 32, 8, 128, "bf16", "bf16"), name="attn_chunk_2048"),
        # prompts of odd lengths with no shared heads, fp32 rows over a bf16 cache
        dict(_step("attention", 3, 5, 301, (0, 700), 9, 32, 12, 12, 64, "f32", "bf16"), name="attn_prompts_odd"),
        # the next token of one sequence: a chat's usual settings
        dict(_sample(1, 32000, "all"), name="sample_1"),
        # a batch whose requests each bring their own settings
        dict(_sample(64, 32000, "each"), name="sample_64_each"),
        # a large batch over a large vocabulary, top-p alone
        dict(_sample(256, 100000, "top_p"), name="sample_256_large"),
    ]


def _log(rng, lo, hi, step=1):
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return max(lo, min(hi, int(round(v / step)) * step))


def draw(rng):
    op = rng.choice(("plan", "append", "attention", "attention", "attention", "sample", "sample"))
    if op == "sample":
        return _sample(_log(rng, 1, 256), _log(rng, 1000, 100000), rng.choice(("all", "each", "top_k", "top_p", "plain")))
    heads = rng.choice(((32, 4, 64), (32, 32, 128), (32, 8, 128), (12, 12, 64), (8, 2, 32)))
    block, spread = rng.choice((16, 16, 32, 64)), rng.randrange(1 << 20)
    x, cache = rng.choice((("f32", "f32"), ("f32", "bf16"), ("bf16", "bf16")))
    if op == "plan":
        single, chunks = _log(rng, 1, 960), rng.choice((0, 0, _log(rng, 1, 40)))
        case = _step(op, single, chunks, _log(rng, 16, 700), (0, _log(rng, 64, 8192)), spread, block, *heads, x, cache)
    elif op == "append":
        single, chunks = _log(rng, 1, 64), rng.choice((0, 0, 1, 2))
        case = _step(op, single, chunks, _log(rng, 16, 4096), (0, _log(rng, 16, 512)), spread, block, *heads, x, cache)
    elif rng.random() < 0.5:                  # a decode step
        hi = _log(rng, 64, 8192)
        case = _step(op, _log(rng, 1, 64), 0, 0, (hi // rng.choice((1, 2, 16)), hi), spread, block, *heads, x, cache)
    else:
        case = _step(op, rng.choice((0, 0, _log(rng, 1, 32))), rng.choice((1, 1, 2, 5)), _log(rng, 16, 2048),
                     (0, _log(rng, 16, 4096)), spread, block, *heads, x, cache)
    top = _MOST[op]
    while any(v > m for v, m in zip(work(case).values(), top)):      # no dearer than the largest listed one
        case["single"], case["new"] = (case["single"] + 1) // 2, max(16, case["new"] * 3 // 4)
        if case["new"] == 16:
            case["past_lo"], case["past_hi"] = case["past_lo"] // 2, case["past_hi"] // 2
    return case


_MOST = {"plan": (217296, 98928), "append": (100696064, 62914560), "attention": (470265856, 103095992320)}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _lens(case):
    """Per request (new, past)."""
    rng = random.Random(case["spread"])

    def past():
        lo, hi = case["past_lo"], case["past_hi"]
        return lo if lo == hi else int(round(math.exp(rng.uniform(math.log(lo + 1), math.log(hi + 1))))) - 1

    out = [(1, past()) for _ in range(case["single"])]
    for i in range(case["chunks"]):
        out.insert(rng.randrange(len(out) + 1), (case["new"] - (rng.randrange(case["new"] // 2) if i else 0), past()))
    return out


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _normal(gen, *shape, std=1.0, dtype=torch.float32):
    return (torch.randn(*shape, generator=gen, device="cuda", dtype=torch.float32) * std).to(dtype)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _blocks(tokens, block):
    return (tokens + block - 1) // block


def _pool(case, seed, with_new):
    """A table of blocks in no order, and how many blocks there are."""
    lens, bs = _lens(case), case["block"]
    held = [_blocks(p + (n if with_new else 0), bs) for n, p in lens]
    spare = sum(_blocks(p + n, bs) for n, p in lens) - sum(held) + 8
    count = sum(held) + spare
    order = np.random.default_rng(seed).permutation(count).astype(np.int32)
    most = max(_blocks(p + n, bs) for n, p in lens) + 1
    table = np.full((len(lens), most), -1, np.int32)
    at = 0
    for b, h in enumerate(held):
        table[b, :h] = order[at:at + h]
        at += h
    return lens, count, table, order[at:]


def _query_start(lens):
    return [0] + np.cumsum([n for n, _ in lens]).tolist()


def _plan_inputs(case, seed):
    lens, count, table, free = _pool(case, seed, False)
    rng = np.random.default_rng(seed + 1)
    # the released requests of the step before, one in sixteen
    new = [-1 if n == 1 and rng.random() < 1 / 16 else n for n, _ in lens]
    stack = np.zeros(count, np.int32)
    stack[:len(free)] = free
    return {"op": "plan", "block": case["block"], "new": _ints(new), "context": _ints([p for _, p in lens]),
            "table": _ints(table), "free": _ints(stack), "height": _ints([len(free)]),
            "tokens": sum(n for n, _ in lens)}


def _cache(gen, count, case):
    shape = (count, case["kv_heads"], case["block"], case["head_dim"])
    return [_normal(gen, *shape, dtype=_TYPES[case["cache"]]) for _ in range(2)]


def _append_inputs(case, seed):
    lens, count, table, _ = _pool(case, seed, True)
    gen, bs, hd = _generator(seed), case["block"], case["head_dim"]
    keys, values = _cache(gen, count, case)
    positions = np.concatenate([np.arange(p, p + n) for n, p in lens])
    rows = np.repeat(np.arange(len(lens)), [n for n, _ in lens])
    slots = table[rows, positions // bs].astype(np.int64) * bs + positions % bs
    # q, k and v lie side by side in a row, as one projection writes them
    nq, nk = case["heads"] * hd, case["kv_heads"] * hd
    qkv = _normal(gen, len(rows), nq + 2 * nk, dtype=_TYPES[case["x"]])
    return {"op": "append", "keys": keys, "values": values, "slots": _ints(slots), "positions": _ints(positions),
            "q": qkv[:, :nq], "k": qkv[:, nq:nq + nk], "v": qkv[:, nq + nk:], "kv_heads": case["kv_heads"]}


def _attention_inputs(case, seed):
    lens, count, table, _ = _pool(case, seed, True)
    gen, starts = _generator(seed), _query_start(lens)
    keys, values = _cache(gen, count, case)
    # scores of standard deviation 2: some positions matter more than others
    q = _normal(gen, starts[-1], case["heads"] * case["head_dim"], std=2.0, dtype=_TYPES[case["x"]])
    return {"op": "attention", "q": q, "keys": keys, "values": values, "table": _ints(table),
            "start": _ints(starts), "context": _ints([n + p for n, p in lens]), "heads": case["heads"],
            "lens": lens, "most_new": max(n for n, _ in lens), "most_context": max(n + p for n, p in lens)}


def _sample_inputs(case, seed):
    gen, rng = _generator(seed), random.Random(seed)
    rows, mix = case["rows"], case["mix"]
    logits = _normal(gen, rows, case["vocab"], std=2.5)
    u = torch.rand(rows, generator=gen, device="cuda", dtype=torch.float32)
    t, k, p, m = [], [], [], []
    for _ in range(rows):
        kind = rng.choice(("greedy", "top_k", "top_p", "all", "plain", "min_p")) if mix == "each" else mix
        t.append(0.0 if kind == "greedy" else rng.choice((0.6, 0.7, 0.8, 1.0, 1.3)))
        k.append(rng.choice((1, 20, 40, 50, 200)) if kind in ("top_k", "all") else 0)
        p.append(rng.choice((0.5, 0.8, 0.9, 0.95, 0.99)) if kind in ("top_p", "all") else 1.0)
        m.append(rng.choice((0.01, 0.05, 0.1)) if kind in ("min_p", "all") else 0.0)

    def floats(v):
        return torch.tensor(v, dtype=torch.float32, device="cuda")

    return {"op": "sample", "logits": logits, "u": u, "temperature": floats(t), "top_k": _ints(k),
            "top_p": floats(p), "min_p": floats(m)}


_INPUTS = {"plan": _plan_inputs, "append": _append_inputs, "attention": _attention_inputs, "sample": _sample_inputs}


def prepare(case, seed):
    return _INPUTS[case["op"]](case, seed)


# ---------------------------------------------------------------------------
# a pass
# ---------------------------------------------------------------------------
def run(state):
    if own:
        return _OWN[state["op"]](backend(), state)
    return _PLAIN[state["op"]](state)


def _own_plan(be, s):
    p = be.paged_plan_device(s["new"], s["context"], s["table"], s["free"], s["height"], s["block"], s["tokens"])
    return {"start": p.queryStart, "context": p.contextLens, "granted": p.granted, "slots": p.slots,
            "positions": p.positions, "height": p.freeCount, "table": s["table"], "free": s["free"]}


def _own_append(be, s):
    q = be.paged_append_device(s["keys"], s["values"], s["slots"], s["k"], s["v"], q=s["q"], positions=s["positions"],
                               ropeBase=_BASE)
    return {"q": q, "keys": s["keys"], "values": s["values"]}


def _own_attention(be, s):
    return be.paged_attention_device(s["q"], s["keys"], s["values"], s["table"], s["start"], s["context"], s["heads"],
                                     maxQueryLen=s["most_new"], maxContextLen=s["most_context"])


def _own_sample(be, s):
    token, prob = be.sample_device(s["logits"], s["u"], temperature=s["temperature"], topK=s["top_k"],
                                   topP=s["top_p"], minP=s["min_p"])
    return {"token": token, "prob": prob}


_OWN = {"plan": _own_plan, "append": _own_append, "attention": _own_attention, "sample": _own_sample}


def _plain_plan(s):
    new, past, table, free, height, bs = s["new"], s["context"], s["table"], s["free"], s["height"], s["block"]
    rows, most = table.shape
    # released requests give their blocks back, on top of the free ones
    held = (past + bs - 1) // bs
    column = torch.arange(most, device=new.device, dtype=torch.int32)
    gone = (new < 0)[:, None] & (column < held[:, None])
    place = height + torch.cumsum(gone.flatten(), 0, dtype=torch.int32) - 1
    place = torch.where(gone.flatten(), place, free.numel())
    stack = torch.cat([free, free.new_zeros(1)])
    stack[place.long()] = table.flatten()            # the last entry takes what stays
    stack = stack[:-1]
    height = height + gone.sum(dtype=torch.int32)
    # who gets blocks, and which
    more = new.clamp(min=0)
    total = past + more
    fits = total <= most * bs
    need = torch.where(fits & (more > 0), (total + bs - 1) // bs - held, 0)
    upto = torch.cumsum(need, 0, dtype=torch.int32)
    ok = fits & (more > 0) & ((need == 0) | (upto <= height))
    taken = torch.where(ok, need, 0)
    before = upto - need
    index = column - held[:, None]
    fresh = ok[:, None] & (index >= 0) & (index < taken[:, None])
    source = (height - 1 - (before[:, None] + index)).clamp(0, free.numel() - 1)
    table = torch.where(fresh, stack[source.long()], table)
    granted = torch.where(ok, more, 0)
    context = torch.where(new < 0, 0, past + granted)
    start = torch.cat([new.new_zeros(1), torch.cumsum(more, 0, dtype=torch.int32)])
    # the tokens' rows
    t = torch.arange(s["tokens"], device=new.device, dtype=torch.int32)
    row = torch.searchsorted(start, t, right=True, out_int32=True) - 1
    live = row < rows
    row = row.clamp(max=rows - 1).long()
    p = past[row] + t - start[row]
    live &= ok[row]
    slot = table[row, (p // bs).clamp(max=most - 1).long()] * bs + p % bs
    return {"start": start, "context": context, "granted": granted, "slots": torch.where(live, slot, -1),
            "positions": torch.where(live, p, -1), "height": height - taken.sum(dtype=torch.int32),
            "table": table, "free": stack}


def _plain_rotate(x, positions, heads):
    # angles of far positions in 64 bits, the rest in 32
    t, hd = x.shape[0], x.shape[1] // heads
    i = torch.arange(0, hd, 2, device=x.device, dtype=torch.float64)
    angle = positions.double()[:, None] * torch.pow(_BASE, -i / hd)
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    pair = x.float().reshape(t, heads, hd // 2, 2)
    a, b = pair[..., 0], pair[..., 1]
    return torch.stack([a * cos - b * sin, a * sin + b * cos], -1).reshape(t, heads, hd)


def _plain_append(s):
    keys, values, n = s["keys"], s["values"], s["kv_heads"]
    bs, hd = keys.shape[2], keys.shape[3]
    slot = s["slots"].long()
    at = (slot // bs, slice(None), slot % bs)
    keys[at] = _plain_rotate(s["k"], s["positions"], n).to(keys.dtype)
    values[at] = s["v"].float().reshape(-1, n, hd).to(values.dtype)
    q = _plain_rotate(s["q"], s["positions"], s["q"].shape[1] // hd).to(s["q"].dtype)
    return {"q": q.reshape(s["q"].shape), "keys": keys, "values": values}


def _plain_attention(s):
    q, heads = s["q"], s["heads"]
    kv_heads, bs, hd = s["keys"].shape[1:]
    out = torch.empty_like(q)
    at = 0
    for b, (new, past) in enumerate(s["lens"]):
        ids = s["table"][b, :_blocks(new + past, bs)].long()
        k, v = (c[ids].float().transpose(0, 1).reshape(kv_heads, -1, hd)[:, :new + past]
                for c in (s["keys"], s["values"]))
        x = q[at:at + new].float().reshape(new, kv_heads, heads // kv_heads, hd).permute(1, 2, 0, 3)
        x = x.reshape(kv_heads, -1, hd)                          # rows: head of the group, token
        score = torch.matmul(x, k.transpose(1, 2)) / math.sqrt(hd)
        if new > 1:
            p = torch.arange(past, past + new, device=q.device)
            seen = torch.arange(new + past, device=q.device) <= p[:, None]
            score = score.reshape(kv_heads, -1, new, new + past).masked_fill(~seen, -math.inf).reshape(score.shape)
        e = torch.exp(score - score.amax(-1, keepdim=True))
        y = torch.matmul(e, v) / e.sum(-1, keepdim=True)
        y = y.reshape(kv_heads, heads // kv_heads, new, hd).permute(2, 0, 1, 3)
        out[at:at + new] = y.reshape(new, heads * hd).to(q.dtype)
        at += new
    return out


def _plain_sample(s):
    logits, u = s["logits"], s["u"]
    rows, vocab = logits.shape
    temperature, greedy = s["temperature"][:, None], s["temperature"][:, None] <= 0
    # sums whose borders decide a token: in 64 bits
    x = logits.double()
    w = torch.exp((x - x.amax(1, keepdim=True)) / torch.where(greedy, 1.0, temperature.double()))
    order = torch.sort(logits, dim=1, descending=True, stable=True).indices      # ties: the lowest index first
    sorted_w = torch.gather(w, 1, order)
    rank = torch.arange(vocab, device=logits.device)
    k = torch.where(greedy, 1, torch.where(s["top_k"][:, None] > 0, s["top_k"][:, None], vocab))
    keep = rank < k
    sorted_w = torch.where(keep, sorted_w, 0.0)
    upto = torch.cumsum(sorted_w, 1)
    p = s["top_p"].double()[:, None]
    keep &= (p >= 1) | (rank == 0) | (upto - sorted_w < p * upto[:, -1:])
    keep &= sorted_w >= s["min_p"].double()[:, None]
    w = torch.where(torch.zeros_like(keep).scatter(1, order, keep), w, 0.0)
    upto = torch.cumsum(w, 1)
    token = (upto <= u.double()[:, None] * upto[:, -1:]).sum(1)
    prob = torch.gather(w, 1, token[:, None])[:, 0] / upto[:, -1]
    return {"token": token.to(torch.int32), "prob": prob.float()}


_PLAIN = {"plan": _plain_plan, "append": _plain_append, "attention": _plain_attention, "sample": _plain_sample}


# ---------------------------------------------------------------------------
# floors, and the same in 64 bits
# ---------------------------------------------------------------------------
def work(case):
    op = case["op"]
    if op == "sample":
        rows, vocab = case["rows"], case["vocab"]
        return {"bytes": rows * (4 * vocab + 28), "flops": 4 * rows * vocab}
    lens, bs, hd = _lens(case), case["block"], case["head_dim"]
    tokens = sum(n for n, _ in lens)
    size = {"f32": 4, "bf16": 2}
    xb, cb = size[case["x"]], size[case["cache"]]
    if op == "plan":
        blocks = sum(_blocks(n + p, bs) - _blocks(p, bs) for n, p in lens)
        return {"bytes": len(lens) * 24 + blocks * 8 + tokens * 8, "flops": 4 * tokens + 8 * len(lens)}
    nq, nk = case["heads"] * hd, case["kv_heads"] * hd
    if op == "append":
        return {"bytes": tokens * (2 * nq * xb + 2 * nk * (xb + cb) + 8), "flops": tokens * 3 * (nq + nk)}
    pairs = sum(n * p + n * (n + 1) // 2 for n, p in lens)
    return {"bytes": 2 * tokens * nq * xb + sum(n + p for n, p in lens) * 2 * nk * cb,
            "flops": 4 * pairs * nq}


def exact(case, seed):
    return _EXACT[case["op"]](prepare(case, seed))


def _exact_plan(s):
    """One request after the other, as the definition says."""
    new, past, table, stack = (s[k].cpu().numpy().copy() for k in ("new", "context", "table", "free"))
    height, bs = int(s["height"][0]), s["block"]
    for b in range(len(new)):
        if new[b] < 0:
            for j in range(-(-int(past[b]) // bs)):
                stack[height] = table[b, j]
                height += 1
    top, asked = height, 0
    start, context, granted, slots, positions = [0], [], [], [], []
    for b in range(len(new)):
        n, p = max(int(new[b]), 0), int(past[b])
        have, want = -(-p // bs), -(-(p + n) // bs)
        need = want - have if n > 0 and want <= table.shape[1] else 0
        ok = n > 0 and want <= table.shape[1] and (need == 0 or asked + need <= height)
        if ok:
            for j in range(need):
                table[b, have + j] = stack[height - 1 - asked - j]
            top -= need
        asked += need
        start.append(start[-1] + n)
        granted.append(n if ok else 0)
        context.append(0 if new[b] < 0 else p + granted[-1])
        for i in range(n):
            slots.append(int(table[b, (p + i) // bs]) * bs + (p + i) % bs if ok else -1)
            positions.append(p + i if ok else -1)
    rest = [-1] * (s["tokens"] - len(slots))
    return {"start": np.array(start), "context": np.array(context), "granted": np.array(granted),
            "slots": np.array(slots + rest), "positions": np.array(positions + rest), "height": np.array([top]),
            "table": table, "free": stack}


def _exact_rotate(x, positions, heads):
    hd = x.shape[1] // heads
    z = torch.view_as_complex(x.double().reshape(x.shape[0], heads, hd // 2, 2).contiguous())
    rate = _BASE ** (-2.0 / hd * torch.arange(hd // 2, dtype=torch.float64, device=x.device))
    angle = positions.double()[:, None, None] * rate
    return torch.view_as_real(z * torch.polar(torch.ones_like(angle), angle)).reshape(x.shape[0], heads, hd)


def _exact_append(s):
    keys, values = s["keys"].double(), s["values"].double()
    n, bs, hd = keys.shape[1:]
    k = _exact_rotate(s["k"], s["positions"], n)
    v = s["v"].double().reshape(-1, n, hd)
    for h in range(n):
        for cache, rows in ((keys, k), (values, v)):
            flat = cache[:, h].reshape(-1, hd)
            flat[s["slots"].long()] = rows[:, h]
            cache[:, h] = flat.reshape(-1, bs, hd)
    q = _exact_rotate(s["q"], s["positions"], s["q"].shape[1] // hd)
    return {"q": q.reshape(s["q"].shape), "keys": keys, "values": values}


def _exact_attention(s):
    q, heads = s["q"], s["heads"]
    kv_heads, bs, hd = s["keys"].shape[1:]
    out = torch.zeros(q.shape[0], heads, hd, dtype=torch.float64, device=q.device)
    x = q.double().reshape(-1, heads, hd)
    start, context = s["start"].tolist(), s["context"].tolist()
    for b, length in enumerate(context):
        lo, hi = start[b], start[b + 1]
        at = torch.arange(length, device=q.device)
        page, row = s["table"][b].long()[at // bs], at % bs
        behind = at[None, :] > (at[length - (hi - lo):])[:, None]
        for h in range(kv_heads):
            k, v = s["keys"][page, h, row].double(), s["values"][page, h, row].double()
            for j in range(h * (heads // kv_heads), (h + 1) * (heads // kv_heads)):
                z = torch.mv(k, x[lo, j])[None] if hi - lo == 1 else x[lo:hi, j].contiguous() @ k.t().contiguous()
                z = (z / math.sqrt(hd)).masked_fill(behind, -math.inf)
                out[lo:hi, j] = torch.softmax(z, -1) @ v
    return out.reshape(q.shape)


def _exact_sample(s):
    logits, u = s["logits"].cpu().numpy().astype(np.float64), s["u"].cpu().numpy().astype(np.float64)
    t, k, p, m = (s[n].cpu().numpy() for n in ("temperature", "top_k", "top_p", "min_p"))
    token, prob = np.empty(len(u), np.int32), np.empty(len(u))
    for r, x in enumerate(logits):
        if t[r] <= 0:
            token[r], prob[r] = int(np.argmax(x)), 1.0
            continue
        first = np.lexsort((np.arange(len(x)), -x))            # largest first, then lowest index
        if 0 < k[r] < len(x):
            first = first[:k[r]]
        w = np.exp((x[first] - x[first[0]]) / np.float64(t[r]))
        if p[r] < 1:
            c = np.cumsum(w)
            w = w[:1 + int(np.searchsorted(c, np.float64(p[r]) * c[-1], side="left"))]
        w = w[w >= np.float64(m[r])]
        kept = np.sort(first[:len(w)])
        w = np.exp((x[kept] - x[first[0]]) / np.float64(t[r]))
        c = np.cumsum(w)
        j = int(np.searchsorted(c, u[r] * c[-1], side="right"))
        token[r], prob[r] = kept[j], w[j] / c[-1]
    return {"token": token, "prob": prob}


_EXACT = {"plan": _exact_plan, "append": _exact_append, "attention": _exact_attention, "sample": _exact_sample}
