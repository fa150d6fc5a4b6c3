"""The operators of a beam-search step of a mixture-of-experts model with 8-bit
floating-point weights, with their plain forms: the product with block-scaled
FP8 weights, a whole mixture-of-experts layer for a few tokens, the selection
over beams and vocabulary, and the reordering of a paged key/value cache by the
selected beams.

``listed()`` names fixed cases, ``draw(rng)`` gives another of the same ranges;
``prepare`` builds what a serving program holds before the call, ``run`` is one
pass through one operator, ``exact`` the same from its definition in float64,
``work`` the bytes and operations one pass cannot do without.

An FP8 matrix is e4m3 data [out][in] with one float32 scale for each block of
128 outputs by 128 inputs.
"""
import math
import random

import numpy as np
import torch

own = False

_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
_SIZE = {"f32": 4, "bf16": 2}
_BLOCK = 128          # of the FP8 scales
_LARGEST = 448.0      # the largest e4m3 value

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
def _fp8(rows, k, n, x, y):
    return {"op": "fp8", "rows": rows, "k": k, "n": n, "x": x, "y": y}


def _moe(tokens, experts, top_k, hidden, inner, normalize, x):
    return {"op": "moe", "tokens": tokens, "experts": experts, "top_k": top_k, "hidden": hidden, "inner": inner,
            "normalize": normalize, "x": x}


def _beam(requests, beams, k, vocab, some_done):
    return {"op": "beam", "requests": requests, "beams": beams, "k": k, "vocab": vocab, "some_done": some_done}


def _reorder(groups, beams, layers, context, shared, block, kv_heads, head_dim, cache, spread):
    return {"op": "reorder", "groups": groups, "beams": beams, "layers": layers, "context": context,
            "shared": shared, "block": block, "kv_heads": kv_heads, "head_dim": head_dim, "cache": cache,
            "spread": spread}


def listed():
    return [
        # one token's keys and values: the smallest product of a decode step
        dict(_fp8(1, 2048, 512, "bf16", "bf16"), name="fp8_kv_1"),
        # one token's logits, kept in fp32
        dict(_fp8(1, 2048, 32000, "f32", "f32"), name="fp8_head_1"),
        # a decode step of 21 running requests into the feed-forward layer
        dict(_fp8(21, 4096, 11008, "bf16", "bf16"), name="fp8_step_21"),
        # a prompt of odd length out of the feed-forward layer, fp32 throughout
        dict(_fp8(333, 5632, 2048, "f32", "f32"), name="fp8_prompt_333"),
        # a batch of long prompts into the feed-forward layer
        dict(_fp8(4096, 4096, 11008, "bf16", "bf16"), name="fp8_prompt_4096"),
        # one token, few large experts, fp32 throughout
        dict(_moe(1, 8, 2, 2048, 5632, True, "f32"), name="moe_1"),
        # a step of 13 requests, many small experts of an odd width
        dict(_moe(13, 64, 6, 2048, 1000, False, "bf16"), name="moe_13"),
        # a step of 64 requests: every expert has tokens
        dict(_moe(64, 32, 4, 4096, 2048, True, "bf16"), name="moe_64"),
        # one request of four beams
        dict(_beam(1, 4, 4, 32000, False), name="beam_4"),
        # 32 requests of eight beams, some of them done, over a large vocabulary, twice as many candidates as beams
        dict(_beam(32, 8, 16, 100000, True), name="beam_256"),
        # the cache behind one request of four beams, fp32
        dict(_reorder(1, 4, 2, 301, 100, 16, 4, 64, "f32", 1), name="reorder_4"),
        # eight requests of eight beams, long prompts and long answers, bf16
        dict(_reorder(8, 8, 2, 1500, 700, 16, 8, 128, "bf16", 2), name="reorder_64"),
    ]


def _log(rng, lo, hi, step=1):
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return max(lo, min(hi, int(round(v / step)) * step))


def draw(rng):
    op = rng.choice(("fp8", "fp8", "fp8", "moe", "moe", "beam", "reorder"))
    if op == "fp8":
        step = rng.choice((1, 8, 128))
        case = _fp8(_log(rng, 1, 4096), _log(rng, 512, 11008, step), _log(rng, 512, 32000, step),
                    rng.choice(("f32", "bf16")), rng.choice(("f32", "bf16")))
        smaller = ("rows", "n")
    elif op == "moe":
        experts, step = rng.choice((4, 8, 16, 32, 60, 64, 128)), rng.choice((1, 8, 128))
        case = _moe(_log(rng, 1, 64), experts, min(experts, rng.choice((1, 2, 4, 6, 8))), _log(rng, 512, 4096, step),
                    _log(rng, 512, 5632, step), rng.choice((True, False)), rng.choice(("f32", "bf16")))
        smaller = ("inner",)
    elif op == "beam":
        beams = rng.choice((1, 2, 3, 4, 5, 8, 16))
        case = _beam(_log(rng, 1, 256 // beams), beams, rng.choice((beams, beams, 2 * beams)),
                     _log(rng, 1000, 100000), rng.choice((True, False)))
        smaller = ("vocab",)
    else:
        beams, context = rng.choice((2, 3, 4, 8)), _log(rng, 16, 1500)
        heads = rng.choice(((4, 64), (8, 64), (8, 128), (12, 64)))
        case = _reorder(_log(rng, 1, 64 // beams), beams, rng.choice((1, 2)), context, rng.randrange(context),
                        rng.choice((16, 16, 32, 64)), *heads, rng.choice(("f32", "bf16")), rng.randrange(1 << 20))
        smaller = ("context", "shared")
    top = [work(c) for c in listed() if c["op"] == op]
    while any(work(case)[n] > max(t[n] for t in top) for n in ("bytes", "flops")):   # no dearer than the largest
        for n in smaller:
            case[n] = max(1, case[n] * 7 // 8)
    return case


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _normal(gen, *shape, std=1.0, dtype=torch.float32):
    return (torch.randn(*shape, generator=gen, device="cuda", dtype=torch.float32) * std).to(dtype)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _ceil(a, b):
    return (a + b - 1) // b


def _fp8_matrix(gen, out, inner):
    """A matrix as a converter stores it: e4m3 data [out][in], its scales the
    largest magnitude of a block over 448."""
    std = 1.0 / math.sqrt(inner)
    w = _normal(gen, out, inner, std=std)
    padded = torch.zeros(_ceil(out, _BLOCK) * _BLOCK, _ceil(inner, _BLOCK) * _BLOCK, device="cuda")
    padded[:out, :inner] = w
    blocks = padded.view(_ceil(out, _BLOCK), _BLOCK, _ceil(inner, _BLOCK), _BLOCK)
    scales = blocks.abs().amax((1, 3)) / _LARGEST
    data = (blocks / scales[:, None, :, None]).clamp(-_LARGEST, _LARGEST).view(padded.shape)[:out, :inner]
    return data.to(torch.float8_e4m3fn).contiguous(), scales.contiguous()


def _activations(gen, rows, width, dtype):
    """Rows as they come from a norm: of unit size, some columns larger than the rest."""
    gain = torch.exp(_normal(gen, width, std=0.5))
    return (_normal(gen, rows, width) * gain).to(dtype)


def _fp8_inputs(case, seed):
    gen = _generator(seed)
    data, scales = _fp8_matrix(gen, case["n"], case["k"])
    x = _activations(gen, case["rows"], case["k"], _TYPES[case["x"]])
    state = {"op": "fp8", "x": x, "data": data, "scales": scales, "y": _TYPES[case["y"]]}
    if own:
        state["weight"] = backend().fp8_weight(data, scales)
    return state


def _moe_inputs(case, seed):
    gen = _generator(seed)
    e, h, i = case["experts"], case["hidden"], case["inner"]

    def stack(out, inner):
        parts = [_fp8_matrix(gen, out, inner) for _ in range(e)]
        return torch.stack([d.view(torch.uint8) for d, _ in parts]).view(torch.float8_e4m3fn), \
            torch.stack([s for _, s in parts])

    gate, up, down = stack(i, h), stack(i, h), stack(h, i)
    state = {"op": "moe", "router": _normal(gen, e, h, std=1.0 / math.sqrt(h)), "gate": gate, "up": up, "down": down,
             "x": _activations(gen, case["tokens"], h, _TYPES[case["x"]]), "top_k": case["top_k"],
             "normalize": case["normalize"]}
    if own:
        state["layer"] = backend().moe_layer(state["router"], *gate, *up, *down)
    return state


def _beam_inputs(case, seed):
    gen, rng = _generator(seed), random.Random(seed)
    rows = case["requests"] * case["beams"]
    logits = _normal(gen, rows, case["vocab"], std=2.5)
    # sums of log probabilities after some tens of tokens; beams of a request lie near each other
    scores = torch.empty(rows, device="cuda")
    scores.uniform_(-4.0, 0.0, generator=gen)
    base = torch.empty(case["requests"], device="cuda").uniform_(-60.0, -5.0, generator=gen)
    scores += base.repeat_interleave(case["beams"])
    done = [int(case["some_done"] and rng.random() < 0.1) for _ in range(rows)]
    return {"op": "beam", "logits": logits, "scores": scores, "done": _ints(done), "beams": case["beams"],
            "k": case["k"], "eos": 2}


def _choices(case):
    """Per request of several beams: length, shared length; per beam its parent."""
    rng, g, b, most = random.Random(case["spread"]), case["groups"], case["beams"], case["context"]
    # requests of different lengths; the listed length is the longest
    context = [most] + [rng.randint(most * 3 // 4 + 1, most) if most > 3 else most for _ in range(g - 1)]
    parents = []
    for i in range(g):                        # good beams are continued more than once
        weight = [math.exp(rng.gauss(0, 1)) for _ in range(b)]
        parents += [i * b + p for p in rng.choices(range(b), weight, k=b)]
    return context, [min(c, case["shared"]) for c in context], parents


def _reorder_inputs(case, seed):
    gen = _generator(seed)
    g, b, bs = case["groups"], case["beams"], case["block"]
    context, shared, parents = _choices(case)
    most = _ceil(case["context"], bs) + 1
    held = [_ceil(c, bs) for c in context for _ in range(b)]
    count = sum(held) + 8
    order = np.random.default_rng(seed).permutation(count).astype(np.int32)
    table = np.full((g * b, most), -1, np.int32)
    at = 0
    for r, n in enumerate(held):
        table[r, :n] = order[at:at + n]
        at += n
    shape = (count, case["kv_heads"], bs, case["head_dim"])
    keys, values = ([_normal(gen, *shape, dtype=_TYPES[case["cache"]]) for _ in range(case["layers"])]
                    for _ in range(2))
    return {"op": "reorder", "keys": keys, "values": values, "table": _ints(table), "beams": b,
            "context": _ints([c for c in context for _ in range(b)]), "parents": _ints(parents),
            "shared": _ints(shared), "new_table": torch.empty(g * b, most, dtype=torch.int32, device="cuda")}


_INPUTS = {"fp8": _fp8_inputs, "moe": _moe_inputs, "beam": _beam_inputs, "reorder": _reorder_inputs}


def prepare(case, seed):
    return _INPUTS[case["op"]](case, seed)


# ---------------------------------------------------------------------------
# a pass
# ---------------------------------------------------------------------------
def run(state):
    if own:
        return _OWN[state["op"]](backend(), state)
    return _PLAIN[state["op"]](state)


def _own_fp8(be, s):
    return be.fp8_matmul_device(s["x"], s["weight"], dtype=s["y"])


def _own_moe(be, s):
    y, experts, weights = be.moe_device(s["x"], s["layer"], s["top_k"], normalize=s["normalize"])
    return {"y": y, "experts": experts, "weights": weights}


def _own_beam(be, s):
    tokens, parents, scores, done = be.beam_select_device(s["logits"], s["scores"], s["beams"], k=s["k"],
                                                          done=s["done"], eos=s["eos"])
    return {"tokens": tokens, "parents": parents, "scores": scores, "done": done}


def _own_reorder(be, s):
    table = be.paged_reorder_device(s["keys"], s["values"], s["table"], s["context"], s["parents"], s["beams"],
                                    sharedLens=s["shared"], tableOut=s["new_table"])
    return {"table": table, "keys": s["keys"], "values": s["values"]}


_OWN = {"fp8": _own_fp8, "moe": _own_moe, "beam": _own_beam, "reorder": _own_reorder}


def _plain_matrix(data, scales):
    """The float32 values of FP8 matrices [..., out, in]."""
    wide = scales.repeat_interleave(_BLOCK, -2)[..., :data.shape[-2], :]
    return data.float() * wide.repeat_interleave(_BLOCK, -1)[..., :data.shape[-1]]


def _plain_fp8(s):
    x = s["x"].float()
    rows, k = x.shape
    blocks = torch.nn.functional.pad(x, (0, -k % _BLOCK)).view(rows, -1, _BLOCK)
    # the least power of two that brings a row's block within e4m3's range: found in 64 bits
    part, power = torch.frexp(blocks.abs().amax(-1, keepdim=True).double() / _LARGEST)
    power = torch.where(part == 0.5, power - 1, power).clamp(min=-126)
    scale = torch.ldexp(torch.ones_like(part), power).float()
    x = ((blocks / scale).to(torch.float8_e4m3fn).float() * scale).view(rows, -1)[:, :k]
    return torch.matmul(x, _plain_matrix(s["data"], s["scales"]).t()).to(s["y"])


def _plain_moe(s):
    x, top_k = s["x"].float(), s["top_k"]
    tokens, (e, inner, hidden) = x.shape[0], s["gate"][0].shape
    # which experts: a border between values, in 64 bits
    z = torch.matmul(s["x"].double(), s["router"].double().t())
    experts = torch.sort(z, dim=1, descending=True, stable=True).indices[:, :top_k]
    w = torch.exp(z - z.amax(1, keepdim=True))
    w = w / w.sum(1, keepdim=True)
    weights = torch.gather(w, 1, experts)
    if s["normalize"]:
        weights = weights / weights.sum(1, keepdim=True)
    weights = weights.float()
    share = torch.zeros(tokens, e, device=x.device).scatter(1, experts, weights)
    # every expert for every token; those that a token has not chosen weigh nothing
    g = torch.matmul(x, _plain_matrix(*s["gate"]).view(-1, hidden).t())
    u = torch.matmul(x, _plain_matrix(*s["up"]).view(-1, hidden).t())
    h = (g / (1 + torch.exp(-g)) * u).view(tokens, e, inner) * share[:, :, None]
    y = torch.matmul(h.view(tokens, -1), _plain_matrix(*s["down"]).transpose(1, 2).reshape(-1, hidden))
    return {"y": y.to(s["x"].dtype), "experts": experts.to(torch.int32), "weights": weights}


def _plain_beam(s):
    # orders of sums over a whole vocabulary: in 64 bits
    x, beams, k = s["logits"].double(), s["beams"], s["k"]
    rows, vocab = x.shape
    top = x.amax(1, keepdim=True)
    total = top + torch.log(torch.exp(x - top).sum(1, keepdim=True))
    key = s["scores"].double()[:, None] + (x - total)
    done = s["done"].bool()[:, None]
    only = torch.where(torch.arange(vocab, device=x.device) == s["eos"], s["scores"].double()[:, None], -math.inf)
    key = torch.where(done, only, key).view(-1, beams * vocab)
    best = torch.sort(key, dim=1, descending=True, stable=True)
    index, none = best.indices[:, :k], best.values[:, :k] == -math.inf
    tokens = index % vocab
    parents = index // vocab + beams * torch.arange(rows // beams, device=x.device)[:, None]
    ended = ((tokens == s["eos"]) | s["done"].bool()[parents]) & ~none
    return {"tokens": tokens.masked_fill(none, -1).to(torch.int32),
            "parents": parents.masked_fill(none, -1).to(torch.int32),
            "scores": best.values[:, :k].float(), "done": ended.to(torch.int32)}


def _plain_reorder(s):
    table, beams, bs = s["table"], s["beams"], s["keys"][0].shape[2]
    rows, most = table.shape
    row = torch.arange(rows, device=table.device)
    parent = s["parents"].long()
    # a parent's own row goes to itself if it goes on, else to its first child
    first = torch.full_like(row, rows).scatter_reduce(0, parent, row, "amin")
    first = torch.where(parent == row, row, first)
    heir = first[parent] == row
    # the others take the rows that nobody continues, in order
    dropped = torch.ones_like(heir).scatter(0, parent, False).view(-1, beams)
    free = torch.sort((~dropped).int(), dim=1, stable=True).indices + beams * (row[::beams] // beams)[:, None]
    turn = (torch.cumsum((~heir).view(-1, beams), 1) - 1).clamp(min=0)
    source = torch.where(heir, parent, torch.gather(free, 1, turn).view(-1))
    s["new_table"].copy_(table[source])
    # and get their parent's positions behind the shared ones
    p = torch.arange(most * bs, device=table.device)
    copied = ~heir[:, None] & (p >= (s["shared"] // bs * bs).repeat_interleave(beams)[:, None]) \
        & (p < s["context"][:, None])
    child, p = torch.nonzero(copied, as_tuple=True)
    to, since = s["new_table"][child, p // bs].long(), table[parent[child], p // bs].long()
    for cache in s["keys"] + s["values"]:
        cache[to, :, p % bs] = cache[since, :, p % bs]
    return {"table": s["new_table"], "keys": s["keys"], "values": s["values"]}


_PLAIN = {"fp8": _plain_fp8, "moe": _plain_moe, "beam": _plain_beam, "reorder": _plain_reorder}


# ---------------------------------------------------------------------------
# floors, and the same in 64 bits
# ---------------------------------------------------------------------------
def _matrix_bytes(out, inner):
    return out * inner + 4 * _ceil(out, _BLOCK) * _ceil(inner, _BLOCK)


def work(case):
    op = case["op"]
    if op == "fp8":
        m, k, n = case["rows"], case["k"], case["n"]
        return {"bytes": _matrix_bytes(n, k) + m * (k * _SIZE[case["x"]] + n * _SIZE[case["y"]]),
                "flops": 2 * m * k * n}
    if op == "moe":
        t, e, h, i = case["tokens"], case["experts"], case["hidden"], case["inner"]
        # experts that at least one token chooses, on the average
        used = e * (1 - (1 - case["top_k"] / e) ** t)
        each = 2 * _matrix_bytes(i, h) + _matrix_bytes(h, i)
        return {"bytes": int(used * each) + 4 * e * h + t * (2 * h * _SIZE[case["x"]] + 8 * case["top_k"]),
                "flops": 2 * t * (e * h + 3 * case["top_k"] * h * i)}
    if op == "beam":
        rows = case["requests"] * case["beams"]
        return {"bytes": rows * (4 * case["vocab"] + 8) + case["requests"] * case["k"] * 16,
                "flops": 4 * rows * case["vocab"]}
    g, b = case["groups"], case["beams"]
    context, shared, parents = _choices(case)
    copied = sum((b - len(set(parents[i * b:i * b + b]))) * (context[i] - shared[i]) for i in range(g))
    position = 2 * case["kv_heads"] * case["head_dim"] * _SIZE[case["cache"]] * case["layers"]
    return {"bytes": 2 * copied * position + 8 * g * b * (_ceil(case["context"], case["block"]) + 2),
            "flops": 8 * g * b}


def exact(case, seed):
    return _EXACT[case["op"]](prepare(case, seed))


def _exact_matrix(data, scales):
    out, inner = data.shape
    at = [torch.arange(n, device=data.device) // _BLOCK for n in (out, inner)]
    return data.float().double() * scales.double()[at[0]][:, at[1]]


def _exact_fp8(s):
    x = s["x"].double()
    rows, k = x.shape
    for at in range(0, k, _BLOCK):
        block = x[:, at:at + _BLOCK]
        most = block.abs().amax(1, keepdim=True)
        scale = torch.full_like(most, 2.0 ** -126)
        while bool((most > _LARGEST * scale).any()):
            scale = torch.where(most > _LARGEST * scale, 2 * scale, scale)
        v = block / scale
        # e4m3: three bits behind the leading one, steps of 2^-9 below 2^-6
        power = torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6)))
        step = torch.exp2(power - 3)
        x[:, at:at + _BLOCK] = torch.round(v / step) * step * scale
    return x @ _exact_matrix(s["data"], s["scales"]).t().contiguous()


def _exact_moe(s):
    x = s["x"].double()
    z = (x @ s["router"].double().t().contiguous()).cpu().numpy()
    y, e = torch.zeros_like(x), z.shape[1]
    experts = np.stack([np.lexsort((np.arange(e), -row))[:s["top_k"]] for row in z])
    w = np.exp(z - z.max(1, keepdims=True))
    w = np.take_along_axis(w / w.sum(1, keepdims=True), experts, 1)
    if s["normalize"]:
        w /= w.sum(1, keepdims=True)
    for j in np.unique(experts):
        t, place = np.nonzero(experts == j)
        rows = torch.tensor(t, device=x.device)
        g, u = (x[rows] @ _exact_matrix(*(v[j] for v in s[n])).t().contiguous() for n in ("gate", "up"))
        h = g * torch.sigmoid(g) * u * torch.tensor(w[t, place], device=x.device)[:, None]
        y[rows] += h @ _exact_matrix(*(v[j] for v in s["down"])).t().contiguous()
    return {"y": y, "experts": experts, "weights": w}


def _exact_beam(s):
    x, score = s["logits"].cpu().numpy().astype(np.float64), s["scores"].cpu().numpy().astype(np.float64)
    done, beams, k, eos = s["done"].cpu().numpy(), s["beams"], s["k"], s["eos"]
    answer = {n: [] for n in ("tokens", "parents", "scores", "done")}
    for r in range(0, len(x), beams):
        found = []
        for b in range(r, r + beams):
            if done[b]:
                found.append((-score[b], b, eos))
                continue
            m = x[b].max()
            total = m + math.log(np.exp(x[b] - m).sum())
            best = np.lexsort((np.arange(x.shape[1]), -x[b]))[:k]
            found += [(-(score[b] + (x[b, j] - total)), b, int(j)) for j in best]
        found = sorted(found)[:k]
        found += [(math.inf, -1, -1)] * (k - len(found))
        answer["tokens"].append([j for _, _, j in found])
        answer["parents"].append([b for _, b, _ in found])
        answer["scores"].append([-v for v, _, _ in found])
        answer["done"].append([int(b >= 0 and (j == eos or done[b] != 0)) for _, b, j in found])
    return {n: np.array(v) for n, v in answer.items()}


def _exact_reorder(s):
    """One request after the other, as the definition says."""
    table, parents, context, shared = (s[n].cpu().numpy() for n in ("table", "parents", "context", "shared"))
    beams, bs = s["beams"], s["keys"][0].shape[2]
    new = np.full_like(table, -1)
    moves = []
    for g in range(0, len(parents), beams):
        taken = {}
        for p in range(g, g + beams):
            children = [c for c in range(g, g + beams) if parents[c] == p]
            if children:
                taken[p if p in children else children[0]] = p
        left = [p for p in range(g, g + beams) if p not in taken.values()]
        for c in range(g, g + beams):
            if c in taken:
                new[c] = table[taken[c]]
                continue
            new[c] = table[left.pop(0)]
            for at in range(shared[g // beams] // bs, -(-context[c] // bs)):
                moves.append((table[parents[c], at], new[c, at], min(bs, context[c] - at * bs)))
    keys, values = [c.double() for c in s["keys"]], [c.double() for c in s["values"]]
    for cache in keys + values:
        for n in {m[2] for m in moves}:
            since, to = (torch.tensor([m[i] for m in moves if m[2] == n], device=cache.device) for i in (0, 1))
            cache[to, :, :n] = cache[since, :, :n]
    return {"table": new, "keys": keys, "values": values}


_EXACT = {"fp8": _exact_fp8, "moe": _exact_moe, "beam": _exact_beam, "reorder": _exact_reorder}
