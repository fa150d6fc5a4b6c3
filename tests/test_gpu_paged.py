"""GPU tests of the paged-cache calls (tbh_paged_plan_device,
tbh_paged_append_device, tbh_paged_attention_device) against
oracle/paged_ref.py in float64.  Whole numbers are equal; where results are
rounded, each tolerance is an error bound worked out from the case's own
numbers (P._bound, and half a step per rounding to a narrower type)."""
import numpy as np
import pytest

import tinybrain_amd as T
from oracle import paged_ref as P
from tinybrain_amd.quantized import PreconditionFailure

pytestmark = pytest.mark.gpu
U32, U16 = 2.0 ** -24, 2.0 ** -8        # half a step of fp32 and of bf16, relative


@pytest.fixture(scope="module")
def backend():
    b = T.HIPBackend(0)
    yield b
    b.close()


@pytest.fixture(scope="module")
def torch():
    import torch

    return torch


def _ints(torch, a):
    return torch.tensor(np.asarray(a), dtype=torch.int32, device="cuda")


def _np(t):
    return t.double().cpu().numpy() if t.is_floating_point() else t.cpu().numpy()


# ---------------------------------------------------------------------------
# plan
# ---------------------------------------------------------------------------
def _plan_case(seed, rows, most, bs, spare, shares=(-1, 0, 1, 1, 1, 7, 50)):
    rng = np.random.default_rng(seed)
    ctx = rng.integers(0, most * bs + 1, rows).astype(np.int32)
    ctx[rng.random(rows) < 0.1] = 0
    new = rng.choice(shares, rows).astype(np.int32)
    held = -(-ctx // bs)
    blocks = int(held.sum()) + spare
    order = rng.permutation(blocks).astype(np.int32)
    table = np.full((rows, most), -1, np.int32)
    at = 0
    for b in range(rows):
        table[b, :held[b]] = order[at:at + held[b]]
        at += held[b]
    stack = np.full(blocks, -7, np.int32)
    stack[:spare] = order[at:]
    return new, ctx, table, stack, spare


def _check_plan(torch, backend, case, bs, max_tokens, in_place=False):
    new, ctx, table, stack, height = case
    want = P.plan(new, ctx, table, stack, height, bs, max_tokens)
    d = [_ints(torch, a) for a in (new, ctx, table, stack, [height])]
    kw = dict(contextOut=d[1], freeCountOut=d[4]) if in_place else {}
    for _ in range(1 if in_place else 2):          # a plan that is not taken over changes nothing it depends on
        p = backend.paged_plan_device(*d, bs, max_tokens, **kw)
    got = {"start": p.queryStart, "granted": p.granted, "context": p.contextLens, "slots": p.slots,
           "positions": p.positions, "table": d[2], "free": d[3]}
    for name, t in got.items():
        np.testing.assert_array_equal(_np(t), want[name], err_msg=name)
    assert int(p.freeCount[0]) == want["count"]
    if not in_place:
        np.testing.assert_array_equal(_np(d[1]), ctx)
        assert int(d[4][0]) == height


@pytest.mark.parametrize("rows,most,bs,spare,slack", [
    (1, 1, 1, 0, 0), (1, 4, 16, 3, 5), (5, 8, 16, 2, -9), (64, 16, 16, 40, 0), (65, 9, 1, 11, 7),
    (200, 3, 1024, 90, 0), (1024, 12, 16, 500, 3), (1025, 12, 8, 100, 0), (3001, 5, 32, 2000, 129),
])
@pytest.mark.parametrize("in_place", [False, True])
def test_plan(torch, backend, rows, most, bs, spare, slack, in_place):
    case = _plan_case(rows + most, rows, most, bs, spare)
    total = int(np.maximum(case[0], 0).sum())
    _check_plan(torch, backend, case, bs, max(total + slack, 0), in_place)


@pytest.mark.parametrize("shares", [(0,), (-1,), (1,), (-1, 400), (0, 0, 0, 1500)])
def test_plan_uniform_batches(torch, backend, shares):
    # everyone idle, released, or adding; long lists of blocks per row
    case = _plan_case(3, 96, 120, 16, 4000, shares)
    _check_plan(torch, backend, case, 16, int(np.maximum(case[0], 0).sum()) + 1)


def test_plan_many_steps(torch, backend):
    # a cache in use: every step's state follows from the one before
    rng = np.random.default_rng(5)
    rows, most, bs, blocks = 40, 10, 4, 150
    cache = T.PagedKVCache(backend, 1, blocks, bs, 1, 8, rows, most)
    table, ctx = np.full((rows, most), -1, np.int32), np.zeros(rows, np.int32)
    free, count = np.arange(blocks)[::-1].astype(np.int32), blocks
    for _ in range(40):
        new = rng.choice([-1, 0, 1, 1, 1, 2, 9], rows).astype(np.int32)
        p = cache.plan(_ints(torch, new), 250)
        want = P.plan(new, ctx, table, free, count, bs, 250)
        table, ctx, free, count = want["table"], want["context"], want["free"], want["count"]
        for got, name in ((cache.blockTable, "table"), (cache.contextLens, "context"), (cache.freeBlocks, "free"),
                          (p.slots, "slots"), (p.positions, "positions"), (p.queryStart, "start"),
                          (p.granted, "granted")):
            np.testing.assert_array_equal(_np(got), want[name], err_msg=name)
        assert int(cache.freeCount[0]) == count


def test_plan_of_values_out_of_range(torch, backend):
    # negative lengths count as 0, a height outside the stack is clamped, a
    # length beyond the table row is never granted: nothing is followed anywhere
    table = np.array([[3, -1], [9, 99], [1, 2]], np.int32)
    d = [_ints(torch, a) for a in ([2, 1, 1], [-5, 3, 1 << 30], table, [0, 4, 5, 6], [77])]
    p = backend.paged_plan_device(*d, 4, 6)
    np.testing.assert_array_equal(_np(p.granted), [2, 1, 0])
    np.testing.assert_array_equal(_np(p.contextLens), [2, 4, 1 << 30])
    # the cache has 4 blocks: 6, popped for row 0, and 9, held by row 1, are none of them
    np.testing.assert_array_equal(_np(p.slots), [-1] * 6)
    np.testing.assert_array_equal(_np(p.positions), [0, 1, 3, -1, -1, -1])
    assert int(p.freeCount[0]) == 3


# ---------------------------------------------------------------------------
# append
# ---------------------------------------------------------------------------
def _close(got, want, tol):
    err = np.abs(got - want)
    assert np.all((err <= tol) | (np.isnan(got) & np.isnan(want))), float(np.nanmax(err - tol))


@pytest.mark.parametrize("x,cache,qt", [("float32", "float32", "float32"), ("float32", "bfloat16", "float32"),
                                        ("float32", "bfloat16", "bfloat16"), ("bfloat16", "bfloat16", "bfloat16"),
                                        ("bfloat16", "float32", "float32"), ("float32", "float32", "bfloat16"),
                                        ("bfloat16", "float32", "bfloat16"), ("bfloat16", "bfloat16", "float32")])
@pytest.mark.parametrize("tokens,nh,nkv,hd,bs,base", [
    (1, 32, 4, 64, 16, 10000.0), (37, 8, 2, 128, 16, 500000.0), (5, 3, 3, 6, 1, 10000.0), (9, 4, 1, 80, 64, 0.0),
    (11, 5, 5, 7, 4, 0.0), (70, 2, 1, 256, 8, 10000.0),
])
def test_append(torch, backend, x, cache, qt, tokens, nh, nkv, hd, bs, base):
    rng = np.random.default_rng(tokens * hd)
    blocks = tokens // bs + 3
    xt, ct, qtt = (getattr(torch, n) for n in (x, cache, qt))
    kc, vc = (torch.tensor(rng.normal(size=(blocks, nkv, bs, hd)), dtype=ct, device="cuda") for _ in range(2))
    # q, k and v side by side in a row, with three columns more
    width = (nh + 2 * nkv) * hd + 3
    rows = torch.tensor(rng.normal(size=(tokens, width)), dtype=xt, device="cuda")
    q, k, v = rows[:, :nh * hd], rows[:, nh * hd:(nh + nkv) * hd], rows[:, (nh + nkv) * hd:width - 3]
    slots = rng.permutation(blocks * bs)[:tokens].astype(np.int32)
    positions = rng.integers(0, 1 << 17, tokens).astype(np.int32)
    if tokens > 3:
        slots[[1, 3]] = -1, blocks * bs                # not stored
        positions[2] = -1                              # rotated as 0
    before = _np(kc), _np(vc)
    out = backend.paged_append_device(kc, vc, _ints(torch, slots), k, v, q=q, positions=_ints(torch, positions),
                                      ropeBase=base, qOut=torch.empty(tokens, nh * hd, dtype=qtt, device="cuda"))
    rot = (lambda a, n: P.rotate(a, positions, n, base)) if base else (lambda a, n: a)
    wk, wv = P.append(before[0], rot(_np(k), nkv), slots), P.append(before[1], _np(v), slots)

    # A rotated value x0 c - x1 s: c and s are off by the angle's 2^-24 pi (it is
    # rounded once, in half turns, below 1) and their own 2 half steps, each
    # product and the sum round once: 8 half steps of |x0| + |x1| <= 2 max |x|.
    # What is copied is exact; then one rounding to the narrower type.
    def tol(want, src, t):
        return (16 * U32 * np.abs(src).max() if base else 0) + (U16 if t == torch.bfloat16 else 0) * np.abs(want)

    wq = rot(_np(q), nh)
    _close(_np(out), wq, tol(wq, _np(q), qtt))
    _close(_np(kc), wk, np.where(wk == before[0], 0, tol(wk, _np(k), ct)))
    narrowed = x == "float32" and cache == "bfloat16"
    _close(_np(vc), wv, np.where(wv == before[1], 0, U16 * np.abs(wv) if narrowed else 0))


def test_append_in_place_and_without_queries(torch, backend):
    rng = np.random.default_rng(8)
    rows = torch.tensor(rng.normal(size=(6, 4 * 64)), dtype=torch.float32, device="cuda")
    q, k, v = rows[:, :128], rows[:, 128:192], rows[:, 192:]
    src = _np(rows)
    kc, vc = torch.zeros(2, 2, 1, 4, 64, device="cuda")
    slots, pos = _ints(torch, np.arange(6)), _ints(torch, np.arange(6) * 1000)
    assert backend.paged_append_device(kc, vc, slots, k, v, positions=pos, ropeBase=10000.0) is None
    k_alone = kc.clone()
    out = backend.paged_append_device(kc, vc, slots, k, v, q=q, positions=pos, ropeBase=10000.0, qOut=q)
    assert out is q and torch.equal(kc, k_alone)
    _close(_np(rows[:, :128]), P.rotate(src[:, :128], _np(pos), 2, 10000.0), 16 * U32 * np.abs(src).max())
    np.testing.assert_array_equal(_np(rows[:, 128:]), src[:, 128:])
    np.testing.assert_array_equal(_np(vc).reshape(8, 64)[:6], src[:, 192:])


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------
def _attention_case(torch, seed, lens, nh, nkv, hd, bs, x, cache, extra_rows=0, holes=False, wide=0, q_std=2.0):
    """lens: (new, context with them) per request.  Places behind a request's
    length hold NaN, as an uninitialised cache may."""
    rng = np.random.default_rng(seed)
    xt, ct = getattr(torch, x), getattr(torch, cache)
    held = [-(-c // bs) for _, c in lens]
    blocks = sum(held) + 2
    order = rng.permutation(blocks).astype(np.int32)
    most = max(held + [1]) + 1
    table = rng.choice([-1, blocks, 1 << 30, -(1 << 31)], (len(lens), most)).astype(np.int64)
    keys, values = (torch.full((blocks, nkv, bs, hd), float("nan"), dtype=ct, device="cuda") for _ in range(2))
    at = 0
    for b, (n, c) in enumerate(lens):
        table[b, :held[b]] = order[at:at + held[b]]
        at += held[b]
        for j in range(held[b]):
            m = min(bs, c - j * bs)
            for a in (keys, values):
                a[int(table[b, j]), :, :m] = torch.tensor(rng.normal(size=(nkv, m, hd)), dtype=ct, device="cuda")
        if holes and held[b] > 2:
            table[b, rng.integers(0, held[b] - 1)] = -1
    start = np.concatenate([[0], np.cumsum([n for n, _ in lens])]).astype(np.int32)
    tokens = int(start[-1]) + extra_rows
    q = torch.tensor(rng.normal(size=(tokens, nh * hd + wide)) * q_std, dtype=xt, device="cuda")[:, :nh * hd]
    return dict(q=q, keys=keys, values=values, table=table.astype(np.int32), start=start,
                context=np.array([c for _, c in lens], np.int32), heads=nh)


def _run_attention(torch, backend, c, **kw):
    return backend.paged_attention_device(c["q"], c["keys"], c["values"], _ints(torch, c["table"]),
                                          _ints(torch, c["start"]), _ints(torch, c["context"]), c["heads"], **kw)


def _tolerance(want, bound, x, cache):
    """The formula's fp32 bound; bf16 rows round the result once, and over a
    bf16 cache each probability too: U16 of sum p |v|, which the bound holds
    at least 8 U32 of."""
    t = bound + U32 * np.abs(want)
    if x == "bfloat16":
        t = t + U16 * np.abs(want)
    return t


def _check_attention(torch, backend, c, x, cache, scale=0.0, **kw):
    rows = int(c["start"][-1])
    out = torch.full(c["q"].shape, 7.0, dtype=c["q"].dtype, device="cuda")
    got = _np(_run_attention(torch, backend, c, out=out, scale=scale, **kw))
    keys, values = _np(c["keys"]), _np(c["values"])
    want, bound = P.attention(_np(c["q"]), keys, values, c["table"], c["start"], c["context"], c["heads"],
                              scale or None)
    tol = _tolerance(want, bound, x, cache)
    if x == "bfloat16" and cache == "bfloat16":        # p rounded to bf16: U16 of sum p |v|
        mass, _ = P.attention(_np(c["q"]), keys, np.abs(values), c["table"], c["start"], c["context"], c["heads"],
                              scale or None)
        tol = tol + U16 * mass
    _close(got[:rows], want[:rows], tol[:rows])
    assert np.all(got[rows:] == 7.0)                   # rows behind the last request
    return got


TYPES = [("float32", "float32"), ("float32", "bfloat16"), ("bfloat16", "bfloat16"), ("bfloat16", "float32")]
MIXED = [(1, 1), (1, 77), (0, 50), (5, 5), (0, 0), (33, 90), (1, 130), (2, 64), (17, 17), (1, 16), (3, 300)]


@pytest.mark.parametrize("x,cache", TYPES)
@pytest.mark.parametrize("nh,nkv,hd,bs", [
    (8, 2, 64, 16), (4, 4, 128, 16), (32, 4, 64, 32), (6, 1, 32, 1), (3, 3, 6, 8), (4, 2, 80, 16), (2, 1, 256, 64),
    (10, 2, 96, 4), (5, 5, 1, 16), (20, 1, 128, 128), (4, 2, 16, 1024), (2, 2, 48, 2), (2, 1, 100, 16),
])
def test_attention_mixed_batch(torch, backend, x, cache, nh, nkv, hd, bs):
    c = _attention_case(torch, nh * hd + bs, MIXED, nh, nkv, hd, bs, x, cache, extra_rows=3)
    a = _check_attention(torch, backend, c, x, cache)
    # what is said of the lengths changes the launches at most
    _check_attention(torch, backend, c, x, cache, maxQueryLen=33, maxContextLen=300)
    _check_attention(torch, backend, c, x, cache, maxQueryLen=1, maxContextLen=1)
    b = _np(_run_attention(torch, backend, c))
    np.testing.assert_array_equal(a[:int(c["start"][-1])], b[:int(c["start"][-1])])


@pytest.mark.parametrize("x,cache", TYPES)
@pytest.mark.parametrize("lens", [
    [(1, 1)], [(1, 64)], [(1, 65)], [(1, 1000)], [(1, 2049)], [(1, 5000)], [(1, 700)] * 5, [(2, 640), (1, 1)],
    [(64, 64)], [(65, 65)], [(130, 500)], [(100, 100), (1, 900), (31, 31)], [(15, 15)], [(16, 16)], [(250, 251)],
])
@pytest.mark.parametrize("nh,nkv,hd", [(8, 2, 64), (4, 1, 128)])
def test_attention_lengths(torch, backend, x, cache, lens, nh, nkv, hd):
    c = _attention_case(torch, len(lens) + lens[0][1], lens, nh, nkv, hd, 16, x, cache)
    _check_attention(torch, backend, c, x, cache, maxQueryLen=max(n for n, _ in lens),
                     maxContextLen=max(t for _, t in lens))


@pytest.mark.parametrize("x,cache", TYPES)
@pytest.mark.parametrize("nh,nkv,hd,bs", [(4, 2, 80, 16), (2, 2, 256, 16), (4, 4, 64, 8), (6, 2, 33, 32), (8, 1, 8, 1)])
def test_attention_of_other_heads_over_several_passes(torch, backend, x, cache, nh, nkv, hd, bs):
    # head dimensions and blocks that no matrix kernel takes, lengths around the waves' passes of 64
    c = _attention_case(torch, 32, [(1, 64), (1, 65), (3, 256), (2, 257), (1, 700), (70, 130), (1, 1)], nh, nkv, hd, bs,
                        x, cache, holes=bs > 1)
    _check_attention(torch, backend, c, x, cache)


@pytest.mark.parametrize("x,cache", TYPES)
def test_attention_strides_holes_and_scale(torch, backend, x, cache):
    # rows of a wider matrix whose starts are not 16-byte aligned; pages that are
    # missing; a scale of the caller's
    c = _attention_case(torch, 4, [(3, 200), (40, 100), (1, 90), (1, 33)], 4, 2, 64, 16, x, cache, holes=True, wide=3)
    _check_attention(torch, backend, c, x, cache, scale=0.03)
    c = _attention_case(torch, 5, [(1, 200)], 4, 2, 64, 16, x, cache, wide=3)
    _check_attention(torch, backend, c, x, cache, scale=-0.2)


@pytest.mark.parametrize("hd", [64, 128, 6])
@pytest.mark.parametrize("x,cache", TYPES)
def test_attention_rows_with_nothing_to_see(torch, backend, x, cache, hd):
    # more rows than positions (the first rows lie before position 0), requests
    # without a block, with no length, and lengths beyond their table row
    c = _attention_case(torch, 6, [(5, 3), (1, 40), (20, 0), (2, 100), (70, 30)], 4, 2, hd, 16, x, cache)
    c["table"][1] = -1
    got = _check_attention(torch, backend, c, x, cache)
    assert not got[:2].any() and not got[5:26].any()
    c["context"][3] = 1 << 30
    out = _np(_run_attention(torch, backend, c))
    assert np.isfinite(out[:5]).all()                   # the other requests are not touched by it


@pytest.mark.parametrize("x,cache", TYPES)
def test_attention_of_chunks_without_a_position(torch, backend, x, cache):
    # requests of many rows that hold nothing yet, beside one that does
    c = _attention_case(torch, 30, [(90, 0), (200, 0), (70, 150), (40, 0)], 4, 2, 128, 16, x, cache)
    got = _check_attention(torch, backend, c, x, cache)
    assert not got[:290].any() and not got[360:].any() and got[290:360].all()


@pytest.mark.parametrize("hd", [64, 128, 6])
@pytest.mark.parametrize("new", [1, 5, 40])
def test_attention_rows_before_the_first_request(torch, backend, hd, new):
    # a step's rows may start behind others of the same matrix, which stay as they are
    c = _attention_case(torch, 31, [(new, 60), (0, 20), (1, 33)], 4, 2, hd, 16, "float32", "float32")
    want = _run_attention(torch, backend, c)
    out = torch.full((new + 4, 4 * hd), 7.0, device="cuda")
    moved = dict(c, q=torch.cat([c["q"].new_full((3, 4 * hd), float("nan")), c["q"]]), start=c["start"] + 3)
    got = _run_attention(torch, backend, moved, out=out)
    assert torch.equal(got[3:], want) and bool((got[:3] == 7.0).all())


@pytest.mark.parametrize("x,cache", TYPES)
def test_attention_extreme_scores(torch, backend, x, cache):
    # one key far ahead of the others, and scores that all lie far from 0
    c = _attention_case(torch, 7, [(1, 333), (40, 70)], 4, 2, 64, 16, x, cache, q_std=40.0)
    _check_attention(torch, backend, c, x, cache)
    # NaN or inf in a place that is seen reaches exactly the rows that see it
    c = _attention_case(torch, 8, [(1, 100), (70, 80)], 4, 2, 64, 16, x, cache)
    p = 75                                               # of the second request: rows 65 .. see it
    c["keys"][int(c["table"][1, p // 16]), 0, p % 16] = float("nan")
    c["values"][int(c["table"][1, p // 16]), 1, p % 16, 3] = float("inf")
    got = _np(_run_attention(torch, backend, c)).reshape(71, 4, 64)
    bad = ~np.isfinite(got)
    assert not bad[:66].any()
    assert bad[66:, :2].all() and bad[66:, 2:, 3].all() and not bad[66:, 2:, :3].any() and not bad[66:, 2:, 4:].any()


def _attention64(torch, c, hd):
    """The formula in float64 on the device, a head at a time: (out, sum p |v|,
    bound of fp32 arithmetic), rows x heads x hd."""
    q = c["q"].double().reshape(c["q"].shape[0], -1, hd)
    rep = q.shape[1] // c["keys"].shape[1]
    out, mass, bound = torch.zeros_like(q), torch.zeros_like(q), torch.zeros_like(q)
    for b, n in enumerate(c["context"]):
        lo, hi, bs = int(c["start"][b]), int(c["start"][b + 1]), c["keys"].shape[2]
        pages = torch.tensor(c["table"][b, :P.ceil_div(int(n), bs)].astype(np.int64), device="cuda")
        see = torch.arange(int(n), device="cuda")[None] <= torch.arange(hi - lo, device="cuda")[:, None] + int(n) - (hi - lo)
        for h in range(q.shape[1]):
            k = c["keys"][pages, h // rep].reshape(-1, hd)[:int(n)].double()
            v = c["values"][pages, h // rep].reshape(-1, hd)[:int(n)].double()
            x = q[lo:hi, h]
            s = (x @ k.T) * hd ** -0.5
            top = s.masked_fill(~see, -float("inf")).max(1, keepdim=True).values
            p = torch.where(see, torch.exp(s - top), torch.zeros_like(s))
            p /= p.sum(1, keepdim=True)
            e = ((hd + 2) * U32 * (x.abs() @ k.abs().T) * hd ** -0.5 + U32 * (s - top).abs()) * see
            out[lo:hi, h], mass[lo:hi, h] = p @ v, p @ v.abs()
            bound[lo:hi, h] = (2 * e.max(1, keepdim=True).values + (int(n) + 8) * U32) * mass[lo:hi, h]
    return out.reshape(c["q"].shape), mass.reshape(c["q"].shape), bound.reshape(c["q"].shape)


@pytest.mark.parametrize("nh,nkv,hd", [(16, 16, 128), (64, 32, 64)])
def test_attention_of_a_long_chunk(torch, backend, nh, nkv, hd):
    # enough rows for the widest tiles, beside a short chunk and a single token
    lens = [(1, 300), (3800 * nkv // nh, 3900), (70, 90)]
    c = _attention_case(torch, 50, lens, nh, nkv, hd, 16, "bfloat16", "bfloat16")
    want, mass, bound = _attention64(torch, c, hd)
    # the result rounded once, and each p: by U16 of sum p |v - out|, at most mass + |out|
    tol = bound + (U32 + 2 * U16) * want.abs() + U16 * mass
    out = torch.full(c["q"].shape, 7.0, dtype=torch.bfloat16, device="cuda")
    got = _run_attention(torch, backend, c, out=out).double()
    rows = int(c["start"][-1])
    assert bool(((got - want).abs() <= tol)[:rows].all()) and bool((got[rows:] == 7.0).all())
    # an inf that only the chunk's last rows see
    p = 3850
    c["values"][int(c["table"][1, p // 16]), nkv - 1, p % 16, 5] = float("inf")
    got = _run_attention(torch, backend, c, out=out).double()
    first = int(c["start"][2]) - (3900 - p)                  # the first row that sees it
    at = [h * hd + 5 for h in range(nh - nh // nkv, nh)]
    assert bool((got[first:int(c["start"][2])][:, at] == float("inf")).all())
    got[first:int(c["start"][2]), at] = want[first:int(c["start"][2]), at]
    assert bool(((got - want).abs() <= tol)[:rows].all())


def test_attention_past_32_bits(torch, backend):
    # blocks whose elements lie beyond 2^31 (and bytes beyond 2^32)
    nkv, bs, hd = 8, 16, 128
    blocks = (1 << 31) // (nkv * bs * hd) + 40
    lens = [(1, 300), (50, 200)]
    small = _attention_case(torch, 9, lens, 16, nkv, hd, bs, "bfloat16", "bfloat16")
    want = _run_attention(torch, backend, small)
    n = small["keys"].shape[0]
    big = {k: torch.empty(blocks, nkv, bs, hd, dtype=torch.bfloat16, device="cuda") for k in ("keys", "values")}
    for k in big:
        big[k][blocks - n:] = small[k]
    t = small["table"].astype(np.int64)
    moved = dict(small, **big, table=np.where((t >= 0) & (t < n), t + blocks - n, -1).astype(np.int32))
    got = _run_attention(torch, backend, moved)
    assert torch.equal(got, want)
    rows = torch.randn(2, 2 * nkv * hd, device="cuda").to(torch.bfloat16)
    k, v = rows[:, :nkv * hd], rows[:, nkv * hd:]
    backend.paged_append_device(big["keys"], big["values"], _ints(torch, [blocks * bs - 1, 5]), k, v)
    assert torch.equal(big["keys"][-1, :, -1].reshape(-1), k[0]) and torch.equal(big["values"][0, :, 5].reshape(-1), v[1])


@pytest.mark.parametrize("hd,bs", [(32, 16), (8, 1)])
def test_more_blocks_than_a_grid_has_across(torch, backend, hd, bs):
    # 2^20 and some rows: requests of one position, so that each row's result is its value
    n, nkv = (1 << 20) + 7, 1
    rows = torch.randn(n, 2 * hd, device="cuda").to(torch.bfloat16)
    k, v = rows[:, :hd], rows[:, hd:]
    keys, values = torch.zeros(2, n, nkv, bs, hd, dtype=torch.bfloat16, device="cuda")
    order = torch.randperm(n, device="cuda").to(torch.int32)
    backend.paged_append_device(keys, values, order * bs, k, v)
    at = order.long()
    assert torch.equal(keys[at, 0, 0], k) and torch.equal(values[at, 0, 0], v)
    start, ones = torch.arange(n + 1, dtype=torch.int32, device="cuda"), torch.ones(n, dtype=torch.int32, device="cuda")
    for kw in ({}, dict(maxQueryLen=1, maxContextLen=1)):
        got = backend.paged_attention_device(k.contiguous(), keys, values, order[:, None].contiguous(), start, ones, 1, **kw)
        assert torch.equal(got, v)


def test_attention_split_partials_of_two_streams(torch, backend):
    # calls that split their contexts on two streams at once, each with its workspace
    c = [_attention_case(torch, 20 + i, [(1, 4000 + i)], 8, 2, 64, 16, "float32", "bfloat16") for i in range(2)]
    args = [[_ints(torch, d[k]) for k in ("table", "start", "context")] for d in c]

    def call(i, stream=None):
        d = c[i]
        return backend.paged_attention_device(d["q"], d["keys"], d["values"], *args[i], d["heads"],
                                              maxContextLen=4100, stream=stream)

    want = [call(i).clone() for i in range(2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(20):
        got = [call(i, streams[i]) for i in range(2)]
        torch.cuda.synchronize()
        assert all(torch.equal(g, w) for g, w in zip(got, want))


def test_attention_captured_before_any_eager_call(torch, backend):
    # a stream without a workspace: whole contexts, and the same formula
    c = _attention_case(torch, 40, [(1, 3000), (60, 900)], 8, 2, 64, 16, "float32", "bfloat16")
    args = [_ints(torch, c[k]) for k in ("table", "start", "context")]
    out = torch.empty_like(c["q"])
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        backend.paged_attention_device(c["q"], c["keys"], c["values"], *args, c["heads"], out=out)
    keys, values = _np(c["keys"]), _np(c["values"])
    want, bound = P.attention(_np(c["q"]), keys, values, c["table"], c["start"], c["context"], c["heads"])
    for _ in range(3):
        out.fill_(7.0)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        _close(_np(out), want, _tolerance(want, bound, "float32", "bfloat16"))
        eager = _run_attention(torch, backend, c)            # with parts
        _close(_np(eager), want, _tolerance(want, bound, "float32", "bfloat16"))


@pytest.mark.parametrize("x,cache", TYPES)
@pytest.mark.parametrize("hd", [64, 128, 32])
def test_attention_of_long_contexts_in_one_part(torch, x, cache, hd):
    # without a workspace a block takes a whole context: past the 4096 positions whose blocks it
    # looks up at once (single tokens), the 1024 of a tile's window, and with pages missing
    c = _attention_case(torch, 43, [(1, 9000), (40, 2600), (1, 4097), (3, 4230)], 4, 2, hd, 16, x, cache, holes=True)
    c["table"][0, [255, 256, 300]] = -1                    # of the positions around the 4096th
    args = [_ints(torch, c[k]) for k in ("table", "start", "context")]
    out = torch.empty_like(c["q"])
    fresh, stream, graph = T.HIPBackend(0), torch.cuda.Stream(), torch.cuda.CUDAGraph()
    try:
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            fresh.paged_attention_device(c["q"], c["keys"], c["values"], *args, c["heads"], out=out)
        keys, values = _np(c["keys"]), _np(c["values"])
        want, bound = P.attention(_np(c["q"]), keys, values, c["table"], c["start"], c["context"], c["heads"])
        tol = _tolerance(want, bound, x, cache)
        if x == cache == "bfloat16":
            tol = tol + U16 * P.attention(_np(c["q"]), keys, np.abs(values), c["table"], c["start"], c["context"], 4)[0]
        for _ in range(2):
            out.fill_(7.0)
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            _close(_np(out), want, tol)
        _check_attention(torch, fresh, c, x, cache)        # and in parts
    finally:
        fresh.close()


@pytest.mark.parametrize("x,cache", TYPES)
@pytest.mark.parametrize("requests", [64, 65, 129, 200])
@pytest.mark.parametrize("nh,nkv,hd", [(8, 2, 64), (4, 1, 96), (4, 2, 32), (3, 3, 40)])
def test_attention_of_many_requests(torch, backend, x, cache, requests, nh, nkv, hd):
    # chunks and single tokens among more requests than a wave looks over at once
    rng = np.random.default_rng(requests)
    lens = [(1, int(rng.integers(1, 120))) for _ in range(requests)]
    for b in {3, 40, 63, 64, 70, 127, 128, 150, requests - 1} & set(range(requests)):
        n = int(rng.integers(2, 40))
        lens[b] = (n, n + int(rng.integers(0, 90)))
    for b in {0, 62, 65, 126} & set(range(requests)):
        lens[b] = (0, int(rng.integers(0, 50)))
    c = _attention_case(torch, requests + hd, lens, nh, nkv, hd, 16, x, cache, extra_rows=2)
    got = _check_attention(torch, backend, c, x, cache)
    again = _check_attention(torch, backend, c, x, cache, maxQueryLen=40, maxContextLen=130)
    np.testing.assert_array_equal(got[-2:], again[-2:])


@pytest.mark.parametrize("x,cache", TYPES)
def test_attention_past_parts_of_1024_positions(torch, backend, x, cache):
    # contexts past 65536 positions: 64 parts hold more than 1024 each
    hd = 64
    c = _attention_case(torch, 45, [(1, 70001), (1, 300), (20, 66000)], 4, 2, hd, 1024, x, cache)
    want, mass, bound = _attention64(torch, c, hd)
    tol = bound + (U32 + (2 * U16 if x == "bfloat16" else 0)) * want.abs()
    if x == cache == "bfloat16":
        tol = tol + U16 * mass
    for kw in ({}, dict(maxQueryLen=20, maxContextLen=70001), dict(maxQueryLen=1)):
        got = _run_attention(torch, backend, c, **kw).double()
        assert bool(((got - want).abs() <= tol).all())


def test_two_captured_steps_take_turns(torch, backend):
    # two graphs of one stream share its workspace; replayed in turn, with eager calls between
    cs = [_attention_case(torch, 41 + i, [(1, 2500 - 700 * i), (30, 800)], 8, 2, 64, 16, "float32", "float32")
          for i in range(2)]
    args = [[_ints(torch, c[k]) for k in ("table", "start", "context")] for c in cs]
    outs = [torch.empty_like(c["q"]) for c in cs]
    stream = torch.cuda.Stream()

    def call(i, out):
        return backend.paged_attention_device(cs[i]["q"], cs[i]["keys"], cs[i]["values"], *args[i], 8, out=out)

    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        want = [call(i, torch.empty_like(outs[i])) for i in range(2)]
        stream.synchronize()
        graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
        for i in range(2):
            with torch.cuda.graph(graphs[i], stream=stream):
                call(i, outs[i])
        for _ in range(4):
            for o in outs:
                o.zero_()
            graphs[0].replay()
            graphs[1].replay()
            again = call(0, torch.empty_like(outs[0]))
            graphs[0].replay()
            stream.synchronize()
            assert all(torch.equal(o, w) for o, w in zip([*outs, again], [*want, want[0]]))


def test_calls_of_nothing(torch, backend):
    # no request, no block, no entry in the table, no row
    i = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")      # noqa: E731
    p = backend.paged_plan_device(i(0), i(0), i(0, 4), i(6), i(1) + 6, 16, 3)
    assert _np(p.queryStart).tolist() == [0] and _np(p.slots).tolist() == [-1] * 3 and int(p.freeCount) == 6
    p = backend.paged_plan_device(i(2) + 1, i(2), i(2, 0), i(0), i(1), 16, 3)
    assert _np(p.queryStart).tolist() == [0, 1, 2] and _np(p.granted).tolist() == [0, 0]
    assert _np(p.slots).tolist() == [-1] * 3 and _np(p.contextLens).tolist() == [0, 0]
    q, rows = torch.randn(3, 256, device="cuda"), torch.randn(3, 128, device="cuda")
    for blocks, entries in ((0, 2), (4, 0), (0, 0)):
        k = torch.ones(blocks, 2, 16, 64, device="cuda")
        for new in (1, 3):
            start = i(3) + new
            start[0] = 0
            got = backend.paged_attention_device(q[:new], k, k, i(2, entries), start, i(2) + 5, 4)
            assert not got.any()
        assert torch.equal(backend.paged_append_device(k, k, i(3) - 1, rows, rows, q=q), q) and bool((k == 1).all())
    k = torch.ones(4, 2, 16, 64, device="cuda")
    assert backend.paged_attention_device(q[:0], k, k, i(2, 1), i(3), i(2), 4).shape == (0, 256)
    assert backend.paged_append_device(k, k, i(0), rows[:0], rows[:0], q=q[:0]).shape == (0, 256)
    out = torch.full_like(q, 7.0)
    assert bool((backend.paged_attention_device(q, k, k, i(0, 1), i(1), i(0), 4, out=out) == 7.0).all())


# ---------------------------------------------------------------------------
# refusals of the Python entry points
# ---------------------------------------------------------------------------
def test_preconditions(torch, backend):
    k = torch.zeros(4, 2, 16, 64, device="cuda")
    i = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")      # noqa: E731
    q = torch.zeros(3, 256, device="cuda")
    r = torch.zeros(3, 128, device="cuda")
    for call in (
        lambda: backend.paged_plan_device(i(3), i(2), i(3, 4), i(4), i(1), 16, 4),
        lambda: backend.paged_plan_device(i(3).long(), i(3), i(3, 4), i(4), i(1), 16, 4),
        lambda: backend.paged_plan_device(i(3), i(3), i(3, 4), i(4), i(1), 16, -1),
        lambda: backend.paged_plan_device(i(3), i(3), i(4, 3).t(), i(4), i(1), 16, 4),
        lambda: backend.paged_append_device(k, k.bfloat16(), i(3), r, r),
        lambda: backend.paged_append_device(k, k, i(2), r, r),
        lambda: backend.paged_append_device(k, k, i(3), r, r[:2]),
        lambda: backend.paged_append_device(k, k, i(3), r.bfloat16(), r),
        lambda: backend.paged_append_device(k, k, i(3), q, r),
        lambda: backend.paged_append_device(k, k, i(3), r, r, q=q, ropeBase=1e4),
        lambda: backend.paged_append_device(k, k, i(3), r, r, q=q, qOut=q.half()),
        lambda: backend.paged_append_device(k.transpose(0, 1), k.transpose(0, 1), i(3), r, r),
        lambda: backend.paged_attention_device(q, k, k, i(2, 4), i(2), i(2), 4),
        lambda: backend.paged_attention_device(q, k, k, i(2, 4), i(3), i(2), 3),
        lambda: backend.paged_attention_device(q.half(), k, k, i(2, 4), i(3), i(2), 4),
        lambda: backend.paged_attention_device(q, k, k, i(2, 4), i(3), i(2), 4, out=q.bfloat16()),
        lambda: backend.paged_attention_device(q.cpu(), k, k, i(2, 4), i(3), i(2), 4),
        lambda: T.PagedKVCache(backend, 1, 4, 24, 2, 64, 2, 4),
        lambda: T.PagedKVCache(backend, 1, 4, 16, 2, 64, 2, 4, dtype=torch.float16),
    ):
        with pytest.raises(PreconditionFailure):
            call()
    with pytest.raises(T.HIPBackendError):
        backend.paged_plan_device(i(3), i(3), i(3, 4), i(4), i(1), 24, 4)
    for call in (lambda: backend.paged_plan_device(i(3), i(3), i(3, 4), i(4), i(1), 1 << 35, 4),
                 lambda: backend.paged_attention_device(q, k, k, i(2, 4), i(3), i(2), 4, maxContextLen=1 << 31)):
        with pytest.raises(PreconditionFailure):
            call()
    with pytest.raises(T.HIPBackendError):
        backend.paged_append_device(k, k, i(3), r, r, positions=i(3), ropeBase=1e300)


# ---------------------------------------------------------------------------
# the calls together
# ---------------------------------------------------------------------------
class _Model:
    """One attention layer of a served model: rows of x -> q | k | v -> cache -> attention."""

    def __init__(self, torch, backend, seed, nh, nkv, hd, width):
        self.backend, self.nh, self.nkv, self.hd = backend, nh, nkv, hd
        w = (np.random.default_rng(seed).normal(size=(width, (nh + 2 * nkv) * hd)) * width ** -0.5).astype(np.float32)
        self.w = T.DeviceWeight(backend, T.quantize(w, T.QuantizationMode.perChannel))

    def step(self, cache, plan, x, q_type=None, **kw):
        nq, nk = self.nh * self.hd, self.nkv * self.hd
        y = self.backend.matmul_device(x, self.w)
        rows, q = y.clone(), y[:, :nq]         # fp32 queries are rotated in place
        if q_type is not None:
            q = q.new_empty(q.shape, dtype=q_type)
        q = cache.append(0, plan, y[:, nq:nq + nk], y[:, nq + nk:], y[:, :nq], ropeBase=10000.0, qOut=q)
        return rows, cache.attention(0, plan, q, self.nh, **kw)


def test_served_requests_equal_whole_sequences(torch, backend):
    # Requests of different lengths, their prompts in chunks beside other
    # requests' single tokens, some waiting for blocks that others give back:
    # every granted row equals causal attention over its own sequence.
    nh, nkv, hd, width = 8, 2, 64, 96
    model = _Model(torch, backend, 3, nh, nkv, hd, width)
    rows, bs = 6, 8
    cache = T.PagedKVCache(backend, 1, 15, bs, nkv, hd, rows, 12)
    rng = np.random.default_rng(4)
    history = {b: np.zeros((0, (nh + 2 * nkv) * hd)) for b in range(rows)}   # each request's rows of q | k | v
    checked = waited = 0
    for step in range(40):
        new = [-1 if len(history[b]) > 27 or rng.random() < 0.06 else int(rng.choice([0, 1, 1, 1, 5, 23]))
               for b in range(rows)]
        total = sum(max(n, 0) for n in new)
        plan = cache.plan(_ints(torch, new), total)
        y, out = model.step(cache, plan, torch.randn(total, width, device="cuda"))
        y, out = _np(y), _np(out)
        granted, at = _np(plan.granted), 0
        for b, n in enumerate(new):
            if n < 0:
                history[b] = history[b][:0]
                continue
            if n and granted[b] == n:
                history[b] = np.concatenate([history[b], y[at:at + n]])
                _check_rows(out[at:at + n], history[b], nh, nkv, hd)
                checked += n
            elif n:
                waited += 1
            at += n
        assert (_np(cache.contextLens) == [len(history[b]) for b in range(rows)]).all()
    assert checked > 200 and waited > 2


def _check_rows(got, y, nh, nkv, hd):
    """The newest rows of a sequence whose projections are y, all fp32."""
    n, pos = len(got), np.arange(len(y))
    q = P.rotate(y[:, :nh * hd], pos, nh, 10000.0)[-n:]
    k = P.rotate(y[:, nh * hd:(nh + nkv) * hd], pos, nkv, 10000.0).reshape(-1, nkv, hd)
    v = y[:, (nh + nkv) * hd:].reshape(-1, nkv, hd)
    case = (np.zeros((1, 1), int), [0, n], [len(y)], nh)
    keys, values = k.transpose(1, 0, 2)[None], v.transpose(1, 0, 2)[None]
    want, bound = P.attention(q, keys, values, *case)
    mass, _ = P.attention(q, keys, np.abs(values), *case)
    # rotated values are off by 16 half steps of the largest (test_append), so a
    # score by that times sum |k| and sum |q|, and a probability by twice that
    qm, km = np.abs(q).max(), np.abs(k).max()
    qs, ks = np.abs(q.reshape(n, nh, hd)).sum(-1).max(), np.abs(k).sum(-1).max()
    _close(got, want, bound + U32 * np.abs(want) + 2 * 16 * U32 * (qm * ks + km * qs) / hd ** 0.5 * mass)


@pytest.mark.parametrize("rows,most_tokens", [(4, 60), (1030, 1200)])
def test_requests_past_the_steps_entries_wait(torch, backend, rows, most_tokens):
    # A step of more tokens than it has entries: who passes them keeps its length (its keys are
    # never stored), is served later, and no row meets a place that was not written (NaN here).
    nh, nkv, hd, bs = 4, 2, 64, 16
    cache = T.PagedKVCache(backend, 1, 3 * rows, bs, nkv, hd, rows, 3)
    for a in (cache.keys[0], cache.values[0]):
        a.fill_(float("nan"))
    rng = np.random.default_rng(rows)
    want_len = rng.integers(1, 40, rows)
    history = [np.zeros((0, (nh + 2 * nkv) * hd))] * rows
    waited = 0
    for step in range(60):
        new = np.where([len(h) == 0 for h in history], want_len, 0).astype(np.int32)
        if not new.any():
            break
        plan = cache.plan(_ints(torch, new), most_tokens)
        y = torch.randn(most_tokens, (nh + 2 * nkv) * hd, device="cuda")
        nq, nk = nh * hd, nkv * hd
        q = cache.append(0, plan, y[:, nq:nq + nk], y[:, nq + nk:], y[:, :nq], ropeBase=10000.0)
        out, y, granted, start = _np(cache.attention(0, plan, q, nh)), _np(y), _np(plan.granted), _np(plan.queryStart)
        np.testing.assert_array_equal(granted, np.where(start[1:] <= most_tokens, new, 0))
        for b in np.flatnonzero(granted):
            history[b] = y[start[b]:start[b + 1]]
            if b % max(rows // 8, 1) == 0:
                _check_rows(out[start[b]:start[b + 1]], history[b], nh, nkv, hd)
        assert np.isfinite(out[:min(int(granted.sum()), most_tokens)]).all()
        waited += int(((granted == 0) & (new > 0)).sum())
        np.testing.assert_array_equal(_np(cache.contextLens), [len(h) for h in history])
    assert waited > 0 and all(len(h) for h in history)


@pytest.mark.parametrize("dtype,q_type", [("float32", None), ("bfloat16", "bfloat16")])
def test_captured_step_replays_with_new_lengths(torch, backend, dtype, q_type):
    # plan, product, append, attention and sampling of one decode step captured
    # once and replayed: each replay equals the same step made eagerly on a copy
    nh, nkv, hd, width, rows = 8, 2, 64, 96, 5
    model = _Model(torch, backend, 6, nh, nkv, hd, width)
    dt, qt = getattr(torch, dtype), None if q_type is None else getattr(torch, q_type)
    caches = [T.PagedKVCache(backend, 1, 200, 16, nkv, hd, rows, 30, dtype=dt) for _ in range(2)]
    prompt = _ints(torch, [100, 3, 0, 260, 17])
    x = torch.randn(380, width, device="cuda")
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        for c in caches:
            model.step(c, c.plan(prompt, 380), x, qt)
        new, xs, u = _ints(torch, [1] * rows), torch.randn(rows, width, device="cuda"), torch.rand(rows, device="cuda")

        def step(c):
            p = c.plan(new, rows)
            y = model.step(c, p, xs, qt, maxQueryLen=1, maxContextLen=480)[1].float()
            return y, backend.sample_device(y, u, topP=torch.full((rows,), 0.9, device="cuda"))

        step(caches[0]), step(caches[1])
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            got = step(caches[0])
        for i in range(6):
            new.copy_(_ints(torch, [1, int(i != 2), 1, -1 if i == 3 else 1, 1]))
            xs.copy_(torch.randn(rows, width, device="cuda"))
            u.copy_(torch.rand(rows, device="cuda"))
            want = step(caches[1])
            want = [t.clone() for t in (want[0], *want[1])]
            stream.synchronize()
            graph.replay()
            stream.synchronize()
            n = int(sum(max(v, 0) for v in _np(new)))
            for g, w in zip((got[0], *got[1]), want):
                assert torch.equal(g[:n], w[:n])
            assert torch.equal(caches[0].contextLens, caches[1].contextLens)
            assert torch.equal(caches[0].keys[0], caches[1].keys[0])
