"""FP8 weights, the mixture-of-experts layer, beam search and cache reordering
without a GPU: the oracle (oracle/experts_ref.py) against closed forms, the host
quantizer, and what the C ABI refuses, launches and allocates."""
import ctypes

import numpy as np
import pytest

import tinybrain_amd as T
from oracle import experts_ref as E
from test_host_launches import stand_in  # noqa: F401
from tinybrain_amd import _abi
from tinybrain_amd.fp8 import E4M3
from tinybrain_amd.quantized import PreconditionFailure


# ---------------------------------------------------------------------------
# the oracle and the quantizer
# ---------------------------------------------------------------------------
def test_e4m3_values_are_torchs():
    torch = pytest.importorskip("torch")
    want = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).float().numpy()
    np.testing.assert_array_equal(E4M3, want)
    np.testing.assert_array_equal(E.e4m3_value(np.arange(256)), want.astype(np.float64))


def test_rounding_to_e4m3_is_torchs():
    torch = pytest.importorskip("torch")
    rng = np.random.default_rng(0)
    v = np.concatenate([E4M3[:127], (E4M3[:126] + E4M3[1:127]) / 2, rng.normal(size=4000) * 100,
                        rng.normal(size=4000) * 2.0 ** -7, rng.uniform(-448, 448, 2000)]).astype(np.float32)
    v = np.clip(np.concatenate([v, -v]), -448, 448)
    want = torch.tensor(v).to(torch.float8_e4m3fn)
    np.testing.assert_array_equal(E.round_e4m3(v.astype(np.float64)), want.float().numpy())
    from tinybrain_amd.fp8 import _to_e4m3

    np.testing.assert_array_equal(_to_e4m3(v), want.view(torch.uint8).numpy())


def test_rows_scales():
    x = np.zeros((6, 130))
    x[0, 3], x[1, 3], x[2, 3], x[3, 129], x[4, 0], x[5, :3] = 448, 448.0001, 224, 1.0, 2.0 ** -140, [np.inf, np.nan, 7]
    q, s = E.quantize_rows(x)
    np.testing.assert_array_equal(s, [[1, 2.0 ** -126], [2, 2.0 ** -126], [0.5, 2.0 ** -126], [2.0 ** -126, 2.0 ** -8],
                                      [2.0 ** -126, 2.0 ** -126], [2.0 ** -6, 2.0 ** -126]])
    assert q[0, 3] == 448 and q[1, 3] == 224 and q[2, 3] == 448 and q[3, 129] == 256 and q[4, 0] == 0 and q[5, 2] == 448
    assert np.isnan(q[5, :2]).all()


@pytest.mark.parametrize("k,n", [(1, 1), (128, 128), (130, 7), (200, 300)])
def test_quantizer(k, n):
    rng = np.random.default_rng(k)
    w = (rng.normal(size=(k, n)) * np.exp(rng.normal(size=n))).astype(np.float32)
    w[:, n // 2] = 0
    t = T.quantize_fp8(w)
    d = t.dequantize()
    np.testing.assert_allclose(d, E.widen(t.data, t.scales).T, rtol=2.0 ** -23)
    # half a step of e4m3 (2^-4 relative, 2^-10 of the scale below its normal range), and the division's rounding
    scale = np.repeat(np.repeat(t.scales, 128, 0)[:n], 128, 1)[:, :k].T
    assert (np.abs(d - w) <= np.abs(w) * 2.0 ** -4 * 1.001 + scale * 2.0 ** -10).all()
    assert np.abs(E4M3[t.data]).max() == (448 if n > 1 else 0)       # (1 x 1: its one column is zeroed)


def test_quantizer_refuses():
    for bad in (np.zeros(3), np.array([[np.inf]]), np.array([[np.nan]])):
        with pytest.raises(PreconditionFailure):
            T.quantize_fp8(bad)
    t = T.quantize_fp8(np.zeros((5, 3)))
    assert (t.data == 0).all() and (t.dequantize() == 0).all()
    for kw in (dict(shape=(5, 4)), dict(scales=np.ones((1, 2))), dict(shape=(15,)), dict(shape=(0, 3))):
        with pytest.raises(PreconditionFailure):
            T.FP8Tensor(**{"shape": t.shape, "data": t.data, "scales": t.scales, **kw})


def test_oracle_moe_of_one_expert_is_a_dense_layer():
    rng = np.random.default_rng(1)
    h, i = 20, 12
    parts = [[((rng.integers(0, 100, size=s)).astype(np.uint8), np.full((1, 1), 0.01, np.float32))]
             for s in ((i, h), (i, h), (h, i))]
    x = rng.normal(size=(3, h))
    y, experts, weights, _ = E.moe(x, np.zeros((1, h)), *parts, 1, True, 0.0)
    g, u, d = (E.widen(*p[0]) for p in parts)
    z = x @ g.T
    np.testing.assert_allclose(y, (z / (1 + np.exp(-z)) * (x @ u.T)) @ d.T)
    assert (experts == 0).all() and (weights == 1).all()


def test_oracle_routing():
    # two experts of equal logits: the first; weights over all experts, or over the chosen ones
    router = np.array([[0.0], [1.0], [1.0], [-1.0]])
    e, w = E.route(np.array([[2.0]]), router, 2, False)
    p = np.exp([0, 2, 2, -2]) / np.exp([0, 2, 2, -2]).sum()
    np.testing.assert_array_equal(e, [[1, 2]])
    np.testing.assert_allclose(w, [p[1:3]])
    np.testing.assert_allclose(E.route(np.array([[2.0]]), router, 2, True)[1], [[0.5, 0.5]])


def test_oracle_beams_over_two_steps_are_the_best_pairs():
    # with as many beams as tokens nothing is lost: the best of all pairs
    rng = np.random.default_rng(2)
    v = 5
    first, second = rng.normal(size=v), rng.normal(size=(v, v))
    lp = lambda x: x - np.log(np.exp(x).sum(-1, keepdims=True))  # noqa: E731
    t1, p1, s1, _ = E.beam_select(np.tile(first, (v, 1)), [0.0] + [-np.inf] * (v - 1), v, v)
    assert (p1 == 0).all()
    t2, p2, s2, _ = E.beam_select(second[t1[0]], s1[0], v, v)
    every = sorted(((lp(first)[a] + lp(second[a])[b], a, b) for a in range(v) for b in range(v)), reverse=True)[:v]
    assert [(t1[0][p], t) for p, t in zip(p2[0], t2[0])] == [(a, b) for _, a, b in every]
    np.testing.assert_allclose(s2[0], [s for s, _, _ in every])


def test_oracle_reorder_known_answer():
    table = np.array([[0, 1], [2, 3], [4, 5], [6, 7]])
    # row 2 goes on twice, row 0 once (as row 3), rows 1 and 3 are dropped
    new, moves, fine = E.reorder(table, [2, 2, 2, 0], [5] * 4, 4, 4, 8)
    np.testing.assert_array_equal(new, [[2, 3], [6, 7], [4, 5], [0, 1]])
    assert moves == [(4, 2, 4), (5, 3, 1), (4, 6, 4), (5, 7, 1)] and fine.tolist() == [1]
    assert E.reorder(table, [2, 2, 2, 0], [5] * 4, 4, 4, 8, [4])[1] == [(5, 3, 1), (5, 7, 1)]
    assert E.reorder(table, [2, 2, 4, 0], [5] * 4, 4, 4, 8)[2].tolist() == [0]


# ---------------------------------------------------------------------------
# refusals that read no handle
# ---------------------------------------------------------------------------
_HANDLE = ctypes.create_string_buffer(4096)
DEV = ctypes.addressof(_HANDLE)
_BUF = (ctypes.c_char * 8192)()
PTR = (ctypes.addressof(_BUF) + 255) // 256 * 256


def test_creating_refuses():
    L, out = _abi.lib(), ctypes.c_void_p()
    def fp8(**kw):
        d = _abi.FP8Desc(**{**dict(K=4, N=4, data=PTR, scales=PTR), **kw})
        return L.tbh_fp8_weight_create(DEV, ctypes.byref(d), ctypes.byref(out))
    for kw in (dict(K=0), dict(N=-1), dict(data=None), dict(scales=None)):
        assert fp8(**kw) == _abi.E_INVALID
    assert fp8(K=(1 << 20) + 1) == fp8(N=(1 << 24) + 1) == _abi.E_UNSUPPORTED
    assert L.tbh_fp8_weight_create(None, None, ctypes.byref(out)) == _abi.E_INVALID
    assert L.tbh_fp8_weight_create(DEV, None, None) == _abi.E_INVALID
    assert L.tbh_fp8_weight_destroy(None) == L.tbh_moe_destroy(None) == _abi.OK

    def moe(**kw):
        f = dict(hidden=4, intermediate=4, experts=2, **{n: PTR for n in (
            "router", "gate", "up", "down", "gate_scales", "up_scales", "down_scales")})
        f.update(kw)
        d = _abi.MoEDesc(**f)
        return L.tbh_moe_create(DEV, ctypes.byref(d), ctypes.byref(out))
    for n, _ in _abi.MoEDesc._fields_:
        if n != "reserved":
            assert moe(**{n: 0 if n in ("hidden", "intermediate", "experts") else None}) == _abi.E_INVALID
    for kw in (dict(hidden=(1 << 17) + 1), dict(intermediate=1 << 18), dict(experts=513)):
        assert moe(**kw) == _abi.E_UNSUPPORTED
    assert L.tbh_moe_create(DEV, None, None) == _abi.E_INVALID
    assert L.tbh_fp8_matmul_device(None, PTR, 0, 1, 4, 4, PTR, 0, 4, None, 0, None) == _abi.E_INVALID
    assert L.tbh_moe_device(None, PTR, 0, 1, 4, 1, 1, PTR, 4, None, None, None, 0, None) == _abi.E_INVALID


def _select(**kw):
    a = dict(dev=DEV, logits=PTR, ld=10, requests=2, beams=2, vocab=10, scores=PTR, done=None, eos=-1, k=2, tokens=PTR,
             parents=PTR, out=PTR, done_out=PTR, ws=None, bytes=0)
    a.update(kw)
    return _abi.lib().tbh_beam_select_device(
        a["dev"], a["logits"], a["ld"], a["requests"], a["beams"], a["vocab"], a["scores"], a["done"], a["eos"], a["k"],
        a["tokens"], a["parents"], a["out"], a["done_out"], a["ws"], a["bytes"], None)


@pytest.mark.parametrize("change", [
    dict(dev=None), dict(logits=None), dict(ld=9), dict(requests=-1), dict(beams=0), dict(vocab=0), dict(scores=None),
    dict(done=PTR), dict(done=PTR, eos=10), dict(k=0), dict(tokens=None), dict(parents=None), dict(out=None),
    dict(ws=PTR + 8, bytes=1 << 20), dict(ws=PTR, bytes=10), dict(ws=PTR, bytes=-1),
])
def test_select_refuses(change):
    assert _select(**change) == _abi.E_INVALID
    assert "tbh_beam_select" in _abi.last_error()


def test_select_limits():
    for kw in (dict(beams=65), dict(k=65), dict(vocab=(1 << 20) + 1, ld=1 << 21), dict(requests=(1 << 19) + 1)):
        assert _select(**kw) == _abi.E_UNSUPPORTED
    assert _select(requests=0, logits=None) == _abi.OK
    n = ctypes.c_int64()
    f = _abi.lib().tbh_beam_select_workspace
    assert f(DEV, 3, 4, 32000, 4, ctypes.byref(n)) == _abi.OK and n.value > 0
    for requests, beams, vocab, k in ((1, 64, 1 << 20, 64), (1 << 14, 64, 1 << 20, 64), (1 << 20, 1, 1, 1)):
        assert f(DEV, requests, beams, vocab, k, ctypes.byref(n)) == _abi.OK and 0 < n.value <= (128 << 20) + _abi.WORKSPACE_COUNTERS
    assert f(DEV, 3, 4, 32000, 4, None) == _abi.E_INVALID


def _reorder(layout=None, **kw):
    f = dict(num_blocks=8, block_size=16, num_kv_heads=2, head_dim=64, type=0, max_requests=4, max_blocks=4)
    f.update(layout or {})
    a = dict(dev=DEV, beams=2, parents=PTR, ctx=PTR, shared=None, table=PTR, out=PTR + 256, layers=1, k=[PTR], v=[PTR],
             flag=None)
    a.update(kw)
    arrays = [None if c is None else (ctypes.c_void_p * max(1, len(c)))(*c) for c in (a["k"], a["v"])]
    return _abi.lib().tbh_paged_reorder_device(a["dev"], ctypes.byref(_abi.PagedLayout(**f)), a["beams"], a["parents"],
                                               a["ctx"], a["shared"], a["table"], a["out"], a["layers"], *arrays,
                                               a["flag"], None)


@pytest.mark.parametrize("change", [
    dict(dev=None), dict(beams=0), dict(beams=3), dict(beams=65), dict(parents=None), dict(ctx=None), dict(table=None),
    dict(out=None), dict(layers=-1), dict(k=None), dict(v=None), dict(k=[None]), dict(v=[None]), dict(k=[PTR + 8]),
    dict(v=[PTR + 4]), dict(out=PTR + 60), dict(out=PTR - 60),
])
def test_reorder_refuses(change):
    assert _reorder(**change) == _abi.E_INVALID
    assert "tbh_paged_reorder" in _abi.last_error()


@pytest.mark.parametrize("change,status", [
    (dict(block_size=24), _abi.E_INVALID), (dict(num_blocks=-1), _abi.E_INVALID), (dict(head_dim=0), _abi.E_INVALID),
    (dict(type=2), _abi.E_INVALID), (dict(head_dim=257), _abi.E_UNSUPPORTED), (dict(max_blocks=-1), _abi.E_INVALID)])
def test_reorder_refuses_layouts(change, status):
    assert _reorder(change) == status


def test_reorder_of_nothing():
    assert _reorder(dict(max_requests=0), parents=None) == _abi.OK


# ---------------------------------------------------------------------------
# with handles, over the stand-in for the HIP runtime
# ---------------------------------------------------------------------------
MAKE = """
import tinybrain_amd as T
backend = T.HIPBackend(0)
dev = backend._dev
rng = np.random.default_rng(0)
w = backend.fp8_weight(T.quantize_fp8(rng.normal(size=(300, 200))))
def stack(k, n):
    ts = [T.quantize_fp8(rng.normal(size=(k, n))) for _ in range(6)]
    return np.stack([t.data for t in ts]), np.stack([t.scales for t in ts])
layer = backend.moe_layer(np.zeros((6, 40), np.float32), *stack(40, 50), *stack(40, 50), *stack(50, 40))
def fp8(m, ws=None, size=0, stream=STREAM, x=P, xt=0, k=300, xs=300, y=P + (1 << 38), yt=0, ys=200, handle=w.handle):
    return L.tbh_fp8_matmul_device(handle, x, xt, m, k, xs, y, yt, ys, ws, size, stream)
def moe(t, ws=None, size=0, stream=STREAM, x=P, xt=0, xs=40, k=2, y=P + (1 << 38), ys=40, e=None, p=None):
    return L.tbh_moe_device(layer.handle, x, xt, t, xs, k, 1, y, ys, e, p, ws, size, stream)
def select(r, ws=None, size=0, stream=STREAM, vocab=9000):
    return L.tbh_beam_select_device(dev, P, vocab, r, 4, vocab, P, None, -1, 4, P, P, P, None, ws, size, stream)
def reorder(l, beams=4, layers=2, stream=STREAM, out=P):
    arrays = (ctypes.c_void_p * layers)(*[P] * layers)
    return L.tbh_paged_reorder_device(dev, ctypes.byref(l), beams, P, P, None, P, out, layers, arrays, arrays, None, stream)
"""


def test_calls_refuse_arguments(stand_in):  # noqa: F811
    stand_in(MAKE + """
I, U = _abi.E_INVALID, _abi.E_UNSUPPORTED
for kw in (dict(m=-1), dict(xt=2), dict(yt=-1), dict(k=299), dict(x=None), dict(y=None), dict(xs=299), dict(ys=199),
           dict(ws=P + 8, size=1 << 30), dict(ws=P, size=10, m=40), dict(ws=P, size=-1, m=40), dict(x=P + 2), dict(y=P + 1),
           dict(xt=1, x=P + 1), dict(y=P), dict(y=P + 2396), dict(y=P - 1596), dict(xs=500, y=P)):
    assert fp8(**{"m": 2, **kw}) == I, kw
    assert "tbh_fp8_matmul" in _abi.last_error()
assert fp8(0, x=None) == 0 and fp8(1, xs=0, ys=0) == 0
assert fp8(2, y=P + 2400) == 0 and fp8(2, y=P - 1600) == 0 and fp8(2, xs=500, y=P + 1200, ys=500) == 0
for kw in (dict(t=-1), dict(xt=2), dict(k=0), dict(k=7), dict(x=None), dict(y=None), dict(xs=39), dict(ys=39),
           dict(ws=P + 8, size=1 << 30), dict(ws=P, size=10), dict(x=P + 2), dict(e=P + 2), dict(p=P + 1),
           dict(y=P), dict(y=P + 316), dict(y=P - 316)):
    assert moe(**{"t": 2, **kw}) == I, kw
    assert "tbh_moe" in _abi.last_error()
assert moe(0, x=None) == 0 and moe(2, y=P + 320) == 0 and moe(2, xs=80, ys=80, y=P + 160) == 0
n = ctypes.c_int64()
assert L.tbh_moe_workspace(layer.handle, 0, 5, 2, None) == I and L.tbh_fp8_matmul_workspace(w.handle, 5, None) == I
assert L.tbh_moe_workspace(layer.handle, 0, 5, 9, ctypes.byref(n)) == I
assert L.tbh_fp8_matmul_workspace(w.handle, -1, ctypes.byref(n)) == I
launches()
for t in (1, 5, 64, 1000):
    assert L.tbh_moe_workspace(layer.handle, 0, t, 2, ctypes.byref(n)) == 0
    assert moe(t, ws=P, size=n.value) == 0 and moe(t, ws=P, size=n.value - 1) == I
    assert L.tbh_fp8_matmul_workspace(w.handle, t, ctypes.byref(n)) == 0
    assert fp8(t, ws=P, size=n.value) == 0 and (t <= 32 or fp8(t, ws=P, size=n.value - 1) == I)
""")


def test_memory_and_captures(stand_in):  # noqa: F811
    stand_in(MAKE + """
launches()
S.stand_in_capturing(1)                       # streams without a workspace
assert fp8(70, stream=0x3000) == 0 and ["fp8_rows" in l[3] for l in launches()] == [True]
assert moe(3, stream=0x3000) == _abi.E_OOM and select(3, stream=0x3000) == _abi.E_OOM and launches() == []
assert "eager" in _abi.last_error()
S.stand_in_capturing(0)
assert moe(3, stream=0x3000) == 0 and select(3, stream=0x3000) == 0 and launches()
S.stand_in_capturing(1)
assert moe(3, stream=0x3000) == 0 and select(3, stream=0x3000) == 0 and launches()
S.stand_in_capturing(0)
S.stand_in_limits(0, ALL)
assert fp8(70, stream=0x5000) == 0 and moe(3, stream=0x5000) == _abi.E_OOM and select(3, stream=0x5000) == _abi.E_OOM
assert fp8(70) == 0                           # the failed allocation's error is no launch's
for make in (lambda: backend.fp8_weight(T.quantize_fp8(np.ones((3, 3)))),
             lambda: backend.moe_layer(np.zeros((6, 40), np.float32), *stack(40, 50), *stack(40, 50), *stack(50, 40))):
    try:
        make()
        raise SystemExit("made without memory")
    except T.HIPBackendError as e:
        assert e.status == _abi.E_OOM
    assert fp8(70) == 0
S.stand_in_limits(ALL, ALL)
before = S.stand_in_bytes()
for limit in (100, 5000, 30000, 100000):     # whatever it fails at, nothing is kept
    S.stand_in_limits(limit, ALL)
    try:
        backend.moe_layer(np.zeros((6, 40), np.float32), *stack(40, 50), *stack(40, 50), *stack(50, 40))
    except T.HIPBackendError:
        assert S.stand_in_bytes() == before, limit
S.stand_in_limits(ALL, ALL)
layer.close(), w.close()
""")


def test_parts_and_grids(stand_in):  # noqa: F811
    stand_in(MAKE + """
for m in (1, 33, (1 << 14) + 1, 1 << 22):
    launches()
    assert fp8(m) == 0, _abi.last_error()
    assert launches()
for t in (1, 64, 65, 5000):
    assert moe(t) == 0 and len(launches()) == 3 * -(-t // 64)
for r in (1, 1000, 1 << 18):
    assert select(r) == 0, _abi.last_error()
    assert S.stand_in_bytes() < 600 << 20 and launches()
for rows in (4, 1 << 20):
    for layers in (1, 24, 25, 60):
        assert reorder(layout(max_requests=rows, max_blocks=8), layers=layers) == 0, _abi.last_error()
        assert len(launches()) == -(-layers // 24) + 1          # and the table in place
        assert reorder(layout(max_requests=rows, max_blocks=8), layers=layers, out=P + (1 << 36)) == 0
        assert len(launches()) == -(-layers // 24)
assert reorder(layout(max_requests=1 << 22, max_blocks=8)) == _abi.E_UNSUPPORTED and launches() == []
""")


def test_threads_on_one_stream(stand_in):  # noqa: F811
    stand_in(MAKE + """
calls = [lambda: fp8(70), lambda: moe(5), lambda: select(20000), lambda: reorder(layout())]
launches()
one = []
for c in calls:
    assert c() == 0
    one.append([n for _, _, _, n in launches()])
assert all(len(x) > 1 for x in one)
def work(t):
    for r in range(12):
        for i in range(len(calls)):
            assert calls[(i + t + r) % len(calls)]() == 0
threads = [threading.Thread(target=work, args=(t,)) for t in range(6)]
[t.start() for t in threads], [t.join() for t in threads]
got, at = [n for _, _, _, n in launches()], 0
assert len(got) == 6 * 12 * sum(map(len, one))
while at < len(got):
    at += next(len(x) for x in one if got[at:at + len(x)] == x)
""")
