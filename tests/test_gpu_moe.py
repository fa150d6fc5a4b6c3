"""GPU tests of the mixture-of-experts layer (tbh_moe_device) against
oracle/experts_ref.py in float64, whose bound says how far fp32 sums may be."""
from types import SimpleNamespace

import numpy as np
import pytest

import tinybrain_amd as T
from oracle import experts_ref as E
from tinybrain_amd.quantized import PreconditionFailure

pytestmark = pytest.mark.gpu
HALF = {"float32": 2.0 ** -24, "bfloat16": 2.0 ** -8}


@pytest.fixture(scope="module")
def backend():
    b = T.HIPBackend(0)
    yield b
    b.close()


@pytest.fixture(scope="module")
def torch():
    import torch

    return torch


def _np(t):
    return t.double().cpu().numpy() if t.is_floating_point() else t.cpu().numpy()


class Model:
    def __init__(self, backend, seed, experts, hidden, inner, same=False):
        rng = np.random.default_rng(seed)
        self.router = (rng.normal(size=(experts, hidden)) / np.sqrt(hidden)).astype(np.float32)
        if same:
            self.router[:] = self.router[0]
        self.gate, self.up, self.down = (
            [T.quantize_fp8(rng.normal(size=(k, n)) * 2 / np.sqrt(k)) for _ in range(experts)]
            for k, n in ((hidden, inner), (hidden, inner), (inner, hidden)))
        args = [self.router]
        for part in (self.gate, self.up, self.down):
            args += [np.stack([w.data for w in part]), np.stack([w.scales for w in part])]
        self.args = args
        self.layer = backend.moe_layer(*args)

    def check(self, x, got, top_k, normalize, dtype):
        y, experts, weights = got
        parts = [[(w.data, w.scales) for w in p] for p in (self.gate, self.up, self.down)]
        # h is rounded to x's type; an fp32 one is kept in pieces
        want, chosen, share, bound = E.moe(_np(x), self.router, *parts, top_k, normalize,
                                           HALF[dtype] if dtype == "bfloat16" else 0.0)
        np.testing.assert_array_equal(_np(experts), chosen)
        # exp, sums of up to 512 and a division in fp32, logits rounded once from 64 bits
        z = np.abs(_np(x) @ self.router.T.astype(np.float64)).max(1, keepdims=True)
        assert (np.abs(_np(weights) - share) <= share * (540 + 2 * z) * 2.0 ** -24 + 2.0 ** -140).all()
        bound = bound + np.abs(want) * (540 + 2 * z) * 2.0 ** -24
        bound = bound + HALF[dtype] * (np.abs(want) + bound)
        err = np.abs(_np(y) - want)
        assert (err <= bound).all(), (err - bound).max()
        rms = np.sqrt((want ** 2).mean())
        assert np.sqrt((err ** 2).mean()) <= (1e-5 if dtype == "float32" else 5e-3) * rms


def _rows(torch, seed, tokens, hidden, dtype):
    rng = np.random.default_rng(seed)
    x = rng.normal(size=(tokens, hidden)) * np.exp(0.5 * rng.normal(size=hidden))
    return torch.tensor(x, dtype=torch.float32).to(getattr(torch, dtype)).cuda()


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("tokens,experts,top_k,hidden,inner,normalize", [
    (1, 1, 1, 1, 1, True), (1, 4, 2, 256, 128, True), (1, 8, 8, 130, 72, False), (2, 7, 3, 100, 260, True),
    (5, 60, 4, 384, 17, False), (13, 64, 6, 256, 200, False), (16, 3, 2, 129, 128, True), (17, 2, 1, 640, 384, True),
    (33, 2, 2, 128, 130, True), (50, 16, 4, 200, 100, False), (64, 8, 8, 130, 260, True), (65, 5, 2, 128, 128, False),
    (130, 9, 3, 64, 300, True), (6, 512, 32, 64, 40, True), (66, 512, 30, 40, 24, True), (64, 100, 32, 48, 40, False), (3, 5, 5, 1000, 1400, True),
])
def test_layer(torch, backend, dtype, tokens, experts, top_k, hidden, inner, normalize):
    model = Model(backend, tokens * 31 + experts, experts, hidden, inner)
    x = _rows(torch, tokens, tokens, hidden, dtype)
    got = backend.moe_device(x, model.layer, top_k, normalize=normalize)
    model.check(x, got, top_k, normalize, dtype)
    again = backend.moe_device(x, model.layer, top_k, normalize=normalize)
    assert all(torch.equal(a, b) for a, b in zip(got, again))


def test_equal_experts_are_taken_in_order(torch, backend):
    model = Model(backend, 3, 6, 96, 64, same=True)
    x = _rows(torch, 4, 40, 96, "float32")
    got = backend.moe_device(x, model.layer, 4)
    assert bool((got[1] == torch.arange(4, device="cuda", dtype=torch.int32)).all())
    model.check(x, got, 4, True, "float32")


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_rows_that_are_not_finite_touch_no_other(torch, backend, dtype):
    model = Model(backend, 5, 4, 200, 150)
    x = _rows(torch, 6, 30, 200, dtype)
    want = backend.moe_device(x, model.layer, 2)
    z = x.clone()
    z[3, 7], z[9, 199], z[20, 0], z[29] = float("inf"), float("nan"), float("-inf"), float("nan")
    y, experts, weights = backend.moe_device(z, model.layer, 2)
    bad = torch.zeros(30, dtype=torch.bool, device="cuda")
    bad[[3, 9, 20, 29]] = True
    assert bool(torch.isnan(y[bad]).all())
    assert bool(((experts >= 0) & (experts < 4)).all())
    for a, b in zip((y, experts, weights), want):
        assert torch.equal(a[~bad], b[~bad])


def test_an_expert_that_is_not_finite_touches_its_own_tokens(torch, backend):
    model = Model(backend, 7, 5, 150, 130)
    x = _rows(torch, 8, 40, 150, "float32")
    want = backend.moe_device(x, model.layer, 2)
    args = [a.copy() for a in model.args]
    args[5][2, 11, 4] = 0x7F            # down of expert 2: output 11
    args[1][3, 0, 0] = 0x7F             # gate of expert 3: its first inner column
    y, experts, _ = backend.moe_device(x, backend.moe_layer(*args), 2)
    has2, has3 = ((experts == e).any(1) for e in (2, 3))
    assert bool(has2.any()) and bool(has3.any()) and bool((~has2 & ~has3).any())
    assert bool(torch.isnan(y[has3]).all()) and bool(torch.isnan(y[has2][:, 11]).all())
    free = ~has2 & ~has3
    assert torch.equal(y[free], want[0][free])
    keep = torch.arange(150, device="cuda") != 11
    only2 = has2 & ~has3
    assert torch.equal(y[only2][:, keep], want[0][only2][:, keep])


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_strided_rows_and_given_outputs(torch, backend, dtype):
    model = Model(backend, 9, 6, 101, 90)
    wide = _rows(torch, 10, 7, 150, dtype)
    x = wide[:, 5:106]
    out = torch.full((7, 140), 3.0, dtype=x.dtype, device="cuda")
    experts = torch.full((7, 3), -9, dtype=torch.int32, device="cuda")
    weights = torch.zeros(7, 3, device="cuda")
    got = backend.moe_device(x, model.layer, 3, out=out[:, 7:108], experts=experts, weights=weights)
    assert got[1] is experts and got[2] is weights
    model.check(x, got, 3, True, dtype)
    assert bool((out[:, :7] == 3).all()) and bool((out[:, 108:] == 3).all())


def test_captured_before_any_eager_call(torch):
    backend = T.HIPBackend(0)
    model = Model(backend, 11, 12, 160, 120)
    x = _rows(torch, 12, 9, 160, "float32")
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(backend.moe_device(x, model.layer, 3))
        graphs.append(g)
    for seed in range(4):
        x.copy_(_rows(torch, 20 + seed, 9, 160, "float32"))
        for g, out in zip(graphs, outs):
            g.replay()
            torch.cuda.synchronize()
            model.check(x, out, 3, True, "float32")
        eager = backend.moe_device(x, model.layer, 3)
        assert all(torch.equal(a, b) for a, b in zip(eager, outs[0]))
    backend.close()


def test_two_streams(torch, backend):
    model = Model(backend, 13, 16, 300, 260)
    xs = [_rows(torch, 14 + i, 20, 300, "bfloat16") for i in range(2)]
    want = [backend.moe_device(x, model.layer, 4) for x in xs]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [backend.moe_device(x, model.layer, 4, stream=s) for _ in range(10) for x, s in zip(xs, streams)]
    torch.cuda.synchronize()
    for i, g in enumerate(got):
        assert all(torch.equal(a, b) for a, b in zip(g, want[i % 2]))


def test_preconditions(torch, backend):
    model = Model(backend, 15, 3, 32, 16)
    x = torch.zeros(2, 32, device="cuda")
    assert tuple(backend.moe_device(x[:0], model.layer, 1)[0].shape) == (0, 32)
    for bad in (x[0], x[:, :31], x.cpu(), x.half()):
        with pytest.raises(PreconditionFailure):
            backend.moe_device(bad, model.layer, 1)
    for kw in (dict(topK=0), dict(topK=4), dict(topK=1, out=torch.zeros(2, 31, device="cuda")),
               dict(topK=1, out=torch.zeros(2, 32, device="cuda", dtype=torch.bfloat16)),
               dict(topK=2, experts=torch.zeros(2, 1, dtype=torch.int32, device="cuda")),
               dict(topK=2, experts=torch.zeros(2, 2, device="cuda")),
               dict(topK=2, weights=torch.zeros(2, 2, dtype=torch.float64, device="cuda"))):
        with pytest.raises(PreconditionFailure):
            backend.moe_device(x, model.layer, **kw)
    with pytest.raises(PreconditionFailure):
        backend.moe_device(x, SimpleNamespace(hidden=32, experts=3, backend=SimpleNamespace(device=1)), 1)
    with pytest.raises(T.HIPBackendError):
        backend.moe_device(x, model.layer, 1, out=x)
    a = model.args
    for i, bad in ((0, a[0][:2]), (0, a[0].astype(np.float64)), (1, a[1][:, :15]), (2, a[2][:2]),
                   (3, a[3][:, :, :31]), (5, a[3]), (6, a[6][:, :, :0])):
        with pytest.raises(PreconditionFailure):
            backend.moe_layer(*a[:i], bad, *a[i + 1:])
