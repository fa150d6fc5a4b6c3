"""GPU tests of the mixture-of-experts layer at the widths of real models: logits
summed over one to four parts of the inputs, with up to 64 experts and with more."""
import numpy as np
import pytest

import tinybrain_amd as T
from oracle import experts_ref as E

pytestmark = pytest.mark.gpu
HALF = {"float32": 2.0 ** -24, "bfloat16": 2.0 ** -8}


@pytest.fixture(scope="module")
def backend():
    b = T.HIPBackend(0)
    yield b
    b.close()


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("hidden", [700, 1409, 1500, 1921, 2000, 2048, 4100])      # 1, 2, 3, 3, 4, 4, 4 parts
@pytest.mark.parametrize("tokens,experts,top_k", [(1, 8, 2), (19, 64, 4), (7, 65, 6), (3, 130, 8), (2, 512, 3)])
def test_layer(backend, dtype, hidden, tokens, experts, top_k):
    torch = pytest.importorskip("torch")
    inner = 24
    rng = np.random.default_rng(hidden + experts)
    router = (rng.normal(size=(experts, hidden)) / np.sqrt(hidden)).astype(np.float32)
    # few different matrices, by the experts in turn
    parts = [[T.quantize_fp8(rng.normal(size=(k, n)) * 2 / np.sqrt(k)) for _ in range(5)]
             for k, n in ((hidden, inner), (hidden, inner), (inner, hidden))]
    args, lists = [router], []
    for part in parts:
        every = [part[e % 5] for e in range(experts)]
        lists.append([(w.data, w.scales) for w in every])
        args += [np.stack([w.data for w in every]), np.stack([w.scales for w in every])]
    layer = backend.moe_layer(*args)
    x = torch.tensor(rng.normal(size=(tokens, hidden)), dtype=getattr(torch, dtype), device="cuda")
    rows = x.double().cpu().numpy()
    y, chosen, weights = backend.moe_device(x, layer, top_k, normalize=False)
    want, experts_, share, bound = E.moe(rows, router, *lists, top_k, False, 0.0)
    np.testing.assert_array_equal(chosen.cpu().numpy(), experts_)
    # exp, sums of up to 512 and a division in fp32, logits rounded once from 64 bits
    z = np.abs(rows @ router.T.astype(np.float64)).max(1, keepdims=True)
    of_weights = (540 + 2 * z) * 2.0 ** -24
    assert (np.abs(weights.double().cpu().numpy() - share) <= share * of_weights).all()
    bound = bound + np.abs(want) * of_weights
    err = np.abs(y.double().cpu().numpy() - want)
    assert (err <= bound + HALF[dtype] * (np.abs(want) + bound)).all()
    if dtype == "float32":
        # Gate, up and down each add a block of 32 inputs to an fp32 sum at a time, off by at most 2^-23 of it, a
        # random walk of 3 hidden / 32 such steps at most (inner is the shorter); h's exp, division and product and
        # the weights' own are some 20 more.
        rms = np.sqrt((want ** 2).mean())
        assert np.sqrt((err ** 2).mean()) <= np.sqrt(3 * hidden / 32 + 20) * 2.0 ** -23 * rms
    layer.close()
