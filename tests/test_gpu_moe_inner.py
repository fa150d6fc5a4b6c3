"""GPU tests of what the mixture-of-experts layer holds between its products,
h = silu(gate) * up: more than the type of its rows."""
import numpy as np
import pytest

import tinybrain_amd as T
from oracle import experts_ref as E

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def backend():
    b = T.HIPBackend(0)
    yield b
    b.close()


@pytest.fixture(scope="module")
def torch():
    import torch

    return torch


def _stack(ts):
    return np.stack([t.data for t in ts]), np.stack([t.scales for t in ts])


@pytest.mark.parametrize("tokens,experts,top_k,hidden,inner", [
    (1, 4, 2, 96, 200), (13, 64, 6, 160, 130), (64, 4, 2, 64, 260), (70, 3, 3, 130, 72),
])
def test_rows_of_bf16_are_rounded_once(torch, backend, tokens, experts, top_k, hidden, inner):
    """y is off by its own rounding, half a step of bf16 at y's size, by what fp32 sums are off, and
    by what h is, 2^-16 of itself."""
    rng = np.random.default_rng(tokens)
    router = (rng.normal(size=(experts, hidden)) / np.sqrt(hidden)).astype(np.float32)
    gate, up, down = ([T.quantize_fp8(rng.normal(size=(k, n)) * 2 / np.sqrt(k)) for _ in range(experts)]
                      for k, n in ((hidden, inner), (hidden, inner), (inner, hidden)))
    layer = backend.moe_layer(router, *_stack(gate), *_stack(up), *_stack(down))
    x = torch.tensor(rng.normal(size=(tokens, hidden)), dtype=torch.bfloat16, device="cuda")
    y, chosen, weights = backend.moe_device(x, layer, top_k)
    rows = x.double().cpu().numpy()
    want, experts_, share, bound = E.moe(rows, router, *([(w.data, w.scales) for w in p] for p in (gate, up, down)),
                                         top_k, True, 2.0 ** -16)
    np.testing.assert_array_equal(chosen.cpu().numpy(), experts_)
    # weights: exp, sums and a division in fp32, logits rounded once from 64 bits
    z = np.abs(rows @ router.T.astype(np.float64)).max(1, keepdims=True)
    bound = bound + np.abs(want) * (540 + 2 * z) * 2.0 ** -24
    largest = np.abs(want) + bound
    half = np.exp2(np.floor(np.log2(largest)) - 8)
    err = np.abs(y.double().cpu().numpy() - want)
    assert (err <= half + bound).all(), (err / half).max()
    # Errors spread over half a step either way have a square of a third of half squared, here within five standard
    # deviations (0.3 of half squared for one) of the mean over so many.  The sums are a random walk of blocks of 32
    # inputs, each step off by 2^-23 at most; h's errors of 2^-16 at most have signs of their own.
    count = (half ** 2).sum() ** 2 / (half ** 4).sum()
    rounding = np.sqrt((half ** 2).mean() * (1 / 3 + 5 * 0.3 / np.sqrt(count)))
    of_sums = (np.sqrt(3 * max(hidden, inner) / 32 + 20) * 2.0 ** -23 + 2.0 ** -16) * np.sqrt((want ** 2).mean())
    assert np.sqrt((err ** 2).mean()) <= rounding + of_sums
    # and the same rows in fp32 give the same before that rounding
    y32 = backend.moe_device(x.float(), layer, top_k)[0].double().cpu().numpy()
    assert (np.abs(y.double().cpu().numpy() - y32) <= half + 2 * bound).all()


ONE, MINUS = 0x38, 0xB8                      # e4m3 of 1 and -1


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("tokens", [1, 20])
def test_h_past_the_largest_float(torch, backend, dtype, tokens):
    """An infinite h weighs like any other infinity: y is infinite, of its sign, and other tokens' are as they were."""
    hidden, inner = 40, 30
    ones = np.full((1, inner, hidden), ONE, np.uint8)
    up = ones.copy()
    up[:, 1::2] = MINUS                      # h of odd columns is -inf, which `down` turns
    down = np.full((1, hidden, inner), ONE, np.uint8)
    down[:, :, 1::2] = MINUS
    down[:, 1::2] ^= 0x80                    # odd outputs: -inf
    scale = np.ones((1, 1, 1), np.float32)
    layer = backend.moe_layer(np.zeros((1, hidden), np.float32), ones, scale, up, scale, down, scale)
    x = torch.ones(tokens, hidden, dtype=getattr(torch, dtype), device="cuda")
    plain = backend.moe_device(x, layer, 1)[0]
    x[::2] = 2.0 ** 70
    y = backend.moe_device(x, layer, 1)[0]
    assert bool((y[::2, ::2] == float("inf")).all()) and bool((y[::2, 1::2] == -float("inf")).all())
    assert torch.equal(y[1::2], plain[1::2])
