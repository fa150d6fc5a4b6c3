"""GPU tests of what the mixture-of-experts layer holds between its products,
h = silu(gate) * up."""
import numpy as np
import pytest

import tinybrain_amd as T

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
