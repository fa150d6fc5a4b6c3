"""GPU tests of how exact a row's sum of exp(logit) is in beam selection, which
decides the order of candidates of different rows.  Its terms are off by at most 2e-12
of themselves (a polynomial within 1.1e-12, and 64-bit roundings of arguments of
at most some hundred), the sums of up to 2^20 of them in 64 bits by less than 1e-12, so that the
logarithm and a score before its rounding to fp32 are within 4e-12."""
import numpy as np
import pytest

import tinybrain_amd as T
from oracle import experts_ref as E

pytestmark = pytest.mark.gpu
OFF = 4e-12


@pytest.fixture(scope="module")
def backend():
    b = T.HIPBackend(0)
    yield b
    b.close()


@pytest.fixture(scope="module")
def torch():
    import torch

    return torch


def _log_sum(x):
    x = x.astype(np.float64)
    top = x.max(-1, keepdims=True)
    return (top + np.log(np.exp(x - top).sum(-1, keepdims=True)))[..., 0]


def _flat_tails(rng, rows, vocab):
    """One large logit, all others equal and some way below."""
    x = np.repeat(rng.uniform(-11, -5, (rows, 1)), vocab, 1)
    x[np.arange(rows), rng.integers(0, vocab, rows)] = rng.uniform(0, 0.5, rows)
    return x.astype(np.float32)


ROWS = {
    "flat": _flat_tails,
    "normal": lambda rng, rows, vocab: (rng.normal(size=(rows, vocab)) * 2.5).astype(np.float32),
    "wide": lambda rng, rows, vocab: (rng.normal(size=(rows, vocab)) * 40).astype(np.float32),
    "ascending": lambda rng, rows, vocab: np.sort(rng.normal(size=(rows, vocab)) * 3).astype(np.float32),
    "far": lambda rng, rows, vocab: (1e3 + rng.integers(-900, 5, (rows, vocab)) / 64).astype(np.float32),
}


def _rows(kind, rows, vocab):
    """Logits, and scores next to the negative of the best candidates' log
    probability: sums next to 0, whose rounding to fp32 hides nothing."""
    x = ROWS[kind](np.random.default_rng(rows + vocab), rows, vocab)
    return x, (_log_sum(x) - x.max(1)).astype(np.float32)


@pytest.mark.parametrize("kind", sorted(ROWS))
@pytest.mark.parametrize("rows,vocab", [(3, 1), (4, 300), (4, 100000), (300, 30001), (256, 70000), (2, 1 << 20)])
def test_scores(torch, backend, kind, rows, vocab):
    # the last two but one: parts of some steps, a block of 16 waves a row (k = 16)
    x, s = _rows(kind, rows, vocab)
    got = backend.beam_select_device(torch.tensor(x, device="cuda"), torch.tensor(s, device="cuda"), 1, k=16)
    want = E.beam_select(x, s, 1, 16)[2]
    best = got[2].cpu().numpy()
    fine = np.isfinite(want)
    np.testing.assert_array_equal(np.isfinite(best), fine)
    assert (np.abs(best[fine] - want[fine]) <= np.abs(want[fine]) * 2.0 ** -24 + OFF).all()


def test_order_between_rows(torch, backend):
    """Best candidates of eight rows whose sums lie some 1e-8 apart."""
    requests, beams, vocab = 32, 8, 20000
    x, s = _rows("flat", requests * beams, vocab)
    key = s.astype(np.float64) + (x.max(1).astype(np.float64) - _log_sum(x))
    gaps = np.diff(np.sort(key.reshape(requests, beams), 1), axis=1)
    assert np.median(gaps) < 1e-7 and gaps.min() > 2 * OFF
    got = backend.beam_select_device(torch.tensor(x, device="cuda"), torch.tensor(s, device="cuda"), beams)
    want = E.beam_select(x, s, beams, beams)
    for g, w in zip(got[:2], want[:2]):
        np.testing.assert_array_equal(g.cpu().numpy(), w)
