"""GPU tests of beam selection where candidates of different logits are equal: a
sum score + (logit - log sum) in 64 bits that is much larger than a logit absorbs
it.  Equal ones go to the lowest row, then the lowest token, as in the oracle,
which sorts a request's sums by nothing else.  Logits are taken so small (2^-60, and
sums of 1 and more, whose steps are 2^-52 and more) or scores so large that an
error of the sums' last bits makes no difference to what is equal."""
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


def _check(torch, backend, x, scores, beams, k, done=None, eos=-1):
    x, scores = np.asarray(x, np.float32), np.asarray(scores, np.float32)
    d = None if done is None else torch.tensor(np.asarray(done), dtype=torch.int32, device="cuda")
    got = backend.beam_select_device(torch.tensor(x, device="cuda"), torch.tensor(scores, device="cuda"), beams, k=k,
                                     done=d, eos=eos)
    want = E.beam_select(x, scores, beams, k, done, eos)
    for g, w, name in zip(got, want, ("tokens", "parents", "scores", "done")):
        if name != "scores":
            np.testing.assert_array_equal(g.cpu().numpy(), w, err_msg=name)
    return got


def _tiny(rng, rows, vocab):
    return rng.normal(size=(rows, vocab)) * 2.0 ** -60


# one list, several parts of a row, a block of 16 waves a row
SHAPES = [(4, 300, 4, 6), (8, 9000, 4, 8), (12, 40001, 3, 7), (256, 33000, 2, 32), (2, 1 << 20, 1, 64)]


@pytest.mark.parametrize("rows,vocab,beams,k", SHAPES)
def test_logits_that_the_sum_absorbs(torch, backend, rows, vocab, beams, k):
    rng = np.random.default_rng(vocab)
    x = _tiny(rng, rows, vocab)
    got = _check(torch, backend, x, np.full(rows, -1.5), beams, k)
    assert got[0][0].tolist() == list(range(k)) and bool((got[1] % beams == 0).all())
    x[:, :vocab // 2] = np.nan
    x[:, vocab - 9::2] = -np.inf
    _check(torch, backend, x, -rng.integers(1, 4, rows), beams, k)


@pytest.mark.parametrize("rows,vocab,beams,k", SHAPES[:4])
def test_some_of_a_rows_candidates_are_equal(torch, backend, rows, vocab, beams, k):
    rng = np.random.default_rng(vocab + 1)
    x = _tiny(rng, rows // beams, vocab)
    # fewer than k larger ones, of equal and of different size; the rest below zero or absorbed
    for row in x:
        row[rng.choice(vocab, k // 2, replace=False)] = rng.integers(1, 4, k // 2)
        row[rng.choice(vocab, vocab // 3, replace=False)] = -1.0
    # A request's rows are copies, and scores either equal or no whole numbers apart: sums of the same terms in another
    # order, and 1 + (2 - total) beside 2 + (1 - total), differ in their last bits by rounding alone, whoever adds them.
    x = x.repeat(beams, 0)
    _check(torch, backend, x, np.full(rows, -2.0), beams, k)
    _check(torch, backend, x, -1.25 - 0.37 * rng.integers(0, 3, rows), beams, k, (rng.random(rows) < 0.3).astype(np.int32),
           vocab - 1)


@pytest.mark.parametrize("vocab", [3, 40, 5000])
def test_zeros_and_what_is_next_to_them(torch, backend, vocab):
    rng = np.random.default_rng(vocab)
    x = rng.choice(np.array([0.0, -0.0, 1e-45, -1e-45, 1e-40, -1e-38], np.float32), size=(6, vocab))
    _check(torch, backend, x, np.zeros(6), 3, 5)


def test_scores_that_absorb_every_logit(torch, backend):
    # beams that a caller parks far below the others, and no others
    rng = np.random.default_rng(7)
    x = rng.normal(size=(8, 700))
    _check(torch, backend, x, np.full(8, -1e30), 4, 9)
    _check(torch, backend, x, [0.0, -1e30, -1e30, -1e30] * 2, 4, 8)
    # one live row of three tokens, then the parked rows' lowest
    x[:] = -np.inf
    x[0, [5, 9, 600]], x[4, [1, 2, 3]] = [1, 2, 3], [3, 2, 1]
    for r in (1, 2, 3, 5, 6, 7):
        x[r, 100:] = rng.normal(size=600)
    got = _check(torch, backend, x, [0.0, -1e30, -1e30, -1e30] * 2, 4, 6)
    assert got[0].tolist() == [[600, 9, 5, 100, 101, 102], [1, 2, 3, 100, 101, 102]]
    assert got[1].tolist() == [[0, 0, 0, 1, 1, 1], [4, 4, 4, 5, 5, 5]]


def test_ended_tokens_follow_the_tokens_taken(torch, backend):
    rng = np.random.default_rng(8)
    got = _check(torch, backend, _tiny(rng, 4, 5000), [-1.0, -1.0, -2.0, -2.0], 2, 4, np.zeros(4, np.int32), 2)
    assert got[3].tolist() == [[0, 0, 1, 0]] * 2
