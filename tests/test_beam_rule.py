"""The oracle's order of candidates in a beam selection (no GPU)."""
import numpy as np

from oracle import experts_ref as E


def test_equal_sums_go_to_the_lowest_row_and_token():
    # logits that score + (logit - log sum) absorbs: all candidates are equal
    x = (np.random.default_rng(0).normal(size=(4, 300)) * 2.0 ** -60).astype(np.float32)
    tokens, parents, scores, _ = E.beam_select(x, np.full(4, -1.0), 4, 6)
    assert tokens.tolist() == [[0, 1, 2, 3, 4, 5]] and parents.tolist() == [[0] * 6]
    assert (scores == -1.0 - np.log(300.0)).all()
    x[0, 7], x[2, 9] = 1.0, 1.0
    tokens, parents, _, _ = E.beam_select(x, [-1.0, -1e30, -3.0, -1e30], 4, 4)
    assert tokens.tolist() == [[7, 0, 1, 2]] and parents.tolist() == [[0, 0, 0, 0]]
    tokens, parents, _, _ = E.beam_select(x[1::2], [-1e30, -1e30], 2, 2)
    assert tokens.tolist() == [[0, 1]] and parents.tolist() == [[0, 0]]
