"""GPU tests of beam selection and cache reordering (tbh_beam_select_device,
tbh_paged_reorder_device) against oracle/experts_ref.py.  Tokens, parents and
copies are equal.  Scores are rounded once from 64 bits, and a row's sum of exp(d),
d = logit - largest, has terms off by (2 + |d|) 2^-23 of themselves and steps of 16 fp32
additions: its logarithm is off by the mean of that over the row's probabilities,
and the mean of |d| is at most their entropy, at most ln(vocab)."""
import numpy as np
import pytest

import tinybrain_amd as T
from oracle import experts_ref as E
from tinybrain_amd.quantized import PreconditionFailure

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


def _ints(torch, a):
    return torch.tensor(np.asarray(a), dtype=torch.int32, device="cuda")


def _select(torch, backend, logits, scores, beams, k, done=None, eos=-1):
    x = torch.tensor(np.asarray(logits, np.float32), device="cuda")
    s = torch.tensor(np.asarray(scores, np.float32), device="cuda")
    d = None if done is None else _ints(torch, done)
    got = backend.beam_select_device(x, s, beams, k=k, done=d, eos=eos)
    _compare(got, E.beam_select(np.asarray(logits, np.float32), np.asarray(scores, np.float32), beams, k, done, eos),
             np.shape(logits)[1])
    return got


def _compare(got, want, vocab=1 << 20):
    for g, w, name in zip(got, want, ("tokens", "parents", "scores", "done")):
        g = g.cpu().numpy()
        if name == "scores":
            fine = np.isfinite(w)
            np.testing.assert_array_equal(np.isfinite(g), fine)
            assert (np.abs(g[fine] - w[fine]) <= np.abs(w[fine]) * 2.0 ** -24 + (2 + 16 + np.log(vocab)) * 2.0 ** -23).all()
        else:
            np.testing.assert_array_equal(g, w, err_msg=name)


@pytest.mark.parametrize("requests,beams,k,vocab", [
    (1, 1, 1, 1), (1, 1, 1, 2), (1, 4, 4, 5), (3, 2, 4, 3), (1, 4, 4, 32000), (5, 3, 6, 1000), (2, 8, 16, 4096),
    (2, 8, 8, 4095), (2, 5, 5, 4097), (1, 64, 64, 9000), (3, 1, 64, 50), (40, 4, 8, 700), (1, 2, 2, 1 << 20),
    (7, 16, 32, 20001), (64, 4, 40, 30011),
])
@pytest.mark.parametrize("ended", [False, True])
def test_selection(torch, backend, requests, beams, k, vocab, ended):
    rng = np.random.default_rng(requests * 7919 + beams * 104729 + vocab + ended)
    rows = requests * beams
    x = rng.normal(size=(rows, vocab)).astype(np.float32) * 2.5
    s = (-20 * rng.random(rows)).astype(np.float32)
    done = (rng.random(rows) < 0.3).astype(np.int32) if ended else None
    _select(torch, backend, x, s, beams, k, done, vocab // 2 if ended else -1)


@pytest.mark.parametrize("vocab", [6, 300, 4097, 9000])
def test_equal_candidates_go_to_the_lowest(torch, backend, vocab):
    rng = np.random.default_rng(vocab)
    # beams that are copies of each other, logits of few values, zeros of both signs
    x = rng.integers(0, 3, size=(1, vocab)).astype(np.float32).repeat(12, 0)
    x[:, ::2] *= -1.0
    _select(torch, backend, x, np.full(12, -1.5), 4, 8)
    _select(torch, backend, np.zeros((12, vocab)), np.full(12, -1.5), 6, 12)
    _select(torch, backend, np.full((12, vocab), -np.float32(3e38)), np.zeros(12), 3, 3)


def test_values_that_are_not_finite(torch, backend):
    rng = np.random.default_rng(2)
    for vocab in (40, 5000):
        x = rng.normal(size=(16, vocab)).astype(np.float32)
        x[0, :], x[1, 3:] = np.nan, -np.inf
        x[2, [1, 5, vocab - 1]] = np.inf
        x[3, ::2] = -np.inf
        x[4:8] = -np.inf
        x[8, :] = np.inf
        x[9, 7] = np.nan
        x[12, 1], x[13, 2] = np.inf, np.nan
        s = -3 * rng.random(16).astype(np.float32)
        s[10], s[11], s[14] = -np.inf, np.nan, np.inf
        for done in (None, np.array([0, 1] * 8), np.ones(16, np.int32)):
            for k in (1, 4, 9):
                _select(torch, backend, x, s, 4, k, done, 0)


@pytest.mark.parametrize("rows,vocab,k", [(2, 20000, 8), (100, 30000, 8), (128, 40000, 8), (132, 16385, 8),
                                          (256, 40000, 32), (260, 16385, 64)])
@pytest.mark.parametrize("order", ["ascending", "descending", "constant", "late", "nan", "waves"])
def test_orders_that_fill_the_lists(torch, backend, rows, vocab, k, order):
    # 2 rows in many parts, 100 and more in parts of several steps, 256 and more in one
    rng = np.random.default_rng(rows + vocab)
    x = np.sort(rng.normal(size=(rows, vocab)).astype(np.float32), 1)
    if order == "descending":
        x = x[:, ::-1].copy()
    elif order == "constant":
        x[:] = 1.0
        x[1::3, vocab // 3] = 2.0
    elif order == "late":
        x[:, :vocab - 300] = -np.inf
    elif order == "nan":
        x[:, ::2], x[:, vocab // 2:] = np.nan, -5.0
    elif order == "waves":                       # some waves' elements all above the others'
        x += 50.0 * ((np.arange(vocab) // 256) % 4 == 1)
    s = -rng.random(rows).astype(np.float32)
    _select(torch, backend, x, s, 4 if rows % 4 == 0 else 2, k)


def test_first_step_of_a_search(torch, backend):
    # one live beam of each request
    rng = np.random.default_rng(3)
    x = rng.normal(size=(2, 500)).astype(np.float32).repeat(5, 0)
    got = _select(torch, backend, x, [0.0] + [-np.inf] * 4 + [0.0] + [-np.inf] * 4, 5, 5)
    assert got[1].cpu().tolist() == [[0] * 5, [5] * 5]


def test_large_ranges_of_logits(torch, backend):
    rng = np.random.default_rng(4)
    x = (rng.normal(size=(8, 3000)) * np.exp2(rng.integers(-60, 100, size=(8, 1)))).astype(np.float32)
    _select(torch, backend, x, -rng.random(8), 4, 6)


def test_strided_logits(torch, backend):
    rng = np.random.default_rng(5)
    wide = torch.tensor(rng.normal(size=(6, 5003)).astype(np.float32), device="cuda")
    x, s = wide[:, 1:4801], torch.zeros(6, device="cuda")
    _compare(backend.beam_select_device(x, s, 3), E.beam_select(x.cpu().numpy(), np.zeros(6), 3, 3))


def test_requests_past_one_part(torch, backend):
    # 64 beams of 64 candidates: some 1300 requests' lists are 128 MiB
    requests, vocab = 1400, 8200
    x = torch.randn(requests * 64, vocab, device="cuda", generator=torch.Generator("cuda").manual_seed(6))
    s = -torch.rand(requests * 64, device="cuda")
    got = backend.beam_select_device(x, s, 64)
    for r in (0, 700, 1270, 1271, 1272, 1273, 1399):
        at = slice(64 * r, 64 * r + 64)
        want = E.beam_select(x[at].cpu().numpy(), s[at].cpu().numpy(), 64, 64)
        want = (want[0], want[1] + 64 * r, *want[2:])
        _compare([g[r:r + 1] for g in got], want)


def test_selection_preconditions(torch, backend):
    x, s = torch.zeros(4, 10, device="cuda"), torch.zeros(4, device="cuda")
    assert tuple(backend.beam_select_device(x[:0], s[:0], 4)[0].shape) == (0, 4)
    for args, kw in (((x.half(), s, 2), {}), ((x, s, 3), {}), ((x, s, 0), {}), ((x, s[:3], 2), {}),
                     ((x, s.double(), 2), {}), ((x, s, 2), dict(k=0)), ((x, s, 2), dict(done=s)), ((x[0], s, 1), {}),
                     ((x, s.cpu(), 2), {}), ((x, s, 2), dict(eos=1 << 40))):
        with pytest.raises(PreconditionFailure):
            backend.beam_select_device(*args, **kw)
    with pytest.raises(T.HIPBackendError):
        backend.beam_select_device(x, s, 2, done=torch.zeros(4, dtype=torch.int32, device="cuda"))
    with pytest.raises(T.HIPBackendError):
        backend.beam_select_device(x, s, 2, k=65)


# ---------------------------------------------------------------------------
# reordering
# ---------------------------------------------------------------------------
def _cache_case(torch, seed, groups, beams, context, bs, heads, hd, dtype, layers, most=None):
    rng = np.random.default_rng(seed)
    lens = [int(rng.integers(0, context + 1)) for _ in range(groups)]
    lens[0] = context
    held = [-(-n // bs) for n in lens for _ in range(beams)]
    blocks = sum(held) + 3
    most = max(held) + 1 if most is None else most
    order = rng.permutation(blocks)
    table = np.full((groups * beams, most), -1, np.int32)
    at = 0
    for r, n in enumerate(held):
        table[r, :n] = order[at:at + n]
        at += n
    arrays = [torch.randn(blocks, heads, bs, hd, device="cuda").to(getattr(torch, dtype)) for _ in range(2 * layers)]
    ctx = np.repeat(np.array(lens, np.int32), beams)
    parents = np.concatenate([g * beams + rng.integers(0, beams, beams) for g in range(groups)]).astype(np.int32)
    return rng, table, ctx, parents, arrays


def _check_reorder(torch, backend, case, beams, shared=None, in_place=False):
    _, table, ctx, parents, arrays = case
    bs, blocks = arrays[0].shape[2], arrays[0].shape[0]
    new, moves, fine = E.reorder(table, parents, ctx, beams, bs, blocks, shared)
    want = [a.cpu().clone() for a in arrays]
    for a in want:
        old = a.clone()
        for since, to, n in moves:
            a[to, :, :n] = old[since, :, :n]
    t = _ints(torch, table)
    flag = torch.full((len(fine),), 5, dtype=torch.int32, device="cuda")
    out = backend.paged_reorder_device(arrays[::2], arrays[1::2], t, _ints(torch, ctx), _ints(torch, parents), beams,
                                       sharedLens=None if shared is None else _ints(torch, shared),
                                       tableOut=t if in_place else None, reordered=flag)
    np.testing.assert_array_equal(out.cpu().numpy(), new)
    np.testing.assert_array_equal(flag.cpu().numpy(), fine)
    if not in_place:
        np.testing.assert_array_equal(t.cpu().numpy(), table)
    for a, w in zip(arrays, want):
        assert torch.equal(a.cpu(), w)


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("groups,beams,context,bs,heads,hd,layers", [
    (1, 1, 5, 16, 2, 64, 1), (1, 2, 1, 1, 1, 1, 1), (3, 4, 100, 16, 2, 64, 2), (2, 8, 333, 16, 3, 33, 1),
    (5, 3, 40, 8, 2, 6, 3), (1, 64, 50, 16, 1, 16, 1), (2, 5, 1500, 1024, 1, 32, 1), (4, 2, 64, 64, 8, 128, 25),
    (30, 4, 20, 4, 1, 5, 1),
])
def test_reorder(torch, backend, in_place, dtype, groups, beams, context, bs, heads, hd, layers):
    case = _cache_case(torch, groups * 100 + beams, groups, beams, context, bs, heads, hd, dtype, layers)
    rng, ctx = case[0], case[2]
    _check_reorder(torch, backend, case, beams, None, in_place)
    shared = [int(rng.integers(0, ctx[g * beams] + 1)) for g in range(groups)]
    case = _cache_case(torch, groups * 100 + beams + 1, groups, beams, context, bs, heads, hd, dtype, layers)
    _check_reorder(torch, backend, case, beams, shared, in_place)


@pytest.mark.parametrize("parents", [(0, 1, 2, 3), (3, 2, 1, 0), (1, 1, 1, 1), (0, 0, 0, 0), (3, 3, 0, 0), (2, 0, 1, 3),
                                     (-1, 0, 0, 3), (-1, -1, -1, -1), (-5, 2, -1, 2)])
@pytest.mark.parametrize("in_place", [False, True])
def test_reorder_by_given_parents(torch, backend, parents, in_place):
    rng, table, ctx, _, arrays = _cache_case(torch, 7, 1, 4, 50, 16, 2, 8, "float32", 2)
    _check_reorder(torch, backend, (rng, table, ctx, np.array(parents, np.int32), arrays), 4, None, in_place)


@pytest.mark.parametrize("in_place", [False, True])
def test_groups_that_cannot_be_reordered_stay(torch, backend, in_place):
    rng, table, ctx, parents, arrays = _cache_case(torch, 8, 6, 4, 60, 16, 2, 16, "bfloat16", 1)
    parents[1], parents[6], parents[9], parents[14] = 4, 3, 1 << 30, 24
    ctx[16] -= 1
    _check_reorder(torch, backend, (rng, table, ctx, parents, arrays), 4, None, in_place)


def test_reorder_of_bad_tables_and_lengths(torch, backend):
    rng, table, ctx, parents, arrays = _cache_case(torch, 9, 4, 4, 70, 16, 1, 16, "float32", 1)
    parents[:] = np.repeat(np.arange(4) * 4, 4)
    table[0, 1], table[2, 0], table[5, 0] = 1 << 29, -4, 10 ** 6
    ctx[4:8] = 1 << 30                     # longer than the table
    ctx[8:12] = -7
    _check_reorder(torch, backend, (rng, table, ctx, parents, arrays), 4, [0, -3, 0, 1 << 30])


def test_reorder_without_layers_of_blocks(torch, backend):
    a = torch.zeros(0, 2, 16, 8, device="cuda")
    t = torch.full((4, 3), -1, dtype=torch.int32, device="cuda")
    z = torch.zeros(4, dtype=torch.int32, device="cuda")
    assert torch.equal(backend.paged_reorder_device([a], [a], t, z, z, 4), t)
    assert backend.paged_reorder_device([a], [a], t[:, :0].contiguous(), z, z, 4).numel() == 0


def test_reorder_preconditions(torch, backend):
    a = torch.zeros(4, 1, 16, 8, device="cuda")
    t, z = torch.zeros(4, 1, dtype=torch.int32, device="cuda"), torch.zeros(4, dtype=torch.int32, device="cuda")
    bad = [(([], [], t, z, z, 4), {}), (([a], [a, a], t, z, z, 4), {}), (([a, a[:3]], [a, a], t, z, z, 4), {}),
           (([a], [a.bfloat16()], t, z, z, 4), {}), (([a], [a], t, z, z, 3), {}), (([a], [a], t, z, z, 0), {}),
           (([a], [a], t, z[:3], z, 1), {}), (([a], [a], t, z, z[:3], 4), {}), (([a], [a], t.long(), z, z, 4), {}),
           (([a], [a], t, z, z, 4), dict(sharedLens=z)), (([a], [a], t, z, z, 2), dict(reordered=z)),
           (([a], [a], t, z, z, 4), dict(tableOut=z))]
    for args, kw in bad:
        with pytest.raises(PreconditionFailure):
            backend.paged_reorder_device(*args, **kw)
