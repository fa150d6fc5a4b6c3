"""GPU tests of beam selection beside itself: several parts of a row and done rows
on two streams, in captured graphs between eager calls, and with a caller's workspace,
whose counters are zero again after every call."""
import ctypes

import numpy as np
import pytest

import tinybrain_amd as T
from oracle import experts_ref as E
from tinybrain_amd import _abi

pytestmark = pytest.mark.gpu
BEAMS, K, EOS = 4, 8, 3
SHAPES = [(3, 40000), (25, 20001), (80, 70000)]      # requests, vocab: parts of a row, fewer, a block of 16 waves a row


@pytest.fixture(scope="module")
def torch():
    import torch

    return torch


def _case(torch, seed, requests, vocab):
    gen = torch.Generator("cuda").manual_seed(seed)
    rows = requests * BEAMS
    x = torch.randn(rows, vocab, device="cuda", generator=gen) * 2.5
    s = -5 * torch.rand(rows, device="cuda", generator=gen)
    done = (torch.rand(rows, device="cuda", generator=gen) < 0.3).int()
    return x, s, done


def _check(got, case, some=None):
    x, s, done = (t.cpu().numpy() for t in case)
    rows = slice(0, len(x) if some is None else some * BEAMS)
    want = E.beam_select(x[rows], s[rows], BEAMS, K, done[rows], EOS)
    for g, w, name in zip(got, want, ("tokens", "parents", "scores", "done")):
        g = g.cpu().numpy()[:len(w)]
        if name == "scores":
            np.testing.assert_allclose(g, w, rtol=2.0 ** -23, atol=1e-6)
        else:
            np.testing.assert_array_equal(g, w, err_msg=name)


@pytest.mark.parametrize("requests,vocab", SHAPES)
def test_two_streams(torch, requests, vocab):
    backend = T.HIPBackend(0)
    cases = [_case(torch, 10 + i, requests, vocab) for i in range(2)]
    want = [backend.beam_select_device(c[0], c[1], BEAMS, k=K, done=c[2], eos=EOS) for c in cases]
    for w, c in zip(want, cases):
        _check(w, c, 5)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [backend.beam_select_device(c[0], c[1], BEAMS, k=K, done=c[2], eos=EOS, stream=s)
           for _ in range(12) for c, s in zip(cases, streams)]
    torch.cuda.synchronize()
    for i, g in enumerate(got):
        assert all(torch.equal(a, b) for a, b in zip(g, want[i % 2]))
    backend.close()


@pytest.mark.parametrize("requests,vocab", SHAPES)
def test_two_graphs_between_eager_calls(torch, requests, vocab):
    backend = T.HIPBackend(0)
    x, s, done = _case(torch, 20, requests, vocab)
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(backend.beam_select_device(x, s, BEAMS, k=K, done=done, eos=EOS))
        graphs.append(g)
    for seed in range(4):
        for t, new in zip((x, s, done), _case(torch, 30 + seed, requests, vocab)):
            t.copy_(new)
        for g, out in zip(graphs, outs):
            g.replay()
            eager = backend.beam_select_device(x, s, BEAMS, k=K, done=done, eos=EOS)
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, eager))
        _check(eager, (x, s, done), 3)
    backend.close()


@pytest.mark.parametrize("requests,vocab", SHAPES)
def test_a_callers_workspace(torch, requests, vocab):
    backend, lib = T.HIPBackend(0), _abi.lib()
    need = ctypes.c_int64()
    assert lib.tbh_beam_select_workspace(backend._dev, requests, BEAMS, vocab, K, ctypes.byref(need)) == _abi.OK
    room = torch.full((need.value + 64,), 0x5A, dtype=torch.uint8, device="cuda")
    room[:_abi.WORKSPACE_COUNTERS] = 0
    for seed in range(3):
        case = x, s, done = _case(torch, 40 + seed, requests, vocab)
        made = torch.full((4, requests, K), -9, dtype=torch.int32, device="cuda")
        at = [made[i].data_ptr() for i in range(4)]
        assert lib.tbh_beam_select_device(backend._dev, x.data_ptr(), vocab, requests, BEAMS, vocab, s.data_ptr(),
                                          done.data_ptr(), EOS, K, *at, room.data_ptr(), need.value,
                                          backend._raw_stream(None)) == _abi.OK, _abi.last_error()
        torch.cuda.synchronize()
        assert not bool(room[:_abi.WORKSPACE_COUNTERS].any()) and bool((room[need.value:] == 0x5A).all())
        tokens, parents, scores, ended = made.unbind(0)
        _check((tokens, parents, scores.view(torch.float32), ended), case, 4)
    backend.close()


def test_scores_in_place(torch):
    """A request's scores written over those it came with, where k = beams."""
    backend, lib = T.HIPBackend(0), _abi.lib()
    for requests, vocab in SHAPES:
        x, s, done = _case(torch, 50, requests, vocab)
        want = backend.beam_select_device(x, s, BEAMS, done=done, eos=EOS)
        made = torch.full((3, requests, BEAMS), -9, dtype=torch.int32, device="cuda")
        at = [made[i].data_ptr() for i in range(3)]
        assert lib.tbh_beam_select_device(backend._dev, x.data_ptr(), vocab, requests, BEAMS, vocab, s.data_ptr(),
                                          done.data_ptr(), EOS, BEAMS, at[0], at[1], s.data_ptr(), at[2], None, 0,
                                          backend._raw_stream(None)) == _abi.OK, _abi.last_error()
        for a, b in zip(want, (made[0], made[1], s.view(requests, BEAMS), made[2])):
            assert torch.equal(a, b)
    backend.close()
