"""GPU tests of tbh_sample / tbh_sample_device against oracle/paged_ref.py:
tokens are equal, probabilities within fp32's rounding."""
import numpy as np
import pytest

import tinybrain_amd as T
from oracle import paged_ref as P
from tinybrain_amd.quantized import PreconditionFailure

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def backend():
    b = T.HIPBackend(0)
    yield b
    b.close()


def _check(backend, x, u, t=1.0, k=0, p=1.0, m=0.0):
    rows = x.shape[0]
    t, k, p, m, u = (np.broadcast_to(np.asarray(a), rows) for a in (t, k, p, m, u))
    f32 = lambda a: a.astype(np.float32)      # noqa: E731
    tokens, probs = backend.sample(x, f32(u), f32(t), k.astype(np.int32), f32(p), f32(m))
    want = [P.sample(x[r], f32(u)[r], f32(t)[r], int(k[r]), f32(p)[r], f32(m)[r]) for r in range(rows)]
    np.testing.assert_array_equal(tokens, [w[0] for w in want])
    # the probability is formed in 64 bits (weights and their sum to 2^-43 each of
    # the largest) and rounded to fp32 once; as fp32 has it, half a step and 2^-40
    np.testing.assert_allclose(probs, [w[1] for w in want], rtol=2.0 ** -24 + 2.0 ** -38, atol=1e-45)


SETTINGS = [dict(), dict(t=0.7), dict(t=0.0), dict(k=1), dict(k=5), dict(k=40), dict(k=700), dict(k=1 << 30),
            dict(p=0.9), dict(p=0.5, t=1.5), dict(p=0.999), dict(p=0.0), dict(p=-1.0), dict(m=0.05), dict(m=1.0),
            dict(t=0.8, k=50, p=0.95, m=0.02), dict(k=3000, p=0.3), dict(t=100.0, k=200, p=0.7), dict(t=1e-3), dict(t=1e-30, k=30, p=0.9),
            dict(t=-1.0), dict(t=float("nan")), dict(p=float("nan"), k=-3, m=float("nan")), dict(t=float("inf"), p=0.6)]


@pytest.mark.parametrize("vocab", [1, 2, 7, 63, 64, 257, 1000, 4097, 32000, 50001])
@pytest.mark.parametrize("s", SETTINGS)
def test_sample(backend, vocab, s):
    rng = np.random.default_rng(vocab)
    x = (rng.normal(size=(6, vocab)) * 2.5).astype(np.float32)
    _check(backend, x, [0.0, 1e-7, 0.3, 0.77, 0.9999, 1 - 2.0 ** -24], **s)


@pytest.mark.parametrize("s", SETTINGS)
def test_sample_equal_logits(backend, s):
    # borders that lie inside many equal logits: the lowest indices stay
    rng = np.random.default_rng(1)
    flat = np.zeros((3, 5000), np.float32)
    few = rng.integers(0, 3, (3, 5000)).astype(np.float32)
    zeros = np.where(rng.random((3, 5000)) < 0.5, -0.0, 0.0).astype(np.float32)
    for x in (flat, few, zeros):
        _check(backend, x, [0.1, 0.5, 0.93], **s)


@pytest.mark.parametrize("s", SETTINGS)
def test_sample_masked_rows(backend, s):
    # infinities, NaN and the type's lowest value: as a mask leaves them
    rng = np.random.default_rng(2)
    low = np.finfo(np.float32).min
    x = np.tile((rng.normal(size=3000) * 2).astype(np.float32), (8, 1))
    x[0, rng.random(3000) < 0.9] = -np.inf
    x[1] = -np.inf
    x[2] = np.nan
    x[3, 5:] = -np.inf
    x[4, rng.random(3000) < 0.5] = np.nan
    x[5, [7, 100, 2999]] = np.inf
    x[6, rng.random(3000) < 0.9] = low
    x[7, :] = low
    x[7, 1234] = -np.inf
    with np.errstate(invalid="ignore", over="ignore"):
        _check(backend, x, 0.6, **s)


def test_sample_large_vocab_and_batch(backend):
    rng = np.random.default_rng(3)
    x = (rng.normal(size=(2, 1 << 20)) * 3).astype(np.float32)
    _check(backend, x, [0.2, 0.8], t=0.9, p=0.8)
    x = (rng.normal(size=(300, 999)) * 3).astype(np.float32)
    _check(backend, x, rng.random(300), t=rng.choice([0, 0.5, 1], 300), k=rng.choice([0, 5, 80], 300),
           p=rng.choice([0.4, 0.9, 1], 300), m=rng.choice([0, 0.1], 300))


@pytest.mark.parametrize("std", [0.02, 0.3, 2.0])
def test_sample_around_a_thousand_candidates(backend, std):
    # kept sets below, at and above what a block holds, in few bins and in many
    rng = np.random.default_rng(6)
    k = np.array([0, 64, 500, 511, 513, 900, 1000, 1023, 1024, 1025, 1500, 2999] * 4)
    x = (rng.normal(size=(len(k), 2999)) * std).astype(np.float32)
    x[1::2, ::3] = x[1::2, :1]                         # a third of every other row is equal
    _check(backend, x, rng.random(len(k)), t=np.repeat([0.7, 1.0, 1.0, 1.3], 12), k=k,
           p=np.repeat([1.0, 0.3, 0.9, 0.35], 12), m=np.tile([0, 0, 0.2], 16))


def test_sample_device_rows(backend):
    # strided rows and rows that start off 16 bytes give the host call's tokens
    import torch

    rng = np.random.default_rng(4)
    x = (rng.normal(size=(9, 1003)) * 2).astype(np.float32)
    u = rng.random(9).astype(np.float32)
    wide = torch.zeros(9, 1010, device="cuda")
    wide[:, 3:1006] = torch.from_numpy(x).cuda()
    k = torch.full((9,), 30, dtype=torch.int32, device="cuda")
    want = backend.sample(x, u, topK=30)
    tokens, probs = backend.sample_device(wide[:, 3:1006], torch.from_numpy(u).cuda(), topK=k)
    np.testing.assert_array_equal(tokens.cpu().numpy(), want[0])
    np.testing.assert_array_equal(probs.cpu().numpy(), want[1])
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    again, _ = backend.sample_device(wide[:, 3:1006], torch.from_numpy(u).cuda(), topK=k, stream=s)
    s.synchronize()
    assert torch.equal(again, tokens)
    one = backend.sample(x[0], 0.5)
    assert one[0].shape == () and one[0] == backend.sample(x[:1], 0.5)[0][0]
    assert backend.sample_device(wide[:0], torch.zeros(0, device="cuda"))[0].numel() == 0
    none = backend.sample_device(wide[:, :0], torch.from_numpy(u).cuda())
    assert (none[0] == -1).all() and (none[1] == 0).all()


def test_sample_more_rows_than_a_grid_has_across(backend):
    import torch

    n = (1 << 20) + 3
    want = torch.randint(0, 3, (n,), device="cuda")
    x = torch.full((n, 3), -float("inf"), device="cuda").scatter_(1, want[:, None], 1.0)
    tokens, probs = backend.sample_device(x, torch.rand(n, device="cuda"))
    assert torch.equal(tokens.long(), want) and bool((probs == 1).all())


@pytest.mark.parametrize("s", [dict(), dict(k=2), dict(k=40), dict(k=1500, p=0.9), dict(p=0.7), dict(p=0.999), dict(m=0.02),
                               dict(k=30, p=0.8, m=0.01)])
@pytest.mark.parametrize("t", [1.0, 2.0, 1e37, 4e37, 1e38, 3e38, float("inf")])
def test_sample_differences_past_the_largest_float(backend, s, t):
    # logits whose distance to the largest is past fp32's range, at temperatures at which that counts
    rng = np.random.default_rng(7)
    x = (rng.uniform(-3.4, 3.4, (5, 3000)) * 1e38).astype(np.float32)
    x[1, :2900] = -3.3e38
    x[2] = np.float32(-3.4e38)
    x[2, [3, 50]] = 3.4e38, 3.3e38
    x[3, ::2] = -np.inf
    x[4, 5] = np.inf
    _check(backend, x, [0.2, 0.6, 0.99, 0.5, 0.3], t=t, **s)


def test_sample_preconditions(backend):
    import torch

    x, u = torch.zeros(2, 8, device="cuda"), torch.zeros(2, device="cuda")
    for call in (lambda: backend.sample(np.zeros((2, 2, 2)), 0.5), lambda: backend.sample(np.zeros((2, 8)), [0.5] * 3),
                 lambda: backend.sample_device(x.half(), u), lambda: backend.sample_device(x.t(), u),
                 lambda: backend.sample_device(x, u[:1]), lambda: backend.sample_device(x, u, topK=u),
                 lambda: backend.sample_device(x.cpu(), u), lambda: backend.sample_device(x, u, topP=u.double())):
        with pytest.raises(PreconditionFailure):
            call()


def test_decoder_and_sampler(backend):
    # a generation loop: the decode step's logits, drawn from on the device
    import torch

    rng = np.random.default_rng(5)
    cfg = T.DecoderConfig(1, 64, 4, 2, 128, 500, max_seq=32)

    def weight(k, n):
        return T.quantize((rng.normal(size=(k, n)) * k ** -0.5).astype(np.float32), T.QuantizationMode.perChannel)

    d = T.Decoder(backend, cfg, rng.normal(size=(500, 64)).astype(np.float32), np.ones(64, np.float32), weight(64, 500))
    d.set_layer(0, np.ones(64, np.float32), np.ones(64, np.float32),
                [weight(64, n) for n in (64, 32, 32, 64, 128, 128)] + [weight(128, 64)])
    u = rng.random(12).astype(np.float32)
    token, seen = 1, []
    for i in range(12):
        logits = torch.empty(500, device="cuda")
        d.step_device(token, logits)
        t, _ = backend.sample_device(logits[None], torch.tensor(u[i:i + 1], device="cuda"),
                                     topK=torch.full((1,), 20, dtype=torch.int32, device="cuda"))
        token = int(t[0])
        assert token == P.sample(logits.cpu().numpy(), u[i], top_k=20)[0]
        seen.append(token)
    d.reset()
    token = 1
    for i in range(12):
        token = int(backend.sample(d.step(token), u[i], topK=20)[0])
        assert token == seen[i]
