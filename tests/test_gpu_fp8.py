"""GPU tests of the FP8 product (tbh_fp8_matmul_device) against
oracle/experts_ref.py in float64.  x's quantization is exact up to its one
rounding, so that results differ by sums alone: at most 2^-23 of the sum of
magnitudes for each of 128 additions inside the matrix instructions (which may
cut), each block's addition and scale, and half a step of the result's type.  A
bf16 result comes from the FP8 instruction, which aligns its
products to the largest and keeps some 17 bits of each: 128 cuts of 2^-17 of the
largest product of a block at the most."""
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
    return t.double().cpu().numpy()


def _weight(rng, k, n):
    w = T.quantize_fp8(rng.normal(size=(k, n)) * np.exp(rng.normal(size=n)) / np.sqrt(k))
    return w


def _rows(torch, rng, m, k, dtype):
    x = rng.normal(size=(m, k)) * np.exp(2 * rng.normal(size=(1, k)))
    return torch.tensor(x, dtype=torch.float32).to(getattr(torch, dtype)).cuda()


def _check(y, x, w, dtype):
    want, size, largest = E.fp8_matmul(_np(x), w.data, w.scales)
    k = w.shape[0]
    tol = (128 + 3 * (-(-k // 128)) + 4) * 2.0 ** -23 * size
    if dtype == "bfloat16":
        tol = tol + 128 * 2.0 ** -17 * largest
    tol += HALF[dtype] * (np.abs(want) + tol)
    err = np.abs(_np(y) - want)
    assert (err <= tol).all(), (err - tol).max()
    rms = np.sqrt((want ** 2).mean())
    assert np.sqrt((err ** 2).mean()) <= (1e-5 if dtype == "float32" else 4e-3) * rms


SHAPES = [(1, 1, 1), (1, 128, 16), (1, 2048, 512), (2, 130, 17), (5, 127, 129), (15, 1000, 300), (16, 256, 128),
          (17, 384, 200), (31, 640, 48), (32, 129, 257), (33, 1000, 300), (48, 128, 128), (64, 129, 128),
          (100, 2048, 130), (129, 520, 1000), (300, 5632, 256), (700, 256, 520),
          # outputs past one, and past two, blocks a CU, in each count of rows
          (1, 300, 4500), (3, 1300, 8200), (16, 260, 9000), (20, 300, 4500), (32, 140, 9000), (60, 300, 9000),
          (60, 140, 21000), (90, 140, 20000), (330, 400, 2048), (330, 140, 5000)]


@pytest.mark.parametrize("xt,yt", [("float32", "float32"), ("bfloat16", "bfloat16"), ("float32", "bfloat16"),
                                   ("bfloat16", "float32")])
@pytest.mark.parametrize("m,k,n", SHAPES)
def test_product(torch, backend, m, k, n, xt, yt):
    rng = np.random.default_rng(m * 1000003 + k * 1009 + n)
    w = _weight(rng, k, n)
    x = _rows(torch, rng, m, k, xt)
    y = backend.fp8_matmul_device(x, backend.fp8_weight(w), dtype=getattr(torch, yt))
    assert y.dtype == getattr(torch, yt) and tuple(y.shape) == (m, n)
    _check(y, x, w, yt)


# enough results to fill the device with blocks of 128 x 256, with larger ones, and with
# larger ones over more than 64 blocks of 128 inputs
@pytest.mark.parametrize("xt,yt", [("float32", "float32"), ("bfloat16", "bfloat16"), ("float32", "bfloat16"),
                                   ("bfloat16", "float32")])
@pytest.mark.parametrize("m,k,n", [(700, 130, 7000), (1100, 300, 7000), (1500, 8330, 4500)])
def test_large_product(torch, backend, m, k, n, xt, yt):
    rng = np.random.default_rng(m + k + n)
    w = _weight(rng, k, n)
    x = _rows(torch, rng, m, k, xt)
    y = backend.fp8_matmul_device(x, backend.fp8_weight(w), dtype=getattr(torch, yt))
    for at in (0, 250, m // 2, m - 24):
        _check(y[at:at + 24], x[at:at + 24], w, yt)


def _one_at(n):
    # W = identity: y is x as quantized
    return T.FP8Tensor((n, n), np.where(np.eye(n) > 0, 0x38, 0).astype(np.uint8),
                       np.ones((-(-n // 128), -(-n // 128)), np.float32))


@pytest.mark.parametrize("m", [3, 40])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_quantization_is_exact(torch, backend, m, dtype):
    rng = np.random.default_rng(5)
    n = 260
    x = rng.normal(size=(m, n)) * np.exp2(rng.integers(-20, 20, size=(m, n)))
    x[0, :128] = 0.0
    x[0, 128:256] = rng.choice([1.75, 1.7500001, 1.8125, 1.9375, 0.0625, 1e-30, -1.75, 2.0 ** -10], 128)
    x[1] = np.float32(3.4e38) * rng.uniform(-1, 1, n)
    x[2] = rng.uniform(-1, 1, n) * 2.0 ** -136            # below fp32's normal range
    x = torch.tensor(x, dtype=torch.float32).to(getattr(torch, dtype)).cuda()
    y = backend.fp8_matmul_device(x, backend.fp8_weight(_one_at(n)), dtype=torch.float32)
    q, s = E.quantize_rows(_np(x))
    # a product of a scale and q is a float, or, where 255 * 2^120 is rounded to 256 * 2^120, past the largest
    # one: equal to what its conversion to a float gives
    with np.errstate(over="ignore"):
        want = (q * np.repeat(s, 128, 1)[:, :n]).astype(np.float32)
    # (a value near the largest float may become an infinity as bf16: its row is NaN)
    want[np.isnan(q).any(1)] = np.nan
    np.testing.assert_array_equal(_np(y), want)


@pytest.mark.parametrize("m", [6, 50])
def test_not_finite(torch, backend, m):
    rng = np.random.default_rng(6)
    w = _weight(rng, 300, 70)
    w.data[7, 200] = 0x7F
    w.data[9, 1] = 0xFF
    x = rng.normal(size=(m, 300))
    x[1, 5], x[2, 290], x[4, 130] = np.inf, np.nan, -np.inf
    x = torch.tensor(x, dtype=torch.float32).cuda()
    y = _np(backend.fp8_matmul_device(x, backend.fp8_weight(w)))
    bad = np.zeros((m, 70), bool)
    bad[[1, 2, 4]] = True
    bad[:, [7, 9]] = True
    np.testing.assert_array_equal(np.isnan(y), bad)
    # the other rows and columns are those of the same call without them
    w.data[7, 200] = w.data[9, 1] = 0
    x = torch.nan_to_num(x, nan=1.0, posinf=1.0, neginf=1.0)
    z = _np(backend.fp8_matmul_device(x, backend.fp8_weight(w)))
    np.testing.assert_array_equal(y[~bad], z[~bad])


@pytest.mark.parametrize("m", [4, 40])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("k,n", [(256, 96), (255, 97)])
def test_strided_rows(torch, backend, m, dtype, k, n):
    rng = np.random.default_rng(7)
    w = _weight(rng, k, n)
    wide = _rows(torch, rng, m, k + 41, dtype)
    x = wide[:, 3:3 + k]
    out = torch.full((m, n + 30), 7.0, dtype=wide.dtype, device="cuda")
    y = backend.fp8_matmul_device(x, backend.fp8_weight(w), out=out[:, 5:5 + n])
    _check(y, x, w, dtype)
    assert bool((out[:, :5] == 7).all()) and bool((out[:, 5 + n:] == 7).all())


def test_weights_of_device_and_host_tensors_are_one(torch, backend):
    rng = np.random.default_rng(8)
    w = _weight(rng, 200, 150)
    x = _rows(torch, rng, 9, 200, "float32")
    ys = [backend.fp8_matmul_device(x, backend.fp8_weight(*d)) for d in (
        (w,), (w.data, w.scales), (torch.tensor(w.data), torch.tensor(w.scales)),
        (torch.tensor(w.data).cuda().view(torch.float8_e4m3fn), torch.tensor(w.scales).cuda()))]
    for y in ys[1:]:
        assert torch.equal(y, ys[0])


def test_rows_past_one_part(torch, backend):
    rng = np.random.default_rng(9)
    w = _weight(rng, 130, 33)
    x = _rows(torch, rng, (1 << 14) + 77, 130, "float32")
    y = backend.fp8_matmul_device(x, backend.fp8_weight(w))
    for at in (0, 1000, (1 << 14) - 40, (1 << 14), (1 << 14) + 37):
        _check(y[at:at + 40], x[at:at + 40], w, "float32")


@pytest.mark.parametrize("m", [5, 70])
def test_captured_before_any_eager_call(torch, m):
    backend = T.HIPBackend(0)
    rng = np.random.default_rng(10)
    w = _weight(rng, 500, 220)
    d = backend.fp8_weight(w)
    x = _rows(torch, rng, m, 500, "float32")
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = backend.fp8_matmul_device(x, d)
    for seed in range(4):
        x.copy_(_rows(torch, np.random.default_rng(seed), m, 500, "float32"))
        g.replay()
        torch.cuda.synchronize()
        _check(y, x, w, "float32")
        assert torch.equal(y, backend.fp8_matmul_device(x, d))
    # the C call without a workspace takes the rows 16 at a time
    s = torch.cuda.Stream()
    out = torch.empty_like(y)
    g = torch.cuda.CUDAGraph()
    lib = backend._lib
    with torch.cuda.stream(s):
        g.capture_begin()
        st = lib.tbh_fp8_matmul_device(d.handle, x.data_ptr(), 0, m, 500, 500, out.data_ptr(), 0, 220, None, 0,
                                       torch.cuda.current_stream().cuda_stream)
        g.capture_end()
    assert st == 0
    g.replay()
    torch.cuda.synchronize()
    _check(out, x, w, "float32")
    backend.close()


def test_two_streams(torch, backend):
    rng = np.random.default_rng(11)
    w = _weight(rng, 700, 300)
    d = backend.fp8_weight(w)
    xs = [_rows(torch, rng, 90, 700, "bfloat16") for _ in range(2)]
    want = [backend.fp8_matmul_device(x, d) for x in xs]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for _ in range(10):
        for x, s in zip(xs, streams):
            got.append(backend.fp8_matmul_device(x, d, stream=s))
    torch.cuda.synchronize()
    for i, y in enumerate(got):
        assert torch.equal(y, want[i % 2])


def test_preconditions(torch, backend):
    w = backend.fp8_weight(_weight(np.random.default_rng(12), 64, 32))
    x = torch.zeros(2, 64, device="cuda")
    assert tuple(backend.fp8_matmul_device(x[:0], w).shape) == (0, 32)
    for bad in (x[0], x[:, :63], x.cpu(), x.half(), x.t().contiguous().t()):
        with pytest.raises(PreconditionFailure):
            backend.fp8_matmul_device(bad, w)
    for kw in (dict(dtype=torch.float16), dict(out=torch.zeros(2, 31, device="cuda")),
               dict(out=torch.zeros(3, 32, device="cuda")),
               dict(out=torch.zeros(2, 32, device="cuda"), dtype=torch.bfloat16)):
        with pytest.raises(PreconditionFailure):
            backend.fp8_matmul_device(x, w, **kw)
    elsewhere = SimpleNamespace(K=64, N=32, backend=SimpleNamespace(device=1))
    with pytest.raises(PreconditionFailure):
        backend.fp8_matmul_device(x, elsewhere)
    square = backend.fp8_weight(_weight(np.random.default_rng(13), 64, 64))
    with pytest.raises(T.HIPBackendError):
        backend.fp8_matmul_device(x, square, out=x)
    data, scales = torch.zeros(32, 64, dtype=torch.uint8), torch.ones(1, 1)
    for d, s in ((data[0], scales), (data, scales[0]), (data.float(), scales), (data, scales.double()),
                 (data.t(), scales), (data, torch.ones(1, 2)), (data.numpy(), scales), (data[:0], scales)):
        with pytest.raises(PreconditionFailure):
            backend.fp8_weight(d, s)
