"""Block-scaled FP8 weights (e4m3, a float32 scale per 128 x 128 block) and the
mixture-of-experts layer on them.

A stored format beside the reference's INT8 and INT4
(Sources/TinyBrainRuntime/QuantizedTensor.swift:62-166), which has no
counterpart of it.  Everything here prepares data; products run in
libtinybrain_hip.so.
"""
from __future__ import annotations

import ctypes
from dataclasses import dataclass
from typing import Tuple

import numpy as np

from . import _abi
from .quantized import PreconditionFailure

FP8_BLOCK = 128
FP8_MAX = 448.0


def _blocks(n: int) -> int:
    return -(-n // FP8_BLOCK)


def _e4m3_values() -> np.ndarray:
    code = np.arange(256)
    e, m = (code >> 3) & 15, code & 7
    v = np.where(e == 0, np.ldexp(m.astype(np.float64), -9), np.ldexp((8 + m).astype(np.float64), e - 10))
    v = np.where((code & 0x7F) == 0x7F, np.nan, v)
    return np.where(code & 0x80, -v, v).astype(np.float32)


E4M3 = _e4m3_values()      # the value of each byte


def _to_e4m3(v: np.ndarray) -> np.ndarray:
    """Bytes of the nearest e4m3 values, ties to even; |v| <= 448."""
    a = np.abs(v).astype(np.float64)
    step = np.exp2(np.maximum(np.floor(np.log2(np.maximum(a, 2.0 ** -9))), -6) - 3)
    a = np.minimum(np.rint(a / step) * step, FP8_MAX)
    code = np.searchsorted(E4M3[:127].astype(np.float64), a)
    return (code | np.where(np.signbit(v), 0x80, 0)).astype(np.uint8)


@dataclass
class FP8Tensor:
    """A [K, N] = [in, out] weight on the host: e4m3 bytes [N, K] and scales
    [ceil(N / 128), ceil(K / 128)]."""
    shape: Tuple[int, int]
    data: np.ndarray
    scales: np.ndarray

    def __post_init__(self):
        self.shape = tuple(int(d) for d in self.shape)
        if len(self.shape) != 2 or min(self.shape) <= 0:
            raise PreconditionFailure("Weights must be 2D")
        k, n = self.shape
        self.data = np.ascontiguousarray(self.data, dtype=np.uint8)
        self.scales = np.ascontiguousarray(self.scales, dtype=np.float32)
        if self.data.shape != (n, k):
            raise PreconditionFailure("FP8: data must be [N, K]")
        if self.scales.shape != (_blocks(n), _blocks(k)):
            raise PreconditionFailure("FP8: need one scale per block of 128 x 128")

    def dequantize(self) -> np.ndarray:
        """The float32 [K, N] matrix."""
        k, n = self.shape
        s = np.repeat(np.repeat(self.scales, FP8_BLOCK, 0)[:n], FP8_BLOCK, 1)[:, :k]
        return np.ascontiguousarray((E4M3[self.data] * s).T)


def quantize_fp8(weight: np.ndarray) -> FP8Tensor:
    """A finite float [K, N] weight as e4m3, each block of 128 x 128 scaled by
    its largest magnitude over 448."""
    w = np.asarray(weight, np.float32)
    if w.ndim != 2:
        raise PreconditionFailure("Weights must be 2D")
    if not np.isfinite(w).all():
        raise PreconditionFailure("FP8: weights must be finite")
    k, n = w.shape
    padded = np.zeros((_blocks(n) * FP8_BLOCK, _blocks(k) * FP8_BLOCK), np.float32)
    padded[:n, :k] = w.T
    blocks = padded.reshape(_blocks(n), FP8_BLOCK, _blocks(k), FP8_BLOCK)
    most = np.abs(blocks).max((1, 3))
    # (a block of zeros, or of values below fp32's normal range, keeps a scale that can be divided by)
    scales = np.maximum(most / np.float32(FP8_MAX), np.float32(2.0 ** -126))
    scaled = blocks.astype(np.float64) / scales[:, None, :, None].astype(np.float64)
    data = _to_e4m3(np.clip(scaled, -FP8_MAX, FP8_MAX)).reshape(padded.shape)[:n, :k]
    return FP8Tensor((k, n), np.ascontiguousarray(data), scales)


def _bytes_and_scales(backend, data, scales, shape, what):
    """Pointers of e4m3 data and its scales, host arrays or tensors on the device,
    with what has to be kept until they are copied."""
    lead = shape[:-2]
    expected = lead + (_blocks(shape[-2]), _blocks(shape[-1]))
    if isinstance(data, np.ndarray) and isinstance(scales, np.ndarray):
        if data.dtype != np.uint8 or scales.dtype != np.float32:
            raise PreconditionFailure(f"{what}: data must be uint8 and scales float32")
        data, scales = np.ascontiguousarray(data), np.ascontiguousarray(scales)
        at = (data.ctypes.data, scales.ctypes.data)
    else:
        import torch

        for t in (data, scales):
            if not isinstance(t, torch.Tensor) or not t.is_contiguous() or (
                    t.is_cuda and t.get_device() != backend.device):
                raise PreconditionFailure(f"{what}: expected numpy arrays, or contiguous tensors on this device")
        if data.dtype not in (torch.uint8, torch.float8_e4m3fn) or scales.dtype != torch.float32:
            raise PreconditionFailure(f"{what}: data must be float8_e4m3fn or uint8 and scales float32")
        at = (data.data_ptr(), scales.data_ptr())
    if tuple(data.shape) != shape or tuple(scales.shape) != expected:
        raise PreconditionFailure(f"{what}: need data {list(shape)} and one scale per block of 128 x 128")
    return at, (data, scales)


def _wait_for_device(backend) -> None:
    """What the caller's current stream still writes has to be there before a copy on another."""
    import torch

    if torch.cuda.is_available():
        torch.cuda.current_stream(torch.device("cuda", backend.device)).synchronize()


class _Handle:
    """A C object of a device, destroyed before it."""
    _destroy = ""

    def __init__(self, backend, handle: ctypes.c_void_p):
        self._lib = _abi.lib()
        self._h = handle
        self.backend = backend
        backend._own(self)

    @property
    def handle(self) -> ctypes.c_void_p:
        return self._h

    def close(self) -> None:
        if self._h:
            getattr(self._lib, self._destroy)(self._h)
            self._h = ctypes.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


class FP8Weight(_Handle):
    """A block-scaled FP8 weight on the device (tbh_fp8_weight)."""
    _destroy = "tbh_fp8_weight_destroy"

    def __init__(self, backend, data, scales=None):
        from .backend import _check

        self._h = ctypes.c_void_p()
        if isinstance(data, FP8Tensor):
            data, scales = data.data, data.scales
        if getattr(data, "ndim", 0) != 2 or min(data.shape) <= 0:
            raise PreconditionFailure("Weights must be 2D")
        n, k = (int(v) for v in data.shape)
        at, keep = _bytes_and_scales(backend, data, scales, (n, k), "fp8_weight")
        if not isinstance(data, np.ndarray):
            _wait_for_device(backend)
        desc, h = _abi.FP8Desc(k, n, *at), ctypes.c_void_p()
        _check(_abi.lib().tbh_fp8_weight_create(backend._dev, ctypes.byref(desc), ctypes.byref(h)))
        del keep
        super().__init__(backend, h)
        self.K, self.N = k, n


class MoELayer(_Handle):
    """Router and experts of a mixture-of-experts layer on the device (tbh_moe)."""
    _destroy = "tbh_moe_destroy"

    def __init__(self, backend, router, gate, gateScales, up, upScales, down, downScales):
        from .backend import _check

        self._h = ctypes.c_void_p()
        if getattr(router, "ndim", 0) != 2 or getattr(gate, "ndim", 0) != 3:
            raise PreconditionFailure("moe: router must be [experts, hidden] and gate [experts, intermediate, hidden]")
        e, h = (int(v) for v in router.shape)
        i = int(gate.shape[1])
        if min(e, h, i) <= 0:
            raise PreconditionFailure("moe: sizes must be positive")
        if isinstance(router, np.ndarray):
            if router.dtype != np.float32:
                raise PreconditionFailure("moe: router must be float32")
            router = np.ascontiguousarray(router)
            at = router.ctypes.data
        else:
            import torch

            if router.dtype != torch.float32 or not router.is_contiguous() or (
                    router.is_cuda and router.get_device() != backend.device):
                raise PreconditionFailure("moe: router must be a contiguous float32 tensor on this device")
            at = router.data_ptr()
        parts = [_bytes_and_scales(backend, d, s, shape, "moe") for d, s, shape in (
            (gate, gateScales, (e, i, h)), (up, upScales, (e, i, h)), (down, downScales, (e, h, i)))]
        if not all(isinstance(t, np.ndarray) for t in (router, gate, up, down)):
            _wait_for_device(backend)
        (g, gs), (u, us), (d, ds) = (p[0] for p in parts)
        desc, out = _abi.MoEDesc(h, i, e, 0, at, g, u, d, gs, us, ds), ctypes.c_void_p()
        _check(_abi.lib().tbh_moe_create(backend._dev, ctypes.byref(desc), ctypes.byref(out)))
        del parts
        super().__init__(backend, out)
        self.hidden, self.intermediate, self.experts = h, i, e
