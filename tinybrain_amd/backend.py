"""HIPBackend: the QuantizedMatMulBackend of TinyBrainHIP.

Mirrors the reference operator interface
``protocol QuantizedMatMulBackend { func matmulQuantized(_ input: Tensor<Float>,
_ quantized: QuantizedTensor) throws -> Tensor<Float> }``
(Sources/TinyBrainRuntime/Backend.swift:173-175) and the way MetalBackend
implements it (Sources/TinyBrainMetal/MetalBackend.swift:894-1048):

  * shape violations are preconditions (traps in Swift; PreconditionFailure
    here), checked before anything else (MetalBackend.swift:895-897);
  * every backend failure raises HIPBackendError -- the Swift wrapper's
    `throw`, on which the unchanged runtime falls back to its CPU path
    (QuantizedTensor.swift:630-642);
  * weights are uploaded once per QuantizedTensor.identifier and kept for the
    backend's lifetime, under a lock (MetalBackend.swift:1282-1308) -- for
    INT4 too, where the reference re-uploads on every call (:1322-1359);
  * results are returned host-resident (numpy), because the reference's
    TensorStorage can only sync from an MTLBuffer (TensorStorage.swift:82-97).

The same class also implements the reference's other backend protocols
(Backend.swift:177-228) -- SoftmaxBackend.softmax, RMSNormBackend.rmsnorm,
ActivationBackend.silu / gelu and AttentionBackend.attention -- with the
shape rules of MetalBackend's implementations (MetalBackend.swift:1062-1260,
1362-1525).

All compute runs in libtinybrain_hip.so; nothing here computes a product.
"""
from __future__ import annotations

import ctypes
import struct
import threading
import uuid
import weakref
from typing import Dict, Optional, Sequence

import numpy as np

from . import _abi
from .fp8 import FP8Weight, MoELayer
from .paged import PagedPlan
from .quantized import PreconditionFailure, QuantizedTensor


_PAGED_TYPES: Dict = {}          # the types of _paged_type, once there was a tensor


class HIPBackendError(RuntimeError):
    """A non-zero tbh_status (the reference backend's `throws`)."""

    def __init__(self, status: int, message: str):
        self.status = status
        super().__init__(f"{_abi.status_name(status)}: {message}")


def _check(st: int) -> None:
    if st != _abi.OK:
        raise HIPBackendError(st, _abi.last_error())


class DeviceWeight:
    """A weight uploaded and repacked on the device (tbh_weight)."""

    def __init__(self, backend: "HIPBackend", quantized: Optional[QuantizedTensor], _handle=None):
        self._lib = _abi.lib()
        self._h = ctypes.c_void_p()
        if _handle is None:
            desc = quantized.desc()
            _check(self._lib.tbh_weight_create(backend._dev, ctypes.byref(desc), ctypes.byref(self._h)))
        else:
            self._h = _handle
        self.backend = backend
        backend._own(self)
        info = _abi.WeightInfo()
        _check(self._lib.tbh_weight_get_info(self._h, ctypes.byref(info)))
        self.K, self.N = info.K, info.N
        self.path = _abi.PATH_NAMES[info.path]
        self.device_bytes = info.device_bytes
        self.stream_bytes = info.stream_bytes
        self.has_zero_points = bool(info.has_zero_points)

    @classmethod
    def concat(cls, backend: "HIPBackend", parts: Sequence[QuantizedTensor]) -> "DeviceWeight":
        """One weight computing every part's outputs side by side
        (tbh_weight_create_concat): x . [W_0 | W_1 | ...] in one launch, for
        projections that read the same input (q, k, v; gate, up)."""
        lib = _abi.lib()
        descs = [p.desc() for p in parts]
        arr = (ctypes.POINTER(_abi.QTensorDesc) * len(descs))(*[ctypes.pointer(d) for d in descs])
        h = ctypes.c_void_p()
        _check(lib.tbh_weight_create_concat(backend._dev, len(descs), arr, ctypes.byref(h)))
        return cls(backend, None, _handle=h)

    @property
    def handle(self) -> ctypes.c_void_p:
        return self._h

    def close(self) -> None:
        if self._h:
            self._lib.tbh_weight_destroy(self._h)
            self._h = ctypes.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


class HIPBackend:
    """QuantizedMatMulBackend on one gfx950 device."""

    def __init__(self, device: int = 0):
        self._lib = _abi.lib()
        self._dev = ctypes.c_void_p()
        _check(self._lib.tbh_device_open(int(device), ctypes.byref(self._dev)))
        ordinal, cus = ctypes.c_int32(), ctypes.c_int32()
        _check(self._lib.tbh_device_get_info(self._dev, ctypes.byref(ordinal), ctypes.byref(cus)))
        self.device = ordinal.value
        self.cu_count = cus.value
        self._cache: Dict[uuid.UUID, DeviceWeight] = {}
        self._lock = threading.Lock()
        # every weight and decoder made on this device: closed before the
        # device, whose handle their own teardown reads.  A lock of its own:
        # weight() holds _lock while it builds the DeviceWeight that registers.
        self._children = weakref.WeakSet()
        self._children_lock = threading.Lock()

    def _own(self, child) -> None:
        with self._children_lock:
            self._children.add(child)

    def set_option(self, option: int, value: int) -> None:
        """tbh_device_set_option: a launch-rule override (e.g.
        ``_abi.OPT_SGEMV_MIN_ROWS``; 0 restores the rule)."""
        _check(self._lib.tbh_device_set_option(self._dev, int(option), int(value)))

    @staticmethod
    def isAvailable(device: int = 0) -> bool:
        """MetalBackend.isAvailable: a gfx950 device can be opened."""
        try:
            L = _abi.lib()
        except OSError:
            return False
        h = ctypes.c_void_p()
        if L.tbh_device_open(int(device), ctypes.byref(h)) != _abi.OK:
            return False
        L.tbh_device_close(h)
        return True

    # -- weights ------------------------------------------------------------
    def weight(self, quantized: QuantizedTensor) -> DeviceWeight:
        """Upload-once cache keyed by QuantizedTensor.identifier."""
        with self._lock:
            w = self._cache.get(quantized.identifier)
            if w is None:
                w = DeviceWeight(self, quantized)
                self._cache[quantized.identifier] = w
            return w

    def evict(self, quantized: QuantizedTensor) -> None:
        with self._lock:
            w = self._cache.pop(quantized.identifier, None)
        if w is not None:
            w.close()

    # -- QuantizedMatMulBackend ----------------------------------------------
    def matmulQuantized(self, input: np.ndarray, quantized: QuantizedTensor) -> np.ndarray:
        """y[M, N] = input[M, K] . dequantize(quantized)[K, N], fp32."""
        x = np.asarray(input)
        if x.ndim != 2:
            raise PreconditionFailure("Input must be 2D")
        if len(quantized.shape) != 2:
            raise PreconditionFailure("Weights must be 2D")
        if x.shape[1] != quantized.shape[0]:
            raise PreconditionFailure("Dimensions must match")
        x = np.ascontiguousarray(x, np.float32)       # makeContiguousCopy
        w = self.weight(quantized)
        m = x.shape[0]
        y = np.empty((m, quantized.shape[1]), np.float32)
        _check(self._lib.tbh_matmul(self._dev, x.ctypes.data, m, x.shape[1], w.handle, y.ctypes.data))
        return y

    def dequantize(self, quantized: QuantizedTensor) -> np.ndarray:
        """The uploaded weight as fp32 [K, N] (see tbh_dequantize)."""
        w = self.weight(quantized)
        out = np.empty(quantized.shape, np.float32)
        _check(self._lib.tbh_dequantize(self._dev, w.handle, out.ctypes.data))
        return out

    # -- device-resident entry (torch tensors on this device) -----------------
    def matmul_device(self, x, weight: DeviceWeight, out=None, stream=None):
        """Enqueue y = x . W on a HIP stream with GPU-resident torch tensors.

        x: float32 [M, K] contiguous cuda tensor; returns float32 [M, N]."""
        import torch

        if x.dim() != 2 or x.shape[1] != weight.K:
            raise PreconditionFailure("Dimensions must match")
        if x.dtype != torch.float32 or not x.is_contiguous() or not x.is_cuda:
            raise PreconditionFailure("x must be a contiguous float32 device tensor")
        if out is None:
            out = self._made(stream, torch.empty, (x.shape[0], weight.N), dtype=torch.float32, device=x.device)
        s = stream if stream is not None else torch.cuda.current_stream(x.device)
        _check(self._lib.tbh_matmul_device(weight.handle, x.data_ptr(), x.shape[0], x.shape[1],
                                           out.data_ptr(), ctypes.c_void_p(s.cuda_stream)))
        return out

    def matmul_device_noalloc(self, x, weight: DeviceWeight, out=None, stream=None):
        """matmul_device through tbh_matmul_device_noalloc: no device memory
        is allocated by the call (for code under graph capture); `out` must
        then be given.  Calls overlapping on one GPU race on its scratch."""
        import torch

        if x.dim() != 2 or x.shape[1] != weight.K:
            raise PreconditionFailure("Dimensions must match")
        if x.dtype != torch.float32 or not x.is_contiguous() or not x.is_cuda:
            raise PreconditionFailure("x must be a contiguous float32 device tensor")
        if out is None or tuple(out.shape) != (x.shape[0], weight.N) or not out.is_contiguous():
            raise PreconditionFailure("out must be a contiguous float32 [M, N] device tensor")
        s = stream if stream is not None else torch.cuda.current_stream(x.device)
        _check(self._lib.tbh_matmul_device_noalloc(weight.handle, x.data_ptr(), x.shape[0], x.shape[1],
                                                   out.data_ptr(), ctypes.c_void_p(s.cuda_stream)))
        return out

    def linear_device(self, x, weight: DeviceWeight, bias=None, out=None, stream=None):
        """Enqueue y = x . W (+ bias[n] on every row) on a HIP stream
        (tbh_linear_device; LinearLayerWeights.apply(toRow:),
        ModelWeights.swift:47-68).  bias: None or a float32 [N] cuda tensor."""
        import torch

        if x.dim() != 2 or x.shape[1] != weight.K:
            raise PreconditionFailure("Dimensions must match")
        if x.dtype != torch.float32 or not x.is_contiguous() or not x.is_cuda:
            raise PreconditionFailure("x must be a contiguous float32 device tensor")
        if bias is not None:
            if tuple(bias.shape) != (weight.N,):
                raise PreconditionFailure("Bias must match output dimension")
            if bias.dtype != torch.float32 or not bias.is_contiguous() or not bias.is_cuda:
                raise PreconditionFailure("bias must be a contiguous float32 device tensor")
        if out is None:
            out = self._made(stream, torch.empty, (x.shape[0], weight.N), dtype=torch.float32, device=x.device)
        s = stream if stream is not None else torch.cuda.current_stream(x.device)
        _check(self._lib.tbh_linear_device(weight.handle, x.data_ptr(), x.shape[0], x.shape[1],
                                           None if bias is None else bias.data_ptr(), out.data_ptr(),
                                           ctypes.c_void_p(s.cuda_stream)))
        return out

    def matmul_bf16_device(self, x, weight: DeviceWeight, out=None, stream=None):
        """Prefill: enqueue y = x . W for bf16 activations on bf16 MFMA.

        x: bfloat16 [M, K] contiguous cuda tensor (K % 8 == 0); returns
        float32 [M, N].  See tbh_matmul_bf16_device."""
        import torch

        if x.dim() != 2 or x.shape[1] != weight.K:
            raise PreconditionFailure("Dimensions must match")
        if x.dtype != torch.bfloat16 or not x.is_contiguous() or not x.is_cuda:
            raise PreconditionFailure("x must be a contiguous bfloat16 device tensor")
        if out is None:
            out = self._made(stream, torch.empty, (x.shape[0], weight.N), dtype=torch.float32, device=x.device)
        s = stream if stream is not None else torch.cuda.current_stream(x.device)
        _check(self._lib.tbh_matmul_bf16_device(weight.handle, x.data_ptr(), x.shape[0], x.shape[1],
                                                out.data_ptr(), ctypes.c_void_p(s.cuda_stream)))
        return out

    def dequantize_device(self, weight: DeviceWeight, out=None, stream=None):
        import torch

        if out is None:
            out = self._made(stream, torch.empty, (weight.K, weight.N), dtype=torch.float32,
                             device=torch.device("cuda", self.device))
        s = stream if stream is not None else torch.cuda.current_stream(out.device)
        _check(self._lib.tbh_dequantize_device(weight.handle, out.data_ptr(),
                                               ctypes.c_void_p(s.cuda_stream)))
        return out

    # -- SoftmaxBackend / RMSNormBackend / ActivationBackend / AttentionBackend --
    def softmax(self, input: np.ndarray) -> np.ndarray:
        """Softmax along the last dimension, rows summing to 1
        (MetalBackend.swift:1073-1134; empty input is returned as is)."""
        x = np.ascontiguousarray(input, np.float32)
        if x.size == 0:
            return x
        if x.ndim == 0:
            raise PreconditionFailure("Cannot apply softmax to empty tensor")
        y = np.empty_like(x)
        cols = x.shape[-1]
        _check(self._lib.tbh_softmax(self._dev, x.ctypes.data, x.size // cols, cols, y.ctypes.data))
        return y

    def rmsnorm(self, input: np.ndarray, weight: np.ndarray, eps: float = 1e-5) -> np.ndarray:
        """x / rms(x) * weight per row of a [tokens, hidden] tensor
        (MetalBackend.swift:1146-1207)."""
        x = np.ascontiguousarray(input, np.float32)
        g = np.ascontiguousarray(weight, np.float32).reshape(-1)
        if x.ndim != 2:
            raise PreconditionFailure("rmsnorm input must be 2-D [tokens, hidden]")
        if g.size != x.shape[1]:
            raise PreconditionFailure("weight size must equal hiddenDim")
        y = np.empty_like(x)
        _check(self._lib.tbh_rmsnorm(self._dev, x.ctypes.data, x.shape[0], x.shape[1], g.ctypes.data,
                                     float(eps), y.ctypes.data))
        return y

    def _elementwise(self, fn, input: np.ndarray) -> np.ndarray:
        x = np.ascontiguousarray(input, np.float32)
        if x.size == 0:
            return x
        y = np.empty_like(x)
        _check(fn(self._dev, x.ctypes.data, x.size, y.ctypes.data))
        return y

    def silu(self, input: np.ndarray) -> np.ndarray:
        """out = x * sigmoid(x) (MetalBackend.swift:1214-1216)."""
        return self._elementwise(self._lib.tbh_silu, input)

    def gelu(self, input: np.ndarray) -> np.ndarray:
        """GELU, tanh approximation (MetalBackend.swift:1221-1223)."""
        return self._elementwise(self._lib.tbh_gelu, input)

    @staticmethod
    def _attention_shape(q, k, v, mask, headDim, numHeads, numKVHeads):
        if not (numHeads >= numKVHeads and numKVHeads > 0 and numHeads % numKVHeads == 0):
            raise PreconditionFailure("numHeads must be a multiple of numKVHeads")
        if q.ndim == 3:
            batch, seq, kv = q.shape[0], q.shape[1], k.shape[1]
        else:
            batch, seq, kv = 1, q.shape[0], k.shape[0]
        if (q.shape[-1] != numHeads * headDim or k.shape[-1] != numKVHeads * headDim
                or tuple(v.shape) != tuple(k.shape) or k.ndim != q.ndim
                or (q.ndim == 3 and k.shape[0] != batch)):
            raise PreconditionFailure("attention: query/keys/values shapes do not match the heads")
        if mask is not None and (mask.numel() if hasattr(mask, "numel") else mask.size) != kv:
            raise PreconditionFailure("attention: mask must have kvSeqLen elements")
        return _abi.AttentionShape(batch, seq, kv, headDim, numHeads, numKVHeads)

    def attention(self, query: np.ndarray, keys: np.ndarray, values: np.ndarray,
                  mask: Optional[np.ndarray], headDim: int, numHeads: int, numKVHeads: int) -> np.ndarray:
        """softmax(Q K^T / sqrt(headDim) + mask) V per head with GQA
        (MetalBackend.swift:1381-1525); returns an array shaped like query."""
        q = np.ascontiguousarray(query, np.float32)
        k = np.ascontiguousarray(keys, np.float32)
        v = np.ascontiguousarray(values, np.float32)
        m = None if mask is None else np.ascontiguousarray(mask, np.float32).reshape(-1)
        sh = self._attention_shape(q, k, v, m, headDim, numHeads, numKVHeads)
        out = np.empty_like(q)
        _check(self._lib.tbh_attention(self._dev, ctypes.byref(sh), q.ctypes.data, k.ctypes.data,
                                       v.ctypes.data, None if m is None else m.ctypes.data, out.ctypes.data))
        return out

    def _made(self, stream, make, *args, **kw):
        """A new tensor that `stream` writes, from that stream's own memory:
        memory freed on torch's current stream may still be used by work that
        is queued there.  Once freed it is kept until what the current stream
        then has queued is done, as the caller may read it there."""
        if stream is None:
            return make(*args, **kw)
        import torch

        if stream.cuda_stream == torch._C._cuda_getCurrentRawStream(self.device):
            return make(*args, **kw)
        with torch.cuda.stream(stream):
            t = make(*args, **kw)
        t.record_stream(torch.cuda.current_stream(self.device))
        return t

    # device-resident variants: contiguous float32 torch tensors on this device
    def _stream(self, t, stream):
        import torch

        return ctypes.c_void_p((stream if stream is not None else torch.cuda.current_stream(t.device)).cuda_stream)

    @staticmethod
    def _dev_tensor(t):
        import torch

        if t.dtype != torch.float32 or not t.is_contiguous() or not t.is_cuda:
            raise PreconditionFailure("expected a contiguous float32 device tensor")
        return t

    def softmax_device(self, x, out=None, stream=None):
        import torch

        x = self._dev_tensor(x)
        out = self._made(stream, torch.empty_like, x) if out is None else self._dev_tensor(out)
        if x.numel():
            cols = x.shape[-1]
            _check(self._lib.tbh_softmax_device(self._dev, x.data_ptr(), x.numel() // cols, cols,
                                                out.data_ptr(), self._stream(x, stream)))
        return out

    def rmsnorm_device(self, x, weight, eps: float = 1e-5, out=None, stream=None):
        import torch

        x, weight = self._dev_tensor(x), self._dev_tensor(weight)
        if x.dim() != 2 or weight.numel() != x.shape[1]:
            raise PreconditionFailure("rmsnorm: x [tokens, hidden] and weight [hidden]")
        out = self._made(stream, torch.empty_like, x) if out is None else self._dev_tensor(out)
        _check(self._lib.tbh_rmsnorm_device(self._dev, x.data_ptr(), x.shape[0], x.shape[1], weight.data_ptr(),
                                            float(eps), out.data_ptr(), self._stream(x, stream)))
        return out

    def silu_device(self, x, out=None, stream=None):
        import torch

        x = self._dev_tensor(x)
        out = self._made(stream, torch.empty_like, x) if out is None else self._dev_tensor(out)
        _check(self._lib.tbh_silu_device(self._dev, x.data_ptr(), x.numel(), out.data_ptr(),
                                         self._stream(x, stream)))
        return out

    def gelu_device(self, x, out=None, stream=None):
        import torch

        x = self._dev_tensor(x)
        out = self._made(stream, torch.empty_like, x) if out is None else self._dev_tensor(out)
        _check(self._lib.tbh_gelu_device(self._dev, x.data_ptr(), x.numel(), out.data_ptr(),
                                         self._stream(x, stream)))
        return out

    def attention_device(self, query, keys, values, mask, headDim: int, numHeads: int, numKVHeads: int,
                         out=None, stream=None):
        import torch

        q, k, v = self._dev_tensor(query), self._dev_tensor(keys), self._dev_tensor(values)
        m = None if mask is None else self._dev_tensor(mask)
        sh = self._attention_shape(q, k, v, m, headDim, numHeads, numKVHeads)
        out = self._made(stream, torch.empty_like, q) if out is None else self._dev_tensor(out)
        _check(self._lib.tbh_attention_device(self._dev, ctypes.byref(sh), q.data_ptr(), k.data_ptr(),
                                              v.data_ptr(), None if m is None else m.data_ptr(),
                                              out.data_ptr(), self._stream(q, stream)))
        return out

    # -- serving many requests from one paged cache (see paged.py) --------------
    # A decode step makes these calls once per layer, and its kernels take a few
    # microseconds: the structs are packed in one go and the stream's handle read
    # directly (us per call of the plan, append and attention of a small step, with
    # ctypes.Structure, stream objects and torch.empty: 14.5, 16.6, 16.6; so: 10.0, 9.8, 11.1).
    _layout = struct.Struct("@7i")                       # tbh_paged_layout
    _rows = struct.Struct("@q2i3P3qPqif2P")              # tbh_paged_rows
    _queries = struct.Struct("@q2i2P2q2Pf2i4x")          # tbh_paged_queries

    def paged_plan_device(self, newLens, contextLens, blockTable, freeBlocks, freeCount, blockSize: int,
                          maxTokens: int, contextOut=None, freeCountOut=None, stream=None) -> PagedPlan:
        """tbh_paged_plan_device: which blocks, slots and positions a step's
        new tokens take.  int32 cuda tensors: newLens and contextLens
        [requests], blockTable [requests, blocks], freeBlocks [blocks of the
        cache], freeCount [1].  blockTable and freeBlocks are updated in
        place; lengths and height come back in the plan, or go to contextOut
        and freeCountOut (contextLens and freeCount themselves: in place)."""
        import torch

        self._ints(torch.int32, newLens, contextLens, blockTable, freeBlocks, freeCount)
        b = newLens.numel()
        if contextLens.numel() != b or blockTable.dim() != 2 or blockTable.shape[0] != b or freeCount.numel() != 1:
            raise PreconditionFailure("plan: lengths and block table must have one row per request")
        if maxTokens < 0:
            raise PreconditionFailure("plan: maxTokens must not be negative")
        out = self._made(stream, newLens.new_empty, 3 * b + 2 + 2 * maxTokens)
        start, granted, slots, positions, ctx, count = torch.split_with_sizes(
            out, (b + 1, b, maxTokens, maxTokens, b, 1))
        if contextOut is not None:
            self._ints(torch.int32, contextOut)
            ctx = contextOut
        if freeCountOut is not None:
            self._ints(torch.int32, freeCountOut)
            count = freeCountOut
        if ctx.numel() != b or count.numel() != 1:
            raise PreconditionFailure("plan: contextOut [requests] and freeCountOut [1]")
        at = out.data_ptr()
        try:
            layout = self._layout.pack(freeBlocks.numel(), blockSize, 0, 0, 0, b, blockTable.shape[1])
        except struct.error:
            raise self._past_32_bits() from None
        _check(self._lib.tbh_paged_plan_device(
            self._dev, layout, newLens.data_ptr(), contextLens.data_ptr(), blockTable.data_ptr(), freeBlocks.data_ptr(),
            freeCount.data_ptr(), maxTokens, at, at + 4 * (b + 1), ctx.data_ptr(), count.data_ptr(),
            at + 4 * (2 * b + 1), at + 4 * (2 * b + 1 + maxTokens), self._raw_stream(stream)))
        return PagedPlan(start, granted, slots, positions, ctx, count)

    def paged_append_device(self, keys, values, slots, k, v, q=None, positions=None, ropeBase: float = 0.0,
                            qOut=None, stream=None):
        """tbh_paged_append_device: rows k, v [tokens, kvHeads * headDim] to
        their slots of the cache arrays keys, values [blocks, kvHeads,
        blockSize, headDim]; with ropeBase > 0 keys and queries q [tokens,
        heads * headDim] are rotated by their positions.  Rows may be slices
        of a wider matrix (only the last dimension must be contiguous).
        Returns the queries: qOut, which may be q itself or of the other type,
        else a new tensor of q's type; None without q."""
        import torch

        n, nkv, bs, hd, ct = self._kv_arrays(keys, values)
        tokens, width = self._row_shape(k)
        if width != nkv * hd or self._row_shape(v) != (tokens, width):
            raise PreconditionFailure("append: k and v must be rows [tokens, kvHeads * headDim]")
        if v.dtype != k.dtype or (q is not None and q.dtype != k.dtype):
            raise PreconditionFailure("append: q, k and v must have one type")
        self._ints(torch.int32, slots)
        if slots.numel() != tokens:
            raise PreconditionFailure("append: slots must have one entry per row")
        at = 0
        if positions is not None:
            self._ints(torch.int32, positions)
            at = positions.data_ptr()
            if positions.numel() != tokens:
                raise PreconditionFailure("append: positions must have one entry per row")
        elif ropeBase:
            raise PreconditionFailure("append: positions are needed to rotate")
        xt = self._paged_type(k)
        heads, qp, qs, op, os, ot = 0, 0, 0, 0, 0, xt
        if q is not None:
            rows, width = self._row_shape(q)
            if rows != tokens or width % hd:
                raise PreconditionFailure("append: q must be rows [tokens, heads * headDim]")
            if qOut is None:
                qOut = self._made(stream, torch.empty_like, q)
            else:
                if self._row_shape(qOut) != (rows, width):
                    raise PreconditionFailure("append: qOut must be shaped like q")
                ot = self._paged_type(qOut)
            heads, qp, qs, op, os = width // hd, q.data_ptr(), q.stride(0), qOut.data_ptr(), qOut.stride(0)
        try:
            layout = self._layout.pack(n, bs, nkv, hd, ct, 0, 0)
            r = self._rows.pack(tokens, xt, heads, qp, k.data_ptr(), v.data_ptr(), qs, k.stride(0), v.stride(0), op,
                                os, ot, ropeBase, slots.data_ptr(), at)
        except struct.error:
            raise self._past_32_bits() from None
        _check(self._lib.tbh_paged_append_device(
            self._dev, layout, r, keys.data_ptr(), values.data_ptr(), self._raw_stream(stream)))
        return qOut if q is not None else None

    def paged_attention_device(self, q, keys, values, blockTable, queryStart, contextLens, numHeads: int,
                               scale: float = 0.0, maxQueryLen: int = 0, maxContextLen: int = 0, out=None,
                               stream=None):
        """tbh_paged_attention_device: q [tokens, numHeads * headDim] (float32
        or bfloat16), request b's rows queryStart[b] .. queryStart[b + 1], its
        newest positions of contextLens[b], over the cache; returns a tensor
        like q (rows behind the last request are left as they were in out).
        maxQueryLen and maxContextLen, if known, choose launch shapes only."""
        import torch

        n, nkv, bs, hd, ct = self._kv_arrays(keys, values)
        tokens, width = shape = self._row_shape(q)
        self._ints(torch.int32, blockTable, queryStart, contextLens)
        b = contextLens.numel()
        if width != numHeads * hd or numHeads <= 0 or numHeads % nkv:
            raise PreconditionFailure("attention: query shape does not match the heads")
        if blockTable.dim() != 2 or blockTable.shape[0] != b or queryStart.numel() != b + 1:
            raise PreconditionFailure("attention: block table and query starts must have one row per request")
        xt = self._paged_type(q)
        if out is None:
            out = self._made(stream, torch.empty_like, q)
        elif self._row_shape(out) != shape or out.dtype != q.dtype:
            raise PreconditionFailure("attention: out must be like the queries")
        try:
            layout = self._layout.pack(n, bs, nkv, hd, ct, b, blockTable.shape[1])
            queries = self._queries.pack(tokens, xt, numHeads, q.data_ptr(), out.data_ptr(), q.stride(0),
                                         out.stride(0), queryStart.data_ptr(), contextLens.data_ptr(), scale,
                                         maxQueryLen, maxContextLen)
        except struct.error:
            raise self._past_32_bits() from None
        _check(self._lib.tbh_paged_attention_device(
            self._dev, layout, queries, keys.data_ptr(), values.data_ptr(), blockTable.data_ptr(), self._raw_stream(stream)))
        return out

    @staticmethod
    def _past_32_bits() -> PreconditionFailure:
        return PreconditionFailure("a size does not fit the call's 32 bits")

    def _raw_stream(self, stream) -> int:
        if stream is not None:
            return stream.cuda_stream
        import torch

        return torch._C._cuda_getCurrentRawStream(self.device)

    def _ints(self, dtype, *tensors) -> None:
        for t in tensors:
            if t.dtype != dtype or not t.is_contiguous() or t.get_device() != self.device:
                raise PreconditionFailure("expected a contiguous int32 tensor on this device")

    def _row_shape(self, t):
        shape = tuple(t.shape)
        if len(shape) != 2 or t.get_device() != self.device or (shape[1] > 1 and t.stride(1) != 1):
            raise PreconditionFailure("expected rows on this device, contiguous along the last dimension")
        return shape

    @staticmethod
    def _paged_type(t) -> int:
        code = _PAGED_TYPES.get(t.dtype)
        if code is None:
            import torch

            _PAGED_TYPES.update({torch.float32: _abi.F32, torch.bfloat16: _abi.BF16})
            code = _PAGED_TYPES.get(t.dtype)
            if code is None:
                raise PreconditionFailure("expected float32 or bfloat16")
        return code

    def _kv_arrays(self, keys, values):
        """blocks, kvHeads, blockSize, headDim, type of the cache arrays."""
        shape = tuple(keys.shape)
        if len(shape) != 4 or shape != tuple(values.shape) or keys.dtype != values.dtype:
            raise PreconditionFailure("the cache is two equal arrays [blocks, kvHeads, blockSize, headDim]")
        if not (keys.is_contiguous() and values.is_contiguous() and keys.get_device() == self.device
                and values.get_device() == self.device):
            raise PreconditionFailure("the cache must be contiguous tensors on this device")
        n, nkv, bs, hd = shape
        return n, nkv, bs, hd, self._paged_type(keys)

    # -- products with block-scaled FP8 weights, mixture of experts (see fp8.py) ----
    def fp8_weight(self, data, scales=None) -> FP8Weight:
        """An FP8 weight, repacked once: an FP8Tensor, or e4m3 data [N, K] with
        scales [ceil(N / 128), ceil(K / 128)] (numpy arrays, or torch tensors)."""
        return FP8Weight(self, data, scales)

    def fp8_matmul_device(self, x, weight: FP8Weight, dtype=None, out=None, stream=None):
        """tbh_fp8_matmul_device: y = x . W with x [M, K] (float32 or bfloat16;
        rows may be strided) quantized to e4m3 per row and 128 inputs; y [M, N]
        of `dtype` (x's unless given) or like out."""
        rows, k = self._row_shape(x)
        if k != weight.K:
            raise PreconditionFailure("Dimensions must match")
        if weight.backend.device != self.device:
            raise PreconditionFailure("fp8: the weight is on another device")
        if out is None:
            out = self._made(stream, x.new_empty, (rows, weight.N), dtype=x.dtype if dtype is None else dtype)
        elif self._row_shape(out) != (rows, weight.N) or (dtype is not None and out.dtype != dtype):
            raise PreconditionFailure("fp8: out must be [M, N] of the type asked for")
        xt, yt = self._paged_type(x), self._paged_type(out)
        room, size = None, 0
        if rows > 16:
            import torch

            if torch.cuda.is_current_stream_capturing():
                need = ctypes.c_int64()
                _check(self._lib.tbh_fp8_matmul_workspace(weight.handle, rows, ctypes.byref(need)))
                room, size = self._room(stream, x, need.value)
        _check(self._lib.tbh_fp8_matmul_device(
            weight.handle, x.data_ptr(), xt, rows, k, x.stride(0), out.data_ptr(), yt, out.stride(0),
            None if room is None else room.data_ptr(), size, self._raw_stream(stream)))
        return out

    def moe_layer(self, router, gate, gateScales, up, upScales, down, downScales) -> MoELayer:
        """A mixture-of-experts layer, repacked once: router float32 [experts,
        hidden], e4m3 gate and up [experts, intermediate, hidden] and down
        [experts, hidden, intermediate], each with its scales per block of 128 x 128
        (numpy arrays, or torch tensors)."""
        return MoELayer(self, router, gate, gateScales, up, upScales, down, downScales)

    def moe_device(self, x, layer: MoELayer, topK: int, normalize: bool = True, out=None, experts=None, weights=None,
                   stream=None):
        """tbh_moe_device on rows x [tokens, hidden] (float32 or bfloat16, may be
        strided): (y like x, experts int32 [tokens, topK], weights float32
        [tokens, topK]); normalize: a token's weights sum to 1."""
        import torch

        tokens, width = shape = self._row_shape(x)
        if width != layer.hidden:
            raise PreconditionFailure("moe: x must be [tokens, hidden]")
        if layer.backend.device != self.device:
            raise PreconditionFailure("moe: the layer is on another device")
        xt = self._paged_type(x)
        if not 0 < topK <= layer.experts:
            raise PreconditionFailure("moe: topK must be 1 .. experts")
        if out is None:
            out = self._made(stream, x.new_empty, shape)
        elif self._row_shape(out) != shape or out.dtype != x.dtype:
            raise PreconditionFailure("moe: out must be like x")
        if experts is None:
            experts = self._made(stream, x.new_empty, (tokens, topK), dtype=torch.int32)
        if weights is None:
            weights = self._made(stream, x.new_empty, (tokens, topK), dtype=torch.float32)
        for t, dtype in ((experts, torch.int32), (weights, torch.float32)):
            if t.dtype != dtype or tuple(t.shape) != (tokens, topK) or not t.is_contiguous() \
                    or t.get_device() != self.device:
                raise PreconditionFailure("moe: experts int32 and weights float32 must be contiguous [tokens, topK]")
        room, size = None, 0
        if torch.cuda.is_current_stream_capturing():
            need = ctypes.c_int64()
            _check(self._lib.tbh_moe_workspace(layer.handle, xt, tokens, topK, ctypes.byref(need)))
            room, size = self._room(stream, x, need.value)
        _check(self._lib.tbh_moe_device(
            layer.handle, x.data_ptr(), xt, tokens, x.stride(0), topK, bool(normalize), out.data_ptr(), out.stride(0),
            experts.data_ptr(), weights.data_ptr(), None if room is None else room.data_ptr(), size,
            self._raw_stream(stream)))
        return out, experts, weights

    def _room(self, stream, like, size: int):
        """A graph under capture gets memory of its own (its pool's), so that it
        needs no eager call before it and shares nothing with other graphs."""
        import torch

        def make():
            room = like.new_empty(max(size, 1), dtype=torch.uint8)
            room[:_abi.WORKSPACE_COUNTERS].zero_()
            return room

        return self._made(stream, make), size

    # -- Sampler (Sampler.swift) with the caller's random numbers ----------------
    def sample(self, logits: np.ndarray, u, temperature=1.0, topK=0, topP=1.0, minP=0.0):
        """tbh_sample on host arrays: logits [rows, vocab] or [vocab], u and
        the settings one number or one per row.  Returns (tokens int32, probs
        float32), shaped like the rows."""
        x = np.ascontiguousarray(logits, np.float32)
        if x.ndim not in (1, 2):
            raise PreconditionFailure("sample: logits must be [vocab] or [rows, vocab]")
        rows, vocab = (1, x.shape[0]) if x.ndim == 1 else x.shape

        def per_row(value, dtype):
            a = np.asarray(value, dtype)
            if a.ndim > 1 or (a.ndim == 1 and a.shape[0] != rows):
                raise PreconditionFailure("sample: settings must be one number or one per row")
            return np.ascontiguousarray(np.broadcast_to(a, (rows,)))

        args = [per_row(temperature, np.float32), per_row(topK, np.int32), per_row(topP, np.float32),
                per_row(minP, np.float32), per_row(u, np.float32)]
        tokens, probs = np.empty(rows, np.int32), np.empty(rows, np.float32)
        _check(self._lib.tbh_sample(self._dev, x.ctypes.data, rows, vocab, *[a.ctypes.data for a in args],
                                    tokens.ctypes.data, probs.ctypes.data))
        return (tokens[0], probs[0]) if x.ndim == 1 else (tokens, probs)

    def sample_device(self, logits, u, temperature=None, topK=None, topP=None, minP=None, tokens=None, probs=None,
                      stream=None):
        """tbh_sample_device on torch tensors: logits float32 [rows, vocab]
        (rows may be strided), u float32 [rows], settings None or [rows]
        (float32; topK int32).  Returns (tokens int32, probs float32)."""
        import torch

        if logits.dtype != torch.float32:
            raise PreconditionFailure("sample: logits must be float32")
        rows, vocab = self._row_shape(logits)
        for t, dtype in ((u, torch.float32), (temperature, torch.float32), (topK, torch.int32), (topP, torch.float32),
                         (minP, torch.float32), (tokens, torch.int32), (probs, torch.float32)):
            if t is not None and (t.dtype != dtype or t.numel() != rows or not t.is_contiguous()
                                  or t.get_device() != self.device):
                raise PreconditionFailure("sample: u and settings must be contiguous device tensors, one entry per row")
        if tokens is None:
            tokens = self._made(stream, u.new_empty, rows, dtype=torch.int32)
        if probs is None:
            probs = self._made(stream, u.new_empty, rows)
        _check(self._lib.tbh_sample_device(
            self._dev, logits.data_ptr(), logits.stride(0), rows, vocab,
            temperature.data_ptr() if temperature is not None else None, topK.data_ptr() if topK is not None else None,
            topP.data_ptr() if topP is not None else None, minP.data_ptr() if minP is not None else None, u.data_ptr(),
            tokens.data_ptr(), probs.data_ptr(), self._raw_stream(stream)))
        return tokens, probs

    # -- beam search ----------------------------------------------------------------
    def beam_select_device(self, logits, scores, beams: int, k: Optional[int] = None, done=None, eos: int = -1,
                           stream=None):
        """tbh_beam_select_device: the k (beams unless given) best continuations of
        each request's `beams` rows of logits float32 [requests * beams, vocab]
        (rows may be strided), scores float32 and done int32 (or None)
        [requests * beams].  Returns (tokens int32, parents int32, scores float32,
        done int32), each [requests, k]; a missing one is -1, -1, -inf, 0."""
        import torch

        if logits.dtype != torch.float32:
            raise PreconditionFailure("beam search: logits must be float32")
        rows, vocab = self._row_shape(logits)
        k = beams if k is None else k
        if beams <= 0 or rows % beams or k <= 0:
            raise PreconditionFailure("beam search: rows must be a multiple of beams, k positive")
        if max(beams, k, abs(eos)) >= 1 << 31:
            raise self._past_32_bits()
        for t, dtype in ((scores, torch.float32), (done, torch.int32)):
            if t is not None and (t.dtype != dtype or t.numel() != rows or not t.is_contiguous()
                                  or t.get_device() != self.device):
                raise PreconditionFailure("beam search: scores float32 and done int32 must be contiguous, one entry per row")
        n = rows // beams
        # one allocation for the four: each takes as long as half of the launch
        made = self._made(stream, scores.new_empty, (4, n, k), dtype=torch.int32)
        room, size = None, 0
        if torch.cuda.is_current_stream_capturing():
            need = ctypes.c_int64()
            _check(self._lib.tbh_beam_select_workspace(self._dev, n, beams, vocab, k, ctypes.byref(need)))
            room, size = self._room(stream, scores, need.value)
        at, step = made.data_ptr(), 4 * n * k
        _check(self._lib.tbh_beam_select_device(
            self._dev, logits.data_ptr(), logits.stride(0), n, beams, vocab, scores.data_ptr(),
            None if done is None else done.data_ptr(), eos, k, at, at + step, at + 2 * step, at + 3 * step,
            None if room is None else room.data_ptr(), size, self._raw_stream(stream)))
        tokens, parents, best, ended = made.unbind(0)
        return tokens, parents, best.view(torch.float32), ended

    def paged_reorder_device(self, keys, values, blockTable, contextLens, parents, beams: int, sharedLens=None,
                             tableOut=None, reordered=None, stream=None):
        """tbh_paged_reorder_device: rows of blockTable [requests, blocks] (groups of
        `beams`) go on where their parents [requests] stood, in the cache arrays of
        every layer (sequences keys and values).  sharedLens [requests / beams]:
        positions that are the same in a group, not copied.  Returns the new table:
        tableOut (blockTable itself: in place), else a new tensor."""
        import torch

        if len(keys) != len(values) or not len(keys):
            raise PreconditionFailure("reorder: one array of keys and one of values per layer")
        n, nkv, bs, hd, ct = self._kv_arrays(keys[0], values[0])
        layers, shape, dtype, device = len(keys), keys[0].shape, keys[0].dtype, self.device
        if layers > 1:
            for a in (*keys[1:], *values[1:]):
                if a.shape != shape or a.dtype != dtype or not a.is_contiguous() or a.get_device() != device:
                    raise PreconditionFailure("reorder: every layer's arrays must be alike")
        self._ints(torch.int32, blockTable, contextLens, parents, *(t for t in (sharedLens, reordered, tableOut) if t is not None))
        b = contextLens.numel()
        if beams <= 0 or b % beams:
            raise PreconditionFailure("reorder: requests must be a multiple of beams")
        if blockTable.dim() != 2 or blockTable.shape[0] != b or parents.numel() != b:
            raise PreconditionFailure("reorder: parents and block table must have one row per request")
        for t in (sharedLens, reordered):
            if t is not None and t.numel() != b // beams:
                raise PreconditionFailure("reorder: sharedLens and reordered must have one entry per group")
        if tableOut is None:
            tableOut = self._made(stream, torch.empty_like, blockTable)
        elif tableOut.shape != blockTable.shape:
            raise PreconditionFailure("reorder: tableOut must be like the block table")
        try:
            layout = self._layout.pack(n, bs, nkv, hd, ct, b, blockTable.shape[1])
        except struct.error:
            raise self._past_32_bits() from None
        pointers = "%dP" % layers
        _check(self._lib.tbh_paged_reorder_device(
            self._dev, layout, beams, parents.data_ptr(), contextLens.data_ptr(),
            None if sharedLens is None else sharedLens.data_ptr(), blockTable.data_ptr(), tableOut.data_ptr(), layers,
            struct.pack(pointers, *[a.data_ptr() for a in keys]), struct.pack(pointers, *[a.data_ptr() for a in values]),
            None if reordered is None else reordered.data_ptr(), self._raw_stream(stream)))
        return tableOut

    def close(self) -> None:
        with self._lock:
            cached = list(self._cache.values())
            self._cache.clear()
        with self._children_lock:
            children = list(self._children) + cached
            self._children.clear()
        for c in children:
            c.close()
        if self._dev:
            self._lib.tbh_device_close(self._dev)
            self._dev = ctypes.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass
