"""Results that the Python entry points allocate when a call names a stream:
they come from that stream's memory (on the CPU: what torch is asked for, with
the library and torch's streams stood in for)."""
import contextlib
import types

import pytest
import torch

import tinybrain_amd as T

CURRENT, OTHER = types.SimpleNamespace(cuda_stream=1), types.SimpleNamespace(cuda_stream=2)


@pytest.fixture
def asked(monkeypatch):
    """(backend on CPU tensors, list of the streams that allocations were made on, list of the streams recorded)."""
    now, made, recorded = [CURRENT], [], []

    @contextlib.contextmanager
    def on(stream):
        now.append(stream)
        yield
        now.pop()

    def noting(f):
        def make(*args, **kw):
            made.append(now[-1])
            return f(*args, **kw)
        return make

    monkeypatch.setattr(torch.cuda, "stream", on)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: now[-1])
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda device: now[-1].cuda_stream)
    monkeypatch.setattr(torch, "empty_like", noting(torch.empty_like))
    monkeypatch.setattr(torch.Tensor, "new_empty", noting(torch.Tensor.new_empty))
    monkeypatch.setattr(torch.Tensor, "record_stream", lambda self, s: recorded.append(s))
    b = T.HIPBackend.__new__(T.HIPBackend)
    b.device, b._dev = -1, None                     # Tensor.get_device() of CPU tensors
    b._lib = types.SimpleNamespace()
    for name in ("tbh_paged_plan_device", "tbh_paged_append_device", "tbh_paged_attention_device", "tbh_sample_device",
                 "tbh_softmax_device", "tbh_rmsnorm_device", "tbh_silu_device", "tbh_gelu_device", "tbh_attention_device"):
        setattr(b._lib, name, lambda *a: 0)
    b._dev_tensor = lambda t: t
    return b, made, recorded


def _calls(b):
    i = lambda *s: torch.zeros(*s, dtype=torch.int32)       # noqa: E731
    k, q, r = torch.zeros(4, 2, 16, 64), torch.zeros(3, 256), torch.zeros(3, 128)
    return {
        "plan": lambda **kw: b.paged_plan_device(i(3), i(3), i(3, 4), i(4), i(1), 16, 4, **kw),
        "append": lambda **kw: b.paged_append_device(k, k, i(3), r, r, q=q, **kw),
        "paged_attention": lambda **kw: b.paged_attention_device(q, k, k, i(2, 4), i(3), i(2), 4, **kw),
        "sample": lambda **kw: b.sample_device(r, torch.zeros(3), **kw),
        "softmax": lambda **kw: b.softmax_device(r, **kw),
        "rmsnorm": lambda **kw: b.rmsnorm_device(r, r[0], **kw),
        "silu": lambda **kw: b.silu_device(r, **kw),
        "gelu": lambda **kw: b.gelu_device(r, **kw),
        "attention": lambda **kw: b.attention_device(q, r, r, None, 64, 4, 2, **kw),
    }


NAMES = ["plan", "append", "paged_attention", "sample", "softmax", "rmsnorm", "silu", "gelu", "attention"]


@pytest.mark.parametrize("name", NAMES)
def test_results_come_from_the_streams_own_memory(asked, name):
    b, made, recorded = asked
    _calls(b)[name](stream=OTHER)
    assert made and all(s is OTHER for s in made)
    assert recorded == [CURRENT] * len(made)         # and stay while the caller's stream reads them


@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("kw", [{}, {"stream": CURRENT}])
def test_results_of_the_current_stream(asked, name, kw):
    b, made, recorded = asked
    _calls(b)[name](**kw)
    assert made and all(s is CURRENT for s in made) and not recorded
