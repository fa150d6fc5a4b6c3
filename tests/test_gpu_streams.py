"""Calls that name a stream while torch's current stream still uses memory that
was freed on it: the result may not lie there."""
import numpy as np
import pytest

import tinybrain_amd as T

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def calls():
    import torch

    b = T.HIPBackend(0)
    i = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")       # noqa: E731
    rng = np.random.default_rng(1)
    w = T.DeviceWeight(b, T.quantize(rng.normal(size=(512, 1024)).astype(np.float32), T.QuantizationMode.perChannel))
    k, q, r = torch.randn(40, 2, 16, 64, device="cuda"), torch.randn(300, 512, device="cuda"), torch.randn(300, 128, device="cuda")
    table, start, context = i([list(range(40))]), i([0, 300]), i([600])
    lens, ctx, u = i([100, 200]), i([0, 0]), torch.rand(300, device="cuda")
    pages, stack, height, q16 = i([[-1] * 20] * 2), i(list(range(40))), i([40]), q.bfloat16()
    kv = torch.zeros(40, 2, 16, 64, device="cuda")
    slots = torch.arange(300, dtype=torch.int32, device="cuda")
    yield {      # inputs are there before: nothing but results is made in a call
        "matmul": lambda **kw: b.matmul_device(q, w, **kw),
        "linear": lambda **kw: b.linear_device(q, w, **kw),
        "matmul_bf16": lambda **kw: b.matmul_bf16_device(q16, w, **kw),
        "dequantize": lambda **kw: b.dequantize_device(w, **kw),
        "softmax": lambda **kw: b.softmax_device(q, **kw),
        "silu": lambda **kw: b.silu_device(q, **kw),
        "attention": lambda **kw: b.attention_device(q, r, r, None, 64, 8, 2, **kw),
        "plan": lambda **kw: b.paged_plan_device(lens, ctx, pages, stack, height, 16, 300, **kw).slots,
        "append": lambda **kw: b.paged_append_device(kv, kv, slots, r, r, q=q, positions=slots, ropeBase=1e4, **kw),
        "paged_attention": lambda **kw: b.paged_attention_device(q, k, k, table, start, context, 8, **kw),
        "sample": lambda **kw: b.sample_device(q, u, **kw)[0],
    }
    w.close()
    b.close()


@pytest.mark.parametrize("name", ["matmul", "linear", "matmul_bf16", "dequantize", "softmax", "silu", "attention", "plan",
                                  "append", "paged_attention", "sample"])
def test_result_outlives_what_the_current_stream_still_writes(calls, name):
    import torch

    call = calls[name]
    want = call().clone()
    s, a = torch.cuda.Stream(), torch.randn(4096, 4096, device="cuda")
    call(stream=s)                                   # its workspace and code
    torch.cuda.synchronize()
    sizes = [want.untyped_storage().nbytes(), 4 * (3 * 2 + 2 + 2 * 300)]
    freed = [torch.empty(n, dtype=torch.uint8, device="cuda") for n in sizes for _ in range(8)]
    for _ in range(40):
        a = a @ a * 1e-2                             # some milliseconds of work, then writes to memory that is freed now
    for t in freed:
        t.fill_(255)
    del freed, t
    got = call(stream=s)
    torch.cuda.synchronize()
    assert torch.equal(got, want)
