"""What the library's host code launches and allocates, without a GPU: the C ABI
over a stand-in for the HIP runtime (hip_stand_in.cpp), in a process of its own.

Each test gives a body of Python that finds `L` (the library), `dev` (an open
device), launches() (those since the last call: stream, grid, block, name) and
the calls below, on addresses that nothing reads.
"""
import os
import shutil
import subprocess
import sys
import textwrap

import pytest

from tinybrain_amd import _abi

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)

PRELUDE = r"""
import ctypes, sys, threading
import numpy as np
S = ctypes.CDLL(sys.argv[1], ctypes.RTLD_GLOBAL)
S.stand_in_bytes.restype = S.stand_in_launches.restype = ctypes.c_size_t
S.stand_in_launches.argtypes = [ctypes.c_char_p, ctypes.c_size_t]
S.stand_in_limits.argtypes = [ctypes.c_size_t, ctypes.c_size_t]
ALL = (1 << 64) - 1
sys.modules["torch"] = None      # its own runtime stays out
from tinybrain_amd import _abi
L = _abi.lib()
dev = ctypes.c_void_p()
assert L.tbh_device_open(0, ctypes.byref(dev)) == 0, _abi.last_error()
P = 1 << 40                      # a device address
STREAM = 0x2000
room = ctypes.create_string_buffer(1 << 20)


def launches():
    assert S.stand_in_launches(room, len(room)) < len(room)
    return [(int(s), (int(x), int(y)), int(b), name) for s, x, y, b, name in
            (line.split(" ", 4) for line in room.value.decode().splitlines())]


def layout(**kw):
    f = dict(num_blocks=4096, block_size=16, num_kv_heads=8, head_dim=128, type=1, max_requests=4, max_blocks=512)
    f.update(kw)
    return _abi.PagedLayout(**f)


def attention(l, tokens, heads=32, stream=STREAM, **kw):
    f = dict(tokens=tokens, type=0, num_heads=heads, q=P, out=P + (1 << 38), q_stride=heads * l.head_dim,
             out_stride=heads * l.head_dim, query_start=P, context_lens=P, scale=0.0, max_query_len=0,
             max_context_len=0)
    f.update(kw)
    q = _abi.PagedQueries(**f)
    return L.tbh_paged_attention_device(dev, ctypes.byref(l), ctypes.byref(q), P, P, P, stream)


def plan(l, tokens, stream=STREAM):
    return L.tbh_paged_plan_device(dev, ctypes.byref(l), P, P, P, P, P, tokens, P, P, P, P, P, P, stream)


def append(l, tokens, stream=STREAM, **kw):
    w = l.num_kv_heads * l.head_dim
    f = dict(tokens=tokens, x_type=0, num_heads=0, q=None, k=P, v=P, q_stride=0, k_stride=w, v_stride=w, q_out=None,
             q_out_stride=0, q_out_type=0, rope_base=0.0, slots=P, positions=None)
    f.update(kw)
    rows = _abi.PagedRows(**f)
    return L.tbh_paged_append_device(dev, ctypes.byref(l), ctypes.byref(rows), P, P, stream)


def sample(rows, vocab, stream=STREAM):
    return L.tbh_sample_device(dev, P, vocab, rows, vocab, None, None, None, None, P, P, None, stream)


def contiguous_attention(queries, positions, stream=STREAM):
    shape = _abi.AttentionShape(1, queries, positions, 64, 8, 2)
    return L.tbh_attention_device(dev, ctypes.byref(shape), P, P, P, None, P + (1 << 38), stream)
"""


@pytest.fixture(scope="session")
def stand_in(tmp_path_factory):
    if not os.path.exists(_abi.LIB_PATH) or shutil.which("g++") is None:
        pytest.skip("needs the built library and g++")
    so = str(tmp_path_factory.mktemp("stand_in") / "stand_in.so")
    subprocess.run(["g++", "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include", "-std=c++17", "-O1", "-shared", "-fPIC", "-o",
                    so, os.path.join(HERE, "hip_stand_in.cpp")], check=True, timeout=120)

    def run(body):
        r = subprocess.run([sys.executable, "-c", PRELUDE + textwrap.dedent(body), so], cwd=ROOT, timeout=120,
                           capture_output=True, text=True)
        assert r.returncode == 0, r.stdout + r.stderr

    return run


def test_stand_in_takes_the_runtimes_place(stand_in):
    stand_in("""
        assert attention(layout(), 4, max_query_len=1) == 0, _abi.last_error()
        l = launches()
        assert ["paged_split" in l[0][3], "paged_split_merge" in l[1][3]] == [True, True] and len(l) == 2, l
        assert {x[0] for x in l} == {STREAM}
        S.stand_in_capturing(1)                  # no workspace on this stream yet: whole contexts, one launch
        assert attention(layout(), 4, max_query_len=1, stream=0x3000) == 0 and len(launches()) == 1
    """)


def test_threads_on_one_stream_do_not_mix_their_launches(stand_in):
    # A call in parts leaves partial results in its stream's workspace and joins them in its last launch:
    # no other thread's launch on that stream may come between.
    stand_in("""
        import tinybrain_amd as T
        backend = T.HIPBackend(0)
        dev = backend._dev                   # one handle: each has its own workspaces
        rng = np.random.default_rng(0)
        w = [T.DeviceWeight(backend, T.quantize(rng.normal(size=s).astype(np.float32), T.QuantizationMode.perChannel))
             for s in ((2048, 256), (4096, 512))]
        calls = [lambda: attention(layout(), 4, max_query_len=1),
                 lambda: attention(layout(), 300),
                 lambda: contiguous_attention(1, 4096),
                 lambda: contiguous_attention(64, 2048),
                 lambda: plan(layout(), 9000)]
        for x in w:
            for rows in (8, 64, 200):
                calls.append(lambda x=x, m=rows: L.tbh_matmul_device(x.handle, P, m, x.K, P, STREAM))
                calls.append(lambda x=x, m=rows: L.tbh_matmul_bf16_device(x.handle, P, m, x.K, P, STREAM))
        launches()
        one = []
        for c in calls:
            assert c() == 0, _abi.last_error()
            one.append([(grid, block, name) for _, grid, block, name in launches()])
        several = [i for i, x in enumerate(one) if len(x) > 1]
        assert several[:5] == [0, 1, 2, 3, 4] and len(several) > 6, [[n[2] for n in x] for x in one]

        def work(t):
            for r in range(12):
                for i in range(len(several)):
                    assert calls[several[(i * 3 + t + r) % len(several)]]() == 0
            done.append(t)

        done = []
        threads = [threading.Thread(target=work, args=(t,)) for t in range(6)]
        [t.start() for t in threads], [t.join() for t in threads]
        assert len(done) == 6
        got = [(grid, block, name) for _, grid, block, name in launches()]
        ends = {0}                           # where whole calls, one after the other, can end
        for at in range(len(got)):
            if at in ends:
                ends |= {at + len(one[i]) for i in several if got[at:at + len(one[i])] == one[i]}
        assert len(got) in ends, got[max(ends):max(ends) + 4]
    """)


def test_memory_that_cannot_be_had_fails_no_call_that_does_without(stand_in):
    # The runtime keeps a failed allocation's error until it is read, and a launch's check reads it.
    stand_in("""
        import tinybrain_amd as T
        backend = T.HIPBackend(0)
        dev = backend._dev
        w = T.quantize(np.random.default_rng(0).normal(size=(4096, 512)).astype(np.float32), T.QuantizationMode.perChannel)
        d = T.DeviceWeight(backend, w)
        S.stand_in_limits(0, ALL)
        calls = [lambda s: attention(layout(), 4, max_query_len=1, stream=s), lambda s: attention(layout(), 300, stream=s),
                 lambda s: contiguous_attention(1, 4096, s), lambda s: contiguous_attention(64, 2048, s),
                 lambda s: L.tbh_matmul_device(d.handle, P, 64, d.K, P, s)]
        for i, call in enumerate(calls):
            assert call(0x4000 + 64 * i) == 0, (i, _abi.last_error())     # whole contexts, whole K
        S.stand_in_limits(ALL, 0)                                         # nor page-locked memory
        backend.matmulQuantized(np.zeros((1, 4096), np.float32), w)
        backend.matmulQuantized(np.zeros((64, 4096), np.float32), w)
    """)


def test_partials_stay_within_their_limit(stand_in):
    # They are sized by what the lengths may be; 128 MiB each for tiles and for few rows.
    stand_in("""
        def grown(l, tokens, stream, **kw):
            before = S.stand_in_bytes()
            assert attention(l, tokens, stream=stream, **kw) == 0, _abi.last_error()
            return S.stand_in_bytes() - before

        most, s = 0, 0x10000
        for requests in (1, 64, 256, 1024, 4096):
            for positions in (1024, 8192, 131072, 1 << 20):
                for hd in (32, 64, 96, 128):
                    for ct in (0, 1):
                        l = layout(max_requests=requests, max_blocks=positions // 16, head_dim=hd, type=ct)
                        for tokens in (1, requests, requests + 511, 20000):
                            for kw in ({}, dict(max_query_len=1), dict(max_query_len=300, max_context_len=positions)):
                                s += 64
                                n = grown(l, tokens, s, **kw)
                                assert n <= 256 << 20, (requests, positions, hd, ct, tokens, kw, n)
                                most = max(most, n)
                                L.tbh_device_close(dev)
                                assert L.tbh_device_open(0, ctypes.byref(dev)) == 0
                                launches()
        assert most > 200 << 20              # the limit is what held some of them
        # a batch of usual size keeps its parts: 64 requests of up to 8192 positions
        assert attention(layout(max_requests=64), 64, max_query_len=1, max_context_len=8192, stream=s + 64) == 0
        assert launches()[0][1] == (64 * 8 * 8, 1)
    """)


def test_calls_of_many_blocks_are_launched(stand_in):
    # A grid's x holds below 2^32 threads: up to 2^31 - 1 rows or requests, as the checks take them.
    stand_in("""
        def blocks():                        # of each kernel, in one launch or in several
            n = {}
            for _, (x, y), _, name in launches():
                n[name] = n.get(name, 0) + x * y
            return list(n.values())

        l = layout(num_kv_heads=1, head_dim=64)
        for tokens in (5, 1 << 20, (1 << 20) + 1, 1 << 24, 1 << 31):
            tokens = min(tokens, (1 << 31) - 1)
            assert append(l, tokens) == 0, (tokens, _abi.last_error())
            n, = blocks()
            assert tokens <= n < tokens + (1 << 20)
        for rows in (5, 1 << 22, (1 << 31) - 1):
            assert sample(rows, 7) == 0, (rows, _abi.last_error())
            n, = blocks()
            assert rows <= n < rows + (1 << 20)
        for heads, hd in ((8, 64), (8, 128), (8, 32), (8, 80)):
            for requests, tokens in (((1 << 21) + 5, (1 << 21) + 5), (4, 1 << 27), ((1 << 27) - 1, (1 << 27) - 1)):
                l = layout(max_requests=requests, max_blocks=2, head_dim=hd)
                for kw in ({}, dict(max_query_len=1))[:1 + (requests == tokens)]:
                    assert attention(l, tokens, heads=heads, **kw) == 0, (heads, hd, requests, kw, _abi.last_error())
                    assert max(blocks()) >= tokens * heads // 128
    """)
