"""The oracle of the paged-cache and sampling calls (oracle/paged_ref.py)
against closed forms and independent restatements, and the refusals of the C
ABI, which come before anything touches a GPU."""
import ctypes

import numpy as np
import pytest

from oracle import ops_ref as R
from oracle import paged_ref as P
from tinybrain_amd import _abi


# ---------------------------------------------------------------------------
# plan: an allocator restated with lists
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("seed", range(20))
def test_plan_keeps_blocks_apart(seed):
    # Over random steps no block is ever held twice or lost, slots of held
    # positions are distinct, and a request keeps the blocks it had.
    rng = np.random.default_rng(seed)
    bs, rows, most, blocks = int(rng.choice([1, 4, 16])), 7, 6, 20
    table, ctx = np.full((rows, most), -1, np.int32), np.zeros(rows, np.int32)
    free, count = rng.permutation(blocks).astype(np.int32), blocks
    for _ in range(30):
        new = rng.choice([-1, 0, 1, 1, 1, 3 * bs, 9 * bs], rows)
        before = [table[b, :P.ceil_div(int(ctx[b]), bs)].copy() for b in range(rows)]
        p = P.plan(new, ctx, table, free, count, bs, 80)
        held = []
        for b in range(rows):
            mine = p["table"][b, :P.ceil_div(int(p["context"][b]), bs)]
            if new[b] >= 0:
                np.testing.assert_array_equal(mine[:len(before[b])], before[b])
            held += mine.tolist()
        assert sorted(held + p["free"][:p["count"]].tolist()) == list(range(blocks))
        used = p["slots"][p["slots"] >= 0]
        assert len(set(used)) == len(used)
        table, ctx, free, count = p["table"], p["context"], p["free"], p["count"]


def test_plan_known_answer():
    # block size 4, two requests of 3 and 0 tokens, 5 free blocks 9 8 7 6 5 (5 on top)
    table = np.array([[2, -1, -1], [-1, -1, -1]], np.int32)
    p = P.plan([2, 5], [3, 0], table, np.array([9, 8, 7, 6, 5, 0]), 5, 4, 8)
    np.testing.assert_array_equal(p["table"], [[2, 5, -1], [6, 7, -1]])
    np.testing.assert_array_equal(p["slots"], [11, 20, 24, 25, 26, 27, 28, -1])
    np.testing.assert_array_equal(p["positions"], [3, 4, 0, 1, 2, 3, 4, -1])
    np.testing.assert_array_equal(p["start"], [0, 2, 7])
    np.testing.assert_array_equal(p["context"], [5, 5])
    assert p["count"] == 2


def test_plan_waits_in_order():
    # two free blocks: row 0 needs three and waits, row 1 needs one and may not
    # overtake it, row 2 needs none and runs; row 3 does not fit its table row
    table = np.full((4, 3), 7, np.int32)
    p = P.plan([12, 4, 1, 40], [0, 0, 2, 0], table, np.array([1, 2, 0, 0]), 2, 4, 60)
    np.testing.assert_array_equal(p["granted"], [0, 0, 1, 0])
    np.testing.assert_array_equal(p["context"], [0, 0, 3, 0])
    assert p["count"] == 2 and p["slots"][16] == 7 * 4 + 2 and (p["slots"] >= 0).sum() == 1


def test_plan_grants_what_has_entries():
    # row 1's last token would be the step's eighth: it waits, and row 2 behind it; their lengths stay
    table = np.full((3, 4), -1, np.int32)
    p = P.plan([3, 5, 1], [0, 2, 0], np.array([[-1] * 4, [9, -1, -1, -1], [-1] * 4], np.int32), np.arange(8), 8, 4, 7)
    np.testing.assert_array_equal(p["granted"], [3, 0, 0])
    np.testing.assert_array_equal(p["context"], [3, 2, 0])
    np.testing.assert_array_equal(p["start"], [0, 3, 8, 9])
    np.testing.assert_array_equal(p["slots"], [28, 29, 30, -1, -1, -1, -1])
    np.testing.assert_array_equal(p["positions"], [0, 1, 2, -1, -1, -1, -1])
    assert p["count"] == 7
    p = P.plan([3, 5, 1], [0, 2, 0], table, np.arange(8), 8, 4, 8)
    np.testing.assert_array_equal(p["granted"], [3, 5, 0])


# ---------------------------------------------------------------------------
# rotation, store, attention
# ---------------------------------------------------------------------------
def test_rotate():
    x = np.array([[1.0, 0.0, 0.0, 2.0]])
    np.testing.assert_allclose(P.rotate(x, [3], 1, 10000.0),
                               [[np.cos(3), np.sin(3), -2 * np.sin(0.03), 2 * np.cos(0.03)]], rtol=1e-15)
    # scores depend on the distance alone
    q, k = np.random.default_rng(0).normal(size=(2, 1, 64))
    a = P.rotate(q, [70], 1, 500.0) @ P.rotate(k, [11], 1, 500.0).T
    b = P.rotate(q, [1059], 1, 500.0) @ P.rotate(k, [1000], 1, 500.0).T
    np.testing.assert_allclose(a, b, rtol=1e-9)


def test_attention_is_the_contiguous_one():
    # one request whose blocks lie in any order, one new token per prefix length
    rng = np.random.default_rng(1)
    bs, nkv, nh, hd, n = 4, 2, 6, 8, 11
    keys, values = rng.normal(size=(2, 5, nkv, bs, hd))
    table = np.array([[3, 0, 4]])
    q = rng.normal(size=(n, nh * hd))
    k = np.concatenate([keys[b].transpose(1, 0, 2) for b in table[0]]).reshape(-1, nkv * hd)
    v = np.concatenate([values[b].transpose(1, 0, 2) for b in table[0]]).reshape(-1, nkv * hd)
    got, bound = P.attention(q, keys, values, table, [0, n], [n], nh)
    for i in range(n):
        want = R.attention(q[i:i + 1], k[:i + 1], v[:i + 1], None, hd, nh, nkv, eps=0.0)
        np.testing.assert_allclose(got[i:i + 1], want, rtol=1e-12)
    assert (bound > 0).all() and (bound < 1e-4).all()


def test_attention_of_nothing():
    keys = values = np.ones((2, 1, 4, 2))
    # rows at positions -1, 0; a hole in the table; rows behind the last request
    got, _ = P.attention(np.ones((4, 2)), keys, values, np.array([[1, -1], [-1, 0]]), [0, 2, 3], [1, 6], 1)
    np.testing.assert_array_equal(got[0], [0, 0])
    np.testing.assert_array_equal(got[1], [1, 1])
    np.testing.assert_allclose(got[2], [1, 1])
    assert np.isnan(got[3]).all()


# ---------------------------------------------------------------------------
# sampling
# ---------------------------------------------------------------------------
def test_sample_known_answers():
    x = np.log(np.array([1.0, 4.0, 2.0, 8.0, 1.0]))
    assert P.sample(x, 0.0)[0] == 0 and P.sample(x, 0.999)[0] == 4
    assert P.sample(x, 0.31)[0] == 1 and P.sample(x, 0.32)[0] == 2       # 5 / 16 = 0.3125
    np.testing.assert_allclose(P.sample(x, 0.5), (3, 0.5))
    np.testing.assert_allclose(P.sample(x, 0.0, top_k=2), (1, 1 / 3))
    np.testing.assert_allclose(P.sample(x, 0.99, top_k=4), (3, 8 / 15))  # of the equal 0 and 4 the first stays
    assert P.sample(x, 0.0, top_p=0.4)[0] == 3
    np.testing.assert_allclose(P.sample(x, 0.0, top_p=0.7), (1, 1 / 3))
    np.testing.assert_allclose(P.sample(x, 0.99, min_p=0.24), (3, 8 / 14))
    np.testing.assert_allclose(P.sample(x, 0.1, temperature=0.5, top_k=2), (1, 0.2))
    assert P.sample(x, 0.7, temperature=0.0) == (3, 1.0)
    assert P.sample([-np.inf, np.nan], 0.5) == (-1, 0.0)
    assert P.sample([1.0, np.inf, np.inf], 0.5) == (2, 0.5)
    assert P.sample([1.0, -np.inf, np.nan, 1.0], 0.9) == (3, 0.5)


def test_sample_follows_its_distribution():
    x = np.random.default_rng(2).normal(size=40)
    u = (np.arange(20000) + 0.5) / 20000
    got = np.bincount([P.sample(x, t, temperature=1.5)[0] for t in u], minlength=40) / 20000
    p = np.exp(x / 1.5) / np.exp(x / 1.5).sum()
    np.testing.assert_allclose(got, p, atol=1.01 / 20000)   # two borders, each off by less than a step of u


# ---------------------------------------------------------------------------
# refusals: decided on the host before any HIP call, so the handle is never read
# ---------------------------------------------------------------------------
_HANDLE = ctypes.create_string_buffer(4096)
DEV = ctypes.addressof(_HANDLE)
_BUF = (ctypes.c_char * 8192)()
PTR = (ctypes.addressof(_BUF) + 255) // 256 * 256


def _layout(**kw):
    f = dict(num_blocks=8, block_size=16, num_kv_heads=2, head_dim=64, type=0, max_requests=4, max_blocks=4)
    f.update(kw)
    return _abi.PagedLayout(**f)


LAYOUTS = [
    (dict(block_size=0), _abi.E_INVALID), (dict(block_size=24), _abi.E_INVALID),
    (dict(block_size=2048), _abi.E_INVALID), (dict(num_blocks=-1), _abi.E_INVALID),
    (dict(max_requests=-1), _abi.E_INVALID), (dict(max_blocks=-1), _abi.E_INVALID),
    (dict(num_blocks=1 << 27), _abi.E_INVALID), (dict(max_requests=1 << 20, max_blocks=1 << 12), _abi.E_INVALID),
    (dict(max_blocks=1 << 27, max_requests=1), _abi.E_INVALID),
]
LIMITS = [
    (dict(max_blocks=(1 << 26) + 1, max_requests=1), _abi.E_INVALID),
    (dict(max_requests=(1 << 30) + 1, max_blocks=1), _abi.E_INVALID),
]
CACHES = [
    (dict(num_kv_heads=0), _abi.E_INVALID), (dict(head_dim=0), _abi.E_INVALID), (dict(type=2), _abi.E_INVALID),
    (dict(head_dim=257), _abi.E_UNSUPPORTED),
]


def _plan(layout, **kw):
    a = dict(new=PTR, ctx=PTR, table=PTR, free=PTR, count=PTR, tokens=4, start=PTR, granted=PTR, out=PTR,
             count_out=PTR, slots=PTR, positions=PTR, dev=DEV)
    a.update(kw)
    return _abi.lib().tbh_paged_plan_device(a["dev"], ctypes.byref(layout) if layout is not None else None, a["new"],
                                            a["ctx"], a["table"], a["free"], a["count"], a["tokens"], a["start"],
                                            a["granted"], a["out"], a["count_out"], a["slots"], a["positions"], None)


@pytest.mark.parametrize("change,status", LIMITS)
def test_sizes_whose_tiles_would_pass_32_bits(change, status):
    assert _plan(_layout(**change)) == status
    assert _attention(_layout(**change)) == status
    assert _append(_layout(**change)) == status


@pytest.mark.parametrize("change,status", LAYOUTS)
def test_plan_refuses_layouts(change, status):
    assert _plan(_layout(**change)) == status
    assert "tbh_paged_plan" in _abi.last_error()


@pytest.mark.parametrize("change", [dict(dev=None), dict(new=None), dict(ctx=None), dict(table=None), dict(free=None),
                                    dict(count=None), dict(start=None), dict(granted=None), dict(out=None),
                                    dict(count_out=None), dict(slots=None), dict(positions=None), dict(tokens=-1),
                                    dict(tokens=1 << 31)])
def test_plan_refuses_arguments(change):
    assert _plan(_layout(), **change) == _abi.E_INVALID
    assert _plan(None) == _abi.E_INVALID


def _append(layout, kc=PTR, vc=PTR, dev=DEV, **kw):
    f = dict(tokens=3, x_type=0, num_heads=4, q=PTR, k=PTR, v=PTR, q_stride=256, k_stride=128, v_stride=128,
             q_out=PTR + 4096, q_out_stride=256, q_out_type=0, rope_base=10000.0, slots=PTR, positions=PTR)
    f.update(kw)
    rows = _abi.PagedRows(**f)
    return _abi.lib().tbh_paged_append_device(dev, ctypes.byref(layout), ctypes.byref(rows), kc, vc, None)


@pytest.mark.parametrize("change,status", LAYOUTS + CACHES)
def test_append_refuses_layouts(change, status):
    assert _append(_layout(**change)) == status


@pytest.mark.parametrize("change", [
    dict(dev=None), dict(tokens=-1), dict(tokens=1 << 31), dict(x_type=3), dict(q_out_type=-1), dict(num_heads=0),
    dict(k=None), dict(v=None), dict(slots=None), dict(q_out=None), dict(positions=None), dict(rope_base=-1.0),
    dict(rope_base=float("nan")), dict(rope_base=float("inf")), dict(kc=None), dict(vc=None), dict(kc=PTR + 8),
    dict(vc=PTR + 4), dict(q_stride=255), dict(k_stride=127), dict(v_stride=0), dict(q_out_stride=255),
    dict(q_out=PTR, q_out_type=1), dict(q_out=PTR, q_out_stride=260),
])
def test_append_refuses_arguments(change):
    assert _append(_layout(), **change) == _abi.E_INVALID


def test_append_refuses_to_rotate_an_odd_head():
    assert _append(_layout(head_dim=63)) == _abi.E_INVALID
    assert _append(_layout(), tokens=0, k=None) == _abi.OK


def _attention(layout, kc=PTR, vc=PTR, table=PTR, dev=DEV, **kw):
    f = dict(tokens=3, type=0, num_heads=4, q=PTR, out=PTR + 4096, q_stride=256, out_stride=256, query_start=PTR,
             context_lens=PTR, scale=0.0, max_query_len=0, max_context_len=0)
    f.update(kw)
    args = _abi.PagedQueries(**f)
    return _abi.lib().tbh_paged_attention_device(dev, ctypes.byref(layout), ctypes.byref(args), kc, vc, table, None)


@pytest.mark.parametrize("change,status", LAYOUTS + CACHES)
def test_attention_refuses_layouts(change, status):
    assert _attention(_layout(**change)) == status


@pytest.mark.parametrize("change", [
    dict(dev=None), dict(tokens=-1), dict(type=2), dict(num_heads=0), dict(num_heads=3), dict(q=None), dict(out=None),
    dict(out=PTR), dict(query_start=None), dict(context_lens=None), dict(table=None), dict(kc=None), dict(vc=None),
    dict(kc=PTR + 4), dict(q_stride=255), dict(out_stride=1), dict(scale=float("nan")), dict(scale=float("inf")),
    dict(max_query_len=-1), dict(max_context_len=-1),
])
def test_attention_refuses_arguments(change):
    assert _attention(_layout(), **change) == _abi.E_INVALID


def test_attention_of_no_rows():
    assert _attention(_layout(), tokens=0) == _abi.OK
    assert _attention(_layout(max_requests=0)) == _abi.OK
    assert _attention(_layout(), tokens=1 << 30, num_heads=4) == _abi.E_UNSUPPORTED


def test_sample_refusals():
    f = _abi.lib().tbh_sample_device
    assert f(None, PTR, 10, 2, 10, None, None, None, None, PTR, PTR, None, None) == _abi.E_INVALID
    assert f(DEV, None, 10, 2, 10, None, None, None, None, PTR, PTR, None, None) == _abi.E_INVALID
    assert f(DEV, PTR, 10, 2, 10, None, None, None, None, None, PTR, None, None) == _abi.E_INVALID
    assert f(DEV, PTR, 10, 2, 10, None, None, None, None, PTR, None, None, None) == _abi.E_INVALID
    assert f(DEV, PTR, 9, 2, 10, None, None, None, None, PTR, PTR, None, None) == _abi.E_INVALID
    assert f(DEV, PTR, 10, -1, 10, None, None, None, None, PTR, PTR, None, None) == _abi.E_INVALID
    assert f(DEV, PTR, 10, 1, -1, None, None, None, None, PTR, PTR, None, None) == _abi.E_INVALID
    big = (1 << 20) + 1
    assert f(DEV, PTR, big, 1, big, None, None, None, None, PTR, PTR, None, None) == _abi.E_UNSUPPORTED
    assert f(DEV, PTR, 10, 0, 10, None, None, None, None, PTR, PTR, None, None) == _abi.OK
    g = _abi.lib().tbh_sample
    assert g(None, PTR, 1, 4, None, None, None, None, PTR, PTR, PTR) == _abi.E_INVALID
    assert g(DEV, PTR, 1, big, None, None, None, None, PTR, PTR, PTR) == _abi.E_UNSUPPORTED


def test_packed_structs_are_the_declared_ones():
    # the wrapper packs the C structs' bytes itself
    from tinybrain_amd import HIPBackend

    for packer, struct in ((HIPBackend._layout, _abi.PagedLayout), (HIPBackend._rows, _abi.PagedRows),
                           (HIPBackend._queries, _abi.PagedQueries)):
        values = list(range(1, len(struct._fields_) + 1))
        want = struct(*values)
        got = struct.from_buffer_copy(packer.pack(*values))
        assert packer.size == ctypes.sizeof(struct)
        for name, _ in struct._fields_:
            assert getattr(got, name) == getattr(want, name), name
