"""Outputs that share memory with inputs are refused by the FP8 product, the
mixture-of-experts layer and beam selection, also where rows are strided; rows side by
side in one wider matrix are not.  Over the stand-in for the HIP runtime."""
from test_experts_host import MAKE
from test_host_launches import stand_in  # noqa: F401

ROWS = """
def shared(x0, sx, nx, y0, sy, ny, rows):      # byte by byte
    bytes_of = lambda at, stride, width: {at + r * stride + i for r in range(rows) for i in range(width)}
    return bool(bytes_of(x0, sx, nx) & bytes_of(y0, sy, ny))
"""


def test_strided_rows(stand_in):  # noqa: F811
    # 300 inputs, 200 outputs of the FP8 product; 40 of the layer
    stand_in(MAKE + ROWS + """
I = _abi.E_INVALID
some = [0, 0]
for rows in (1, 2, 3, 5):
    for xs, ys in ((300, 200), (300, 500), (500, 200), (500, 500), (700, 500), (500, 703), (300, 201), (1000, 1000)):
        for off in (4, 296, 299, 300, 301, 495, 500, 504, 700, 800, 1199, 1200, 1500, 1999, 2000, 3000, 5000,
                    -4, -199, -200, -201, -300, -496, -500, -700, -1000, -1200, -2000, -5000):
            want = shared(0, 4 * xs, 1200, 4 * off, 4 * ys, 800, rows)
            got = fp8(rows, xs=xs, ys=ys, y=P + 4 * off)
            assert got == (I if want else 0), (rows, xs, ys, off, got)
            some[want] += 1
assert min(some) > 50
for rows in (1, 2, 4):
    for xs, ys in ((40, 40), (40, 80), (80, 40), (80, 80), (100, 80)):
        for off in (4, 36, 39, 40, 41, 60, 80, 120, 160, 400, -4, -39, -40, -41, -80, -120, -400):
            want = shared(0, 4 * xs, 160, 4 * off, 4 * ys, 160, rows)
            got = moe(rows, xs=xs, ys=ys, y=P + 4 * off)
            assert got == (I if want else 0), (rows, xs, ys, off, got)
# x of bf16 within rows of fp32 and beside them
assert fp8(9, xt=1, xs=1400, y=P + 600, ys=700) == 0 and fp8(9, xt=1, xs=1400, y=P + 596, ys=700) == I
assert fp8(9, xt=1, xs=1400, y=P + 2000, ys=700) == 0 and fp8(9, xt=1, xs=1400, y=P + 2004, ys=700) == I
# the last of very many rows
n = 1 << 22
assert fp8(n, xs=300, y=P + 1200 * n - 4, ys=999) == I and fp8(n, xs=300, y=P + 1200 * n, ys=999) == 0
assert fp8(n, xs=500, y=P + 2000 * n, ys=200) == 0 and fp8(n, xs=500, y=P + 2000 * n - 804, ys=200) == I
""")


def test_choices_of_the_layer(stand_in):  # noqa: F811
    # 5 tokens of 40 fp32; two experts a token: 40 bytes each
    stand_in(MAKE + """
I, far = _abi.E_INVALID, P + (1 << 37)
X, Y, n = P, P + (1 << 38), 5 * 160
for at in (X, Y):
    for kw in (dict(e=at), dict(p=at), dict(e=at + n - 4), dict(p=at + n - 4), dict(e=at - 36), dict(p=at - 36)):
        assert moe(5, **kw) == I, kw
        assert "overlap" in _abi.last_error()
    for kw in (dict(e=at + n), dict(p=at - 40), dict(e=at + n, p=at - 40)):
        assert moe(5, **kw) == 0, kw
assert moe(5, e=far, p=far) == moe(5, e=far, p=far + 36) == moe(5, e=far, p=far - 36) == I
assert moe(5, e=far, p=far + 40) == moe(5, e=far + 40, p=far) == 0
# between the rows of a wider matrix
assert moe(5, xs=80, e=X + 160) == 0 and moe(5, xs=80, e=X + 124) == I and moe(5, ys=80, p=Y + 300) == I
""")


def test_outputs_of_a_selection(stand_in):  # noqa: F811
    # 3 requests of 4 rows, k = 4: 48 bytes of everything but the logits, of 12 rows of 900 in 1000
    stand_in(MAKE + """
I = _abi.E_INVALID
NAMES = ("tokens", "parents", "scores_out", "done_out")
def call(k=4, **kw):
    a = dict(logits=P, scores=P + (1 << 30), done=P + (2 << 30), tokens=P + (3 << 30), parents=P + (4 << 30),
             scores_out=P + (5 << 30), done_out=P + (6 << 30))
    a.update(kw)
    return L.tbh_beam_select_device(dev, a["logits"], 1000, 3, 4, 900, a["scores"], a["done"], 2, k, *(a[n] for n in NAMES),
                                    None, 0, STREAM)
assert call() == 0 and call(done=None) == 0 and call(done_out=None) == 0
SCORES, DONE = P + (1 << 30), P + (2 << 30)
for n in NAMES:                                # what all blocks of a row read
    for off in (0, 44, -44):
        assert call(**{n: DONE + off}) == I, (n, off)
        assert "overlap" in _abi.last_error()
    assert call(**{n: DONE + 48}) == call(**{n: DONE - 48}) == 0
    assert call(done=None, **{n: DONE}) == 0
for off in (4, -4, 44, -44):
    assert call(scores_out=SCORES + off) == I
for off in (0, 4, -4, 44, -44):
    assert call(done_out=SCORES + off) == I and call(done_out=P + 40000 + off) == I
    for n in ("tokens", "parents", "scores_out"):
        assert call(done_out=P + (7 << 30) + off, **{n: P + (7 << 30)}) == I
assert call(scores_out=SCORES) == 0            # a request's scores in place
assert call(k=3, scores_out=SCORES) == call(k=8, scores_out=SCORES) == I
""")
