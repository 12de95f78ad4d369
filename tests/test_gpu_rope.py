"""Rotary positions on the GPU against 64 bits (attn_ref.rope).

Tolerance: sine and cosine within 2^-23 (the angle's last rounding 2^-25 of pi / 4 in f32, three roundings of the series' first
terms, the truncation 2e-9), both products and their sum rounded once each, two multiplications with mscale: 4 * 2^-23 of
|a| + |b| covers them, mscale times."""
import numpy as np
import pytest

import arcinferzero_amd as az
import attn_ref as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def eng(rt):
    e = az.Engine(16, 256)
    yield e
    e.close()


def freqs(p, base=10000.0):
    return [base ** (-i / p) for i in range(p)]


def check(eng, T, heads, hd, pairs, neighbours, axes=1, far=0, ld=None, off=0, in_place=False, mscale=1.0, negative=False, yld=None, yoff=0, ld_pos=None):
    print(f"rope T={T} heads={heads} hd={hd} pairs={pairs} neighbours={neighbours} axes={axes} far={far} ld={ld} off={off} in_place={in_place}", flush=True)
    rng = np.random.default_rng(T + heads + pairs)
    w = heads * hd
    ld, yld, ld_pos = ld or w, yld or w, ld_pos or T
    x = rng.standard_normal((T, ld)).astype(np.float32)
    pos = np.zeros((axes, ld_pos), np.int32)
    pos[:, :T] = rng.integers(0, 5000, size=(axes, T)) + far
    if negative:
        pos = -pos
    axis = [(3 * i) % axes for i in range(pairs)]
    f = freqs(pairs)
    r = eng.make_rope(f, axis, neighbours, mscale)
    xb, pb = az.Runtime.from_numpy(x), az.Runtime.from_numpy(pos)
    y0 = np.full((T, yld), 7.5, np.float32)
    yb = xb if in_place else az.Runtime.from_numpy(y0)
    if in_place:
        y0, yld, yoff = x.copy(), ld, off
    eng.rope(r, xb, ld, off, yb, yld, yoff, T, heads, hd, pb, ld_pos)
    y = yb.read(np.float32, T * yld).reshape(T, yld)
    h = x[:, off:off + w].reshape(T, heads, hd)
    want = ref.rope(h, pos[:, :T], f, axis, neighbours, mscale)
    got = y[:, yoff:yoff + w].reshape(T, heads, hd)
    mag = np.abs(h).astype(np.float64)
    tol = np.zeros_like(mag)
    for i in range(pairs):
        m, n = (2 * i, 2 * i + 1) if neighbours else (i, i + pairs)
        tol[..., m] = tol[..., n] = (mag[..., m] + mag[..., n]) * 4 * 2.0 ** -23 * mscale
    assert (np.abs(got - want) <= tol).all(), (np.abs(got - want) - tol).max()
    rest = np.ones(yld, bool)
    rest[yoff:yoff + w] = False
    assert np.array_equal(y[:, rest], y0[:, rest])
    for b in [r, pb, xb] + ([] if in_place else [yb]):
        b.free()


@pytest.mark.parametrize("T", [1, 2, 37, 300])
@pytest.mark.parametrize("hd,pairs", [(64, 32), (128, 64), (128, 32), (256, 128), (80, 40), (128, 29), (6, 1), (96, 45), (7, 3)])
@pytest.mark.parametrize("neighbours", [False, True])
def test_heads(eng, T, hd, pairs, neighbours):
    check(eng, T, 5, hd, pairs, neighbours)


@pytest.mark.parametrize("axes", [2, 3, 4])
def test_axes(eng, axes):
    check(eng, 45, 12, 128, 64, False, axes=axes)
    check(eng, 45, 3, 128, 40, True, axes=axes, ld_pos=64)


@pytest.mark.parametrize("far", [1 << 20, (1 << 24) + 1, (1 << 31) - 5001])
def test_far_positions(eng, far):
    """An f32 product of such a position and a frequency has no digit of its place on the circle left."""
    check(eng, 20, 4, 128, 64, False, far=far)
    check(eng, 20, 4, 128, 64, True, far=far, negative=True)


@pytest.mark.parametrize("off,ld", [(0, 1000), (128, 1000), (3, 777), (4, 1001), (130, 700)])
def test_columns_and_strides(eng, off, ld):
    check(eng, 9, 4, 128, 64, False, ld=ld, off=off, yld=801, yoff=5)
    check(eng, 9, 4, 128, 48, True, ld=ld, off=off, yld=800, yoff=4)
    check(eng, 9, 4, 128, 64, False, ld=ld, off=off, in_place=True)
    check(eng, 9, 4, 128, 31, True, ld=ld, off=off, in_place=True, mscale=1.25)


def test_back_is_the_inverse(eng):
    rng = np.random.default_rng(3)
    T, w = 50, 512
    x = rng.standard_normal((T, w)).astype(np.float32)
    pos = rng.integers(0, 1 << 20, size=T).astype(np.int32)
    b = [az.Runtime.from_numpy(a) for a in (x, pos, -pos)]
    r = eng.make_rope(freqs(64))
    eng.rope(r, b[0], w, 0, b[0], w, 0, T, 4, 128, b[1])
    eng.rope(r, b[0], w, 0, b[0], w, 0, T, 4, 128, b[2])
    y = b[0].read(np.float32, T * w).reshape(T, w)
    assert np.abs(y - x).max() <= 16 * 2.0 ** -23 * np.abs(x).max()     # (two turns, each 4 * 2^-23 of both values of a pair)
    ref.free(b + [r])


def test_refusals(eng):
    x, pos = az.Runtime.alloc(4 * 8 * 512), az.Runtime.alloc(4 * 8)
    y = az.Runtime.alloc(4 * 8 * 512)
    r = eng.make_rope(freqs(64))
    ok = (r, x, 512, 0, y, 512, 0, 8, 4, 128, pos)
    eng.rope(*ok)

    def refused(*a, **k):
        with pytest.raises(az.ArczError):
            eng.rope(*a, **k)
    refused(r, x, 511, 0, y, 512, 0, 8, 4, 128, pos)          # columns past the row
    refused(r, x, 512, 1, y, 512, 0, 8, 4, 128, pos)
    refused(r, x, 512, -1, y, 512, 0, 8, 4, 128, pos)
    refused(r, x, 512, 0, y, 512, 0, 9, 4, 128, pos)          # rows past the buffers
    refused(r, x, 512, 0, y, 512, 0, -1, 4, 128, pos)
    refused(r, x, 512, 0, y, 512, 0, 8, 4, 126, pos)          # more pairs than the head has
    refused(r, x, 512, 0, y, 512, 0, 8, 0, 128, pos)
    refused(r, x, 512, 0, y, 512, 0, 8, 4, 128, pos, 7)       # positions of fewer rows
    refused(r, x, 512, 0, x, 512, 128, 7, 3, 128, pos)        # x and y share some columns
    eng.rope(r, x, 512, 0, x, 512, 256, 8, 2, 128, pos)       # ... or none
    eng.rope(r, x, 512, 0, y, 512, 0, 0, 4, 128, pos)         # no rows
    r3 = eng.make_rope(freqs(4), [0, 1, 2, 0])
    refused(r3, x, 512, 0, y, 512, 0, 8, 4, 128, pos)         # positions on one axis only
    for bad in ([], [1.0] * 513, [float("nan")], [float("inf")]):
        with pytest.raises(az.ArczError):
            eng.make_rope(bad)
    for b in (r3, r, y, pos, x):
        b.free()
