"""Norms of queries and keys with the rotation in the same pass, on the GPU against 64 bits.

Tolerance: of the sum of squares a lane's part of at most twelve is added in f32, four roundings behind one another at most on the way of any
square (its product or the fused one, the sum of two such, of two of these, of three): 4 * 2^-24 of the sum, half of that of its root, which
is else held in 64 bits; the root's reciprocal, its product with x and the product with the weight are rounded once each: 5 * 2^-24 of the
normed value n, with 2^-40 for the reciprocal's and the products of errors.  The rotation then misses by 4 * 2^-23 of |a| + |b| as tests/test_gpu_rope.py derives it,
and carries the errors of both: 7 * 2^-23 of |a| + |b| covers them, mscale times.  Behind the pairs 5.1 * 2^-24 of the value."""
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


def norms(x, wq, wk, heads, eps):
    x = x.astype(np.float64)
    v = (x * x).mean(-1, keepdims=True) + eps
    n = x * np.divide(1.0, np.sqrt(v), out=np.zeros_like(v), where=v > 0)
    w = np.ones((x.shape[1], x.shape[2]))
    if wq is not None:
        w[:heads] = wq
    if wk is not None:
        w[heads:] = wk
    return n * w


def check(eng, T, heads, kv, hd, pairs, neighbours, axes=1, far=0, ld=None, off=0, in_place=False, mscale=1.0, yld=None, yoff=0, weights=(True, True), eps=1e-6, scale=1.0, x=None):
    print(f"norm_rope T={T} heads={heads}+{kv} hd={hd} pairs={pairs} neighbours={neighbours} axes={axes} ld={ld} off={off} in_place={in_place}", flush=True)
    rng = np.random.default_rng(T + heads + pairs)
    n = heads + kv
    w = n * hd
    ld, yld = ld or w, yld or w
    full = (rng.standard_normal((T, ld)) * scale).astype(np.float32)
    if x is not None:
        full[:, off:off + w] = x.reshape(T, w)
    x = full
    wq, wk = ((1.0 + 0.3 * rng.standard_normal(hd)).astype(np.float32) if given else None for given in weights)
    pos = (rng.integers(0, 5000, size=(axes, T)) + far).astype(np.int32)
    axis, f = [(3 * i) % axes for i in range(pairs)], freqs(pairs)
    r = eng.make_rope(f, axis, neighbours, mscale)
    xb, pb = az.Runtime.from_numpy(x), az.Runtime.from_numpy(pos)
    wb = [None if a is None else az.Runtime.from_numpy(a) for a in (wq, wk)]
    y0 = np.full((T, yld), 7.5, np.float32)
    yb = xb if in_place else az.Runtime.from_numpy(y0)
    if in_place:
        y0, yld, yoff = x.copy(), ld, off
    eng.norm_rope(r, xb, ld, off, yb, yld, yoff, T, heads, kv, hd, wb[0], wb[1], eps, pb)
    y = yb.read(np.float32, T * yld).reshape(T, yld)
    normed = norms(x[:, off:off + w].reshape(T, n, hd), wq, wk, heads, np.float64(np.float32(eps)))
    want = ref.rope(normed, pos, f, axis, neighbours, mscale)
    got = y[:, yoff:yoff + w].reshape(T, n, hd)
    mag = np.abs(normed)
    tol = mag * 5.1 * 2.0 ** -24 + 2.0 ** -148
    for i in range(pairs):
        a, b = (2 * i, 2 * i + 1) if neighbours else (i, i + pairs)
        tol[..., a] = tol[..., b] = (mag[..., a] + mag[..., b]) * 7 * 2.0 ** -23 * mscale + 2.0 ** -146
    assert (np.abs(got - want) <= tol).all(), (np.abs(got - want) / tol).max()
    rest = np.ones(yld, bool)
    rest[yoff:yoff + w] = False
    assert np.array_equal(y[:, rest], y0[:, rest])
    ref.free([r, pb, xb] + [m for m in wb if m] + ([] if in_place else [yb]))
    return got


@pytest.mark.parametrize("T", [1, 2, 37, 300])
@pytest.mark.parametrize("hd,pairs", [(64, 32), (128, 64), (128, 32), (256, 128), (80, 40), (128, 29), (6, 1), (96, 44), (7, 3), (512, 256), (640, 320), (1024, 512), (256, 4), (516, 2)])
@pytest.mark.parametrize("neighbours", [False, True])
def test_heads(eng, T, hd, pairs, neighbours):
    check(eng, T, 4, 2, hd, pairs, neighbours)


@pytest.mark.parametrize("heads,kv", [(1, 0), (0, 1), (1, 1), (32, 8), (5, 3), (17, 0), (70, 30)])
def test_counts_of_heads(eng, heads, kv):
    for T in (1, 5, 260):
        check(eng, T, heads, kv, 128, 64, False)
        check(eng, T, heads, kv, 64, 16, True)


@pytest.mark.parametrize("axes", [2, 3])
def test_axes_and_far_positions(eng, axes):
    check(eng, 45, 6, 2, 128, 64, False, axes=axes, far=1 << 20)
    check(eng, 45, 3, 1, 128, 40, True, axes=axes, far=(1 << 31) - 5001)


@pytest.mark.parametrize("weights", [(False, True), (True, False), (False, False)])
def test_without_weights(eng, weights):
    check(eng, 9, 4, 2, 128, 64, False, weights=weights)
    check(eng, 9, 4, 2, 90, 31, True, weights=weights)


@pytest.mark.parametrize("off,ld", [(0, 1000), (128, 1000), (3, 777), (4, 1001), (130, 700)])
def test_columns_and_strides(eng, off, ld):
    check(eng, 9, 3, 1, 128, 64, False, ld=ld, off=off, yld=801, yoff=5)
    check(eng, 9, 3, 1, 128, 48, True, ld=ld, off=off, yld=800, yoff=4)
    check(eng, 9, 3, 1, 128, 64, False, ld=ld, off=off, in_place=True)
    check(eng, 9, 3, 1, 128, 31, True, ld=ld, off=off, in_place=True, mscale=1.25)
    check(eng, 300, 3, 1, 128, 32, False, ld=ld, off=off, in_place=True)


@pytest.mark.parametrize("scale", [1e-30, 1e-18, 1e18, 1e36])
def test_ends_of_the_range(eng, scale):
    """Squares that f32 does not hold."""
    check(eng, 5, 2, 2, 128, 64, False, scale=scale, eps=0.0)
    check(eng, 5, 2, 2, 100, 30, True, scale=scale, eps=1e-6)


def test_zeros_ones_and_what_is_no_number(eng):
    x = np.random.default_rng(2).standard_normal((6, 4, 128)).astype(np.float32)
    x[0, 1] = 0.0
    x[1, 2] = 0.0
    x[1, 2, 77] = 3e-39        # (below the normal numbers)
    for eps in (0.0, 1e-6):
        got = check(eng, 6, 3, 1, 128, 64, False, eps=eps, x=x)
        assert not got[0, 1].any()
    # an infinity or a NaN is its own head's alone
    x[2, 0, 5], x[3, 3, 100] = np.inf, np.nan
    for nb in (False, True):
        r = eng.make_rope(freqs(64), None, nb)
        b = [az.Runtime.from_numpy(a) for a in (x, np.arange(6, dtype=np.int32))]
        y = az.Runtime.alloc(x.nbytes)
        eng.norm_rope(r, b[0], 512, 0, y, 512, 0, 6, 3, 1, 128, None, None, 1e-6, b[1])
        got = y.read(np.float32).reshape(x.shape)
        bad = ~np.isfinite(got).all(-1)
        assert bad.sum() == 2 and bad[2, 0] and bad[3, 3] and np.isnan(got[3, 3]).all()
        ref.free(b + [y, r])


def test_as_norm_and_rope_apart(eng):
    """One call for q and k where two of the rotation on normed rows would do: the same angles, bit for bit where the norm does nothing."""
    T, heads, kv, hd = 70, 4, 2, 128
    x = np.where(np.random.default_rng(4).random((T, (heads + kv) * hd)) < 0.5, -1.0, 1.0).astype(np.float32)     # (mean square 1)
    pos = np.arange(T, dtype=np.int32) * 31
    b = [az.Runtime.from_numpy(a) for a in (x, pos)]
    y = [az.Runtime.alloc(x.nbytes) for _ in range(2)]
    r = eng.make_rope(freqs(64), None, False, 1.5)
    w = x.shape[1]
    eng.norm_rope(r, b[0], w, 0, y[0], w, 0, T, heads, kv, hd, None, None, 0.0, b[1])
    eng.rope(r, b[0], w, 0, y[1], w, 0, T, heads + kv, hd, b[1])
    assert np.array_equal(y[0].read(np.uint32), y[1].read(np.uint32))
    ref.free(b + y + [r])


def test_refusals(eng):
    x, y, pos, w = az.Runtime.alloc(4 * 8 * 512), az.Runtime.alloc(4 * 8 * 512), az.Runtime.alloc(4 * 8), az.Runtime.alloc(4 * 128)
    for m in (x, pos, w):
        m.fill(0)
    r = eng.make_rope(freqs(64))
    ok = [r, x, 512, 0, y, 512, 0, 8, 3, 1, 128, w, w, 1e-6, pos]
    eng.norm_rope(*ok)
    launches = az.lib.arcz_launch_count()

    def refused(extra=(), **k):
        a = list(ok)
        for i, v in k.items():
            a[int(i[1:])] = v
        with pytest.raises(az.ArczError):
            eng.norm_rope(*a, *extra)
    refused(_2=511)
    refused(_3=1)
    refused(_3=-1)
    refused(_7=9)
    refused(_7=-1)
    refused(_8=-1)
    refused(_9=-1)
    refused(_8=0, _9=0)
    refused(_8=2 ** 31 - 1, _9=2 ** 31 - 1)
    refused(_10=126)
    refused(_10=0)
    refused(_13=-1e-6)
    refused(_13=float("nan"))
    refused(_13=float("inf"))
    refused(_11=pos)                    # a weight of fewer values
    refused(_12=pos)
    refused(extra=(7,))                 # positions of fewer rows
    refused(_4=x, _6=128, _8=2)         # x and y share some columns
    v = y.view(0, 512)
    refused(_11=v)                      # y over a weight, or the positions
    refused(_12=v)
    refused(_14=v)
    r3 = eng.make_rope(freqs(4), [0, 1, 2, 0])
    refused(_0=r3)                      # positions on one axis only
    assert az.lib.arcz_launch_count() == launches
    a = list(ok)
    a[7] = 0
    eng.norm_rope(*a)                   # no rows
    assert az.lib.arcz_launch_count() == launches
    assert az.lib.arcz_engine_norm_rope(eng.h, None, x.h, 512, 0, y.h, 512, 0, 8, 3, 1, 128, None, None, 1e-6, pos.h, 8) == -100
    ref.free([x, y, pos, w, r, r3, v])
