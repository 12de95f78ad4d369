"""How exact norms with the rotation are, by the steps that the kernels take.

Squares, their sum, the mean and the reciprocal of its root are 64-bit: 2^-40 of the factor, and 2^-52 a step, which f32 does not show.  A normed
value is rounded when its product with the factor becomes f32, 2^-24, and once more with a weight, 2^-24.  So behind the pairs the value misses by
2^-24 of itself without a weight and by 2 * 2^-24 + 2^-48 with one; 2^-38 more holds the factor's 2^-40.  Where the rounded values are below the normal ones a
rounding is 2^-150, at most (1 + |w|) of it.
A pair's values have cosines and sines within 2^-23, products rounded once each (2^-24) and their sum (2^-24 of at most |a| + |b|), with mscale 1
multiplications by it that are exact: of |a| + |b| that is 2^-23 + 2 * 2^-24 + products of errors, 2 * 2^-23 and less than 2^-44, on top of the normed values' own."""
import numpy as np
import pytest

import arcinferzero_amd as az
import attn_ref as ref

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T", [1, 40, 700])
@pytest.mark.parametrize("hd,pairs", [(64, 32), (64, 16), (128, 64), (128, 32), (256, 64), (256, 128), (80, 40), (128, 29), (7, 3), (512, 128), (640, 300)])
@pytest.mark.parametrize("neighbours", [False, True])
@pytest.mark.parametrize("weights", [False, True])
def test_within_its_roundings(rt, T, hd, pairs, neighbours, weights):
    eng = az.Engine(16, 256)
    heads, kv = 3, 2
    rng = np.random.default_rng(T + hd + pairs)
    x = (rng.standard_normal((T, heads + kv, hd)) * 10.0 ** rng.uniform(-15, 15, size=(T, heads + kv, 1))).astype(np.float32)
    wq, wk = ((1.0 + 0.3 * rng.standard_normal(hd)).astype(np.float32) for _ in range(2))
    pos = rng.integers(0, 100000, size=(1, T)).astype(np.int32)
    freq = [10000.0 ** (-i / pairs) for i in range(pairs)]
    b = [az.Runtime.from_numpy(a) for a in (x, pos, wq, wk)]
    y, r, w = az.Runtime.alloc(x.nbytes), eng.make_rope(freq, None, neighbours), (heads + kv) * hd
    eng.norm_rope(r, b[0], w, 0, y, w, 0, T, heads, kv, hd, b[2] if weights else None, b[3] if weights else None, 1e-6, b[1])
    got = y.read(np.float32).reshape(x.shape).astype(np.float64)
    ref.free(b + [y, r])
    eng.close()
    n = x.astype(np.float64)
    n /= np.sqrt((n * n).mean(-1, keepdims=True) + np.float64(np.float32(1e-6)))
    if weights:
        n[:, :heads] *= wq
        n[:, heads:] *= wk
    want = ref.rope(n, pos, freq, [0] * pairs, neighbours)
    mag, least = np.abs(n), 2.0 ** -150 * 4
    own = (2 * 2.0 ** -24 + 2.0 ** -48 if weights else 2.0 ** -24) + 2.0 ** -38
    tol = mag * own + least
    for i in range(pairs):
        m, k = (2 * i, 2 * i + 1) if neighbours else (i, i + pairs)
        tol[..., m] = tol[..., k] = (mag[..., m] + mag[..., k]) * (own + 2 * 2.0 ** -23 + 2.0 ** -40) + 4 * least
    assert (np.abs(got - want) <= tol).all(), (np.abs(got - want) / tol).max()
