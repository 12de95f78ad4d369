"""Heads with an infinity: x / sqrt(mean(x^2) + eps) is NaN for it and 0 for the finite values beside it."""
import numpy as np
import pytest

import arcinferzero_amd as az
import attn_ref as ref

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hd,pairs", [(128, 64), (128, 32), (64, 32), (256, 64), (128, 29), (7, 3)])
@pytest.mark.parametrize("neighbours", [False, True])
def test_the_values_beside_it_are_zeros(rt, hd, pairs, neighbours):
    eng = az.Engine(16, 256)
    T, heads = 5, 3
    x = np.random.default_rng(hd).standard_normal((T, heads, hd)).astype(np.float32)
    x[1, 0, 2], x[2, 2, hd - 1], x[3, 1, 0] = np.inf, -np.inf, np.inf
    x[3, 1, 1] = np.nan                       # (a NaN beside it: the head's mean is none)
    b = [az.Runtime.from_numpy(a) for a in (x, np.arange(T, dtype=np.int32) * 7)]
    y = az.Runtime.alloc(x.nbytes)
    r = eng.make_rope([10000.0 ** (-i / pairs) for i in range(pairs)], None, neighbours)
    for eps in (0.0, 1e-6):
        eng.norm_rope(r, b[0], heads * hd, 0, y, heads * hd, 0, T, 2, 1, hd, None, None, eps, b[1])
        got = y.read(np.float32).reshape(x.shape)
        for t, h, i in ((1, 0, 2), (2, 2, hd - 1)):
            nan = {i}
            if i < 2 * pairs:
                nan |= {i ^ 1} if neighbours else {(i + pairs) % (2 * pairs)}
            for d in range(hd):
                assert np.isnan(got[t, h, d]) if d in nan else got[t, h, d] == 0.0, (t, h, d, got[t, h, d])
        assert np.isnan(got[3, 1]).all()
        got[1, 0] = got[2, 2] = got[3, 1] = 0.0
        assert np.isfinite(got).all() and all(np.abs(got[t, h]).max() > 0.1 for t in (0, 4) for h in range(heads))
    ref.free(b + [y, r])
    eng.close()
