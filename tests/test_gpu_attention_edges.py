"""Attention over the 8-bit cache where its parts and its ranges end: against 64 bits, with attn_ref.attention's tolerance of each value."""
import numpy as np
import pytest

import arcinferzero_amd as az
import attn_ref as ref
from test_gpu_attention import check

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def eng(rt):
    e = az.Engine(16, 256)
    yield e
    e.close()


STEP = 0.3   # octaves of a score to one of a key's first value (scored)


def scored(b, page, block, kv, hd, steps):
    """A cache of scale 1 whose position p of sequence 0 has the score steps.get(p, 0) * STEP octaves with every row of `lines`."""
    c = ref.Cache(b.pages, page, block, kv, hd, seed=3)
    c.d[:] = 1.0
    c.q[0] = 0
    for p, v in steps.items():
        c.q[0, b.table[0, p // page], :, p % page, 0] = v
    return c


def lines(T, heads, hd):
    q = np.zeros((T, heads, hd), np.float32)
    q[:, :, 0] = STEP * np.log(2.0)
    return q.reshape(T, heads * hd)


@pytest.mark.parametrize("hd,page,block,heads,kv,seqs", [(64, 64, 64, 1, 1, [(40, 250)]), (64, 16, 4, 2, 1, [(100, 250)]), (128, 64, 16, 2, 2, [(40, 250)]), (128, 64, 64, 1, 1, [(40, 250)]),
                                                         (256, 64, 64, 1, 1, [(40, 250)]), (128, 64, 64, 4, 1, [(300, 4100)]), (64, 64, 64, 8, 8, [(1, 4000)] + [(1, 1)] * 63),
                                                         (128, 16, 1, 16, 8, [(1, 4000)] + [(1, 1)] * 63)])
def test_many_keys_far_below_one(eng, hd, page, block, heads, kv, seqs):
    """One key 24 octaves above all others: each of those is half a step of the sum's f32, all together many of its steps."""
    b = ref.Batch(seqs, page, seed=1)
    rows = seqs[0][0]
    check(eng, seqs, heads, kv, hd, page, block, dict(scale=1.0), b=b, c=scored(b, page, block, kv, hd, {3: 80}), q=lines(b.T, heads, hd), only={0, 1, rows // 2, rows - 1})


@pytest.mark.parametrize("hd,page,block,rows,heads", [(64, 64, 64, 40, 1), (64, 16, 4, 40, 2), (128, 64, 64, 40, 1), (128, 32, 8, 40, 1), (256, 64, 64, 40, 1), (128, 64, 64, 1, 1), (64, 16, 1, 2, 8)])
@pytest.mark.parametrize("jump", [124, 125, 126, 127])
def test_weights_at_the_last_place_of_their_f16(eng, hd, page, block, rows, heads, jump):
    """32 keys 2^-30 to 2^-31 of the largest weight, which alone fill a column of the values: cut off at 2^-32 of it, not above."""
    b = ref.Batch([(rows, 240)], page, seed=1)
    c = scored(b, page, block, 1, hd, {**{64 + j: 23 for j in range(32)}, 3: jump})
    c.q[1, :, :, :, 5] = 0
    for j in range(32):
        c.q[1, b.table[0, (64 + j) // page], :, (64 + j) % page, 5] = 127
    check(eng, [(rows, 240)], heads, 1, hd, page, block, dict(scale=1.0), b=b, c=c, q=lines(b.T, heads, hd))


# heads of 64 with and without a scale for each key, in one work-group and two; heads of 128 in work-groups of eight waves
@pytest.mark.parametrize("hd,page,block,rows,keys,heads", [(64, 64, 64, 40, 240, 1), (64, 16, 4, 40, 240, 1), (64, 64, 32, 100, 400, 2), (128, 64, 64, 300, 4100, 4)])
@pytest.mark.parametrize("jump", [57, 67, 80, 84, 100, 113, 127])
def test_weights_that_a_later_key_of_the_tile_puts_far_behind(eng, hd, page, block, rows, keys, heads, jump):
    """A tile of 64 keys that begins with 32 keys 6.9 octaves above all before it and goes on with one key 17 to 38 octaves above: the
    32 keys' weights have to come along.  One column of the values is filled by them alone."""
    b = ref.Batch([(rows, keys)], page, seed=1)
    t = 33 * 64 if keys > 4000 else 64
    c = scored(b, page, block, 1, hd, {**{t + j: 23 for j in range(32)}, t + 39: jump})
    c.q[1, :, :, :, 5] = 0
    for j in range(32):
        c.q[1, b.table[0, (t + j) // page], :, (t + j) % page, 5] = 127
    only = {0, 1, 31, 32, rows // 2, rows - 1}
    got = check(eng, [(rows, keys)], heads, 1, hd, page, block, dict(scale=1.0), b=b, c=c, q=lines(b.T, heads, hd), only=only)
    assert (got[sorted(only), :, 5] > 0).all()


FORMS = [(64, 64, 16, 8, 2, [(64, 200)]), (128, 32, 8, 8, 2, [(64, 200)]), (128, 64, 64, 8, 2, [(64, 200), (9, 60)]), (256, 32, 16, 4, 2, [(50, 120)]),
         (128, 64, 64, 8, 2, [(300, 4100)]), (128, 32, 8, 8, 2, [(2, 200)]), (64, 16, 16, 32, 1, [(1, 300)])]


@pytest.mark.parametrize("hd,page,block,heads,kv,seqs", FORMS)
@pytest.mark.parametrize("below", [18, 24, 40, 90])
def test_rows_far_smaller_than_their_neighbours(eng, hd, page, block, heads, kv, seqs, below):
    """A row's bits do not hang on the other rows of its work-group: every third one is 2^-below of the others, with a scale that gives
    just those ordinary scores."""
    T = sum(n for n, _ in seqs)
    q = np.random.default_rng(4).standard_normal((T, heads, hd)).astype(np.float32)
    small = np.arange(T) % 3 == 1 if T > 1 else np.array([True])
    q[small] *= np.float32(2.0 ** -below)
    if T == 1:
        q[:, ::2] *= np.float32(2.0 ** below)
    only = set(np.flatnonzero(small).tolist()[:: max(1, T // 60)])
    if T == 1:      # (one row: heads of unlike sizes; the large ones' scores are one-hot)
        only = None
    check(eng, seqs, heads, kv, hd, page, block, dict(scale=0.09 * 2.0 ** below), q=q.reshape(T, -1), only=only)


@pytest.mark.parametrize("hd,page,block,heads,kv", [(64, 64, 16, 8, 2), (128, 32, 8, 8, 2), (128, 64, 64, 8, 2), (256, 32, 16, 4, 2)])
def test_rows_that_see_nothing_are_of_any_size(eng, hd, page, block, heads, kv):
    """Stale rows -- at positions below 0, of a document that begins behind them -- of 1e30 beside rows of 1."""
    rng = np.random.default_rng(4)
    seqs = [(60, 40), (30, 200)]
    q = rng.standard_normal((90, heads * hd)).astype(np.float32)
    first = np.zeros(90, np.int64)
    first[60:90:4] = 10000
    q[:20] *= np.float32(1e30)
    q[60:90:4] *= np.float32(1e30)
    got = check(eng, seqs, heads, kv, hd, page, block, dict(first=first), q=q)
    assert not got[:20].any() and not got[60:90:4].any()


@pytest.mark.parametrize("seqs", [[(1, 300), (2, 40)], [(70, 300), (30, 30)]])
@pytest.mark.parametrize("q_std", [1e-37, 1e36])
def test_rows_at_the_ends_of_f32(eng, seqs, q_std):
    check(eng, seqs, 8, 2, 128, 32, 8, dict(scale=0.09 / q_std), q_std=q_std)


@pytest.mark.parametrize("seqs", [[(1, 300), (2, 40)], [(70, 300), (30, 30)], [(1, 2000)]])
@pytest.mark.parametrize("hd,block", [(64, 1), (128, 8), (128, 32)])
def test_scores_far_below_zero(eng, seqs, hd, block):
    """Every score of a row about -1e31 (they differ by more than f32's steps there): the largest has the weight, as anywhere."""
    b = ref.Batch(seqs, 32, seed=2)
    c = ref.Cache(b.pages, 32, block, 2, hd, seed=3)
    c.q[0] = np.maximum(np.abs(c.q[0]), 1)
    q = -np.abs(np.random.default_rng(5).standard_normal((b.T, 8 * hd))).astype(np.float32) * np.float32(2e30)
    got = check(eng, seqs, 8, 2, hd, 32, block, dict(scale=0.5), b=b, c=c, q=q)
    assert got.any(-1).all()


@pytest.mark.parametrize("rows", [1, 9, 40])
@pytest.mark.parametrize("block", [1, 8, 32])
@pytest.mark.parametrize("kind", ["tiny", "tiny_and_zeros", "one_tiny_then_zeros"])
def test_values_that_hardly_are_any(eng, rows, block, kind):
    """Hundreds of keys whose values' scale is 2^-119, just what the cache holds as more than zeros, or blocks of zeros behind one
    such: they count in the sum of weights as all keys do."""
    b = ref.Batch([(rows, 1100)], 32, seed=2)
    c = ref.Cache(b.pages, 32, block, 2, 128, seed=3)
    for i in range(20):
        c.d[1, b.table[0, i]] = 2.0 ** -119
    if kind != "tiny":
        keep = 1 if kind == "one_tiny_then_zeros" else 10
        for i in range(keep, 20):
            c.d[1, b.table[0, i]] = 0.0
            c.q[1, b.table[0, i]] = 0
    check(eng, [(rows, 1100)], 8, 2, 128, 32, block, b=b, c=c, q_std=0.3)


@pytest.mark.parametrize("seqs", [[(6, 3), (1, 50)], [(50, 30), (40, 70)]])
@pytest.mark.parametrize("window", [0, 11])
def test_rows_before_position_0_behind_a_prefix(eng, seqs, window):
    """Rows whose position is below 0 are left out, zeros, whatever the prefix."""
    T = sum(n for n, _ in seqs)
    n, l = seqs[0]
    out = n - l
    got = check(eng, seqs, 8, 2, 128, 32, 32, dict(prefix=[2, 60], window=window), only=set(range(out, T)))
    assert not got[:out].any()
    got = check(eng, seqs, 8, 2, 128, 32, 32, dict(prefix=[2 ** 31 - 1, 60], window=window), only=set(range(out, T)))
    assert not got[:out].any()


@pytest.mark.parametrize("hd,page,block,rows,keys,heads", [(64, 64, 64, 40, 240, 1), (64, 16, 4, 40, 240, 2), (64, 32, 32, 100, 250, 2), (128, 64, 16, 40, 240, 1), (128, 64, 64, 40, 240, 1),
                                                           (256, 32, 32, 40, 240, 1), (256, 16, 16, 40, 240, 2), (128, 64, 64, 300, 4100, 4), (128, 64, 64, 2, 1000, 4)])
@pytest.mark.parametrize("deep", [2.0, 8.0, 256.0])
@pytest.mark.parametrize("form", ["plain", "cap", "distance"])
def test_first_keys_far_below_the_others(eng, hd, page, block, rows, keys, heads, deep, form):
    """The first 32 keys of a tile of 64 (of the one in front too, in work-groups of eight waves) have scores 76 to 9754 octaves below zero,
    those behind them ordinary ones: no bits of those hang on the first reference."""
    b = ref.Batch([(rows, keys)], page, seed=1)
    rng = np.random.default_rng(2)
    t = 32 * 64 if keys > 4000 else 0
    n = 64 if keys > 4000 else 32
    c = scored(b, page, block, 1, hd, {p: int(v) for p, v in enumerate(rng.integers(-20, 21, size=keys)) if not t <= p < t + n})
    for p in range(t, t + n):
        c.q[0, b.table[0, p // page], :, p % page, 0] = -127
        if block <= 32 or n == 64:
            c.d[0, b.table[0, p // page], :, p % page // block] = deep
    q = lines(b.T, heads, hd)
    f = dict(plain=dict(scale=1.0), cap=dict(scale=1.0, cap=8000.0), distance=dict(scale=1.0, slopes=np.full(heads, 2.0 ** -9)))[form]
    check(eng, [(rows, keys)], heads, 1, hd, page, block, f, b=b, c=c, q=q, only={0, 1, rows // 2, rows - 1})
