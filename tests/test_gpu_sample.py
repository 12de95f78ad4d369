"""Tokens from rows of logits, on the GPU against the definition in 64 bits on the host.

A token is a whole number, so it has to be equal -- unless the draw, or a cut, lies within the weights' rounding of a border between two tokens: weights
are held to 2^-42 (and to 2^-43 of the largest), so a running sum of n of them misses by no more than n * 2^-43 of the largest and 2^-42 of itself.
The check asks for a token that the definition gives for some u within that of the one given, and for some cut by p likewise; where the
borders are further off (all but about one in 10^6 rows) that is one token.  prob: the same relative to the weight, and its rounding to f32, 2^-24."""
import os

import numpy as np
import pytest

import arcinferzero_amd as az
import attn_ref as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", params=["0", "1"])
def eng(rt, request):
    """An engine that gives a row one work-group, or (up to 96 rows a call) sixteen."""
    os.environ["ARCZ_SAMPLE_SPLIT"] = request.param
    e = az.Engine(16, 256)
    del os.environ["ARCZ_SAMPLE_SPLIT"]
    yield e
    e.close()


def kept(x, t, k, p, q, slack=0.0):
    """(indices in the row's order, their weights) by the definition; p moved by `slack` of the sum."""
    with np.errstate(all="ignore"):
        x = np.where(np.isnan(x), -np.inf, x.astype(np.float64))
    if not (x > -np.inf).any():
        return np.zeros(0, int), np.zeros(0)
    top = x.max()
    if not t > 0:
        i = int(np.argmax(x))
        return np.array([i]), np.ones(1)
    with np.errstate(all="ignore"):
        w = np.where(x == np.inf, 1.0, 0.0) if top == np.inf else np.where(x > -np.inf, np.exp((x - top) / np.float64(t)) if np.isfinite(t) else 1.0, 0.0)
    order = np.lexsort((np.arange(x.size), -x))
    order = order[x[order] > -np.inf]
    if 0 < k < x.size:
        order = order[:k]
    if p < 1:
        run = np.cumsum(w[order])
        n = 1 + int(np.searchsorted(run, max(p, 0.0) * run[-1] + slack * run[-1], side="left"))
        order = order[:n]
    if q > 0:
        order = order[(w[order] >= min(q, 1.0)) | (x[order] == top)]
    order = np.sort(order)
    return order, w[order]


def tokens(x, t, k, p, q, u):
    """{token: its probabilities} of every draw, and every cut by p, that the rounding allows (weights that are all equal lie on a border)."""
    out = {}
    n = x.size
    eps = n * 2.0 ** -43 + 2.0 ** -41
    for slack in ((0.0,) if not p < 1 else (0.0, -eps, eps)):
        order, w = kept(x, t, k, p, q, slack)
        if not order.size:
            return {-1: [0.0]}
        run = np.cumsum(w)
        u0 = float(u) if u > 0 else 0.0
        for d in (0.0, -eps, eps):
            i = int(np.searchsorted(run, min(max(u0 + d, 0.0), 1.0) * run[-1], side="right"))
            heavy = np.nonzero(w > 2.0 ** -44)[0]
            i = min(i, int(heavy[-1]))
            out.setdefault(int(order[i]), []).append(w[i] / run[-1])
    return out


def check(eng, x, t=None, k=None, p=None, q=None, u=None, ld=None, off=0, seed=0, prob=True):
    """Parameters: one for all rows, one each, or None."""
    T, V = x.shape
    rng = np.random.default_rng(seed)
    ld = ld or V
    full = np.full((T, ld), np.nan, np.float32)     # (what lies beside the rows does not matter)
    full[:, off:off + V] = x
    u = np.broadcast_to(np.asarray(rng.random(T) if u is None else u, np.float32), T)
    given = [None if a is None else np.ascontiguousarray(np.broadcast_to(np.asarray(a, dt), T)) for a, dt in ((t, np.float32), (k, np.int32), (p, np.float32), (q, np.float32))]
    print(f"sample T={T} V={V} t={t} k={k} p={p} q={q} ld={ld} off={off}", flush=True)
    hold = [az.Runtime.from_numpy(np.ascontiguousarray(a)) for a in (full, u)]
    form = [None if a is None else az.Runtime.from_numpy(a) for a in given]
    tok, pr = az.Runtime.from_numpy(np.full(T, -9, np.int32)), az.Runtime.from_numpy(np.full(T, -9, np.float32))
    eng.sample(hold[0], ld, off, V, T, az.Sampling(*form), hold[1], tok, pr if prob else None)
    got, gp = tok.read(np.int32), pr.read(np.float32)
    for r in range(T):
        a = [d if g is None else g[r] for g, d in zip(given, (1.0, 0, 1.0, 0.0))]
        want = tokens(x[r], float(a[0]), int(a[1]), float(a[2]), float(a[3]), float(u[r]))
        assert int(got[r]) in want, (r, got[r], want, a, u[r])
        if prob:
            assert any(abs(gp[r] - w) <= w * (2.0 ** -24 + 2.0 ** -40) + V * 2.0 ** -43 for w in want[int(got[r])]), (r, gp[r], want)
    assert prob or (gp == -9).all()
    ref.free(hold + [f for f in form if f] + [tok, pr])
    return got


def rows(T, V, seed=0, spread=2.5):
    rng = np.random.default_rng(seed)
    x = rng.standard_normal((T, V)) * spread
    x += (rng.random((T, V)) < 0.003) * rng.exponential(3.0, (T, V))
    x[rng.random((T, V)) < 0.02] = -np.inf
    return x.astype(np.float32)


CUTS = [dict(), dict(k=1), dict(k=50), dict(k=512), dict(k=513), dict(k=960), dict(k=960, p=0.8), dict(k=961), dict(k=961, p=0.8), dict(k=3000), dict(p=0.9), dict(p=0.3), dict(q=0.05), dict(k=40, p=0.95), dict(k=40, p=0.95, q=0.02), dict(k=2000, p=0.7),
        dict(k=900, p=0.999, q=0.001), dict(p=0.97, q=0.01), dict(t=0.0), dict(t=0.2, p=0.9), dict(t=3.0, k=700), dict(t=0.7, k=20, p=0.8, q=0.1)]


@pytest.mark.parametrize("V", [1, 2, 3, 5, 63, 1000, 1023, 4096, 8191, 32001, 50257])
@pytest.mark.parametrize("cut", range(len(CUTS)))
def test_cuts(eng, V, cut):
    check(eng, rows(9, V, seed=V + cut), seed=cut, **CUTS[cut])


def test_large_vocabularies(eng):
    for V in (151936, 262147, 1 << 20):
        for c in (dict(k=50, p=0.9), dict(p=0.95), dict(), dict(k=5000, p=0.9), dict(t=1.5, q=0.001)):
            check(eng, rows(2, V, seed=V), seed=V, **c)


def test_each_row_on_its_own(eng):
    """Other parameters in every row: greedy, cut in every way, not at all, and parameters that are none."""
    rng = np.random.default_rng(3)
    T = 120
    t = rng.choice([0.0, -1.0, np.nan, 0.3, 1.0, 1.7, np.inf, 1e-30, 1e-44], T)
    k = rng.choice([0, -5, 1, 7, 100, 512, 600, 5000, 2 ** 31 - 1, -2 ** 31], T)
    p = rng.choice([1.0, 0.0, -1.0, np.nan, 0.5, 0.9, 0.9999, 7.0, 1e-20, -np.inf], T)
    q = rng.choice([0.0, -1.0, np.nan, 0.01, 0.5, 1.0, 3.0], T)
    u = rng.choice([0.0, 0.5, 0.999999, 1.0 - 2.0 ** -24, 0.123, -1.0, np.nan, 1.0, 2.0, np.inf], T).astype(np.float32)
    check(eng, rows(T, 6001, seed=4), t, k, p, q, np.where(u >= 1, np.float32(1.0), u))
    a = check(eng, rows(T, 6001, seed=4), t, k, p, q, u, prob=False)
    assert (a >= 0).all()


def test_draws_walk_through_the_row(eng):
    """Every token of a row in turn, by draws on both sides of each border."""
    x = rows(1, 40, seed=7)
    order, w = kept(x[0], 0.9, 25, 0.97, 0.01)
    edge = np.cumsum(w)[:-1] / w.sum()
    u = np.sort(np.concatenate([[0.0], edge - 1e-5, edge + 1e-5])).astype(np.float32)
    got = check(eng, np.repeat(x, u.size, 0), 0.9, 25, 0.97, 0.01, u)
    assert (np.diff(got) >= 0).all() and set(got) == set(order)


def test_equal_logits(eng):
    """Ties at the cut: the lower indices stay.  Whole rows of one value, values of few bits, more equals than a work-group's memory takes."""
    for V in (100, 9000, 40000):
        x = np.zeros((6, V), np.float32)
        x[1] = -3.5
        x[2, ::2] = 1.0
        x[3] = np.float32(1e30)
        x[4, V // 2:] = -np.inf
        x[5, 1::2] = -0.0
        for c in (dict(k=10), dict(k=V // 2), dict(p=0.25), dict(k=V - 1, p=0.5), dict(), dict(q=1.0), dict(k=600, p=0.9)):
            check(eng, x, **c)
    rng = np.random.default_rng(5)
    x = (np.round(rng.standard_normal((8, 30000)) * 2) / 2).astype(np.float32)      # (a few dozen values)
    for c in (dict(k=300), dict(k=7000), dict(p=0.6), dict(k=20000, p=0.9), dict(t=30.0, p=0.5), dict(t=30.0, k=11111, p=0.5, q=0.99)):
        check(eng, x, **c)
    y = rows(4, 30000, seed=1)
    for c in (dict(t=1000.0, p=0.5), dict(t=1000.0, k=9999), dict(t=1000.0, k=9999, p=0.123)):    # (one bin holds all)
        check(eng, y, **c)


def test_tokens_side_by_side(eng):
    """The likely ones all in one place of the row, more of them than a wave's share of the list."""
    x = rows(4, 50000, seed=9)
    x[:, :2000] = np.abs(x[:, :2000]) + 9
    x[1, 49000:] = x[1, :1000]
    x[2, :] = x[2, ::-1]
    for c in (dict(k=400), dict(k=512, p=0.9), dict(k=1900), dict(p=0.9), dict(t=20.0, k=1500, p=0.5)):
        check(eng, x, **c)


def test_what_is_no_number(eng):
    x = rows(10, 3000, seed=2)
    x[0, ::3] = np.nan
    x[1] = np.nan
    x[2] = -np.inf
    x[3, 5] = x[3, 700] = x[3, 2999] = np.inf
    x[4] = -np.inf
    x[4, 1234] = -3e38
    x[5, 0] = 3.4e38
    x[6] = -3.4e38
    x[6, 9] = 3.4e38
    x[7, :] = np.inf
    x[8, 1::2] = np.nan
    x[8, 0::2] = -np.inf
    x[9] *= 1e-42
    for c in (dict(), dict(k=2), dict(k=700), dict(p=0.5), dict(k=5, p=0.9, q=0.5), dict(t=0.0), dict(k=1000, p=0.1)):
        got = check(eng, x, **c)
        assert got[1] == got[2] == got[8] == -1 and got[3] in (5, 700, 2999) and got[4] == 1234


@pytest.mark.parametrize("off,ld", [(0, 5000), (1, 5001), (2, 5003), (3, 4999), (900, 6002)])
def test_columns_and_strides(eng, off, ld):
    x = rows(7, 4099 if ld > 4990 else 4000, seed=ld)
    for c in (dict(), dict(k=30, p=0.9), dict(p=0.9), dict(k=800)):
        check(eng, x[:, :ld - off] if x.shape[1] + off > ld else x, ld=ld, off=off, **c)


def test_many_rows_and_the_same_again(eng):
    x = rows(700, 257, seed=1)
    a = check(eng, x, k=13, p=0.9, seed=5)
    assert np.array_equal(a, check(eng, x, k=13, p=0.9, seed=5))
    # a row's token does not hang on the rows beside it
    b = np.concatenate([check(eng, x[i:i + 350], k=13, p=0.9, u=np.random.default_rng(5).random(700).astype(np.float32)[i:i + 350]) for i in (0, 350)])
    assert np.array_equal(a, b)


def test_frequencies(eng):
    """Tokens come as often as their weights say: 200 thousand draws, each count within six standard deviations."""
    x = np.array([[0.0, 1.0, -1.0, 2.0, 0.5, -np.inf, 1.0, -4.0]], np.float32)
    T = 200000
    hold = [az.Runtime.from_numpy(np.repeat(x, T, 0)), az.Runtime.from_numpy(np.random.default_rng(1).random(T).astype(np.float32)), az.Runtime.alloc(4 * T)]
    for form, par in (((None,) * 4, (1.0, 0, 1.0, 0.0)), ((None, 4, None, None), (1.0, 4, 1.0, 0.0)), ((2.0, None, 0.8, None), (2.0, 0, 0.8, 0.0))):
        f = [None if a is None else az.Runtime.from_numpy(np.full(T, a, np.int32 if i == 1 else np.float32)) for i, a in enumerate(form)]
        eng.sample(hold[0], 8, 0, 8, T, az.Sampling(*f), hold[1], hold[2])
        n = np.bincount(hold[2].read(np.int32), minlength=8)
        order, w = kept(x[0], *[np.float32(v) if i != 1 else v for i, v in enumerate(par)])
        pr = np.zeros(8)
        pr[order] = w / w.sum()
        assert (np.abs(n - T * pr) <= 6 * np.sqrt(T * pr * (1 - pr))).all(), (n, T * pr)
        ref.free([m for m in f if m])
    ref.free(hold)


def test_in_a_launch_list(eng):
    x = [rows(5, 20011, seed=s) for s in range(3)]
    b = [az.Runtime.alloc(x[0].nbytes)] + [az.Runtime.alloc(64) for _ in range(6)]
    form = az.Sampling(b[1], b[2], b[3], None)

    def put(i):
        rng = np.random.default_rng(i)
        for m, a in zip(b, (x[i], rng.random(5).astype(np.float32) + 0.5, np.array([0, 3, 50, 600, 9000], np.int32)[rng.permutation(5)], rng.random(5).astype(np.float32), rng.random(5).astype(np.float32))):
            m.write(a)
        b[5].fill(0xFFFFFFFF)

    def call():
        eng.sample(b[0], 20011, 0, 20011, 5, form, b[4], b[5], b[6])
    put(0)
    l = az.Runtime.record(call)
    assert l.launches in (1, 4)
    for i in (0, 1, 2, 1):
        put(i)
        call()
        want = b[5].read(np.int32, 5), b[6].read(np.uint32, 5)
        put(i)
        l.run()
        assert np.array_equal(b[5].read(np.int32, 5), want[0]) and np.array_equal(b[6].read(np.uint32, 5), want[1])
    l.free()
    ref.free(b)


@pytest.mark.parametrize("T,V,launches", [(1, 48000, 4), (16, 48000, 4), (16, 47999, 1), (17, 51000, 4), (17, 50999, 1), (1, 2, 1)])
def test_the_work_groups_of_a_row(T, V, launches):
    """By the sizes; a first call of few long rows needs room, which no list being recorded can make."""
    e = az.Engine(16, 256)
    x = rows(T, V, seed=3)
    b = [az.Runtime.from_numpy(x), az.Runtime.from_numpy(np.full(T, 0.37, np.float32)), az.Runtime.alloc(4 * T)]
    f = az.Sampling(None, None, None, None)

    def call():
        e.sample(b[0], V, 0, V, T, f, b[1], b[2], None)
    if launches > 1:
        with pytest.raises(az.ArczError):
            az.Runtime.record(call)
    check(e, x, t=0.8, p=0.9, seed=5)
    n = az.lib.arcz_launch_count()
    call()
    assert az.lib.arcz_launch_count() - n == launches
    l = az.Runtime.record(call)
    assert l.launches == launches
    want = b[2].read(np.int32)
    for _ in range(3):
        b[2].fill(0)
        l.run()
        assert np.array_equal(b[2].read(np.int32), want)
    l.free()
    ref.free(b)
    e.close()


def test_refusals(eng):
    x, u, tok, pr, small = (az.Runtime.alloc(n) for n in (4 * 8 * 128, 32, 32, 32, 64))
    short = small.view(0, 28)
    for m in (x, u):
        m.fill(0)
    n = az.lib.arcz_launch_count()
    none = az.Sampling()

    def refused(logits=x, ld=128, off=0, V=128, T=8, form=none, u=u, token=tok, prob=pr):
        with pytest.raises(az.ArczError):
            eng.sample(logits, ld, off, V, T, form, u, token, prob)
    refused(V=0)
    refused(V=-1)
    refused(V=(1 << 20) + 1, ld=1 << 21)
    refused(V=129)
    refused(off=1)
    refused(off=-1)
    refused(T=-1)
    refused(T=9)
    refused(u=short)
    refused(token=short)
    refused(prob=short)
    for i in range(4):
        refused(form=az.Sampling(*[short if j == i else None for j in range(4)]))
    refused(prob=tok)
    refused(token=u)
    refused(form=az.Sampling(tok))
    view = x.view(0, 32)
    refused(token=view)
    refused(prob=view)
    assert az.lib.arcz_engine_sample(eng.h, x.h, 128, 0, 128, 8, None, u.h, tok.h, None) == -100
    assert az.lib.arcz_engine_sample(eng.h, None, 128, 0, 128, 8, none.at, u.h, tok.h, None) == -100
    assert az.lib.arcz_engine_sample(eng.h, x.h, 128, 0, 128, 8, none.at, None, tok.h, None) == -100
    assert az.lib.arcz_engine_sample(eng.h, x.h, 128, 0, 128, 8, none.at, u.h, None, None) == -100
    eng.sample(x, 128, 0, 128, 0, none, u, tok, pr)
    assert az.lib.arcz_launch_count() == n
    ref.free([x, small, u, tok, pr, short, view])


@pytest.fixture
def two():
    e = []
    for split in ("0", "1"):
        os.environ["ARCZ_SAMPLE_SPLIT"] = split
        e.append(az.Engine(16, 256))
        del os.environ["ARCZ_SAMPLE_SPLIT"]
    yield e
    for x in e:
        x.close()


@pytest.mark.parametrize("V,off,ld", [(60001, 0, 60001), (151936, 3, 151940), (2049, 1, 2051), (63, 0, 64), (1, 0, 1)])
def test_one_work_group_and_sixteen_give_the_same_bits(rt, two, V, off, ld):
    """Sums of whole numbers: which work-group adds them does not matter."""
    T, rng = 24, np.random.default_rng(V)
    x = np.zeros((T, ld), np.float32)
    x[:, off:off + V] = rows(T, V, seed=2)
    x[5, off:off + V] = 1.25                                     # (all equal)
    x[6, off:off + V] = np.round(x[6, off:off + V])              # (many equal)
    x[7, off:off + V] = -np.inf
    x[8, off + V // 2] = np.inf
    given = [np.array(rng.choice(a, T), d) for a, d in (([0.0, 0.3, 1.0, 1.7, 40.0], np.float32), ([0, 1, 50, 300, 960, 961, 5000], np.int32), ([1.0, 0.95, 0.5, 0.01], np.float32),
                                                        ([0.0, 0.001, 0.2], np.float32))]
    hold = [az.Runtime.from_numpy(a) for a in (x, rng.random(T).astype(np.float32), *given)]
    got = []
    for e in two:
        out = [az.Runtime.from_numpy(np.full(T, -9, np.int32)) for _ in range(2)]
        e.sample(hold[0], ld, off, V, T, az.Sampling(*hold[2:]), hold[1], *out)
        got.append([o.read(np.int32) for o in out])
        ref.free(out)
    assert np.array_equal(got[0], got[1])
    ref.free(hold)


def test_lists_that_share_the_engines_room(rt):
    """Keys shared out and rows in sixteen parts go through one room: recorded lists of both, replayed in turn with eager calls between them."""
    eng, V, hold = az.Engine(16, 256), 50000, []
    c = ref.Cache(40, 128, 64, 2, 128, seed=4)
    kv = ref.device_cache(eng, c, hold)
    rng = np.random.default_rng(6)
    dev = {n: az.Runtime.from_numpy(a) for n, a in dict(rows=np.arange(3, dtype=np.int32), len=np.array([4900, 120], np.int32), table=rng.permutation(80).astype(np.int32) % 40,
                                                       q=rng.standard_normal((2, 8 * 128)).astype(np.float32), out=np.zeros((2, 8 * 128), np.float32), x=rows(3, V, seed=8),
                                                       u=np.array([0.1, 0.5, 0.9], np.float32), p=np.array([0.9, 1.0, 0.4], np.float32), token=np.zeros(3, np.int32)).items()}
    batch, form, how = az.KvBatch(dev["rows"], dev["len"], dev["table"], 2, 40, 2, 1, 4900), az.Attention(0.1), az.Sampling(top_p=dev["p"])

    def attend():
        eng.attention(kv, batch, dev["q"], 8 * 128, 0, 8, dev["out"], 8 * 128, 0, form)

    def draw():
        eng.sample(dev["x"], V, 0, V, 3, how, dev["u"], dev["token"])
    calls, outs = (attend, draw), ("out", "token")
    for f in calls:
        f()
    want = [dev[n].read(np.uint32) for n in outs]
    lists = [az.Runtime.record(f) for f in calls]
    assert lists[1].launches == 4
    for i in range(3):
        for j in ((0, 1), (1, 0), (1, 1))[i]:
            dev[outs[j]].fill(0)
            dev[outs[1 - j]].fill(0)
            lists[j].run()
            calls[1 - j]()
            assert all(np.array_equal(dev[n].read(np.uint32), w) for n, w in zip(outs, want))
    for l in lists:
        l.free()
    ref.free(hold + list(dev.values()))
    eng.close()
