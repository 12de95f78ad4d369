"""Attention over the 8-bit cache on the GPU against 64 bits (attn_ref.attention, which derives the tolerance of each value)."""
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


def run(eng, c, b, q, ldq, q_off, heads, form, hold, ldo=None, o_off=0):
    """(out [T][heads][hd], the whole output buffer)"""
    w = heads * c.hd
    ldo = ldo or w
    kv = ref.device_cache(eng, c, hold)
    qb, ob = az.Runtime.from_numpy(q), az.Runtime.from_numpy(np.full((b.T, ldo), 7.5, np.float32))
    hold += [qb, ob]
    parts = {k: None if form.get(k) is None else az.Runtime.from_numpy(np.ascontiguousarray(form[k], t)) for k, t in
             (("slopes", np.float32), ("prefix", np.int32), ("first", np.int32))}
    hold += [p for p in parts.values() if p]
    a = az.Attention(form["scale"], form.get("cap", 0.0), form.get("window", 0), **parts)
    eng.attention(kv, b.device(hold), qb, ldq, q_off, heads, ob, ldo, o_off, a)
    y = ob.read(np.float32, b.T * ldo).reshape(b.T, ldo)
    return y[:, o_off:o_off + w].reshape(b.T, heads, c.hd), y


def check(eng, seqs, heads, kv, hd, page, block, form=None, q_std=1.3, ld_pad=0, off=0, seed=0, T=None, c=None, b=None, q=None, max_rows=None, only=None):
    print(f"attention seqs={seqs} heads={heads}/{kv} hd={hd} page={page} block={block} form={sorted((form or {}).items(), key=str)}"[:300], flush=True)
    b = b or ref.Batch(seqs, page, seed=seed + page, T=T, max_rows=max_rows)
    c = c or ref.Cache(b.pages, page, block, kv, hd, seed=seed + 3)
    form = dict(form or {})
    form.setdefault("scale", hd ** -0.5)
    w = heads * hd
    ld = w + ld_pad
    if q is None:
        q = np.random.default_rng(seed + 9).standard_normal((b.T, ld)).astype(np.float32) * np.float32(q_std)
    hold = []
    got, whole = run(eng, c, b, q, ld, off, heads, form, hold, ldo=w + ld_pad, o_off=off)
    ref.free(hold)
    want, tol, done = ref.attention(c, q[:, off:off + w].reshape(b.T, heads, hd), b.rows, b.lens, b.table, max_rows=b.max_rows, only=only, **form)
    d = np.abs(got - want)[done]
    assert np.array_equal(np.isnan(got[done]), np.isnan(want[done]))
    bad = ~(d <= tol[done]) & ~np.isnan(want[done])
    assert not bad.any(), (int(bad.sum()), float(np.nanmax(d / np.maximum(tol[done], 1e-30))), float(np.nanmax(d)))
    if only is None and not done.all():
        assert (got[~done] == 7.5).all()
    rest = np.ones(w + ld_pad, bool)
    rest[off:off + w] = False
    assert (whole[:, rest] == 7.5).all()
    return got


# tokens of each sequence and keys in front of them: single tokens (one key, ends inside and at a tile), drafts, prompts, nothing
ONE = [(1, 1), (1, 15), (1, 16), (1, 33), (1, 100), (1, 257), (1, 700)]


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("heads,kv", [(1, 1), (4, 1), (5, 1), (8, 1), (12, 1), (16, 1), (24, 1), (32, 1), (8, 2), (14, 2)])
def test_single_tokens(eng, hd, heads, kv):
    check(eng, ONE, heads, kv, hd, 64, 64)


@pytest.mark.parametrize("page,block", [(16, 16), (16, 1), (32, 2), (32, 32), (64, 4), (128, 128), (128, 1), (256, 64)])
@pytest.mark.parametrize("seqs", [ONE, [(3, 3), (4, 300), (2, 2)], [(40, 40), (33, 210), (1, 90), (17, 17)]])
def test_pages_and_blocks(eng, page, block, seqs):
    check(eng, seqs, 8, 2, 128, page, block)


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("seqs,heads,kv", [([(2, 2), (7, 130), (1, 64)], 4, 1), ([(40, 40)], 4, 1), ([(129, 300), (1, 1), (64, 65), (0, 5)], 2, 1),
                                           ([(33, 190)], 5, 1), ([(70, 70), (9, 400)], 14, 2), ([(150, 150)], 3, 3)])
def test_chunks(eng, hd, seqs, heads, kv):
    check(eng, seqs, heads, kv, hd, 32, 16)


FORMS = {
    "cap": dict(cap=20.0),
    "cap_small": dict(cap=0.5),
    "window": dict(window=37),
    "window_1": dict(window=1),
    "cap_window": dict(cap=30.0, window=64),
    "distance": dict(slopes=2.0 ** -np.arange(1, 9)),
    "cap_distance": dict(cap=15.0, slopes=0.1 * np.arange(8)),
    "scale": dict(scale=0.31),
    "negative_scale": dict(scale=-0.1),
}


@pytest.mark.parametrize("form", sorted(FORMS))
@pytest.mark.parametrize("seqs", [[(1, 200), (1, 1), (2, 90)], [(60, 60), (35, 180), (1, 70)]])
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_forms(eng, form, seqs, hd):
    check(eng, seqs, 8, 2, hd, 64, 16, FORMS[form])


@pytest.mark.parametrize("seqs", [[(1, 90), (2, 33), (3, 3)], [(60, 100), (35, 35), (9, 200)]])
@pytest.mark.parametrize("window", [0, 20])
def test_prefix_and_documents(eng, seqs, window):
    """Prefixes that end behind some rows; documents that begin between rows; rows that see nothing (zeros)."""
    n = sum(r for r, _ in seqs)
    rng = np.random.default_rng(1)
    check(eng, seqs, 8, 2, 128, 32, 32, dict(prefix=[20, 300, 3], window=window))
    check(eng, seqs, 8, 2, 128, 32, 32, dict(prefix=[-5, 0, 2 ** 31 - 1], window=window))
    check(eng, seqs, 8, 2, 128, 32, 32, dict(first=rng.integers(-3, 60, size=n), window=window))
    check(eng, seqs, 8, 2, 128, 32, 32, dict(first=np.full(n, 2 ** 31 - 1), window=window))
    check(eng, seqs, 8, 2, 128, 32, 32, dict(first=rng.integers(0, 40, size=n), prefix=[50, 10, 80], window=window, cap=10.0))


@pytest.mark.parametrize("seqs", [[(1, 60), (2, 40)], [(50, 90), (40, 40)]])
def test_columns_and_strides(eng, seqs):
    for pad, off in ((64, 0), (64, 32), (13, 5), (4, 3)):
        check(eng, seqs, 4, 2, 64, 16, 16, ld_pad=pad, off=off)


@pytest.mark.parametrize("seqs", [[(1, 60), (3, 2), (1, 0)], [(50, 40), (40, 300)]])
def test_rows_before_position_0_rows_past_the_sequences(eng, seqs):
    """More rows than keys: the first ones have no position and no key (zeros); rows of no sequence stay as they are."""
    check(eng, seqs, 4, 2, 128, 16, 16, T=sum(n for n, _ in seqs) + 7)
    check(eng, seqs, 4, 2, 128, 16, 16, max_rows=2)


@pytest.mark.parametrize("seqs", [[(1, 190), (2, 70)], [(64, 190), (40, 70)]])
def test_pages_that_are_none(eng, seqs):
    """Keys on a page outside the cache are not seen; lengths past the table are cut; rows that fall hold none."""
    b = ref.Batch(seqs, 32, seed=2)
    b.table[0, 1], b.table[1, 2] = -1, b.pages
    check(eng, seqs, 8, 2, 128, 32, 16, b=b)
    b.table[0, :], b.table[1, :] = 2 ** 31 - 1, -2 ** 31
    got = check(eng, seqs, 8, 2, 128, 32, 16, b=b)
    assert not got.any()
    b = ref.Batch(seqs, 32, seed=2, tail_page=0)
    c = ref.Cache(b.pages, 32, 16, 2, 128, seed=3)
    q = np.random.default_rng(4).standard_normal((b.T, 8 * 128)).astype(np.float32)
    hold = []
    b.lens[0] = b.ldt * 32
    want, _ = run(eng, c, b, q, 1024, 0, 8, dict(scale=0.1), hold)
    b.lens[0] = 2 ** 31 - 1
    got, _ = run(eng, c, b, q, 1024, 0, 8, dict(scale=0.1), hold)
    assert np.array_equal(got, want)
    b.rows[:] = [2 ** 31 - 1, -5, -9]
    got, _ = run(eng, c, b, q, 1024, 0, 8, dict(scale=0.1), hold)
    assert (got == 7.5).all()
    ref.free(hold)


@pytest.mark.parametrize("seqs", [[(1, 100), (1, 30)], [(70, 100), (30, 30)]])
def test_what_is_masked_has_no_effect(eng, seqs):
    """NaN and infinite scales behind the last key, before a window, before a document: the same bits as with ordinary ones."""
    page = block = 16
    b = ref.Batch(seqs, page, seed=2)
    c = ref.Cache(b.pages, page, block, 2, 128, seed=3)
    for form, spoil in ((dict(), [(0, 7), (1, 2)]), (dict(window=30 if seqs[0][0] == 1 else 20), [(0, 0)]), (dict(first=np.full(b.T, 20)), [(0, 0), (1, 0)])):
        form = dict(form, scale=0.09)
        q = np.random.default_rng(4).standard_normal((b.T, 8 * 128)).astype(np.float32)
        hold = []
        want, _ = run(eng, c, b, q, 1024, 0, 8, form, hold)
        # (rows near the beginning of the first sequence see its spoiled first page through the window: not compared)
        blind = np.ones(b.T, bool)
        if form.get("window"):
            blind[:seqs[0][0]] = seqs[0][1] - seqs[0][0] + np.arange(seqs[0][0]) - form["window"] + 1 >= page
        assert blind.sum() > b.T // 2
        for bad in (np.nan, np.inf, -1.0, 3e38):
            x = ref.Cache(b.pages, page, block, 2, 128, seed=3)
            for s, i in spoil:
                if b.table[s, i] >= 0:
                    x.d[:, b.table[s, i]] = bad
                    x.q[:, b.table[s, i]] = -128
            got, _ = run(eng, x, b, q, 1024, 0, 8, form, hold)
            assert np.array_equal(got[blind], want[blind]), (form, bad)
        ref.free(hold)


@pytest.mark.parametrize("seqs", [[(1, 100), (1, 30)], [(70, 100), (30, 30)]])
def test_nan_where_it_is_seen(eng, seqs):
    """A block whose scale is NaN makes the rows that see it NaN, and no other; so does a row of NaN, its own."""
    page = block = 16
    b = ref.Batch(seqs, page, seed=2)
    for which in (0, 1):
        c = ref.Cache(b.pages, page, block, 2, 128, seed=3)
        c.d[which, b.table[0, 2], 1] = np.nan
        check(eng, seqs, 8, 2, 128, page, block, b=b, c=c)
    c = ref.Cache(b.pages, page, block, 2, 128, seed=3)
    q = np.random.default_rng(4).standard_normal((b.T, 1024)).astype(np.float32)
    q[0, 130] = np.nan
    q[b.T - 1, 1023] = np.nan
    check(eng, seqs, 8, 2, 128, page, block, b=b, c=c, q=q)


@pytest.mark.parametrize("seqs", [[(1, 400), (1, 30)], [(70, 400), (30, 30)]])
@pytest.mark.parametrize("kind", ["zero_blocks", "all_zero", "wide", "tiny", "huge", "first_zero"])
def test_scales_of_every_size(eng, seqs, kind):
    """Blocks of zeros, scales that differ by 2^24, all tiny, all huge: a weight carries its block's scale."""
    page, block = 32, 8
    b = ref.Batch(seqs, page, seed=2)
    c = ref.Cache(b.pages, page, block, 2, 128, seed=3)
    rng = np.random.default_rng(8)
    if kind == "zero_blocks":
        z = rng.random(c.d[1].shape) < 0.4
        c.d[1][z] = 0.0
    if kind == "first_zero":
        c.d[1][:] *= np.float32(2.0 ** -30)
        for s in range(len(seqs)):
            c.d[1][b.table[s, 0]] = 0.0
    if kind == "all_zero":
        c.d[1][:] = 0.0
    c.q[1].reshape(c.d[1].shape + (block, 128))[c.d[1] == 0.0] = 0      # (as kv_write stores such a block)
    if kind == "wide":
        c.d[1][:] *= 2.0 ** rng.integers(-12, 13, size=c.d[1].shape)
    if kind == "tiny":
        c.d[1][:] *= np.float32(2.0 ** -90)
    if kind == "huge":
        c.d[1][:] *= np.float32(2.0 ** 90)
    check(eng, seqs, 8, 2, 128, page, block, b=b, c=c)


@pytest.mark.parametrize("seqs", [[(1, 400), (1, 330)], [(70, 400), (30, 330)]])
@pytest.mark.parametrize("block", [1, 8, 32])
def test_zero_blocks_behind_an_outlier(eng, seqs, block):
    """Blocks of zeros behind keys of huge scales that hardly count or are not seen: the other keys' weights stay what they are."""
    page = 32
    b = ref.Batch(seqs, page, seed=2)
    rng = np.random.default_rng(8)

    def cache(scale):
        c = ref.Cache(b.pages, page, block, 2, 128, seed=3)
        c.d[1][rng.random(c.d[1].shape) < 0.4] = 0.0
        for s in range(len(seqs)):
            c.d[1][b.table[s, :4]] = scale
        c.q[1].reshape(c.d[1].shape + (block, 128))[c.d[1] == 0.0] = 0
        return c
    # (the row's own distance: 2^60 e^-140 and less of the others' weights)
    check(eng, seqs, 8, 2, 128, page, block, dict(slopes=np.ones(8)), b=b, c=cache(2.0 ** 60))
    first = np.full(b.T, 4 * page + 3)
    for huge in (2.0 ** 60, 3e38, np.inf):
        c = cache(huge)
        want = ref.Cache(b.pages, page, block, 2, 128, seed=3)
        want.q, want.d = c.q.copy(), c.d.copy()
        for s in range(len(seqs)):
            want.d[1][b.table[s, :5]] = 0.0
            c.d[1][b.table[s, 4]] = huge
        for f in (dict(first=first + page - 3), dict(first=np.full(b.T, 5 * page - 1))):
            if f["first"][0] == 5 * page - 1:     # (the last key of the spoiled page is seen: as zeros in both)
                for x in (c, want):
                    for s in range(len(seqs)):
                        x.d[1][b.table[s, 4], :, -1] = 0.0
                        x.q[1][b.table[s, 4], :, -block:] = 0
            f = dict(f, scale=0.09)
            q = np.random.default_rng(4).standard_normal((b.T, 1024)).astype(np.float32)
            hold = []
            a, _ = run(eng, want, b, q, 1024, 0, 8, f, hold)
            g, _ = run(eng, c, b, q, 1024, 0, 8, f, hold)
            assert np.array_equal(a, g)
            ref.free(hold)


@pytest.mark.parametrize("seqs", [[(1, 300), (2, 40)], [(70, 300), (30, 30)]])
@pytest.mark.parametrize("q_std", [0.0, 1e-6, 40.0, 1e3, 1e-30, 1e30])
def test_rows_of_every_size(eng, seqs, q_std):
    """Flat and one-hot weights; rows near the ends of f32 (with a scale that brings their scores back)."""
    form = dict(scale=0.09 / q_std if q_std in (1e-30, 1e30) else 0.09)
    check(eng, seqs, 8, 2, 128, 32, 8, form, q_std=q_std)


def test_rows_of_different_sizes_in_one_tile(eng):
    q = np.random.default_rng(4).standard_normal((64, 1024)).astype(np.float32)
    q[::3] *= np.float32(2.0 ** -14)
    q[1] = 0.0
    check(eng, [(64, 200)], 8, 2, 128, 32, 8, q=q)
    check(eng, [(2, 200)], 8, 2, 128, 32, 8, q=q[:2])


@pytest.mark.parametrize("rows", [1, 2, 9, 40])
def test_long_sequences_are_shared_out(eng, rows):
    """Keys in pieces, joined; most of the mass in one piece, or in none more than in another."""
    seqs = [(rows, 5003)]
    check(eng, seqs, 8, 2, 128, 256, 32, q_std=0.3)
    check(eng, seqs, 8, 2, 128, 256, 32, q_std=6.0)
    check(eng, seqs, 8, 2, 128, 256, 32, dict(window=3000), q_std=0.3)
    check(eng, seqs, 8, 2, 128, 256, 32, dict(first=np.full(rows, 4990)), q_std=0.3)
    check(eng, [(rows, 5003), (rows, rows), (1, 800)], 8, 2, 64, 16, 16)


@pytest.mark.parametrize("page,block", [(64, 64), (32, 32), (16, 4)])
@pytest.mark.parametrize("form", ["plain", "cap", "distance", "window", "prefix"])
def test_many_rows_over_thousands_of_keys(eng, page, block, form):
    """Rows from 1024 on that see 2000 keys and more: work-groups of eight waves, here with the last one not full and a sequence that is short;
    rows at the seams of waves and work-groups, and some between."""
    seqs = [(300, 4100), (9, 130), (41, 41)]
    f = dict(plain={}, cap=dict(cap=12.0), distance=dict(slopes=2.0 ** -np.arange(1.0, 9)), window=dict(window=2100), prefix=dict(prefix=[4000, 0, 41]))[form]
    rng = np.random.default_rng(3)
    only = {0, 1, 7, 8, 15, 16, 63, 64, 65, 127, 128, 191, 192, 255, 256, 299, 300, 308, 309, 349} | set(rng.integers(0, 350, size=6).tolist())
    check(eng, seqs, 8, 2, 128, page, block, f, only=only)


def test_far_pages(eng):
    """Pages behind 2^32 bytes of keys."""
    page, heads, hd = 256, 8, 128
    pages = (1 << 32) // (page * heads * hd) + 4
    c = ref.Cache(3, page, 16, heads, hd, seed=1)
    far = [pages - 1, 1, pages - 2]
    for rows in (1, 40):
        b = ref.Batch([(rows, 700)], page, seed=1)
        b.table[0, :3] = [0, 1, 2]
        b.pages = 3
        q = np.random.default_rng(4).standard_normal((rows, heads * hd)).astype(np.float32)
        hold = []
        want, _ = run(eng, c, b, q, heads * hd, 0, heads, dict(scale=0.09), hold)
        kv = eng.make_kv(pages, page, 16, heads, hd)
        hold.append(kv)
        for i, pg in enumerate(far):
            for j in range(4):
                a = (c.q[0], c.q[1], c.d[0], c.d[1])[j][i]
                kv.buffer(j).write(a, offset=pg * a.nbytes)
        b.table[0, :3] = far
        qb, ob = az.Runtime.from_numpy(q), az.Runtime.alloc(q.nbytes)
        hold += [qb, ob]
        eng.attention(kv, b.device(hold), qb, heads * hd, 0, heads, ob, heads * hd, 0, az.Attention(0.09))
        assert np.array_equal(ob.read(np.float32, q.size).reshape(want.shape), want)
        ref.free(hold)


@pytest.mark.parametrize("rows", [1, 2, 40])
@pytest.mark.parametrize("form", ["first", "window"])
def test_the_last_positions_there_are(eng, rows, form):
    """The end of the longest sequence that a table can name: what a row sees there is what it would see at the end of a short one."""
    page, seen, long = 256, 300, 0x7FFFF000
    b = ref.Batch([(rows, 3 * page)], page, seed=1, ld_extra=0)
    c = ref.Cache(b.pages, page, 32, 2, 128, seed=3)
    q = np.random.default_rng(4).standard_normal((rows, 1024)).astype(np.float32)
    f = dict(scale=0.09, window=seen) if form == "window" else dict(scale=0.09, first=np.full(rows, 3 * page - seen))
    want, tol, _ = ref.attention(c, q.reshape(rows, 8, 128), b.rows, b.lens, b.table, **f)
    tail, b.table = b.table, np.full((1, long // page), -1, np.int32)
    b.table[0, -3:] = tail
    b.ldt, b.lens, b.max_len = long // page, np.array([long], np.int32), long
    if form == "first":
        f["first"] = np.full(rows, long - seen)
    hold = []
    got, _ = run(eng, c, b, q, 1024, 0, 8, f, hold)
    assert (np.abs(got - want) <= tol).all()
    ref.free(hold)


@pytest.mark.parametrize("seqs", [[(1, 900), (1, 33)], [(70, 300), (30, 30)]])
def test_same_bits_again_and_in_another_batch(eng, seqs):
    """The same call gives the same bits; so does the first sequence's call with other pages in another order."""
    b = ref.Batch(seqs, 32, seed=2)
    c = ref.Cache(b.pages, 32, 8, 2, 128, seed=3)
    q = np.random.default_rng(4).standard_normal((b.T, 1024)).astype(np.float32)
    hold = []
    one, _ = run(eng, c, b, q, 1024, 0, 8, dict(scale=0.09), hold)
    two, _ = run(eng, c, b, q, 1024, 0, 8, dict(scale=0.09), hold)
    assert np.array_equal(one, two)
    turn = np.arange(b.pages)[::-1].copy()
    x = ref.Cache(b.pages, 32, 8, 2, 128, zeros=True)
    x.q[:, turn], x.d[:, turn] = c.q, c.d
    b.table = np.where(b.table >= 0, turn[np.maximum(b.table, 0)], -1).astype(np.int32)
    three, _ = run(eng, x, b, q, 1024, 0, 8, dict(scale=0.09), hold)
    assert np.array_equal(one, three)
    ref.free(hold)


def test_caps_that_are_refused(eng):
    """A cap's part of a score is formed in f32."""
    kv = eng.make_kv(2, 16, 16, 2, 64)
    i = az.Runtime.from_numpy(np.zeros(8, np.int32))
    x, y = az.Runtime.alloc(4 * 256), az.Runtime.alloc(4 * 256)
    for cap in (1e-38, 1e-45, 2.0 ** 101, 3e38):
        with pytest.raises(az.ArczError):
            eng.attention(kv, az.KvBatch(i, i, i, 1, 2, 1, 1), x, 256, 0, 4, y, 256, 0, az.Attention(0.1, cap=cap))
    for b in (kv, i, x, y):
        b.free()


@pytest.mark.parametrize("cap", [2.0 ** -100, 1e-6, 1e12, 2.0 ** 100])
def test_smallest_and_largest_caps(eng, cap):
    check(eng, [(1, 90), (40, 60)], 4, 2, 64, 16, 16, dict(cap=cap))
    check(eng, [(1, 90), (2, 60)], 4, 2, 64, 16, 16, dict(cap=cap))


def test_refusals(eng):
    kv = eng.make_kv(2, 16, 16, 2, 64)
    i = az.Runtime.from_numpy(np.zeros(8, np.int32))
    x, y = az.Runtime.alloc(4 * 4 * 512), az.Runtime.alloc(4 * 4 * 512)
    ok = az.KvBatch(i, i, i, 1, 2, 4, 4)
    a = az.Attention(0.1)

    def refused(*args):
        with pytest.raises(az.ArczError):
            eng.attention(kv, *args)
    eng.attention(kv, ok, x, 512, 0, 4, y, 512, 0, a)
    refused(ok, x, 512, 0, 3, y, 512, 0, a)                  # heads that do not share out
    refused(ok, x, 512, 0, 0, y, 512, 0, a)
    refused(ok, x, 255, 0, 4, y, 512, 0, a)                  # columns past the row
    refused(ok, x, 512, 257, 4, y, 512, 0, a)
    refused(ok, x, 512, 0, 4, y, 512, 257, a)
    refused(az.KvBatch(i, i, i, 1, 2, 5, 4), x, 512, 0, 4, y, 512, 0, a)   # rows past the buffers
    refused(az.KvBatch(i, i, i, 8, 1, 4, 4), x, 512, 0, 4, y, 512, 0, a)
    refused(az.KvBatch(i, i, i, 1, 2, 4, 4, -1), x, 512, 0, 4, y, 512, 0, a)
    refused(ok, x, 512, 0, 4, x, 512, 128, a)                # out among the rows
    eng.attention(kv, ok, x, 512, 0, 4, x, 512, 256, a)      # ... or beside them
    refused(ok, x, 512, 0, 4, kv.buffer(0), 256, 0, a)
    for bad in (az.Attention(float("nan")), az.Attention(float("inf")), az.Attention(0.1, cap=-1.0), az.Attention(0.1, cap=float("nan")),
                az.Attention(0.1, cap=float("inf")), az.Attention(0.1, window=-1), az.Attention(0.1, slopes=i.view(0, 12)),
                az.Attention(0.1, first=i.view(0, 12)), az.Attention(0.1, prefix=i.view(0, 0))):
        refused(ok, x, 512, 0, 4, y, 512, 0, bad)
        for h in bad.held:
            if h:
                h.free()
    dead = az.KvBatch(i, i, i, 1, 2, 4, 4)
    gone = az.Runtime.alloc(64)
    dead.len = gone.h
    gone.free()
    refused(dead, x, 512, 0, 4, y, 512, 0, a)
    eng.attention(kv, az.KvBatch(i, i, i, 0, 2, 4, 4), x, 512, 0, 4, y, 512, 0, a)
    eng.attention(kv, az.KvBatch(i, i, i, 1, 2, 0, 4), x, 512, 0, 4, y, 512, 0, a)
    for b in (kv, i, x, y):
        b.free()
