"""The 8-bit cache on the GPU: the stored bytes and scales bit for bit against the f32 operations that define them
(attn_ref.Cache.write), and read back."""
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


def rows_of(T, width, seed, amp=1.0):
    rng = np.random.default_rng(seed)
    x = rng.standard_normal((T, width)).astype(np.float32) * np.float32(amp)
    return x * (1.0 + 3.0 * (rng.random((T, 1)) < 0.2)).astype(np.float32)


def write_and_compare(eng, c, b, x, ld, k_off, v_off, hold, kv=None):
    """One kv_write of the rows of x on both sides; the GPU's cache must be the host's, bit for bit."""
    kv = kv or ref.device_cache(eng, c, hold)
    xb = az.Runtime.from_numpy(x)
    hold.append(xb)
    eng.kv_write(kv, b.device(hold), xb, ld, k_off, xb, ld, v_off)
    w = c.heads * c.hd
    for s, (n, l) in enumerate(b.seqs):
        m = min(n, b.max_rows)
        for which, off in ((0, k_off), (1, v_off)):
            c.write(which, b.table[s], l - n, x[b.rows[s]:b.rows[s] + m, off:off + w].reshape(m, c.heads, c.hd))
    q, d = ref.read_cache(kv, c)
    assert np.array_equal(d.view(np.uint32) & 0x7FFFFFFF, c.d.view(np.uint32) & 0x7FFFFFFF)
    assert np.array_equal(q, c.q)
    return kv


@pytest.mark.parametrize("page,block", [(16, 16), (16, 1), (32, 8), (64, 64), (64, 2), (128, 128), (128, 32), (256, 256), (256, 4)])
@pytest.mark.parametrize("hd,heads", [(64, 3), (128, 2), (256, 1)])
def test_write(eng, page, block, hd, heads):
    print(f"kv_write page={page} block={block} hd={hd} heads={heads}", flush=True)
    # a prompt, a chunk behind an odd length, a token on an older block, a token that begins one, nothing, a chunk over pages
    seqs = [(page + 3, page + 3), (70, 111), (1, page // 2 + 1), (1, page + 1), (0, 9), (3 * page - 1, 4 * page + 5)]
    b = ref.Batch(seqs, page, seed=page + block)
    c = ref.Cache(b.pages, page, block, heads, hd, seed=2)
    w = heads * hd
    x = rows_of(b.T, 4 * w, seed=page, amp=2.0)
    hold = []
    kv = write_and_compare(eng, c, b, x, 4 * w, w, 3 * w, hold)
    # the same rows again (drafts taken back and written anew), smaller: the scales of the first block stay
    write_and_compare(eng, c, b, x * np.float32(0.25), 4 * w, w, 3 * w, hold, kv)
    write_and_compare(eng, c, b, x * np.float32(9.0), 4 * w, w, 3 * w, hold, kv)
    ref.free(hold)


@pytest.mark.parametrize("page,block", [(16, 16), (64, 16), (64, 1)])
def test_token_by_token(eng, page, block):
    """A sequence grown by one token a call: the scale of the block under way grows, the older values are rounded again."""
    c = ref.Cache(6, page, block, 2, 128, seed=5)
    hold, kv = [], None
    for step in range(2 * page + 3):
        b = ref.Batch([(1, step + 1), (1, 7 + step)], page, seed=1, ld_extra=0)
        b.ldt = 4
        b.table = np.array([[3, 0, 5, -1], [1, 2, 4, -1]], np.int32)
        x = rows_of(2, 512, seed=step, amp=1.0 + 0.1 * step)
        kv = write_and_compare(eng, c, b, x, 512, 0, 256, hold, kv)
    ref.free(hold)


def test_unaligned_columns(eng):
    b = ref.Batch([(5, 9), (40, 40)], 32, seed=4)
    c = ref.Cache(b.pages, 32, 8, 1, 64, seed=3)
    hold = []
    write_and_compare(eng, c, b, rows_of(45, 203, seed=8), 203, 3, 130, hold)
    ref.free(hold)


def test_values_at_the_edges(eng):
    """Zeros, the smallest and largest numbers, halves of a step, infinities and NaN (the block is NaN until it is begun anew)."""
    page = block = 16
    b = ref.Batch([(16, 16)], page, seed=4)
    hold, kv = [], None
    c = ref.Cache(b.pages, page, block, 1, 64, seed=3)
    base = rows_of(16, 128, seed=1)
    halves = (np.arange(16 * 128).reshape(16, 128) % 255 - 127 + 0.5).astype(np.float32)
    halves[0, 0] = halves[0, 64] = 127.0
    cases = [np.zeros_like(base), np.full_like(base, 1e-42), np.full_like(base, 2.0 ** -113), base * np.float32(1e-30), np.full_like(base, 3.4e38), halves, -np.zeros_like(base)]
    for bad in (np.inf, -np.inf, np.nan):
        a = base.copy()
        a[7, 3] = bad
        a[9, 100] = bad
        cases.append(a)
    cases.append(base)
    for x in cases:
        kv = write_and_compare(eng, c, b, x, 128, 0, 64, hold, kv)
    # a NaN behind older tokens, and a token behind a NaN: the block stays NaN
    for step, bad in enumerate((1.0, np.nan, 1.0)):
        b1 = ref.Batch([(1, 5 + step)], page, seed=4)
        b1.table[0, 0] = b.table[0, 0]
        x = rows_of(1, 128, seed=step)
        x[0, 5] = bad
        kv = write_and_compare(eng, c, b1, x, 128, 0, 64, hold, kv)
    assert np.isnan(c.d[0, b.table[0, 0], 0, 0])
    ref.free(hold)


def test_pages_that_are_none_and_lengths_that_do_not_fit(eng):
    """A page outside the cache is not written; rows before position 0 and rows past max_rows are left out; lengths past the
    table are cut to it.  (The host's restatement takes the same cuts; every access of the kernel is held to the buffers.)"""
    page, block = 16, 8
    b = ref.Batch([(20, 50), (30, 12), (40, 45)], page, seed=6, max_rows=33)
    c = ref.Cache(b.pages, page, block, 2, 64, seed=3)
    b.table[0, 2], b.table[2, 1] = b.pages, -7
    hold = []
    x = rows_of(b.T, 256, seed=2)
    kv = write_and_compare(eng, c, b, x, 256, 0, 128, hold)
    # a length past the table: the newest rows are those at its end
    b.lens[0] = 2 ** 31 - 1
    b.seqs = [(20, b.ldt * page), (30, 12), (40, 45)]
    b.table[0, :] = [t if t >= 0 else 0 for t in b.table[0]]
    b.table[0, -1] = b.table[0, 0]
    b.table[0, 0] = -1
    kv = write_and_compare(eng, c, b, x, 256, 0, 128, hold, kv)
    # rows that fall or pass the buffers hold no rows
    b.rows[:] = [5, -3, 2 ** 31 - 1, 0]
    b.seqs = [(0, 0), (0, 0), (0, 0)]
    b.lens[1] = -5
    before = ref.read_cache(kv, c)
    xb = az.Runtime.from_numpy(x)
    hold.append(xb)
    d = b.device(hold)
    d.T = 2           # (sequence 1 has the two rows of the buffers, at positions below 0)
    eng.kv_write(kv, d, xb, 256, 0, xb, 256, 128)
    after = ref.read_cache(kv, c)
    assert np.array_equal(before[0], after[0]) and np.array_equal(before[1], after[1])
    ref.free(hold)


@pytest.mark.parametrize("page,block,hd,heads", [(16, 16, 64, 3), (64, 1, 128, 2), (256, 64, 256, 5), (32, 32, 128, 8)])
@pytest.mark.parametrize("ld_pad,off", [(0, 0), (8, 4), (7, 3)])
def test_read(eng, page, block, hd, heads, ld_pad, off):
    seqs = [(1, 40), (77, 90), (0, 3), (6, 2)]
    b = ref.Batch(seqs, page, seed=page, T=90)
    c = ref.Cache(b.pages, page, block, heads, hd, seed=7)
    b.table[1, 0] = -1       # (its first page is none: zeros)
    w = heads * hd
    ld = w + ld_pad
    hold = []
    kv = ref.device_cache(eng, c, hold)
    kb, vb = (az.Runtime.from_numpy(np.full((90, ld), 7.5, np.float32)) for _ in range(2))
    hold += [kb, vb]
    eng.kv_read(kv, b.device(hold), kb, ld, off, vb, ld, off)
    for which, buf in ((0, kb), (1, vb)):
        got = buf.read(np.float32, 90 * ld).reshape(90, ld)
        want = np.full((90, ld), 7.5, np.float32)
        for s, (n, l) in enumerate(seqs):
            v = c.values(which, b.table[s], l).astype(np.float32).reshape(l, w)
            for i in range(n):
                if l - n + i >= 0:
                    want[b.rows[s] + i, off:off + w] = v[l - n + i]
        assert np.array_equal(got, want)
    ref.free(hold)


def test_far_pages(eng):
    """Pages behind 2^32 bytes of keys: written and read where they are."""
    page, heads, hd = 256, 8, 128
    pages = (1 << 32) // (page * heads * hd) + 4
    kv = eng.make_kv(pages, page, 1, heads, hd)
    T, w = 300, heads * hd
    x = rows_of(T, 2 * w, seed=1)
    hold = [kv] + [az.Runtime.from_numpy(a) for a in (np.array([0, T], np.int32), np.array([T], np.int32), np.array([[pages - 1, 2]], np.int32), x,
                                                      np.zeros((T, 2 * w), np.float32))]
    b = az.KvBatch(hold[1], hold[2], hold[3], 1, 2, T, T)
    eng.kv_write(kv, b, hold[4], 2 * w, 0, hold[4], 2 * w, w)
    eng.kv_read(kv, b, hold[5], 2 * w, 0, hold[5], 2 * w, w)
    y = hold[5].read(np.float32, T * 2 * w).reshape(T * 2 * heads, hd)
    d = np.abs(x.reshape(T * 2 * heads, hd)).max(1, keepdims=True) / np.float32(127)
    want = np.rint(x.reshape(T * 2 * heads, hd) * (np.float32(1) / d)) * d
    assert np.array_equal(y, want.astype(np.float32))
    # the last page's first row, where a 64-bit offset puts it
    at = (pages - 1) * heads * page * hd
    assert at >= 1 << 32
    assert np.array_equal(kv.buffer(0).read(np.int8, hd, offset=at), np.rint(x[0, :hd] * (np.float32(1) / d[0])).astype(np.int8))
    ref.free(hold)


@pytest.mark.parametrize("hd", [64, 256])
def test_the_last_positions_there_are(eng, hd):
    """Rows at the end of the longest sequence that a table can name, in a batch whose longest is told to be far longer."""
    page, long, rows, w = 256, 0x7FFFF000, 5, 2 * hd
    b = ref.Batch([(rows, 3 * page)], page, seed=1, ld_extra=0, T=rows + 20000, max_rows=rows + 20000)
    c = ref.Cache(b.pages, page, 32, 2, hd, seed=2)
    x = rows_of(b.T, 2 * w, seed=3)
    hold = []
    kv, xb = ref.device_cache(eng, c, hold), az.Runtime.from_numpy(x)
    yb = az.Runtime.from_numpy(np.full(x.shape, 7.5, np.float32))
    hold += [xb, yb]
    for which in (0, 1):
        c.write(which, b.table[0], 3 * page - rows, x[:rows, which * w:which * w + w].reshape(rows, 2, hd))
    tail, b.table = b.table, np.full((1, long // page), -1, np.int32)
    b.table[0, -3:] = tail
    b.ldt, b.lens = long // page, np.array([long], np.int32)
    batch = b.device(hold)
    eng.kv_write(kv, batch, xb, 2 * w, 0, xb, 2 * w, w)
    q, d = ref.read_cache(kv, c)
    assert np.array_equal(d, c.d) and np.array_equal(q, c.q)
    eng.kv_read(kv, batch, yb, 2 * w, 0, yb, 2 * w, w)
    y = yb.read(np.float32, x.size).reshape(x.shape)
    for which in (0, 1):
        v = c.values(which, tail[0], 3 * page)[-rows:].reshape(rows, w)
        assert np.array_equal(y[:rows, which * w:which * w + w], v.astype(np.float32))
    assert (y[rows:] == 7.5).all()
    ref.free(hold)


def test_refusals(eng):
    for pages, page, block, heads, hd in [(0, 16, 1, 1, 64), (1, 8, 1, 1, 64), (1, 48, 16, 1, 64), (1, 512, 1, 1, 64), (1, 16, 32, 1, 64), (1, 16, 3, 1, 64),
                                          (1, 16, 0, 1, 64), (1, 16, 1, 0, 64), (1, 16, 1, 1, 80), (1, 16, 1, 40000, 64)]:
        with pytest.raises(az.ArczError):
            eng.make_kv(pages, page, block, heads, hd)
    small = az.Runtime.alloc(16 * 64 * 2 - 1)
    with pytest.raises(az.ArczError):
        eng.make_kv(2, 16, 16, 1, 64, k=small)
    big = az.Runtime.alloc(1 << 16)
    odd = big.view(8, 16 * 64 * 2)
    with pytest.raises(az.ArczError):
        eng.make_kv(2, 16, 16, 1, 64, k=odd)
    with pytest.raises(az.ArczError):
        eng.make_kv(2, 16, 16, 1, 64, k=big, v=big)
    kv = eng.make_kv(2, 16, 16, 1, 64)
    i = az.Runtime.from_numpy(np.zeros(8, np.int32))
    x = az.Runtime.alloc(4 * 128 * 4)

    def refused(batch, *a):
        for f in (eng.kv_write, eng.kv_read):
            with pytest.raises(az.ArczError):
                f(kv, batch, *a)
    ok = az.KvBatch(i, i, i, 1, 2, 4, 4)
    eng.kv_write(kv, ok, x, 128, 0, x, 128, 64)
    eng.kv_read(kv, ok, x, 128, 0, x, 128, 64)
    refused(az.KvBatch(i, i, i, 8, 1, 4, 4), x, 128, 0, x, 128, 64)        # rows needs nine values
    refused(az.KvBatch(i, i, i, 1, 9, 4, 4), x, 128, 0, x, 128, 64)        # the table nine
    refused(az.KvBatch(i, i, i, -1, 2, 4, 4), x, 128, 0, x, 128, 64)
    refused(az.KvBatch(i, i, i, 1, 0, 4, 4), x, 128, 0, x, 128, 64)
    refused(ok, x, 128, 65, x, 128, 64)                                     # columns past the row
    refused(ok, x, 60, 0, x, 128, 64)
    refused(az.KvBatch(i, i, i, 1, 2, 5, 4), x, 128, 0, x, 128, 64)        # rows past the buffer
    refused(ok, kv.buffer(0), 64, 0, x, 128, 0)                             # rows in the cache itself
    with pytest.raises(az.ArczError):
        eng.kv_read(kv, ok, x, 128, 0, x, 128, 63)                          # k and v share a column
    for e in (az.KvBatch(i, i, i, 0, 2, 4, 4), az.KvBatch(i, i, i, 1, 2, 0, 4), az.KvBatch(i, i, i, 1, 2, 4, 0)):
        eng.kv_write(kv, e, x, 128, 0, x, 128, 64)                          # nothing to do
        eng.kv_read(kv, e, x, 128, 0, x, 128, 64)
    for b in (kv, odd, big, small, i, x):
        b.free()
