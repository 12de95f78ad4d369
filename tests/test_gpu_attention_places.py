"""Which buffers of a call of the attention block may share memory: outputs and what a launch reads may not, pieces of one allocation that
do not meet may."""
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


def test_outputs_over_what_is_read_are_refused(eng):
    """Every output against rows, len, table, pos, slopes, prefix and first: an error, and no launch."""
    hold = []

    def keep(b):
        hold.append(b)
        return b
    # one allocation: [ints 256 | rows of q, k, v | cache]
    big = keep(az.Runtime.alloc(1 << 20).fill(0))
    w, kvw = 4 * 64, 2 * 64
    ints = keep(big.view(0, 1024))
    own = [keep(az.Runtime.from_numpy(np.array(a, np.int32))) for a in ([0, 4], [4], [0, 1])]
    x = keep(az.Runtime.alloc(4 * 2 * w * 4).fill(0))
    kv = keep(eng.make_kv(2, 16, 16, 2, 64))
    rope = keep(eng.make_rope([1.0] * 32))
    a = az.Attention(0.1)
    n = az.lib.arcz_launch_count()

    def batch(*parts):
        return az.KvBatch(*parts, 1, 2, 4, 4)

    def refused(f, *args):
        with pytest.raises(az.ArczError):
            f(*args)
        assert az.lib.arcz_launch_count() == n
    for i in range(3):
        parts = list(own)
        parts[i] = ints
        refused(eng.attention, kv, batch(*parts), x, 2 * w, 0, 4, big, w, 0, a)
        refused(eng.kv_read, kv, batch(*parts), big, kvw, 0, x, kvw, 0)
        refused(eng.kv_read, kv, batch(*parts), x, kvw, 0, big, kvw, 0)
        # (the cache on memory that the batch lies in)
        c = eng.make_kv(2, 16, 16, 2, 64, k=big)
        refused(eng.kv_write, c, batch(*parts), x, kvw, 0, x, kvw, 0)
        c.free()
        c = eng.make_kv(2, 16, 16, 2, 64, vs=big)
        refused(eng.kv_write, c, batch(*parts), x, kvw, 0, x, kvw, 0)
        c.free()
    for part in ("slopes", "prefix", "first"):
        refused(eng.attention, kv, batch(*own), x, 2 * w, 0, 4, big, w, 0, az.Attention(0.1, **{part: ints}))
    refused(eng.rope, rope, x, w, 0, big, w, 0, 4, 4, 64, ints)
    refused(eng.rope, rope, big, w, 0, big, w, 0, 4, 4, 64, ints)
    ref.free(hold)


def test_pieces_of_one_allocation(eng):
    """Cache, rows, outputs and the batch's arrays side by side in one allocation, the cache's handles as large as all of it: the results
    are those of buffers of their own."""
    page, block, kv, hd, heads = 16, 8, 2, 64, 4
    seqs = [(5, 20), (3, 3)]
    b = ref.Batch(seqs, page, seed=2)
    c = ref.Cache(b.pages, page, block, kv, hd, seed=3)
    rng = np.random.default_rng(4)
    w = (heads + 2 * kv) * hd
    x = rng.standard_normal((b.T, w)).astype(np.float32)
    results = []
    for one in (False, True):
        hold = []
        parts = [c.q[0], c.q[1], c.d[0], c.d[1], x, np.zeros((b.T, heads * hd), np.float32), np.zeros((b.T, 2 * kv * hd), np.float32), b.rows, b.lens, b.table]
        if one:
            at = np.cumsum([0] + [-(-p.nbytes // 64) * 64 for p in parts])
            big = az.Runtime.alloc(int(at[-1]))
            hold.append(big)
            m = []
            for o, p in zip(at[:-1], parts):
                big.write(p, offset=int(o))
                # (the cache's buffers: to the end of the allocation, more than it takes)
                m.append(big.view(int(o), int(at[-1] - o) if len(m) < 4 else p.nbytes))
        else:
            m = [az.Runtime.from_numpy(p) for p in parts]
        hold += m
        k = eng.make_kv(c.pages, page, block, kv, hd, *m[:4])
        hold.append(k)
        batch = az.KvBatch(m[7], m[8], m[9], len(seqs), b.ldt, b.T, b.max_rows, b.max_len)
        eng.kv_write(k, batch, m[4], w, heads * hd, m[4], w, (heads + kv) * hd)
        eng.kv_read(k, batch, m[6], 2 * kv * hd, 0, m[6], 2 * kv * hd, kv * hd)
        eng.attention(k, batch, m[4], w, 0, heads, m[5], heads * hd, 0, az.Attention(0.1))
        results.append([p.read(np.uint8, q.nbytes) for p, q in zip(m, parts)])
        ref.free(hold)
    assert all(np.array_equal(p, q) for p, q in zip(*results))
    assert results[0][5].any() and results[0][6].any()


@pytest.mark.parametrize("which", [0, 1, 2, 3])
def test_a_buffer_freed_under_the_cache(eng, which):
    """The caller's buffer freed before the cache, smaller ones made behind it (in its handle's place, as it happens): refused."""
    size = (4 * 2 * 16 * 64, 4 * 2 * 16 * 64, 4 * 2 * 4, 4 * 2 * 4)
    bufs = [az.Runtime.alloc(n).fill(0) for n in size]
    kv = eng.make_kv(4, 16, 16, 2, 64, *bufs)
    own = [az.Runtime.from_numpy(np.array(a, np.int32)) for a in ([0, 1], [1], [3, 3])]
    batch, x, y = az.KvBatch(*own, 1, 2, 1, 1), az.Runtime.alloc(4 * 256).fill(0), az.Runtime.alloc(4 * 256).fill(0)
    eng.kv_write(kv, batch, x, 128, 0, x, 128, 0)
    bufs[which].free()
    small = [az.Runtime.alloc(16) for _ in range(8)]
    n = az.lib.arcz_launch_count()
    for f, args in ((eng.kv_write, (x, 128, 0, x, 128, 0)), (eng.kv_read, (x, 128, 0, y, 128, 0)), (eng.attention, (x, 256, 0, 4, y, 256, 0, az.Attention(0.1)))):
        with pytest.raises(az.ArczError):
            f(kv, batch, *args)
    assert az.lib.arcz_launch_count() == n
    ref.free([b for i, b in enumerate(bufs) if i != which] + own + [x, y] + small + [kv])
