"""Prompts and single tokens in one batch: as one call, and as one call for each kind on views of the same arrays."""
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


@pytest.mark.parametrize("hd,page,block,heads,kv", [(64, 16, 4, 8, 2), (128, 64, 64, 8, 2), (256, 32, 32, 4, 1)])
@pytest.mark.parametrize("seqs,few", [([(70, 300), (1, 900), (1, 1), (2, 40), (1, 333)], 1), ([(1, 700), (3, 90), (130, 130), (40, 600)], 2)])
def test_a_call_for_each_kind(eng, hd, page, block, heads, kv, seqs, few):
    """The batch's sequences [0, few) and [few, end): rows, len and table from where each part begins, T and the rows' buffers as they
    are.  Each call writes its own rows alone; together they are the one call's results."""
    b = ref.Batch(seqs, page, seed=3)
    c = ref.Cache(b.pages, page, block, kv, hd, seed=4)
    w = (heads + 2 * kv) * hd
    x = np.random.default_rng(5).standard_normal((b.T, w)).astype(np.float32)
    first = np.random.default_rng(6).integers(0, 30, size=b.T).astype(np.int32)
    prefix = np.array([20, 0, 1, 60, 7][:len(seqs)], np.int32)
    hold = []
    kvc = ref.device_cache(eng, c, hold)
    xb, fb, pb = (az.Runtime.from_numpy(a) for a in (x, first, prefix))
    one = b.device(hold)
    hold += [xb, fb, pb]
    parts = []
    for s0, s1 in ((0, few), (few, len(seqs))):
        n = s1 - s0
        v = [m.view(4 * o, 4 * k) for m, o, k in zip(one.held, (s0, s0, s0 * b.ldt), (n + 1, n, n * b.ldt))] + [pb.view(4 * s0, 4 * n)]
        hold += v
        parts.append((az.KvBatch(*v[:3], n, b.ldt, b.T, max(r for r, _ in seqs[s0:s1]), max(l for _, l in seqs[s0:s1])), v[3], slice(b.rows[s0], b.rows[s1])))
    want, tol, _ = ref.attention(c, x[:, :heads * hd].reshape(b.T, heads, hd), b.rows, b.lens, b.table, 0.09, prefix=prefix, first=first)
    for turn in range(2):
        out = az.Runtime.from_numpy(np.full((b.T, heads * hd), 7.5, np.float32))
        hold.append(out)

        def call(batch, pre):
            eng.attention(kvc, batch, xb, w, 0, heads, out, heads * hd, 0, az.Attention(0.09, prefix=pre, first=fb))

        def got():
            return out.read(np.float32).reshape(b.T, heads, hd)
        if turn == 0:
            call(one, pb)
        else:
            call(parts[0][0], parts[0][1])
            assert (got()[parts[1][2]] == 7.5).all()
            call(parts[1][0], parts[1][1])
        assert (np.abs(got() - want) <= tol).all()
    # the cache's own calls on the parts, rows of k and v behind those of q: what one call writes and reads
    caches = []
    for batches in ([one], [p[0] for p in parts]):
        kvc = ref.device_cache(eng, c, hold)
        back = az.Runtime.from_numpy(np.full((b.T, 2 * kv * hd), 7.5, np.float32))
        hold.append(back)
        for p in batches:
            eng.kv_write(kvc, p, xb, w, heads * hd, xb, w, (heads + kv) * hd)
        for p in batches:
            eng.kv_read(kvc, p, back, 2 * kv * hd, 0, back, 2 * kv * hd, kv * hd)
        caches.append(ref.read_cache(kvc, c) + (back.read(np.float32),))
    assert all(np.array_equal(a, d) for a, d in zip(*caches))
    ref.free(hold)
