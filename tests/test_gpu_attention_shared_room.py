"""The workspace and the launches of attention behind shared prefixes go by the batch's rows, not by its longest sequence times their number."""
import numpy as np
import pytest

import arcinferzero_amd as az
import attn_ref as ref
from test_gpu_attention_shared import Case, engine

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def eng(rt):
    e = engine("1")
    yield e
    e.close()


def room(eng, seqs, T, max_rows, group_rows, heads=64, kv=8, hd=128, ldt=140, page=64, shared=8000, own=700):
    """The bytes for `seqs` sequences in one group, and those of one piece of all rows."""
    hold = [az.Runtime.alloc(4 * n) for n in (seqs + 1, seqs, seqs * ldt, 2, 1)]
    c = eng.make_kv(4, page, page, kv, hd)
    n = eng.attention_shared_room(c, az.KvBatch(*hold[:3], seqs, ldt, T, max_rows, shared + own), az.KvShared(hold[3], hold[4], 1, group_rows, shared), heads, az.Attention(0.1))
    ref.free(hold + [c])
    return n, T * heads * (hd + 2) * 4


def test_one_long_sequence_beside_many_short_ones(eng):
    """255 tokens and a prompt's chunk: no more than a few pieces a row (blocks for the longest's rows, for each sequence, would be 8.8 GB of 2048 rows)."""
    for chunk in (2048, 4096):
        n, piece = room(eng, 256, 255 + chunk, chunk, 255 + chunk)
        assert n <= 12 * piece, (n, piece)


def test_a_loose_most_of_rows(eng):
    """What max_rows says beyond the batch's rows costs no room."""
    for T in (256, 600):
        n, piece = room(eng, 256, T, 1, T)
        for max_rows, group_rows in ((T, T), (1 << 20, 1 << 20)):
            m, _ = room(eng, 256, T, max_rows, group_rows)
            assert m <= max(2 * n, 12 * piece), (m, n, piece)


def test_buffers_of_more_rows_than_the_batch_may_have(eng):
    """A recorded step's buffers are made for its largest batch: what the sequences can have, seqs * max_rows, is less."""
    n, _ = room(eng, 128, 128, 1, 128)
    m, _ = room(eng, 128, 8192, 1, 128)
    assert m <= n


@pytest.mark.parametrize("hd,kv,heads", [(64, 2, 8), (128, 1, 4), (256, 1, 3)])
@pytest.mark.parametrize("max_rows", [None, 1, 3])
def test_loose_buffers(eng, hd, kv, heads, max_rows):
    """Places by sequences: rows left out of some, sequences of none, a group and sequences of no group."""
    k = Case([(130, [(1, 9), (3, 40), (0, 7), (2, 2), (1, 200)]), (50, [(1, 1), (3, 77)])], 32, 16, kv, hd, heads, T=90, max_rows=max_rows)
    k.run(eng, again=2)
    k.groups, k.shared = [1, 4], [130]
    k.run(eng)


@pytest.mark.parametrize("hd,kv,heads", [(64, 2, 8), (128, 1, 4), (256, 1, 3)])
def test_unlike_sequences(eng, hd, kv, heads):
    """A chunk of 300 rows between tokens, in a group and in none; rows behind the last sequence; a loose max_rows."""
    short = [(1, 1 + 11 * i % 70) for i in range(9)]
    Case([(130, short + [(300, 310)] + short), (60, [(2, 5), (40, 40)])], 32, 16, kv, hd, heads, T=420, max_rows=5000, group_rows=5000).run(eng)
    k = Case([(130, short[:4] + [(150, 160)] + short[4:])], 32, 16, kv, hd, heads, seed=3)
    k.groups, k.shared = [2, 7], [130]
    k.run(eng)


def test_many_rows_and_heads(eng):
    """More than 65535 blocks of rows and heads: 64 heads of 256 values on one of keys, buffers of 4200 rows, of which six belong to sequences."""
    T, heads, hd = 4200, 64, 256
    k = Case([(64, [(3, 9), (2, 40), (1, 1)])], 32, 16, 1, hd, heads)
    hold, w, n = [], heads * hd, k.b.T
    kv, b = ref.device_cache(eng, k.c, hold), k.b.device(hold)
    batch = az.KvBatch(*b.held, 3, b.ld_table, T, 5000, b.max_len)
    q, out = az.Runtime.alloc(T * w * 4), az.Runtime.alloc(T * w * 4)
    q.fill(0)
    out.fill(0x40E80000)     # (7.25)
    q.write(k.x)
    gb, sb = az.Runtime.from_numpy(np.array(k.groups, np.int32)), az.Runtime.from_numpy(np.array(k.shared, np.int32))
    sh, form = az.KvShared(gb, sb, 1, T, 64), az.Attention(0.11)
    rm = az.Runtime.alloc(eng.attention_shared_room(kv, batch, sh, heads, form))
    hold += [q, out, gb, sb, rm]
    launches = az.lib.arcz_launch_count()
    eng.attention_shared(kv, batch, sh, q, w, 0, heads, out, w, 0, form, rm)
    assert az.lib.arcz_launch_count() == launches + 3
    y = out.read(np.float32).reshape(T, heads, hd)
    want, tol, _ = ref.attention(k.c, k.x, k.b.rows, k.b.lens, k.b.table, 0.11)
    assert (np.abs(y[:n] - want) <= tol).all() and (y[n:] == 7.25).all()
    ref.free(hold)


def test_loose_buffers_pay_as_tight_ones_do(rt):
    """256 sequences of a token behind a long prefix are three launches, also in buffers of 8192 rows; the values are the same."""
    e, got = engine(None), []
    for T in (256, 8192):
        k = Case([(64, [(1, 30 + i % 7) for i in range(256)])], 32, 16, 2, 128, 8, T=T)
        hold, w = [], 8 * 128
        k.x[256:] = 0
        kv, batch = ref.device_cache(e, k.c, hold), k.b.device(hold)
        batch.max_len = 9040
        q, out = az.Runtime.from_numpy(k.x), az.Runtime.alloc(k.x.nbytes)
        gb, sb = az.Runtime.from_numpy(np.array(k.groups, np.int32)), az.Runtime.from_numpy(np.array(k.shared, np.int32))
        sh, form = az.KvShared(gb, sb, 1, 256, 9000), az.Attention(0.05)
        rm = az.Runtime.alloc(e.attention_shared_room(kv, batch, sh, 8, form))
        hold += [q, out, gb, sb, rm]
        q.write(np.random.default_rng(1).standard_normal((256, w)).astype(np.float32))
        n = az.lib.arcz_launch_count()
        e.attention_shared(kv, batch, sh, q, w, 0, 8, out, w, 0, form, rm)
        assert az.lib.arcz_launch_count() == n + 3
        got.append(out.read(np.uint32, 256 * w))
        ref.free(hold)
    assert np.array_equal(*got)
    e.close()
