"""The first call of an engine behind a shared prefix may be a recorded one: what it needs is there once its room has been asked for."""
import numpy as np
import pytest

import arcinferzero_amd as az
import attn_ref as ref
from test_gpu_attention_shared import Case, engine

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,hd,heads", [(1, 128, 8), (20, 64, 8)])
@pytest.mark.parametrize("way", ["0", None, "1"])
def test_the_first_call_is_recorded(rt, way, rows, hd, heads):
    """Few sequences of many keys: one launch of attention that shares them out (two, where rows are many), or the three."""
    e = engine(way)
    k = Case([(900, [(rows, 400), (rows, 700)])], 32, 16, 2, hd, heads)
    hold, w = [], heads * hd
    kv, batch = ref.device_cache(e, k.c, hold), k.b.device(hold)
    q, out = az.Runtime.from_numpy(k.x), az.Runtime.alloc(k.x.nbytes)
    gb, sb = az.Runtime.from_numpy(np.array(k.groups, np.int32)), az.Runtime.from_numpy(np.array(k.shared, np.int32))
    sh, form = az.KvShared(gb, sb, 1, 2 * rows, 900), az.Attention(0.07)
    room = az.Runtime.alloc(e.attention_shared_room(kv, batch, sh, heads, form))
    hold += [q, out, gb, sb, room]

    def call():
        e.attention_shared(kv, batch, sh, q, w, 0, heads, out, w, 0, form, room)
    l = az.Runtime.record(call)
    want, tol, _ = ref.attention(k.c, k.x, k.b.rows, k.b.lens, k.b.table, 0.07)
    for _ in range(3):
        out.fill(0xFFFFFFFF)
        l.run()
        y = out.read(np.float32).reshape(k.x.shape)
        assert (np.abs(y - want) <= tol).all()
        out.fill(0xFFFFFFFF)
        call()
        assert np.array_equal(out.read(np.uint32), y.view(np.uint32).ravel())
    l.free()
    ref.free(hold)
    e.close()


def test_room_that_cannot_be_made_while_recording(rt):
    """Asked for while a list is recorded, by an engine that has none yet: an error, and none behind it."""
    e = engine("0")
    k = Case([(900, [(1, 400), (1, 700)])], 32, 16, 2, 128, 8)
    hold = []
    kv, batch = ref.device_cache(e, k.c, hold), k.b.device(hold)
    gb, sb = az.Runtime.from_numpy(np.array(k.groups, np.int32)), az.Runtime.from_numpy(np.array(k.shared, np.int32))
    sh, form = az.KvShared(gb, sb, 1, 2, 900), az.Attention(0.07)
    hold += [gb, sb]

    def ask():
        return e.attention_shared_room(kv, batch, sh, 8, form)
    with pytest.raises(az.ArczError):
        az.Runtime.record(ask)
    n = ask()
    assert n > 0 and ask() == n
    ref.free(hold)
    e.close()
