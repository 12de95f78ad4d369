"""The room that attention shares keys out in: made once, whatever is called behind it."""
import ctypes as C

import numpy as np
import pytest

import arcinferzero_amd as az
import attn_ref as ref

pytestmark = pytest.mark.gpu


@pytest.fixture
def eng(rt):
    e = az.Engine(16, 256)
    yield e
    e.close()


def device_bytes():
    az.lib.arcz_device_bytes.restype = C.c_size_t
    return az.lib.arcz_device_bytes()


class Call:
    """Attention of `rows` tokens behind `keys`, with max_len as the caller knows it then."""

    def __init__(self, eng, hold, rows, keys, heads=8, kv=2, hd=128, seqs=1, page=64):
        self.eng, self.heads, self.hd = eng, heads, hd
        self.b = ref.Batch([(rows, keys)] * seqs, page, seed=rows)
        self.c = ref.Cache(self.b.pages, page, 32, kv, hd, seed=3)
        self.q = np.random.default_rng(keys).standard_normal((self.b.T, heads * hd)).astype(np.float32)
        self.kv, self.batch = ref.device_cache(eng, self.c, hold), self.b.device(hold)
        self.qb, self.out = az.Runtime.from_numpy(self.q), az.Runtime.alloc(self.q.nbytes)
        hold += [self.qb, self.out]

    def run(self):
        w = self.heads * self.hd
        self.eng.attention(self.kv, self.batch, self.qb, w, 0, self.heads, self.out, w, 0, az.Attention(0.09))

    def check(self):
        got = self.out.read(np.float32).reshape(self.b.T, self.heads, self.hd)
        want, tol, _ = ref.attention(self.c, self.q.reshape(got.shape), self.b.rows, self.b.lens, self.b.table, 0.09, only={0, self.b.T - 1})
        assert (np.abs(got - want) <= tol)[[0, self.b.T - 1]].all()


def test_longer_sequences_and_larger_batches_need_no_more(eng):
    """A sequence that grows from step to step, more rows, more heads, wider ones, prompts: the first call that shares keys out makes
    the room, no later one makes any, also not while it is recorded."""
    hold = []
    calls = [Call(eng, hold, *a) for a in ((1, 600), (1, 700), (1, 1500), (1, 9000), (2, 5000, 32, 8), (3, 4000, 32, 8, 64), (2, 3000, 16, 2, 256, 3),
                                           (1, 1300, 16, 2, 128, 64), (40, 900), (300, 4100, 8, 2), (100, 2000, 16, 4, 256), (33, 1200, 8, 8, 64, 4))]
    calls[0].run()
    calls[0].check()
    before, lists = device_bytes(), []
    for k in calls:
        lists.append(az.Runtime.record(k.run))     # (the first time that the engine sees such a batch)
        assert device_bytes() == before
        lists[-1].run()
        k.check()
    for k in calls[::-1]:
        k.run()
        k.check()
        assert device_bytes() == before
    for l in lists:
        l.run()
    for k in calls:
        k.check()
    for l in lists:
        l.free()
    ref.free(hold)


def test_the_room_goes_with_the_engine(rt):
    before = device_bytes()
    for _ in range(2):
        e, hold = az.Engine(16, 256), []
        a, b = Call(e, hold, 1, 600), Call(e, hold, 1, 6000)
        a.run()
        l = az.Runtime.record(a.run)
        b.run()
        l.run()
        a.check()
        b.check()
        l.free()
        ref.free(hold)
        e.close()
        assert device_bytes() == before
