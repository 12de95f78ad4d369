"""A serving step's operators together, as a decode loop uses them: where the new tokens go, the q|k|v product, norms and rotation, the cache, attention
behind shared prefixes, the head's product and the drawn tokens.  Each is held to its own definition on what the one before really left on the
GPU; the whole step, recorded once, is replayed to the same tokens."""
import numpy as np
import pytest

import arcinferzero_amd as az
import attn_ref as ref
from common import make_acts, make_weights
from test_gpu_kv_plan import walk
from test_gpu_norm_rope import norms
from test_gpu_sample import tokens

pytestmark = pytest.mark.gpu

E, HEADS, KV, HD, PAGE, BLOCK, V = 512, 8, 2, 64, 16, 16, 3001
W, SEQS, PAGES, LDT, PREFIX = (HEADS + 2 * KV) * HD, 5, 60, 12, (48, 32)
GROUPS = np.array([0, 3, 5], np.int32)


class Step:
    """The buffers and calls of a step of five sequences in two groups, a token each (or none)."""

    def __init__(self, eng, forced):
        self.eng, self.forced, rng = eng, forced, np.random.default_rng(5)
        self.Mp = 16
        self.wq = eng.make_weight(az.Q8_0, W, E, make_weights(az.Q8_0, W, E, 1))
        self.wo = eng.make_weight(az.Q8_0, V, HEADS * HD, make_weights(az.Q8_0, V, HEADS * HD, 2))
        self.freq = [10000.0 ** (-i / 32) for i in range(32)]
        self.rope = eng.make_rope(self.freq)
        self.nq, self.nk = ((1 + 0.2 * rng.standard_normal(HD)).astype(np.float32) for _ in range(2))
        self.c = ref.Cache(PAGES, PAGE, BLOCK, KV, HD, seed=3)
        self.hold = []
        self.kv = ref.device_cache(eng, self.c, self.hold)
        # the first pages of a group are its sequences' all; each has some tokens of its own behind them
        order = rng.permutation(PAGES).astype(np.int32)
        self.table, at = np.full((SEQS, LDT), -1, np.int32), 5
        self.len = np.array([PREFIX[0] + 5, PREFIX[0], PREFIX[0] + 31, PREFIX[1] + 16, PREFIX[1] + 1], np.int32)
        self.shared = np.array([PREFIX[0]] * 3 + [PREFIX[1]] * 2, np.int32)
        for s in range(SEQS):
            g = int(s >= 3)
            n = PREFIX[g] // PAGE
            self.table[s, :n] = order[:3] if g == 0 else order[3:5]
            m = -(-int(self.len[s]) // PAGE) - n
            self.table[s, n:n + m] = order[at:at + m]
            at += m
        self.ring = np.concatenate([order[at:], np.full(at, -1, np.int32)])
        self.state = np.array([0, PAGES - at, 0, 0], np.int32)
        self.top_p, self.temp = np.array([0.9, 0.5, 1.0, 0.95, 0.8], np.float32), np.array([0.8, 1.0, 0.0, 1.3, 0.7], np.float32)
        self.top_k = np.array([40, 0, 0, 700, 9], np.int32)
        for n, a in dict(rows=np.zeros(SEQS + 1, np.int32), blen=self.len, btable=self.table, bring=self.ring, bstate=self.state, add=np.ones(SEQS, np.int32), bshared=self.shared,
                         pos=np.zeros(SEQS, np.int32), slot=np.zeros(SEQS, np.int32), x=np.zeros((self.Mp, E), np.float32), qkv=np.zeros((self.Mp, W), np.float32),
                         out=np.zeros((self.Mp, HEADS * HD), np.float32), logits=np.zeros((self.Mp, V), np.float32), u=np.zeros(SEQS, np.float32), token=np.zeros(SEQS, np.int32),
                         prob=np.zeros(SEQS, np.float32), bnq=self.nq, bnk=self.nk, groups=GROUPS, prefix=np.array(PREFIX, np.int32), btemp=self.temp, btop_p=self.top_p,
                         btop_k=self.top_k).items():
            setattr(self, n, az.Runtime.from_numpy(a))
            self.hold.append(getattr(self, n))
        self.batch = az.KvBatch(self.rows, self.blen, self.btable, SEQS, LDT, SEQS, 1, LDT * PAGE)
        self.plan = az.KvPlan(PAGES, PAGE, self.add, self.blen, self.bring, self.bstate, self.bstate, self.pos, self.slot, self.bshared)
        self.sh = az.KvShared(self.groups, self.prefix, 2, SEQS, max(PREFIX))
        self.form = az.Attention(HD ** -0.5)
        self.sampling = az.Sampling(self.btemp, self.btop_k, self.btop_p)
        self.room = az.Runtime.alloc(eng.attention_shared_room(self.kv, self.batch, self.sh, HEADS, self.form))
        self.hold += [self.room, self.rope, self.wq, self.wo]

    def put(self, step, add):
        rng = np.random.default_rng(100 + step)
        x = np.zeros((self.Mp, E), np.float32)
        x[:SEQS] = make_acts(SEQS, E, seed=step)
        self.x.write(x)
        self.add.write(np.array(add, np.int32))
        self.draws = rng.random(SEQS).astype(np.float32)
        self.u.write(self.draws)

    def calls(self):
        e, kw = self.eng, HEADS * HD
        yield e.kv_plan(self.batch, self.plan)
        e.quantize(self.x, E, E, self.Mp, SEQS)
        yield e.matmul("qkv", self.wq, self.Mp, self.qkv, W)
        yield e.norm_rope(self.rope, self.qkv, W, 0, self.qkv, W, 0, SEQS, HEADS, KV, HD, self.bnq, self.bnk, 1e-6, self.pos)
        yield e.kv_write(self.kv, self.batch, self.qkv, W, kw, self.qkv, W, kw + KV * HD)
        yield e.attention_shared(self.kv, self.batch, self.sh, self.qkv, W, 0, HEADS, self.out, kw, 0, self.form, self.room)
        e.quantize(self.out, kw, kw, self.Mp, SEQS)
        yield e.matmul("head", self.wo, self.Mp, self.logits, V)
        yield e.sample(self.logits, V, 0, V, SEQS, self.sampling, self.u, self.token, self.prob)

    def run(self):
        for _ in self.calls():
            pass

    def read(self, name, dtype, *shape):
        return getattr(self, name).read(dtype, int(np.prod(shape))).reshape(shape)


@pytest.mark.parametrize("forced", ["0", "1"])
def test_a_decode_loop(rt, forced, monkeypatch):
    monkeypatch.setenv("ARCZ_ATTN_SHARED", forced)       # (attention in one launch, or the prefixes apart)
    eng = az.Engine(64, 1024)
    monkeypatch.delenv("ARCZ_ATTN_SHARED")
    s = Step(eng, forced)
    adds = [[1] * 5, [1, 0, 1, 1, 1], [1] * 5, [0, 1, -16, 1, 1], [1] * 5, [1] * 5]
    seen = []
    for step, add in enumerate(adds):
        s.put(step, add)
        calls = s.calls()
        # ---- the batch
        next(calls)
        rows, s.len, s.table, s.ring, s.state, pos, slot = walk(add, s.len, s.table, s.ring, s.state, s.shared, PAGE, SEQS, 1)
        s.len, s.state, rows, n = np.array(s.len, np.int32), np.array(s.state, np.int32), np.array(rows, np.int32), len(pos)
        for name, want in (("rows", rows), ("blen", s.len), ("btable", s.table.ravel()), ("bring", s.ring), ("bstate", s.state)):
            assert np.array_equal(s.read(name, np.int32, want.size), want), name
        assert np.array_equal(s.read("pos", np.int32, SEQS)[:n], pos) and np.array_equal(s.read("slot", np.int32, SEQS)[:n], slot)
        # ---- norms and rotation
        next(calls)
        before = s.read("qkv", np.float32, SEQS, HEADS + 2 * KV, HD)
        next(calls)
        after = s.read("qkv", np.float32, SEQS, HEADS + 2 * KV, HD)
        nrm = norms(before[:, :HEADS + KV], s.nq, s.nk, HEADS, np.float64(np.float32(1e-6)))
        p = s.read("pos", np.int32, 1, SEQS)
        turned = ref.rope(nrm, p, s.freq, [0] * 32, False)
        mag = np.abs(nrm)
        tol = np.concatenate([mag[..., :32] + mag[..., 32:]] * 2, -1) * 7 * 2.0 ** -23 + 2.0 ** -146
        assert (np.abs(after[:, :HEADS + KV] - turned) <= tol).all() and np.array_equal(after[:, HEADS + KV:], before[:, HEADS + KV:])
        # ---- the cache, and attention over it
        next(calls)
        for q in range(SEQS):
            for which, h0 in ((0, HEADS), (1, HEADS + KV)):
                c = rows[q + 1] - rows[q]
                if c:
                    s.c.write(which, s.table[q], s.len[q] - c, after[rows[q]:rows[q + 1], h0:h0 + KV])
        q, d = ref.read_cache(s.kv, s.c)
        assert np.array_equal(q, s.c.q) and np.array_equal(d, s.c.d)
        next(calls)
        y = s.read("out", np.float32, SEQS, HEADS, HD)
        exact, tol, done = ref.attention(s.c, after[:n, :HEADS], rows, s.len, s.table, HD ** -0.5)
        assert done.all() and (np.abs(y[:n] - exact) <= tol).all()
        # ---- the tokens
        next(calls)
        next(calls)
        logits, tok = s.read("logits", np.float32, SEQS, V), s.read("token", np.int32, SEQS)
        for r in range(n):
            assert int(tok[r]) in tokens(logits[r], float(s.temp[r]), int(s.top_k[r]), float(s.top_p[r]), 0.0, float(s.draws[r]))
        seen.append((tok[:n].copy(), s.read("prob", np.uint32, SEQS)[:n], s.len.copy()))
    lens = s.len.copy()
    ref.free(s.hold)
    # ---- the same loop as a recorded list
    t = Step(eng, forced)
    start = [t.read(n, np.int32, a.size) for n, a in (("blen", t.len), ("btable", t.table), ("bring", t.ring), ("bstate", t.state))]
    t.put(0, adds[0])
    t.run()                                             # (once eagerly: every buffer exists)
    l = az.Runtime.record(t.run)
    for name, a in zip(("blen", "btable", "bring", "bstate"), start):
        getattr(t, name).write(a)
    for i, a in enumerate((t.c.q[0], t.c.q[1], t.c.d[0], t.c.d[1])):
        t.kv.buffer(i).write(a)
    for step, add in enumerate(adds):
        t.put(step, add)
        l.run()
        n = int(t.read("rows", np.int32, SEQS + 1)[-1])
        assert np.array_equal(t.read("token", np.int32, SEQS)[:n], seen[step][0])
        assert np.array_equal(t.read("prob", np.uint32, SEQS)[:n], seen[step][1]) and np.array_equal(t.read("blen", np.int32, SEQS), seen[step][2])
    assert np.array_equal(t.read("blen", np.int32, SEQS), lens)
    l.free()
    ref.free(t.hold)
    eng.close()
