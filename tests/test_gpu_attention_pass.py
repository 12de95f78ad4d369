"""The attention block's operators together, as a forward pass uses them: behind the q|k|v product, in front of the output projection; in
launch lists; on buffers of another allocator."""
import ctypes as C
import importlib.util
import os
import subprocess
import sys

if __name__ == "__main__":   # (a process of its own: torch's HIP runtime has to be the one that the library finds, so torch comes first)
    sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
    import torch
import numpy as np
import pytest

import arcinferzero_amd as az
import attn_ref as ref
import oracle_lib as orc
from common import make_acts, make_weights

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def eng(rt):
    e = az.Engine(512, 2048)
    yield e
    e.close()


def test_a_layer_prompt_then_tokens(eng):
    """Two sequences: prompts of odd lengths, then drafts of three tokens, then single ones.  Every operator is held to its own definition on
    what the one before really left on the GPU; the projections to the oracle."""
    E, heads, kv, hd, page, block = 512, 8, 2, 64, 32, 16
    w = (heads + 2 * kv) * hd
    W, O = make_weights(az.Q8_0, w, E, 1), make_weights(az.Q8_0, E, heads * hd, 2)
    wq, wo = eng.make_weight(az.Q8_0, w, E, W), eng.make_weight(az.Q8_0, E, heads * hd, O)
    freq, axis = [10000.0 ** (-i / 32) for i in range(32)], [0] * 32
    rope = eng.make_rope(freq)
    table = np.array([[3, 1, 6, 0, 7], [2, 8, 4, 5, 9]], np.int32)
    c = ref.Cache(10, page, block, kv, hd, seed=1)
    hold = []
    kvc = ref.device_cache(eng, c, hold)
    lens = np.zeros(2, np.int32)
    for step, counts in enumerate([(70, 41), (3, 3), (1, 1), (1, 1), (17, 2)]):
        T = sum(counts)
        Mp = (T + 15) // 16 * 16 if T < 128 else (T + 127) // 128 * 128
        rows = np.array([0, counts[0], T], np.int32)
        lens += np.array(counts, np.int32)
        pos = np.concatenate([np.arange(l - n, l) for n, l in zip(counts, lens)]).astype(np.int32)
        x = make_acts(T, E, seed=20 + step)
        res = az.gen_normal(70 + step, (Mp, E))
        b = [az.Runtime.from_numpy(a) for a in (x, rows, lens, table, pos, res)]
        qkv, out = az.Runtime.alloc(Mp * w * 4), az.Runtime.from_numpy(np.zeros((Mp, heads * hd), np.float32))
        batch = az.KvBatch(b[1], b[2], b[3], 2, 5, T, max(counts), int(lens.max()))
        eng.quantize(b[0], E, E, Mp, T)
        eng.matmul("qkv", wq, Mp, qkv, w)
        before = qkv.read(np.float32, T * w).reshape(T, heads + 2 * kv, hd)
        raq, rasc, _ = orc.quantize_act(np.concatenate([x, np.zeros((Mp - T, E), np.float32)]))
        want = orc.matmul_ref(az.Q8_0, W, w, E, raq[:T], rasc).reshape(before.shape)
        assert np.abs(before - want).max() <= 1e-5 * np.abs(want).max()
        # q and k turned where they lie, in one call
        eng.rope(rope, qkv, w, 0, qkv, w, 0, T, heads + kv, hd, b[4])
        after = qkv.read(np.float32, T * w).reshape(before.shape)
        turned = ref.rope(before[:, :heads + kv], pos[None], freq, axis, False)
        assert np.abs(after[:, :heads + kv] - turned).max() <= 8 * 2.0 ** -23 * np.abs(before).max()
        assert np.array_equal(after[:, heads + kv:], before[:, heads + kv:])
        eng.kv_write(kvc, batch, qkv, w, heads * hd, qkv, w, (heads + kv) * hd)
        for s in (0, 1):
            for which, h0 in ((0, heads), (1, heads + kv)):
                c.write(which, table[s], lens[s] - counts[s], after[rows[s]:rows[s + 1], h0:h0 + kv])
        q, d = ref.read_cache(kvc, c)
        assert np.array_equal(q, c.q) and np.array_equal(d, c.d)
        eng.attention(kvc, batch, qkv, w, 0, heads, out, heads * hd, 0, az.Attention(hd ** -0.5))
        y = out.read(np.float32, T * heads * hd).reshape(T, heads, hd)
        exact, tol, done = ref.attention(c, after[:, :heads], rows, lens, table, hd ** -0.5)
        assert done.all() and (np.abs(y - exact) <= tol).all()
        # the output projection, added to the residual
        eng.quantize(out, heads * hd, heads * hd, Mp, T)
        eng.matmul("o", wo, Mp, b[5], E, 0, 1)
        raq, rasc, _ = orc.quantize_act(np.concatenate([y.reshape(T, -1), np.zeros((Mp - T, heads * hd), np.float32)]))
        want = res[:T] + orc.matmul_ref(az.Q8_0, O, E, heads * hd, raq[:T], rasc)
        got = b[5].read(np.float32, T * E).reshape(T, E)
        assert np.abs(got - want).max() <= 1e-5 * np.abs(want).max()
        for m in b + [qkv, out]:
            m.free()
    ref.free(hold)
    for m in (rope, wq, wo):
        m.free()


class Step:
    """A pass of rope, kv_write and attention on buffers of its own, eager or recorded."""

    def __init__(self, eng, hold, n, heads=8, kv=2, hd=128, seed=0, pages=40, page=64):
        self.eng, self.n, self.heads, self.kv, self.hd, self.w = eng, n, heads, kv, hd, (heads + 2 * kv) * hd
        self.S, self.ldt = 2, pages // 2
        T = self.T = self.S * n
        self.c = ref.Cache(pages, page, 16, kv, hd, seed=seed)
        self.kvc = ref.device_cache(eng, self.c, hold)
        self.rope = eng.make_rope([10000.0 ** (-i / (hd // 2)) for i in range(hd // 2)])
        self.rows, self.len, self.table, self.pos, self.x, self.y, self.out = (
            az.Runtime.alloc(4 * k) for k in (self.S + 1, self.S, self.S * self.ldt, T, T * self.w, T * self.w, T * heads * hd))
        hold += [self.rope, self.rows, self.len, self.table, self.pos, self.x, self.y, self.out]
        self.batch = az.KvBatch(self.rows, self.len, self.table, self.S, self.ldt, T, n, pages // 2 * page)
        self.form = az.Attention(hd ** -0.5)

    def put(self, seed):
        """Another pass's rows, lengths and pages into the same buffers, and the cache as it was."""
        rng = np.random.default_rng(seed)
        lens = rng.integers(self.n, self.ldt * self.c.page, size=2).astype(np.int32)
        self.rows.write(np.array([0, self.n, 2 * self.n], np.int32))
        self.len.write(lens)
        self.table.write(rng.permutation(self.c.pages).astype(np.int32))
        self.pos.write(np.concatenate([np.arange(l - self.n, l) for l in lens]).astype(np.int32))
        self.x.write(rng.standard_normal((self.T, self.w)).astype(np.float32))
        for i, a in enumerate((self.c.q[0], self.c.q[1], self.c.d[0], self.c.d[1])):
            self.kvc.buffer(i).write(a)
        self.out.fill(0xFFFFFFFF)

    def run(self):
        e, h, k, hd, w = self.eng, self.heads, self.kv, self.hd, self.w
        e.rope(self.rope, self.x, w, 0, self.y, w, 0, self.T, h + 2 * k, hd, self.pos)
        e.kv_write(self.kvc, self.batch, self.y, w, h * hd, self.y, w, (h + k) * hd)
        e.attention(self.kvc, self.batch, self.y, w, 0, h, self.out, h * hd, 0, self.form)

    def got(self):
        return self.out.read(np.uint32), self.kvc.buffer(0).read(np.uint8), self.kvc.buffer(3).read(np.uint32)


def test_launch_lists_replay(eng):
    """Single tokens (pieces joined in the launch), drafts and chunks (pieces joined behind it), recorded once and replayed on new lengths, pages
    and rows, lists in turn on the engine's one room for pieces, with eager calls between: the eager results, bit for bit."""
    hold = []
    steps = [Step(eng, hold, n, seed=n) for n in (1, 5, 40)]
    for s in steps:
        s.put(1)
        s.run()
    lists = [az.Runtime.record(s.run) for s in steps]
    for turn in range(4):
        eager = []
        for i, s in enumerate(steps):
            s.put(10 * turn + i)
            s.run()
            eager.append(s.got())
        for i, s in enumerate(steps):
            s.put(10 * turn + i)
        for l in lists if turn % 2 else lists[::-1]:
            l.run()
        for s, e in zip(steps, eager):
            assert all(np.array_equal(a, b) for a, b in zip(s.got(), e))
        # a larger call than any recorded one: more room for pieces; the lists keep theirs
        big = []
        t = Step(eng, big, 3 + turn, heads=32, kv=8, hd=128, seed=3, pages=200)
        t.put(turn)
        t.run()
        first = t.got()
        for l in lists:
            l.run()
        t.put(turn)
        t.run()
        assert all(np.array_equal(a, b) for a, b in zip(t.got(), first))
        ref.free(big)
    with pytest.raises(az.ArczError):
        steps[0].kvc.buffer(0)          # (a handle only)
        hold[0].free()                  # a buffer of the cache that a list names
    for l in lists:
        l.free()
    ref.free(hold)


def test_nothing_is_allocated_while_recording(eng):
    """A call that needs more room than there is refuses to record, and the engine stays as it was."""
    e = az.Engine(16, 256)
    hold = []
    s = Step(e, hold, 1, seed=1)
    s.put(1)
    with pytest.raises(az.ArczError):
        az.Runtime.record(s.run)
    s.run()
    want = s.got()
    s.put(1)
    l = az.Runtime.record(s.run)
    l.run()
    assert all(np.array_equal(a, b) for a, b in zip(s.got(), want))
    l.free()
    ref.free(hold)
    e.close()


def test_two_engines_and_profile(eng):
    e = az.Engine(16, 256)
    hold, held = [], []
    a, b = Step(eng, hold, 1, seed=4), Step(e, held, 1, seed=4)
    for s in (a, b):
        s.put(3)
    e.profile(True)
    a.run()
    b.run()
    assert all(np.array_equal(x, y) for x, y in zip(a.got(), b.got()))
    e.profile_collect()
    e.profile(False)
    assert [e.profile_get(n)[1] for n in ("rope", "kv_write", "attention")] == [1, 1, 1]
    ref.free(hold)
    ref.free(held)
    e.close()


def test_buffers_of_another_allocator(eng):
    """Tensors of torch as buffers (below, in a process of its own)."""
    if importlib.util.find_spec("torch") is None:   # (not imported here: a second HIP runtime under the first one's name)
        pytest.skip("no torch")
    r = subprocess.run([sys.executable, os.path.abspath(__file__)], capture_output=True, text=True, timeout=110)
    assert r.returncode == 0 and "tensors as buffers: ok" in r.stdout, r.stdout[-2000:] + r.stderr[-4000:]


def tensors_as_buffers(eng):
    """The same results on torch's tensors; calls ordered with torch's default stream, and with another by events."""
    hold = []
    s = Step(eng, hold, 2, seed=6)
    s.put(8)
    s.run()
    want = s.got()[0]
    s.put(8)
    t = {n: torch.from_numpy(getattr(s, n).read(np.float32)).cuda() for n in ("x", "y", "out")}
    kept = [az.Runtime.wrap(t[n].data_ptr(), t[n].numel() * 4) for n in ("x", "y", "out")]
    s.x, s.y, s.out = kept
    # (what torch has queued on its default stream is done before the library's kernels, and they before what it queues next)
    t["out"].fill_(7.0)
    t["x"].mul_(2.0).mul_(0.5)
    s.run()
    again = t["out"].clone()
    assert np.array_equal(again.cpu().numpy().view(np.uint32), want)
    # another stream: ordered by its owner
    mine, theirs = torch.cuda.Stream(), torch.cuda.ExternalStream(az.Runtime.stream())
    s.put(8)
    torch.cuda.synchronize()
    x = t["x"].clone()
    with torch.cuda.stream(mine):
        t["x"].zero_()
        t["x"].add_(x)
    theirs.wait_stream(mine)
    s.run()
    mine.wait_stream(theirs)
    with torch.cuda.stream(mine):
        again = t["out"].clone()
    mine.synchronize()
    assert np.array_equal(again.cpu().numpy().view(np.uint32), want)
    # in a launch list
    s.put(8)
    l = az.Runtime.record(s.run)
    for _ in range(3):
        t["out"].fill_(3.0)
        s.put(8)
        l.run()
        assert np.array_equal(t["out"].cpu().numpy().view(np.uint32), want)
    l.free()
    v = kept[0].view(256, 256)
    assert np.array_equal(v.read(np.float32), t["x"].cpu().numpy()[64:128])
    v.free()
    for b in kept:
        b.free()
    # refused: host memory, past the allocation, nothing
    h = np.zeros(16, np.float32)
    big = torch.zeros(1 << 22, device="cuda")
    for ptr, n in ((h.ctypes.data, 64), (big.data_ptr(), 1 << 40), (0, 64), (big.data_ptr(), 0)):
        with pytest.raises(az.ArczError):
            az.Runtime.wrap(ptr, n)
    assert torch.equal(big + 1, torch.ones_like(big))     # (nothing of it is left behind as an error)
    ref.free(hold)


def test_null_handles_and_freed_ones(eng):
    """At the C boundary: an error, no exception and no launch."""
    lib, n = az.lib, az.lib.arcz_launch_count()
    hold = []
    s = Step(eng, hold, 1, seed=1)
    b, a, k = s.batch.at, s.form.at, s.kvc.h
    assert lib.arcz_engine_rope(eng.h, None, s.x.h, 64, 0, s.y.h, 64, 0, 1, 1, 64, s.pos.h, 1) == -100
    assert lib.arcz_engine_kv_write(eng.h, None, b, s.y.h, 64, 0, s.y.h, 64, 0) == -100
    assert lib.arcz_engine_kv_write(eng.h, k, None, s.y.h, 64, 0, s.y.h, 64, 0) == -100
    assert lib.arcz_engine_kv_read(eng.h, k, b, None, s.w, 0, s.y.h, s.w, 0) == -100
    assert lib.arcz_engine_attention(eng.h, None, b, s.y.h, s.w, 0, 8, s.out.h, 1024, 0, a) == -100
    assert lib.arcz_engine_attention(eng.h, k, b, s.y.h, s.w, 0, 8, s.out.h, 1024, 0, None) == -100
    assert lib.arcz_engine_attention(eng.h, k, b, s.y.h, s.w, 0, 8, None, 1024, 0, a) == -100
    assert lib.arcz_kv_free(eng.h, None) == 0 and lib.arcz_rope_free(eng.h, None) == 0
    assert not lib.arcz_kv_buffer(k, 4) and not lib.arcz_kv_buffer(None, 0)
    assert not lib.arcz_rope_create(eng.h, 2, None, None, 1, 0, C.c_float(1.0))
    assert lib.arcz_launch_count() == n
    ref.free(hold)


if __name__ == "__main__":
    torch.zeros(1, device="cuda")
    az.Runtime.init(0)
    engine = az.Engine(16, 256)
    tensors_as_buffers(engine)
    engine.close()
    print("tensors as buffers: ok", flush=True)
