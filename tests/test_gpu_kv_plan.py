"""A pass's batch made on the GPU against a plain walk over the sequences (all whole numbers: equal)."""
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


def walk(add, before, table, ring, state, shared, page, T, max_rows):
    """The definition: (rows, len, table, ring, after, pos, slot of the rows), a sequence and a page at a time."""
    pages, most = len(ring), table.shape[1] * page
    table, ring, (head, count) = table.copy(), ring.copy(), (int(v) for v in state[:2])
    rows, lens, pos, slot, back, bad = [0], [], [], [], [], False
    take = [0]
    held = [min(max(int(b), 0), most) for b in before]
    for s, (b, a) in enumerate(zip(held, (int(v) for v in add))):
        bad |= a > max_rows or b + a > most
        to = max(0, b + a)
        for e in range(-(-b // page), -(-to // page)):
            take.append((s, e))
        keep = 0 if shared is None else min(max(int(shared[s]), 0), most) // page
        back += [(s, e) for e in range(max(-(-to // page), keep), -(-b // page))]
        rows.append(rows[-1] + max(a, 0))
        lens.append(to)
        pos += list(range(b, b + max(a, 0)))
    take = take[1:]
    bad |= rows[-1] > T or not 0 <= head < pages or not 0 <= count <= pages or count + len(back) > pages
    short = -1 if bad else max(0, len(take) - count)
    if short:
        return [0] * (len(add) + 1), list(before), table, ring, [int(state[0]), int(state[1]), short, 0], [], []
    for i, (s, e) in enumerate(back):
        ring[(head + count + i) % pages] = table[s, e]
    for i, (s, e) in enumerate(take):
        table[s, e] = ring[(head + i) % pages]
    for s in range(len(add)):
        for p in pos[rows[s]:rows[s + 1]]:
            pg = table[s, p // page]
            slot.append(pg * page + p % page if 0 <= pg < pages else -1)
    return rows, lens, table, ring, [(head + len(take)) % pages, count - len(take) + len(back), 0, rows[-1]], pos, slot


class Plan:
    """A batch's buffers; pages in use dealt out in no order, the free ones from `head` on."""

    def __init__(self, lens, page, pages=None, ldt=None, head=0, T=64, max_rows=64, seed=0, shared=None, own=False):
        rng = np.random.default_rng(seed)
        self.page, self.T, self.max_rows, self.seqs = page, T, max_rows, len(lens)
        have = [-(-l // page) for l in lens]
        self.ldt = ldt or max(have) + 4
        self.pages = pages or sum(have) + 40
        order = rng.permutation(self.pages).astype(np.int32)
        self.table, at = np.full((len(lens), self.ldt), -7, np.int32), 0
        for s, n in enumerate(have):
            self.table[s, :n] = order[at:at + n]
            at += n
        self.ring = np.full(self.pages, -9, np.int32)
        free = order[at:]
        self.ring[(head + np.arange(free.size)) % self.pages] = free
        self.len, self.state = np.array(lens, np.int32), np.array([head, free.size, 5, 5], np.int32)
        self.shared = None if shared is None else np.array(shared, np.int32)
        self.own = own     # lengths and state in buffers of their own, or brought on in place

    def run(self, eng, add, want_pos=True, want_slot=True, launch=None):
        hold = []

        def dev(a):
            hold.append(az.Runtime.from_numpy(np.ascontiguousarray(a, np.int32)))
            return hold[-1]
        fill = np.full(max(self.T, 1), -77, np.int32)
        rows, table, ring = dev(np.full(self.seqs + 1, -3)), dev(self.table), dev(self.ring)
        before, state, adds, pos, slot = dev(self.len), dev(self.state), dev(add), dev(fill), dev(fill)
        lens, after = (dev(np.full(self.seqs, -3)), dev(np.full(4, -3))) if self.own else (before, state)
        batch = az.KvBatch(rows, lens, table, self.seqs, self.ldt, self.T, self.max_rows)
        plan = az.KvPlan(self.pages, self.page, adds, before, ring, state, after, pos if want_pos else None, slot if want_slot else None,
                         None if self.shared is None else dev(self.shared))
        print(f"plan of {self.seqs} sequences, {self.T} rows, pages of {self.page}", flush=True)
        eng.kv_plan(batch, plan)
        got = [rows.read(np.int32), lens.read(np.int32), table.read(np.int32).reshape(self.table.shape), ring.read(np.int32), after.read(np.int32), pos.read(np.int32), slot.read(np.int32)]
        want = list(walk(add, self.len, self.table, self.ring, self.state, self.shared, self.page, self.T, self.max_rows))
        for i, given in ((5, want_pos), (6, want_slot)):
            full = fill.copy()
            if given:
                full[:len(want[i])] = want[i]
            want[i] = full
        for name, g, w in zip("rows len table ring after pos slot".split(), got, want):
            assert np.array_equal(g, np.asarray(w, np.int32)), (name, g, w)
        if self.own:
            assert np.array_equal(before.read(np.int32), self.len) and np.array_equal(state.read(np.int32), self.state)
        self.len, self.table, self.ring, self.state = got[1], got[2], got[3], got[4]
        ref.free(hold)
        return got


@pytest.mark.parametrize("page", [16, 64, 256])
@pytest.mark.parametrize("own", [False, True])
def test_tokens_prompts_and_ends(eng, page, own):
    """A conversation's life in many plans one behind the other: prompts, tokens, drafts taken back, sequences that end and begin again."""
    rng = np.random.default_rng(page)
    p = Plan([0, 1, page - 1, page, page + 1, 3 * page, 5], page, pages=61, ldt=12, head=58, T=300, max_rows=200, own=own)
    for step in range(25):
        add = np.array([rng.choice([0, 1, 1, 1, -1, -3, int(rng.integers(1, 40)), -2 ** 31, 8 - int(l) if l > 8 else 2]) for l in p.len], np.int64).astype(np.int32)
        p.run(eng, add)
    assert (p.len >= 0).all()


def test_one_sequence_one_token(eng):
    p = Plan([0], 64, pages=3, ldt=2, T=1, max_rows=1)
    for n in range(1, 129):
        p.run(eng, [1])
        assert p.len[0] == n
    got = p.run(eng, [1])          # the table's row is full
    assert got[4][2] == -1 and p.len[0] == 128


@pytest.mark.parametrize("seqs", [1023, 1024, 1025, 2500])
@pytest.mark.parametrize("rows", [1, 7])
def test_many_sequences(eng, seqs, rows):
    """More sequences than the work-group has threads; the places of many rows are a launch of their own."""
    rng = np.random.default_rng(seqs)
    p = Plan(list(rng.integers(0, 70, size=seqs)), 16, T=seqs * rows + 3, max_rows=rows, pages=seqs * 8, ldt=8, seed=seqs, own=True)
    p.run(eng, rng.integers(1, rows + 1, size=seqs))
    p.run(eng, np.where(rng.random(seqs) < 0.4, -rng.integers(1, 60, size=seqs), rng.integers(0, rows + 1, size=seqs)))
    p.run(eng, np.full(seqs, rows), want_slot=False)
    p.run(eng, np.full(seqs, -2 ** 31))
    assert (p.len == 0).all()


def test_long_prompts(eng):
    p = Plan([0, 3, 200], 32, T=30000, max_rows=20000, pages=1200, ldt=700, own=True)
    p.run(eng, [20000, 1, 9000])
    p.run(eng, [1, 1, 1], want_pos=False)
    p.run(eng, [-19000, 0, 5000])


def test_shared_pages_stay(eng):
    """A prefix that others use too is not given back with the sequence; the page that it ends within is the sequence's own."""
    p = Plan([300, 300, 40, 64], 64, shared=[256, 130, 1000, -5], seed=3)
    got = p.run(eng, [-300, -300, -40, -64])
    assert got[4][1] == 40 + 1 + 3 + 0 + 1


def test_all_or_nothing(eng):
    for lens, add, kw in (([60, 60], [10, 10], dict(pages=3)),                    # one page for two
                          ([60, 60], [10, 4], dict(pages=2)),                     # none for one
                          ([0], [65], dict(max_rows=64)),                         # more than the caller has room for
                          ([3, 3], [40, 40], dict(T=79)),                         # more rows than the buffers have
                          ([100, 5], [200, 1], dict(ldt=4, T=300, max_rows=300))):  # a longer sequence than the table has
        p = Plan(lens, 64, **kw)
        was = p.len.copy()
        got = p.run(eng, add)
        assert got[4][2] != 0 and not got[0].any() and np.array_equal(got[1], was)
    assert got[4][2] == -1
    p = Plan([60, 60], 64, pages=3)
    assert p.run(eng, [10, 10])[4][2] == 1 and p.run(eng, [10, -60])[4][2] == 0


def test_nonsense_in_the_buffers(eng):
    """Lengths, counts and a ring that are none: nothing outside the buffers is looked at or written."""
    for state in ([-1, 3, 0, 0], [50, 3, 0, 0], [0, 51, 0, 0], [0, -1, 0, 0], [2 ** 31 - 1, 2 ** 31 - 1, 0, 0], [3, 50, 0, 0]):
        p = Plan([10, 70], 64, pages=50)
        p.state = np.array(state, np.int32)
        p.run(eng, [1, -70])
    p = Plan([10, 70, 4, 4], 64, pages=50)
    p.len = np.array([-5, 2 ** 31 - 1, -2 ** 31, 300], np.int32)
    p.run(eng, [1, 0, 5, -1])
    p = Plan([10, 70], 64, pages=50)
    p.run(eng, [2 ** 31 - 1, 1])
    p.ring[:] = 2 ** 31 - 1       # pages of no cache: no places
    p.run(eng, [1, 60])
    assert (p.state[2] == 0) and p.table[1, 2] == 2 ** 31 - 1


def test_in_a_launch_list(eng):
    """A decode loop's plan recorded once, replayed with lengths, table and ring brought on where they are, other calls between."""
    rng = np.random.default_rng(8)
    p = Plan(list(rng.integers(0, 200, size=9)), 16, pages=300, ldt=40, T=40, max_rows=4)
    b = {n: az.Runtime.from_numpy(np.ascontiguousarray(a, np.int32)) for n, a in
         dict(rows=np.zeros(10), len=p.len, table=p.table, ring=p.ring, state=p.state, add=np.ones(9), pos=np.full(40, -1), slot=np.full(40, -1)).items()}
    batch = az.KvBatch(b["rows"], b["len"], b["table"], 9, 40, 40, 4)
    plan = az.KvPlan(300, 16, b["add"], b["len"], b["ring"], b["state"], b["state"], b["pos"], b["slot"])
    l = az.Runtime.record(lambda: eng.kv_plan(batch, plan))
    assert l.launches == 1
    pos, slot = np.full(40, -1, np.int32), np.full(40, -1, np.int32)
    for step in range(12):
        add = rng.choice([0, 1, 1, 4, -3], size=9).astype(np.int32)
        b["add"].write(add)
        l.run()
        rows, p.len, p.table, p.ring, p.state, wp, ws = walk(add, p.len, p.table, p.ring, p.state, None, 16, 40, 4)
        pos[:len(wp)], slot[:len(ws)] = wp, ws
        p.len, p.state = np.array(p.len, np.int32), np.array(p.state, np.int32)
        for n, w in (("rows", rows), ("len", p.len), ("table", p.table.ravel()), ("ring", p.ring), ("state", p.state), ("pos", pos), ("slot", slot)):
            assert np.array_equal(b[n].read(np.int32), np.asarray(w, np.int32)), (step, n)
        eng.kv_plan(az.KvBatch(b["rows"], b["len"], b["table"], 0, 40, 40, 4), plan)     # (no sequences: nothing)
    l.free()
    for m in b.values():
        m.free()


def test_refusals(eng):
    n = {k: az.Runtime.alloc(4 * 64) for k in ("rows", "len", "table", "add", "before", "ring", "state", "after", "pos", "slot", "shared")}
    small = az.Runtime.alloc(64)     # (16 values)
    big = az.Runtime.alloc(4 * 600)
    for m in n.values():
        m.fill(0)
    launches = az.lib.arcz_launch_count()

    def call(seqs=20, ldt=3, T=60, max_rows=5, pages=64, page=16, **k):
        d = {**n, **k}
        eng.kv_plan(az.KvBatch(d["rows"], d["len"], d["table"], seqs, ldt, T, max_rows),
                    az.KvPlan(pages, page, d["add"], d["before"], d["ring"], d["state"], d["after"], d["pos"], d["slot"], d["shared"]))

    def refused(**k):
        with pytest.raises(az.ArczError):
            call(**k)
    for name in ("rows", "len", "table", "add", "before", "ring", "pos", "slot", "shared"):
        refused(**{name: small})
    view = big.view(0, 8)
    refused(state=view)
    refused(after=view)
    for kw in (dict(page=15), dict(page=512), dict(page=48), dict(pages=0), dict(pages=-4), dict(pages=65), dict(seqs=-1), dict(seqs=65536), dict(T=-1), dict(T=65), dict(max_rows=-1),
               dict(ldt=0), dict(ldt=4), dict(ldt=1 << 30)):
        refused(**kw)
    a, c, d = big.view(0, 256), big.view(64, 256), big.view(8, 256)     # (partly over one another: 20 lengths take 80 bytes, a state 16)
    refused(len=a, before=c)
    refused(state=a, after=d)
    refused(rows=a, pos=c)
    refused(add=a, slot=c)
    for x, y in (("rows", "len"), ("pos", "slot"), ("table", "ring"), ("add", "rows"), ("shared", "len"), ("before", "table"), ("state", "ring"), ("add", "after")):
        refused(**{x: a, y: a})
    for name in ("rows", "len", "table", "add", "before", "ring", "state", "after"):
        with pytest.raises((az.ArczError, AttributeError)):
            call(**{name: None})
    assert az.lib.arcz_launch_count() == launches
    huge = az.Runtime.alloc(4 << 23)
    refused(pages=1 << 23, page=256, ring=huge)     # (2^31 places)
    call(pages=1 << 23, page=256, ring=huge, slot=None)
    call(seqs=0, rows=small)
    call()
    for m in list(n.values()) + [small, view, a, c, d, big, huge]:
        m.free()
