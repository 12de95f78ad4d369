"""Attention for sequences that share prefixes in groups, on the GPU against 64 bits (attn_ref.attention, which knows no groups, with its bounds:
the two parts of a row's keys are joined as pieces of keys are)."""
import os

import numpy as np
import pytest

import arcinferzero_amd as az
import attn_ref as ref

pytestmark = pytest.mark.gpu


def engine(way):
    """An engine that takes the parts apart always (1), never (0), or where it pays (None)."""
    if way is not None:
        os.environ["ARCZ_ATTN_SHARED"] = way
    try:
        return az.Engine(16, 256)
    finally:
        os.environ.pop("ARCZ_ATTN_SHARED", None)


@pytest.fixture(scope="module")
def eng(rt):
    e = engine("1")
    yield e
    e.close()


class Case:
    """Sequences of (rows, keys behind the prefix) in groups of (shared positions, sequences); shared[i] < 0: sequences of no group."""

    def __init__(self, groups, page=16, block=16, kv=2, hd=64, heads=4, seed=0, max_rows=None, group_rows=None, T=None):
        self.kv, self.hd, self.heads, self.page = kv, hd, heads, page
        seqs, self.groups, self.shared = [], [0], []
        for p, ss in groups:
            seqs += [(n, p + own) for n, own in ss]
            self.groups.append(len(seqs))
            self.shared.append(p)
        self.b = ref.Batch(seqs, page, seed=seed, T=T, max_rows=max_rows)
        self.c = ref.Cache(self.b.pages, page, block, kv, hd, seed=seed + 1)
        for g, (p, ss) in enumerate(groups):
            lead = self.b.table[self.groups[g]]
            for s in range(self.groups[g] + 1, self.groups[g + 1]):
                self.b.table[s, :p // page] = lead[:p // page]
                if p % page and self.b.table[s, p // page] >= 0:     # (the prefix ends within a page: each has a copy of it)
                    for a in (self.c.q, self.c.d):
                        a[:, self.b.table[s, p // page]] = a[:, lead[p // page]]
        self.group_rows = group_rows if group_rows is not None else max([1] + [sum(n for n, _ in ss) for _, ss in groups])
        self.x = np.random.default_rng(seed + 2).standard_normal((self.b.T, heads, hd)).astype(np.float32)

    def run(self, eng, cap=0.0, window=0, slopes=None, prefix=None, first=None, max_len=None, ld=None, off=0, again=1, plain=False):
        print(f"groups {self.groups} shared {self.shared} hd {self.hd} heads {self.heads}/{self.kv} page {self.page} cap {cap} window {window} T {self.b.T}", flush=True)
        hold = []
        w = self.heads * self.hd
        ld = ld or w
        kv, batch = ref.device_cache(eng, self.c, hold), self.b.device(hold)
        if max_len is not None:
            batch.max_len = max_len
        q = np.zeros((self.b.T, ld), np.float32)
        q[:, off:off + w] = self.x.reshape(self.b.T, w)

        def dev(a, t=np.int32):
            if a is None:
                return None
            hold.append(az.Runtime.from_numpy(np.ascontiguousarray(a, t)))
            return hold[-1]
        qb, out = dev(q, np.float32), dev(np.full((self.b.T, ld), 7.25), np.float32)
        form = az.Attention(0.11, cap, window, dev(slopes, np.float32), dev(prefix), dev(first))
        sh = az.KvShared(dev(self.groups), dev(self.shared + [0]), len(self.shared), self.group_rows, 0 if max_len == 0 else max([1] + self.shared))
        room = az.Runtime.alloc(eng.attention_shared_room(kv, batch, sh, self.heads, form))
        hold.append(room)
        got = None
        for _ in range(again):
            room.fill(0xFFFFFFFF)      # (whatever the workspace holds)
            eng.attention_shared(kv, batch, sh, qb, ld, off, self.heads, out, ld, off, form, room)
            y = out.read(np.float32).reshape(self.b.T, ld)
            assert got is None or np.array_equal(y.view(np.uint32), got.view(np.uint32))
            got = y
        rest = np.ones(ld, bool)
        rest[off:off + w] = False
        assert (got[:, rest] == 7.25).all()
        got = got[:, off:off + w].reshape(self.x.shape)
        want, tol, done = ref.attention(self.c, self.x, self.b.rows, self.b.lens, self.b.table, 0.11, cap, window, slopes, prefix, first, self.b.max_rows)
        for g in range(len(self.shared)):     # (rows past the group's most are left as they are)
            r0, r1 = self.b.rows[self.groups[g]], self.b.rows[self.groups[g + 1]]
            done[r0 + self.group_rows:r1] = False
        assert (np.abs(got - want) <= tol)[done].all(), (np.abs(got - want) / (tol + 1e-30))[done].max()
        assert (got[~done] == 7.25).all()
        ref.free(hold)
        return got


@pytest.mark.parametrize("hd,kv,heads", [(64, 2, 4), (128, 1, 5), (128, 2, 16), (256, 2, 6)])
@pytest.mark.parametrize("page,block", [(16, 1), (32, 16), (64, 64), (256, 32)])
def test_tokens_behind_one_prefix(eng, hd, kv, heads, page, block):
    Case([(2 * page + 300, [(1, 1 + 37 * i) for i in range(7)])], page, block, kv, hd, heads).run(eng)


@pytest.mark.parametrize("hd,kv,heads", [(64, 2, 4), (128, 2, 8), (256, 1, 3)])
@pytest.mark.parametrize("form", ["cap", "distance", "cap_distance", "window", "narrow_window", "prefix", "documents"])
def test_forms(eng, hd, kv, heads, form):
    """Whatever a row sees of both parts; a window that begins in either, rows before the prefix's end, documents that begin in it or behind it."""
    for rows in (1, 3, 40):
        k = Case([(200, [(rows, rows + 20 * i) for i in range(4)]), (90, [(rows, rows + 5), (1, 1)])], 32, 16, kv, hd, heads, seed=rows)
        kw = {}
        if "cap" in form:
            kw["cap"] = 9.0
        if "distance" in form:
            kw["slopes"] = np.linspace(0.01, 0.4, heads)
        if "window" in form:
            kw["window"] = 7 if "narrow" in form else 150
        if form == "prefix":
            kw["prefix"] = [k.b.lens[0], 10, 0, 230, 91, 2]
        if form == "documents":
            kw["first"] = np.random.default_rng(3).integers(0, 260, size=k.b.T)
        k.run(eng, **kw)


def test_prefixes_that_end_anywhere(eng):
    """Inside a page, a tile, a step; of one position, of none, longer than the sequence was before its rows."""
    for p in (0, 1, 15, 16, 17, 31, 33, 63, 100, 127):
        Case([(p, [(1, 1), (2, 40), (1, 300)])], 32, 8, 2, 64, 4, seed=p).run(eng)
    Case([(120, [(50, 0), (130, 20), (7, 7)])], 32, 32, 2, 128, 4).run(eng)     # (rows that lie in the prefix themselves)


def test_groups_of_all_sizes(eng):
    """One sequence, many, sequences of no group, groups without sequences; more rows than a tile of rows."""
    Case([(64, [(1, 5)])]).run(eng)
    Case([(256, [(1, 1 + i % 9) for i in range(150)])], 64, 32, 1, 128, 8).run(eng)
    Case([(256, [(9, 9 + i % 9) for i in range(33)]), (70, [(1, 3)]), (500, [(2, 2)] * 40)], 64, 32, 2, 128, 8).run(eng)
    k = Case([(64, [(1, 5), (1, 9)]), (64, [(1, 7)] * 3), (32, [(2, 3)])])
    k.groups, k.shared = [2, 2, 5], [900, 64]            # (an empty one; the first two and the last sequence in none)
    k.run(eng)
    k.groups, k.shared = [0], []                         # (no groups at all)
    k.run(eng)


def test_prompts_behind_a_prefix(eng):
    Case([(300, [(140, 140), (33, 60), (260, 300)]), (40, [(5, 90)])], 64, 64, 2, 128, 4).run(eng)
    Case([(300, [(70, 140), (33, 60)])], 16, 1, 1, 64, 7).run(eng, cap=20.0)
    Case([(130, [(70, 70), (33, 60)])], 16, 2, 1, 256, 2).run(eng)


def test_long_prefix(eng):
    """Enough keys for many pieces in both parts."""
    Case([(5000, [(1, 900 + i) for i in range(3)])], 128, 128, 1, 128, 4).run(eng, again=3)
    Case([(3000, [(2, 2000)])], 64, 16, 2, 64, 8).run(eng, again=2)


def test_columns_and_hints(eng):
    k = Case([(200, [(2, 30), (1, 70)]), (60, [(3, 9)])], 32, 8, 2, 64, 4)
    a = k.run(eng)
    for ld, off in ((300, 4), (301, 3), (256, 0)):
        assert np.array_equal(a.view(np.uint32), k.run(eng, ld=ld, off=off).view(np.uint32))
    k.run(eng, max_len=0)                                # (nothing known of the lengths)
    k.run(eng, max_len=1)


def test_rows_that_are_left_out(eng):
    Case([(100, [(3, 9), (5, 9), (1, 1)])], max_rows=2).run(eng)
    Case([(100, [(3, 9), (5, 9), (1, 1)]), (40, [(1, 1)])], group_rows=6).run(eng)
    Case([(100, [(3, 9), (5, 9)])], T=40).run(eng)       # (rows behind the last sequence)


def test_pages_that_are_none(eng):
    k = Case([(200, [(1, 30), (1, 70), (2, 9)])], 32, 16)
    for s in (1, 2):
        k.b.table[s, 2] = k.b.table[0, 2] = -1
    k.b.table[1, 7] = 2 ** 31 - 1
    k.run(eng)


def test_nonsense_in_the_buffers(eng):
    """Groups, lengths and rows that are none: nothing outside the buffers is looked at or written, and sound sequences come out right."""
    k = Case([(64, [(1, 40), (2, 9)]), (96, [(1, 3), (1, 30)])], 32, 16, T=12)
    hold = []
    kv, batch = ref.device_cache(eng, k.c, hold), k.b.device(hold)
    q = az.Runtime.from_numpy(k.x)
    form = az.Attention(0.11)
    guard = np.full((12 + 64, k.heads * k.hd), 7.25, np.float32)
    hold.append(q)
    for groups, shared in (([0, 2, 4], [-5, 2 ** 31 - 1]), ([-7, 2 ** 31 - 1, 3], [64, 64]), ([4, 2, 0], [64, 64]), ([1, 1, 1], [9, 9]), ([-2 ** 31, -1, 9], [64, -2 ** 31])):
        gb, sb, ob = (az.Runtime.from_numpy(np.array(a, t)) for a, t in ((groups, np.int32), (shared, np.int32), (guard, np.float32)))
        out = ob.view(32 * k.heads * k.hd * 4, 12 * k.heads * k.hd * 4)
        sh = az.KvShared(gb, sb, 2, 5, 96)
        room = az.Runtime.alloc(eng.attention_shared_room(kv, batch, sh, k.heads, form) + 512)
        room.fill(0x5A5A5A5A)
        print("groups", groups, "shared", shared, flush=True)
        eng.attention_shared(kv, batch, sh, q, k.heads * k.hd, 0, k.heads, out, k.heads * k.hd, 0, form, room)
        assert (room.read(np.uint32)[-128:] == 0x5A5A5A5A).all()
        y = ob.read(np.float32).reshape(guard.shape)
        assert (y[:32] == 7.25).all() and (y[32 + 5:] == 7.25).all()      # (five rows belong to sequences)
        for m in (out, gb, sb, ob, room):
            m.free()
    ref.free(hold)


def test_in_a_launch_list(eng):
    """Recorded once (nothing is allocated in a call), replayed on other rows, lengths and groups, with eager calls of the same workspace between."""
    cases = [Case([(p, [(1, 40 + i) for i in range(a)]), (320 - p, [(1, 7)] * (6 - a))], 32, 16, 2, 128, 8, seed=p) for p, a in ((160, 3), (64, 5), (256, 1))]
    hold = []
    pages = max(k.b.pages for k in cases)
    ldt = max(k.b.ldt for k in cases)
    k0 = cases[0]
    c = ref.Cache(pages, 32, 16, 2, 128, seed=1)
    kv = ref.device_cache(eng, c, hold)
    rows, lens, table, groups, shared = (az.Runtime.alloc(4 * n) for n in (7, 6, 6 * ldt, 3, 2))
    x, out = az.Runtime.alloc(k0.x.nbytes), az.Runtime.alloc(k0.x.nbytes)
    batch = az.KvBatch(rows, lens, table, 6, ldt, 6, 1, ldt * 32)
    sh = az.KvShared(groups, shared, 2, 6, 256)
    form = az.Attention(0.11)
    room = az.Runtime.alloc(eng.attention_shared_room(kv, batch, sh, 8, form))
    hold += [rows, lens, table, groups, shared, x, out, room]

    def put(k):
        t = np.full((6, ldt), -1, np.int32)
        t[:, :k.b.ldt] = k.b.table
        for b, a in ((rows, k.b.rows), (lens, k.b.lens), (table, t), (groups, np.array(k.groups, np.int32)), (shared, np.array(k.shared, np.int32)), (x, k.x)):
            b.write(a)
        out.fill(0xFFFFFFFF)

    def call():
        eng.attention_shared(kv, batch, sh, x, 1024, 0, 8, out, 1024, 0, form, room)
    put(k0)
    l = az.Runtime.record(call)
    for turn in range(2):
        for k in cases:
            put(k)
            call()
            want = out.read(np.uint32)
            put(k)
            l.run()
            assert np.array_equal(out.read(np.uint32), want)
            l.run()
            assert np.array_equal(out.read(np.uint32), want)
    with pytest.raises(az.ArczError):
        room.free()
    l.free()
    ref.free(hold)


def test_refusals(eng):
    k = Case([(64, [(1, 40), (2, 9)]), (96, [(1, 3), (1, 30)])], 32, 16)
    hold = []
    kv, batch = ref.device_cache(eng, k.c, hold), k.b.device(hold)
    w = k.heads * k.hd
    gb, sb = az.Runtime.from_numpy(np.array(k.groups, np.int32)), az.Runtime.from_numpy(np.array(k.shared, np.int32))
    q, out, form = az.Runtime.from_numpy(k.x), az.Runtime.alloc(k.x.nbytes), az.Attention(0.11)
    sh = az.KvShared(gb, sb, 2, 3, 96)
    n = eng.attention_shared_room(kv, batch, sh, k.heads, form)
    room, small, big = az.Runtime.alloc(n), az.Runtime.alloc(n - 16 if n > 80 else 64), az.Runtime.alloc(n + k.x.nbytes + 4096)
    hold += [gb, sb, q, out, room, small, big]
    launches = az.lib.arcz_launch_count()

    def view(m, at, size):
        hold.append(m.view(at, size))
        return hold[-1]

    def call(sh=sh, q=q, ldq=w, q_off=0, heads=k.heads, out=out, ldo=w, o_off=0, form=form, room=room):
        eng.attention_shared(kv, batch, sh, q, ldq, q_off, heads, out, ldo, o_off, form, room)

    def refused(**kw):
        with pytest.raises(az.ArczError):
            call(**kw)
    refused(room=view(small, 0, min(small.size, n - 16)))
    refused(room=view(big, 4, n))
    refused(heads=3)
    refused(heads=0)
    refused(ldq=w - 1)
    refused(q_off=1)
    refused(ldo=w - 1)
    refused(out=q)
    refused(out=kv.buffer(0))
    refused(out=view(big, 0, k.x.nbytes), room=view(big, 0, n))
    refused(q=view(big, 0, k.x.nbytes), room=view(big, 64, n))
    refused(sh=az.KvShared(gb, sb, 3, 3, 96))                      # (more groups than the buffers hold)
    refused(sh=az.KvShared(gb, sb, -1, 3, 96))
    refused(sh=az.KvShared(gb, sb, 2, -1, 96))
    refused(sh=az.KvShared(gb, sb, 2, 3, -1))
    refused(sh=az.KvShared(None, sb, 2, 3, 96))
    refused(sh=az.KvShared(gb, None, 2, 3, 96))
    refused(sh=az.KvShared(view(out, 0, 12), sb, 2, 3, 96))          # (out over the groups)
    refused(sh=az.KvShared(gb, view(room, 0, 8), 2, 3, 96))          # (the room over them)
    for f in (az.Attention(float("nan")), az.Attention(0.1, -1.0), az.Attention(0.1, 0.0, -1), az.Attention(0.1, 1e38), az.Attention(0.1, slopes=sb), az.Attention(0.1, first=sb)):
        refused(form=f)
    assert az.lib.arcz_launch_count() == launches
    lib = az.lib
    assert lib.arcz_engine_attention_shared_room(eng.h, None, batch.at, sh.at, 4, form.at) == 0
    assert lib.arcz_engine_attention_shared_room(eng.h, kv.h, batch.at, None, 4, form.at) == 0
    assert lib.arcz_engine_attention_shared(eng.h, kv.h, batch.at, sh.at, q.h, w, 0, 4, out.h, w, 0, None, room.h) == -100
    assert lib.arcz_engine_attention_shared(eng.h, kv.h, batch.at, sh.at, q.h, w, 0, 4, out.h, w, 0, form.at, None) == -100
    call()
    for s0 in (0, 4):     # (no sequences, no rows: nothing to do)
        e = az.KvBatch(*batch.held, s0, batch.ld_table, 0 if s0 else batch.T, batch.max_rows)
        eng.attention_shared(kv, e, sh, q, w, 0, k.heads, out, w, 0, form, room)
    assert az.lib.arcz_launch_count() == launches + 3
    ref.free(hold)


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("block", [1, 16, 64])
@pytest.mark.parametrize("form", range(4))
def test_every_kernel(eng, hd, block, form):
    """Every kernel of both parts, each with more steps than it has in its registers at once: 4, 12, 28 and 40 rows a sequence and head, 16 and 300 a group."""
    for heads, rows in ((4, 1), (4, 3), (7, 4), (8, 5)):
        k = Case([(330, [(rows, 310), (rows, 270), (1, 20)])], 64, block, 1, hd, heads, seed=hd + rows)
        k.run(eng, cap=11.0 if form & 1 else 0.0, slopes=np.linspace(0.002, 0.05, heads) if form & 2 else None)
    k = Case([(330, [(1, 3 + i % 5) for i in range(75)])], 64, block, 1, hd, 4, seed=hd)
    k.run(eng, cap=11.0 if form & 1 else 0.0, slopes=np.linspace(0.002, 0.05, 4) if form & 2 else None)


def test_where_it_pays(rt):
    """By the sizes alone that the caller names: a few sequences are one launch of attention as it is, many behind a long prefix the parts; the results
    are the same."""
    for groups, named, launches in (([(64, [(1, 5), (2, 9)])], 64, 1), ([(64, [(1, 30 + i % 7) for i in range(256)])], 9000, 3), ([(64, [(1, 30)])], 9000, 1)):
        k = Case(groups, 32, 16, 2, 128, 8)
        heads = 8
        got = []
        for way in (None, "1", "0"):
            e = engine(way)
            hold = []
            kvc, batch = ref.device_cache(e, k.c, hold), k.b.device(hold)
            batch.max_len = named + 40
            w = heads * 128
            q, out = az.Runtime.from_numpy(k.x), az.Runtime.alloc(k.x.nbytes)
            gb, sb = az.Runtime.from_numpy(np.array(k.groups, np.int32)), az.Runtime.from_numpy(np.array(k.shared, np.int32))
            sh, form = az.KvShared(gb, sb, len(k.shared), k.group_rows, named), az.Attention(0.05)
            room = az.Runtime.alloc(e.attention_shared_room(kvc, batch, sh, heads, form))
            hold += [q, out, gb, sb, room]
            n = az.lib.arcz_launch_count()
            e.attention_shared(kvc, batch, sh, q, w, 0, heads, out, w, 0, form, room)
            n = az.lib.arcz_launch_count() - n
            if way is None:
                print(groups[0][0], "launches", n, flush=True)
                first = n
            else:
                assert n == 3 if way == "1" else n == 1
            got.append(out.read(np.float32).reshape(k.x.shape))
            ref.free(hold)
            e.close()
        assert first == launches
        assert np.array_equal(got[0].view(np.uint32), got[1 if first == 3 else 2].view(np.uint32))
        only = {0, k.b.T - 1}
        want, tol, _ = ref.attention(k.c, k.x, k.b.rows, k.b.lens, k.b.table, 0.05, only=only)
        for y in got:
            assert all((np.abs(y[t] - want[t]) <= tol[t]).all() for t in only)
