"""Plans of sequences whose first pages are also others': their pages get no rows and are not lost (all whole numbers: equal)."""
import numpy as np
import pytest

import arcinferzero_amd as az
from test_gpu_kv_plan import Plan

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def eng(rt):
    e = az.Engine(16, 256)
    yield e
    e.close()


def refused(p, eng, add):
    """The plan changes nothing, and says so."""
    was = [a.copy() for a in (p.len, p.table, p.ring, p.state)]
    rows, lens, table, ring, after, pos, slot = p_run(p, eng, add)
    assert not rows.any() and np.array_equal(lens, was[0]) and np.array_equal(table, was[1]) and np.array_equal(ring, was[2])
    assert list(after) == [was[3][0], was[3][1], -1, 0] and (pos == -77).all() and (slot == -77).all()


def p_run(p, eng, add):
    """One plan, without a definition to hold it to."""
    hold = []

    def dev(a):
        hold.append(az.Runtime.from_numpy(np.ascontiguousarray(a, np.int32)))
        return hold[-1]
    fill = np.full(p.T, -77, np.int32)
    rows, lens, table, ring, state, adds, pos, slot, shared = (dev(a) for a in (np.full(p.seqs + 1, -3), p.len, p.table, p.ring, p.state, add, fill, fill, p.shared))
    print(f"plan of {p.seqs} sequences, add {list(add)}", flush=True)
    eng.kv_plan(az.KvBatch(rows, lens, table, p.seqs, p.ldt, p.T, p.max_rows), az.KvPlan(p.pages, p.page, adds, lens, ring, state, state, pos, slot, shared))
    got = [rows.read(np.int32), lens.read(np.int32), table.read(np.int32).reshape(p.table.shape), ring.read(np.int32), state.read(np.int32), pos.read(np.int32), slot.read(np.int32)]
    p.len, p.table, p.ring, p.state = got[1:5]
    for m in hold:
        m.free()
    return got


@pytest.mark.parametrize("max_rows", [8, 64])
def test_a_sequence_taken_back_into_its_prefix(eng, max_rows):
    """Pages of 16, 64 positions shared: down to 40, where tokens are refused, to none, where they are as well, and from 64 on again."""
    p = Plan([100, 70], 16, shared=[64, 64], max_rows=max_rows, seed=1)
    free = int(p.state[1])
    kept = p.table[0, :4].copy()
    p.run(eng, [-60, 1])
    assert p.len[0] == 40 and p.state[1] == free + 3 and np.array_equal(p.table[0, :4], kept)
    refused(p, eng, [1, 1])
    refused(p, eng, [8, 0])
    p.run(eng, [0, 1])                                     # (the others' tokens go on)
    p.run(eng, [-2 ** 31, 1])
    assert p.len[0] == 0 and p.state[1] == free + 3
    refused(p, eng, [1, 0])
    refused(p, eng, [min(max_rows, 64), 0])
    p.len[0] = 64
    p.run(eng, [1, 1])
    assert p.len[0] == 65 and np.array_equal(p.table[0, :4], kept)
    p.len[0], p.shared[0] = 40, 0                          # (nobody else's any more)
    p.run(eng, [5, 0])
    assert p.len[0] == 45


@pytest.mark.parametrize("seqs", [7, 1500])
def test_one_such_sequence_holds_back_the_plan(eng, seqs):
    """Also where it is no thread's first one; a prefix that ends within a page refuses its whole pages alone."""
    rng = np.random.default_rng(seqs)
    p = Plan(list(rng.integers(70, 130, size=seqs)), 16, shared=np.full(seqs, 69), T=3 * seqs, max_rows=3, pages=seqs * 12, ldt=12, seed=2)
    p.run(eng, rng.integers(0, 4, size=seqs))
    p.len[seqs - 1] = 64
    p.run(eng, rng.integers(1, 4, size=seqs))
    p.len[seqs - 1] = 63
    add = rng.integers(0, 4, size=seqs).astype(np.int32)
    add[seqs - 1] = 1
    refused(p, eng, add)
    add[seqs - 1] = -1
    p.run(eng, add)
    assert p.len[seqs - 1] == 62
