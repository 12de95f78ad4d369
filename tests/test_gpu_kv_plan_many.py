"""Plans whose rows and pages the work-group shares out (more than eight rows a sequence): one sequence a thread and several rounds of them, positions
and places in the same launch and in one of their own, pages taken and given back in one plan, the ring's end inside it; counts that pass 2^20
of one sequence."""
import numpy as np
import pytest

import arcinferzero_amd as az
from test_gpu_kv_plan import Plan
from test_gpu_kv_plan_shared import p_run

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def eng(rt):
    e = az.Engine(16, 256)
    yield e
    e.close()


@pytest.mark.parametrize("seqs", [1, 255, 256, 257, 1023, 1024, 1025, 2500])
@pytest.mark.parametrize("max_rows", [8, 9, 40])
@pytest.mark.parametrize("few", [False, True])
def test_shared_out(eng, seqs, max_rows, few):
    """few: no more rows than one launch places; else as many as there may be.  Every plan takes, gives and leaves alone."""
    rng = np.random.default_rng(seqs * 100 + max_rows)
    T = min(seqs * max_rows, 1024 if max_rows > 8 else 2048) if few else seqs * max_rows
    p = Plan(list(rng.integers(0, 130, size=seqs)), 16, T=max(T, 1), max_rows=max_rows, pages=seqs * 14 + 9, ldt=14, seed=seqs, head=seqs * 14 + 3, own=True)

    def adds(give):
        a = rng.integers(0, max_rows + 1, size=seqs)
        if few:      # (as many sequences with rows as fit)
            a[rng.permutation(seqs)[max(1, T // max_rows):]] = 0
        a = np.where(p.len + a > 14 * 16, 0, a)
        return np.where(rng.random(seqs) < give, -rng.integers(1, 90, size=seqs), a)
    for give in (0.0, 0.4, 0.1, 0.7):
        got = p.run(eng, adds(give))
        assert got[4][2] == 0
    p.run(eng, adds(0.3), want_slot=False)
    p.run(eng, adds(0.3), want_pos=False)
    p.run(eng, np.full(seqs, -2 ** 31))
    assert (p.len == 0).all() and p.state[1] == p.pages


@pytest.mark.parametrize("seqs", [3, 300, 1500])
def test_all_rows_in_one_sequence(eng, seqs):
    """One prompt among sequences of nothing: every row is found in it, wherever it stands."""
    for at in (0, seqs // 2, seqs - 1):
        p = Plan([5] * seqs, 16, T=900, max_rows=900, pages=seqs + 90, ldt=64, seed=at)
        add = np.zeros(seqs, np.int32)
        add[at] = 900
        got = p.run(eng, add)
        assert got[4][2] == 0 and got[0][at] == 0 and got[0][at + 1] == 900


def test_counts_past_2_20(eng):
    """Sums in 64 bits where a sequence alone has more than 2^20 rows, takes or gives: a plan of it, and ones that do not fit."""
    n = (1 << 20) + 70
    for seqs, at in ((2, 0), (300, 299)):
        p = Plan([3] * seqs, 16, T=n + 8, max_rows=n, pages=n // 16 + seqs + 20, ldt=n // 16 + 4, seed=at)
        add = np.zeros(seqs, np.int64)
        add[at] = n
        short = Plan([3] * seqs, 16, T=n - 1, max_rows=n, pages=n // 16 + seqs + 20, ldt=n // 16 + 4, seed=at)
        got = short.run(eng, add)
        assert got[4][2] == -1 and not got[0].any()
        got = p.run(eng, add)
        assert got[4][2] == 0 and p.len[at] == n + 3
        add[at] = -n
        got = p.run(eng, add)
        assert got[4][2] == 0 and p.len[at] == 3


def test_rows_whose_sum_passes_32_bits(eng):
    p = Plan([0, 0, 9], 256, T=1000, max_rows=2 ** 31 - 1, pages=50, ldt=(2 ** 31 - 4096) // 256, shared=[0, 0, 0])
    was = [a.copy() for a in (p.len, p.ring, p.state)]
    rows, lens, _, ring, after, pos, slot = p_run(p, eng, [2 ** 31 - 5000, 2 ** 31 - 5000, 1])
    assert not rows.any() and np.array_equal(lens, was[0]) and np.array_equal(ring, was[1]) and list(after) == [was[2][0], was[2][1], -1, 0]
    assert (pos == -77).all() and (slot == -77).all()
