"""The operators of a serving step around the products and the attention, as cases whose time can be taken and whose outputs can be
compared: where a pass's new tokens go, the norms of queries and keys with their rotation, attention for sequences that share a prefix,
and the token that a row of logits gives.

Each case is one operator on one batch.  With `own` the calls go through the framework's entry points (arcinferzero_amd.Engine); without
it they are computed from elementary torch operations.

  plan    new tokens of every sequence: rows, lengths, pages out of (and back into) a ring of free ones, positions, places in the cache
  norm    rows of f32 heads brought to unit mean square, weighted, turned by their positions; queries and keys side by side
  shared  the rows of every sequence against the keys in its pages; the sequences of a group have their first pages in common
  sample  a token from each row of logits: temperature, the k likeliest, the likeliest that make p, those above a part of the likeliest

listed() names twelve of them, draw() gives more of the same ranges.
"""
import math
import random

import numpy as np
import torch

own = False


def listed():
    return [
        # -- a pass's batch
        # a decode step: a token for each of 256 conversations
        dict(name="plan_256_tokens", op="plan", seqs=256, rows=1, old=4000, drop=0.0, page=64),
        # drafts of up to eight tokens, a quarter of the sequences takes rejected ones back
        dict(name="plan_drafts_taken_back", op="plan", seqs=777, rows=8, old=2500, drop=0.25, page=16),
        # a burst of ragged prompts
        dict(name="plan_1024_prompts", op="plan", seqs=1024, rows=500, old=1, drop=0.0, page=32),
        # -- norms of queries and keys with the rotation
        # one token of a decode step
        dict(name="norm_1", op="norm", T=1, heads=32, kv=8, hd=128, pairs=64, neighbours=False, axes=1, far=4000),
        # an odd number of tokens, half of each wide head turned, neighbouring values as pairs
        dict(name="norm_half_neighbours_777", op="norm", T=777, heads=16, kv=8, hd=256, pairs=64, neighbours=True, axes=1, far=1000000),
        # the largest prompt chunk
        dict(name="norm_8192", op="norm", T=8192, heads=32, kv=8, hd=128, pairs=64, neighbours=False, axes=1, far=3000),
        # -- attention behind shared prefixes
        # a few conversations behind one short system prompt
        dict(name="shared_5_tokens", op="shared", seqs=5, groups=1, rows=1, shared=1024, own=300, heads=32, kv=8, hd=128, page=64, block=64, form="causal"),
        # many answers to one long document
        dict(name="shared_128_tokens", op="shared", seqs=128, groups=1, rows=1, shared=16384, own=600, heads=32, kv=8, hd=128, page=64, block=64, form="causal"),
        # questions behind three documents, read for the first time; capped scores
        dict(name="shared_questions_3_groups", op="shared", seqs=24, groups=3, rows=90, shared=4000, own=250, heads=16, kv=8, hd=256, page=32, block=16, form="cap"),
        # -- tokens
        # one conversation, the usual cuts
        dict(name="sample_1", op="sample", T=1, V=151936, form="k_p"),
        # drafts of a smaller vocabulary, every row with cuts of its own, some greedy
        dict(name="sample_37_mixed", op="sample", T=37, V=32001, form="mixed"),
        # a large batch, the likeliest that make nine tenths
        dict(name="sample_256_p", op="sample", T=256, V=151936, form="p"),
    ]


FORMS = ("causal", "causal", "causal", "cap", "distance", "window")
SAMPLES = ("k_p", "p", "min_p", "temperature", "greedy", "mixed", "mixed")
MOST = {"plan": 1024 * 500, "norm": 8192 * 40 * 128, "shared": 1.3e11, "sample": 256 * 151936}


def _log(rng, lo, hi):
    """Whole numbers between lo and hi, even over the logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    while True:
        op = rng.choice(("plan", "norm", "shared", "shared", "sample", "sample"))
        if op == "plan":
            c = dict(op=op, seqs=_log(rng, 1, 4096), rows=1 if rng.random() < 0.4 else _log(rng, 2, 4096), old=_log(rng, 1, 16000),
                     drop=rng.choice((0.0, 0.0, 0.2, 0.5)), page=rng.choice((16, 32, 64, 128, 256)))
            if c["seqs"] * c["rows"] <= MOST["plan"] and c["seqs"] * (c["old"] + c["rows"]) <= 6e7:
                return c
            continue
        if op == "norm":
            hd = rng.choice((64, 80, 128, 128, 128, 256))
            kv = rng.choice((1, 2, 4, 8))
            c = dict(op=op, T=_log(rng, 1, 8192), heads=kv * rng.choice((1, 2, 4, 5, 8)), kv=kv, hd=hd, pairs=rng.choice((hd // 2, hd // 2, hd // 4, hd // 4 - 3)),
                     neighbours=rng.random() < 0.3, axes=rng.choice((1, 1, 3)), far=_log(rng, 100, 2000000))
            if c["T"] * (c["heads"] + kv) * hd <= MOST["norm"]:
                return c
            continue
        if op == "sample":
            c = dict(op=op, T=_log(rng, 1, 512), V=_log(rng, 1000, 262144), form=rng.choice(SAMPLES))
            if c["T"] * c["V"] <= MOST["sample"]:
                return c
            continue
        page = rng.choice((16, 32, 64, 128, 256))
        block = rng.choice([b for b in (1, 16, 32, 64, 128, 256) if b <= page])
        kv, hd = rng.choice((1, 2, 4, 8)), rng.choice((64, 128, 128, 128, 256))
        seqs = _log(rng, 2, 192)
        c = dict(op=op, seqs=seqs, groups=min(seqs, rng.choice((1, 1, 2, 5))), rows=rng.choice((1, 1, _log(rng, 2, 8), _log(rng, 8, 256))), shared=_log(rng, 300, 20000),
                 own=_log(rng, 20, 2000), heads=kv * rng.choice((1, 2, 4, 4, 5, 8, 8)), kv=kv, hd=hd, page=page, block=block, form=rng.choice(FORMS))
        c["own"] = max(c["own"], c["rows"])
        scores = seqs * c["rows"] * c["heads"] * (c["shared"] + c["own"])
        if work(c)["flops"] <= MOST["shared"] and scores <= 1.2e9 and seqs * (c["shared"] + c["own"]) * kv * hd <= 2.3e9 and seqs * c["own"] * kv * hd <= 3e8:
            return c


# ---------------------------------------------------------------- a batch's shapes
def _tokens(case):
    """(length before, change) of every sequence of a plan."""
    rng = random.Random(case["seqs"] * 1000003 + case["rows"] * 101 + case["old"])
    out = []
    for s in range(case["seqs"]):
        old = case["old"] if s == 0 else int(rng.uniform(0, case["old"] + 1))
        n = case["rows"] if s == 0 or case["rows"] == 1 else rng.randint(1, case["rows"])
        out.append((old, -min(old, n) if s and rng.random() < case["drop"] else n))
    return out


def _shape(case):
    """(group, shared positions, rows, keys) of every sequence behind shared prefixes: whole pages are shared."""
    rng = random.Random(case["seqs"] * 7919 + case["rows"] * 31 + case["shared"])
    page, n, out = case["page"], case["groups"], []
    shared = [max(page, int(case["shared"] * (1.0 if g == 0 else rng.uniform(0.2, 1.0))) // page * page) for g in range(n)]
    for s in range(case["seqs"]):
        g = s * n // case["seqs"]
        r = case["rows"] if s == 0 or case["rows"] <= 8 else max(1, int(case["rows"] * rng.uniform(0.1, 1.0)))
        out.append((g, shared[g], r, shared[g] + (case["own"] if s == 0 else max(r, int(case["own"] * rng.uniform(0.05, 1.0))))))
    return out


def _window(case):
    return 2048 if case["form"] == "window" else 0


def work(case):
    if case["op"] == "plan":
        t = _tokens(case)
        rows, page = sum(max(n, 0) for _, n in t), case["page"]
        pages = sum(abs(-(-(l + n) // page) - -(-l // page)) for l, n in t)
        # counts, lengths in and out, rows; a page out of the ring and into the table, or back; position and place of each row
        return {"bytes": 16 * len(t) + 8 * pages + 8 * rows, "flops": 4.0 * len(t) + 3.0 * rows}
    if case["op"] == "norm":
        h = case["T"] * (case["heads"] + case["kv"])
        return {"bytes": 8 * h * case["hd"] + 4 * case["axes"] * case["T"] + 8 * case["hd"], "flops": h * (4.0 * case["hd"] + 6.0 * case["pairs"])}
    if case["op"] == "sample":
        return {"bytes": 4 * case["T"] * case["V"] + 28 * case["T"], "flops": 4.0 * case["T"] * case["V"]}
    seqs, kv, hd, w = _shape(case), case["kv"], case["hd"], _window(case)
    rows, pairs, keys = sum(n for _, _, n, _ in seqs), 0, 0
    least = {}
    for g, p, n, l in seqs:
        for q in range(l - n, l):
            pairs += min(q + 1, w) if w else q + 1
        lo = max(0, l - n - w + 1) if w else 0
        keys += l - max(lo, p)
        least[g] = min(least.get(g, p), lo)
    keys += sum(p - min(least[g], p) for g, p in {(g, p) for g, p, _, _ in seqs})
    return {"bytes": 2 * kv * (keys * hd + 4 * keys / case["block"]) + 8 * rows * case["heads"] * hd, "flops": 4.0 * hd * case["heads"] * pairs}


# ---------------------------------------------------------------- inputs
class _State:
    def __init__(self, case):
        self.case, self.held = case, []

    def __del__(self):
        for h in reversed(self.held):
            h.free()


def _frequencies(case):
    return [10000.0 ** (-i / case["pairs"]) for i in range(case["pairs"])]


def _axes(case):
    """The axis of each pair: one for all, or the three in turn for the fast ones and time for the slow rest."""
    p = case["pairs"]
    return [0] * p if case["axes"] == 1 else [i % 3 if i < 3 * (p // 4) else 0 for i in range(p)]


def _quantized(x, block):
    """Rows [..., tokens, hd] in 8 bits with a scale for each block of tokens."""
    b = x.unflatten(-2, (-1, block))
    d = b.abs().amax((-1, -2)) / 127.0
    q = torch.round(b / d[..., None, None]).to(torch.int8).flatten(-3, -2)
    return q, d


def _ints(a):
    return torch.tensor(a, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    s = _State(case)

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda")

    def uniform(*shape):
        return torch.rand(shape, generator=g, device="cuda")

    {"plan": _prepare_plan, "norm": _prepare_norm, "shared": _prepare_shared, "sample": _prepare_sample}[case["op"]](s, seed, g, normal, uniform)
    if own:
        _handles(s)
    torch.cuda.synchronize()
    return s


def _prepare_plan(s, seed, g, normal, uniform):
    c, page = s.case, s.case["page"]
    t = _tokens(c)
    s.new = sum(max(n, 0) for _, n in t)
    s.T, s.max_rows = max(1, s.new), c["rows"]
    s.ldt = -(-max(max(l, l + n) for l, n in t) // page) + 2
    have = [-(-l // page) for l, _ in t]
    need = sum(max(0, -(-(l + n) // page) - h) for (l, n), h in zip(t, have))
    s.pages = sum(have) + need + 5
    # the pages in use, dealt out in no order; the free ones somewhere in the ring
    order = torch.randperm(s.pages, generator=g, device="cuda").int().cpu().numpy()
    table, at = np.full((c["seqs"], s.ldt), -1, np.int32), 0
    for i, h in enumerate(have):
        table[i, :h] = order[at:at + h]
        at += h
    head, free = seed % s.pages, order[at:]
    ring = np.full(s.pages, -1, np.int32)
    ring[(head + np.arange(free.size)) % s.pages] = free
    s.add, s.len0, s.table, s.ring = _ints([n for _, n in t]), _ints([l for l, _ in t]), torch.from_numpy(table).cuda(), torch.from_numpy(ring).cuda()
    s.state0 = _ints([head, free.size, 0, 0])
    s.rows, s.len, s.state = _ints([0] * (c["seqs"] + 1)), torch.zeros_like(s.len0), torch.zeros_like(s.state0)
    s.pos, s.slot = (torch.full((s.T,), -1, dtype=torch.int32, device="cuda") for _ in range(2))


def _prepare_norm(s, seed, g, normal, uniform):
    c = s.case
    T, h, hd = c["T"], c["heads"] + c["kv"], c["hd"]
    # the q and k columns of rows [q | k | v]; heads of unlike sizes
    s.ld = (h + c["kv"]) * hd
    s.x = (normal(T, h + c["kv"], hd) * (0.3 + 3.0 * uniform(1, h + c["kv"], 1))).view(T, s.ld)
    s.y = torch.empty((T, h * hd), device="cuda")
    s.wq, s.wk, s.eps = 1.0 + 0.2 * normal(hd), 1.0 + 0.2 * normal(hd), 1e-6
    t = torch.arange(T, device="cuda") + int(c["far"]) + seed % 17
    if c["axes"] == 1:
        s.pos = t[None].int()
    else:   # text in front, then a picture of 64 patches a row: time stands still, height and width run
        i, text = torch.arange(T, device="cuda"), T // 8
        at = (i - text).clamp_min(0)
        s.pos = torch.stack([torch.where(i < text, t, t[text]), torch.where(i < text, t, t[text] + at // 64), torch.where(i < text, t, t[text] + at % 64)]).int()


def _prepare_shared(s, seed, g, normal, uniform):
    c = s.case
    kv, hd, page, block, h = c["kv"], c["hd"], c["page"], c["block"], c["heads"]
    seqs = _shape(c)
    n = [r for _, _, r, _ in seqs]
    s.T, s.max_rows, s.max_len = sum(n), max(n), max(l for _, _, _, l in seqs)
    s.group_rows = max(sum(r for k, _, r, _ in seqs if k == j) for j in range(c["groups"]))
    s.prefix = [next(p for k, p, _, _ in seqs if k == j) for j in range(c["groups"])]
    own_pages = [-(-l // page) - p // page for _, p, _, l in seqs]
    s.pages = sum(p // page for p in s.prefix) + sum(own_pages) + 3
    order = torch.randperm(s.pages, generator=g, device="cuda").int().cpu()
    table, at, first = torch.full((len(seqs), -(-s.max_len // page)), -1, dtype=torch.int32), 0, []
    for p in s.prefix:
        first.append(order[at:at + p // page])
        at += p // page
    for i, ((k, p, _, _), m) in enumerate(zip(seqs, own_pages)):
        table[i, :p // page] = first[k]
        table[i, p // page:p // page + m] = order[at:at + m]
        at += m
    s.table, s.rows, s.len = table.cuda(), _ints(np.cumsum([0] + n)), _ints([l for _, _, _, l in seqs])
    s.groups, s.shared = _ints(np.cumsum([0] + [sum(k == j for k, _, _, _ in seqs) for j in range(c["groups"])])), _ints(s.prefix)
    # (keys have a few large columns)
    columns = 1.0 + 3.0 * (uniform(kv, 1, hd) < 0.04)
    s.kq, s.ks = _quantized(normal(s.pages, kv, page, hd) * columns, block)
    s.vq, s.vs = _quantized(normal(s.pages, kv, page, hd), block)
    s.ld = (h + 2 * kv) * hd
    s.x = normal(s.T, s.ld) * 1.3
    s.out = torch.empty((s.T, h * hd), device="cuda")
    s.scale, s.cap, s.slopes = hd ** -0.5, 30.0 if c["form"] == "cap" else 0.0, None
    if c["form"] == "distance":
        s.slopes = torch.tensor([2.0 ** (-8.0 * (i + 1) / h) for i in range(h)], device="cuda")


def _prepare_sample(s, seed, g, normal, uniform):
    c = s.case
    T, V, form = c["T"], c["V"], c["form"]
    # a broad floor and some tokens that stand out of it, a few hundredths of the vocabulary ruled out
    s.x = normal(T, V) * 2.5
    s.x -= torch.log(uniform(T, V).clamp_min(1e-6)) * (uniform(T, V) < 0.003) * 2.0
    s.x[uniform(T, V) < 0.02] = -math.inf
    s.u = uniform(T)
    s.temp, s.k, s.p, s.q = torch.ones(T, device="cuda"), torch.zeros(T, dtype=torch.int32, device="cuda"), torch.ones(T, device="cuda"), torch.zeros(T, device="cuda")
    if form in ("k_p", "p", "min_p", "temperature", "mixed"):
        s.temp = 0.6 + 0.6 * uniform(T)
    if form == "greedy":
        s.temp = torch.zeros(T, device="cuda")
    if form in ("k_p", "mixed"):
        s.k = (5 + 95 * uniform(T)).int()
    if form in ("k_p", "p", "mixed"):
        s.p = 0.8 + 0.19 * uniform(T)
    if form in ("min_p", "mixed"):
        s.q = 0.02 + 0.1 * uniform(T)
    if form == "mixed":
        i = torch.arange(T, device="cuda") + seed % 5
        s.k, s.p, s.q = torch.where(i % 2 == 0, s.k, torch.zeros_like(s.k)), torch.where(i % 3 == 0, s.p, torch.ones_like(s.p)), torch.where(i % 4 == 0, s.q, torch.zeros_like(s.q))
        s.temp = torch.where(i % 5 == 0, torch.zeros_like(s.temp), s.temp)
    s.token, s.prob = torch.empty(T, dtype=torch.int32, device="cuda"), torch.empty(T, device="cuda")


# ---------------------------------------------------------------- the framework's calls
_engine = None


def _handles(s):
    """What a program of the framework keeps: its engine, handles of the buffers, the cache, the batch, the rotation, a workspace."""
    global _engine
    import arcinferzero_amd as az
    az.Runtime.init(0)
    if _engine is None:
        _engine = az.Engine(16, 256)

    def keep(h):
        s.held.append(h)
        return h

    def wrap(t):
        return None if t is None else keep(az.Runtime.wrap(t.data_ptr(), t.numel() * t.element_size()))

    c = s.case
    if c["op"] == "plan":
        s.badd, s.blen0, s.bring, s.bstate0, s.bstate, s.bpos, s.bslot = (wrap(t) for t in (s.add, s.len0, s.ring, s.state0, s.state, s.pos, s.slot))
        s.batch = az.KvBatch(wrap(s.rows), wrap(s.len), wrap(s.table), c["seqs"], s.ldt, s.T, s.max_rows)
        s.plan = az.KvPlan(s.pages, c["page"], s.badd, s.blen0, s.bring, s.bstate0, s.bstate, s.bpos, s.bslot)
    elif c["op"] == "norm":
        s.bx, s.by, s.bwq, s.bwk, s.bpos = (wrap(t) for t in (s.x, s.y, s.wq, s.wk, s.pos))
        s.rope = keep(_engine.make_rope(_frequencies(c), _axes(c), c["neighbours"]))
    elif c["op"] == "sample":
        s.bx, s.bu, s.btoken, s.bprob = (wrap(t) for t in (s.x, s.u, s.token, s.prob))
        s.form = az.Sampling(wrap(s.temp), wrap(s.k), wrap(s.p), wrap(s.q))
    else:
        s.bx, s.bout = wrap(s.x), wrap(s.out)
        s.kvc = keep(_engine.make_kv(s.pages, c["page"], c["block"], c["kv"], c["hd"], wrap(s.kq), wrap(s.vq), wrap(s.ks), wrap(s.vs)))
        s.batch = az.KvBatch(wrap(s.rows), wrap(s.len), wrap(s.table), c["seqs"], s.table.shape[1], s.T, s.max_rows, s.max_len)
        s.groups_of = az.KvShared(wrap(s.groups), wrap(s.shared), c["groups"], s.group_rows, max(s.prefix))
        s.form = az.Attention(s.scale, s.cap, _window(c), wrap(s.slopes))
        s.room = keep(az.Runtime.alloc(_engine.attention_shared_room(s.kvc, s.batch, s.groups_of, c["heads"], s.form)))


def _run_own(s):
    c = s.case
    if c["op"] == "plan":
        _engine.kv_plan(s.batch, s.plan)
        return s.rows, s.len, s.table, s.ring, s.state, s.pos, s.slot
    if c["op"] == "norm":
        _engine.norm_rope(s.rope, s.bx, s.ld, 0, s.by, (c["heads"] + c["kv"]) * c["hd"], 0, c["T"], c["heads"], c["kv"], c["hd"], s.bwq, s.bwk, s.eps, s.bpos)
        return s.y
    if c["op"] == "sample":
        _engine.sample(s.bx, c["V"], 0, c["V"], c["T"], s.form, s.bu, s.btoken, s.bprob)
        return s.token, s.prob
    _engine.attention_shared(s.kvc, s.batch, s.groups_of, s.bx, s.ld, 0, c["heads"], s.bout, c["heads"] * c["hd"], 0, s.form, s.room)
    return s.out


# ---------------------------------------------------------------- the plain forms
def _plain_plan(s):
    c, page, S = s.case, s.case["page"], s.case["seqs"]
    new = s.add.clamp_min(0)
    to = (s.len0 + s.add).clamp_min(0)
    had, has = (s.len0 + page - 1) // page, (to + page - 1) // page
    s.rows[1:] = new.cumsum(0)
    s.len.copy_(to)
    head, count = s.state0[0].long(), s.state0[1].long()
    k = torch.arange(s.ldt, device="cuda")
    taken, given = (k >= had[:, None]) & (k < has[:, None]), (k >= has[:, None]) & (k < had[:, None])
    # (the n-th entry that is taken, or given back, in the order of the sequences)
    nth, back = taken.flatten().cumsum(0).view_as(taken), given.flatten().cumsum(0).view_as(given)
    total, freed = nth[-1, -1], back[-1, -1]
    fresh = s.ring[(head + nth - 1) % s.pages]
    j = torch.where(given, (head + count + back - 1) % s.pages, torch.full_like(back, s.pages))   # (behind the ring: nothing)
    grown = torch.cat([s.ring, s.ring[:1]]).scatter_(0, j.flatten(), s.table.flatten())
    s.ring.copy_(grown[:-1])
    s.table.copy_(torch.where(taken, fresh, s.table))
    s.state.copy_(torch.stack([(head + total) % s.pages, count - total + freed, torch.zeros_like(head), s.rows[-1].long()]))
    seq = torch.repeat_interleave(torch.arange(S, device="cuda"), new, output_size=s.new)
    pos = s.len0[seq] + torch.arange(s.new, device="cuda").int() - s.rows[seq]
    s.pos[:s.new] = pos
    s.slot[:s.new] = s.table[seq, (pos // page).long()] * page + pos % page
    return s.rows, s.len, s.table, s.ring, s.state, s.pos, s.slot


def _plain_norm(s):
    c = s.case
    T, h, hd, p = c["T"], c["heads"] + c["kv"], c["hd"], c["pairs"]
    freq = torch.tensor(_frequencies(c), dtype=torch.float64, device="cuda")
    angle = s.pos[torch.tensor(_axes(c), device="cuda")].T.double() * freq   # (far positions: 64 bits)
    co, si = angle.cos().float()[:, None], angle.sin().float()[:, None]
    x = s.x[:, :h * hd].reshape(T, h, hd)
    x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + s.eps)
    x[:, :c["heads"]] *= s.wq
    x[:, c["heads"]:] *= s.wk
    y = x.clone()
    a, b = (x[..., 0:2 * p:2], x[..., 1:2 * p:2]) if c["neighbours"] else (x[..., :p], x[..., p:2 * p])
    u, v = a * co - b * si, a * si + b * co
    if c["neighbours"]:
        y[..., 0:2 * p:2], y[..., 1:2 * p:2] = u, v
    else:
        y[..., :p], y[..., p:2 * p] = u, v
    return y.view(T, h * hd)


def _plain_shared(s):
    """Without the groups: each sequence against all of its keys, as many sequences at a time as memory holds."""
    c = s.case
    kv, hd, h, S, R, L = c["kv"], c["hd"], c["heads"], c["seqs"], s.max_rows, s.max_len
    G, parts = h // kv, []
    step = max(1, int(6e8 // (kv * L * (hd + R * G))))
    j = torch.arange(L, device="cuda")
    for s0 in range(0, S, step):
        s1 = min(S, s0 + step)
        n, l = (s.rows[s0 + 1:s1 + 1] - s.rows[s0:s1]).long()[:, None], s.len[s0:s1].long()[:, None]
        i = torch.arange(R, device="cuda")[None]
        row = (s.rows[s0:s1].long()[:, None] + i).clamp_max(s.T - 1)
        q = s.x[row, :h * hd].view(-1, R, kv, G, hd).permute(0, 2, 1, 3, 4).reshape(-1, kv, R * G, hd)
        pages = s.table[s0:s1].long().clamp_min(0)
        k, v = ((a[pages].float().unflatten(3, (-1, c["block"])) * d[pages][..., None, None]).flatten(3, 4).transpose(1, 2).reshape(s1 - s0, kv, -1, hd)[:, :, :L]
                for a, d in ((s.kq, s.ks), (s.vq, s.vs)))
        p = (l - n + i)[:, :, None]
        seen = (j < l[:, :, None]) & (j <= p)
        if _window(c):
            seen &= p - j < _window(c)
        a = ((q * s.scale) @ k.transpose(-1, -2).contiguous()).view(-1, kv, R, G, L)
        if s.cap:
            a = s.cap * torch.tanh(a / s.cap)
        if s.slopes is not None:
            a = a - s.slopes.view(kv, 1, G, 1) * (p - j).abs().float()[:, None, :, None]
        a = a.masked_fill(~seen[:, None, :, None], -math.inf)
        a = (a - a.amax(-1, keepdim=True).clamp_min(-3e38)).exp()
        a = a / a.sum(-1, keepdim=True).clamp_min(1e-37)
        o = (a.view(-1, kv, R * G, L) @ v).view(-1, kv, R, G, hd).permute(0, 2, 1, 3, 4).reshape(-1, R, h * hd)
        parts.append(o[i.expand(s1 - s0, R) < n])
    return torch.cat(parts)


def _plain_sample(s):
    """In 64 bits: a draw next to a border goes by the last digits of a running sum."""
    V = s.case["V"]
    top = s.x.amax(-1, keepdim=True)
    greedy = s.x.argmax(-1)
    w = ((s.x - top).double() / s.temp.double().clamp_min(1e-30)[:, None]).exp()
    order = torch.sort(s.x, dim=-1, descending=True, stable=True).indices
    sorted_w = w.gather(1, order)
    rank = torch.arange(V, device="cuda")
    k = torch.where(s.k > 0, s.k, V)[:, None]
    kept = (rank < k) & (sorted_w > 0)
    run = (sorted_w * kept).cumsum(-1)
    before = torch.cat([torch.zeros_like(run[:, :1]), run[:, :-1]], -1)
    kept &= (before < s.p.double()[:, None] * run[:, -1:]) | (s.p >= 1)[:, None] | (rank == 0)
    kept &= (sorted_w >= s.q.double()[:, None]) | (rank == 0)
    keep = torch.zeros_like(kept).scatter_(1, order, kept)
    w = w * keep
    run = w.cumsum(-1)
    i = (run <= s.u.double()[:, None] * run[:, -1:]).sum(-1)
    i = torch.where(s.temp > 0, i.clamp_max(V - 1), greedy)
    p = torch.where(s.temp > 0, w.gather(1, i[:, None])[:, 0] / run[:, -1], torch.ones_like(run[:, -1]))
    return i.int(), p.float()


def run(state):
    if own:
        return _run_own(state)
    return {"plan": _plain_plan, "norm": _plain_norm, "shared": _plain_shared, "sample": _plain_sample}[state.case["op"]](state)


# ---------------------------------------------------------------- the definitions in 64 bits
def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    return {"plan": _exact_plan, "norm": _exact_norm, "shared": _exact_shared, "sample": _exact_sample}[case["op"]](s)


def _exact_plan(s):
    c, page = s.case, s.case["page"]
    table, ring = s.table.cpu().numpy().copy(), s.ring.cpu().numpy().copy()
    head, count = (int(v) for v in s.state0[:2].cpu())
    rows, lens, pos, slot, back = [0], [], s.pos.cpu().numpy().copy(), s.slot.cpu().numpy().copy(), []
    for q, (l, n) in enumerate(_tokens(c)):
        to, at = max(0, l + n), rows[-1]
        for e in range(-(-l // page), -(-to // page)):
            table[q, e], head, count = ring[head], (head + 1) % s.pages, count - 1
        back += [table[q, e] for e in range(-(-to // page), -(-l // page))]
        if n > 0:
            p = np.arange(l, to)
            pos[at:at + n] = p
            slot[at:at + n] = table[q, p // page] * page + p % page
        rows.append(at + max(n, 0))
        lens.append(to)
    # (what this pass gives back comes behind all that was free before it)
    for i, v in enumerate(back):
        ring[(head + count + i) % s.pages] = v
    state = [head, count + len(back), 0, rows[-1]]
    return tuple(torch.from_numpy(np.asarray(a, np.int32)).cuda() for a in (rows, lens, table, ring, state, pos, slot))


def _exact_norm(s):
    c = s.case
    T, h, hd, p = c["T"], c["heads"] + c["kv"], c["hd"], c["pairs"]
    x = s.x.double().view(T, -1, hd)[:, :h]
    w = torch.cat([s.wq.double().expand(c["heads"], hd), s.wk.double().expand(c["kv"], hd)])
    y = x / torch.sqrt(x.square().sum(-1, keepdim=True) / hd + s.eps) * w
    x = y.clone()
    for i, (f, a) in enumerate(zip(_frequencies(c), _axes(c))):
        m, n = (2 * i, 2 * i + 1) if c["neighbours"] else (i, i + p)
        z = torch.polar(torch.ones(T, dtype=torch.float64, device="cuda"), s.pos[a].double() * f)[:, None] * torch.complex(x[..., m], x[..., n])
        y[..., m], y[..., n] = z.real, z.imag
    return y.reshape(T, -1)


def _exact_shared(s):
    c = s.case
    kv, hd, h, block = c["kv"], c["hd"], c["heads"], c["block"]
    G, out, at = h // kv, torch.empty((s.T, h, hd), dtype=torch.float64, device="cuda"), 0
    for i, (_, _, n, l) in enumerate(_shape(c)):
        pages = s.table[i, :-(-l // c["page"])].long()
        for g in range(kv):
            k, v = (a[pages, g].double().reshape(-1, hd)[:l] * d[pages, g].double().reshape(-1).repeat_interleave(block)[:l, None] for a, d in ((s.kq, s.ks), (s.vq, s.vs)))
            q = s.x[at:at + n, g * G * hd:(g + 1) * G * hd].double().reshape(n * G, hd)
            a = (q @ k.T.contiguous()).view(n, G, l) * s.scale
            p, j = torch.arange(l - n, l, device="cuda")[:, None], torch.arange(l, device="cuda")
            if s.cap:
                a = torch.tanh(a / s.cap) * s.cap
            if s.slopes is not None:
                a = a - s.slopes[g * G:(g + 1) * G].double()[:, None] * (p - j)[:, None]
            hidden = j > p
            if _window(c):
                hidden = hidden | (j <= p - _window(c))
            out[at:at + n, g * G:(g + 1) * G] = (torch.softmax(a.masked_fill(hidden[:, None], -math.inf), -1).view(n * G, l) @ v).view(n, G, hd)
        at += n
    return out.view(s.T, h * hd)


def _exact_sample(s):
    tokens, probs = [], []
    for r in range(s.case["T"]):
        x = s.x[r].cpu().double().numpy()
        t, k, p, q, u = (float(a[r]) for a in (s.temp, s.k, s.p, s.q, s.u))
        if not t > 0.0:
            tokens.append(int(np.argmax(x)))
            probs.append(1.0)
            continue
        order = np.lexsort((np.arange(x.size), -x))
        order = order[np.isfinite(x[order])][:int(k) if k > 0 else None]
        w = np.exp((x[order] - x[order[0]]) / t)
        if p < 1.0:
            order = order[:1 + int(np.searchsorted(np.cumsum(w), p * w.sum()))]
        w = w[:order.size]
        order = np.sort(order[(w >= q) | (order == order[0])])
        w = np.exp((x[order] - x.max()) / t)
        run = np.cumsum(w)
        i = min(int(np.searchsorted(run, u * run[-1], side="right")), order.size - 1)
        tokens.append(int(order[i]))
        probs.append(w[i] / run[-1])
    return torch.tensor(tokens, dtype=torch.int32, device="cuda"), torch.tensor(probs, dtype=torch.float64, device="cuda")
