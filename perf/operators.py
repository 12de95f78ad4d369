"""The attention block's operators between the q|k|v product and the output projection, as cases whose time can be taken and
whose outputs can be compared: rotary positions, the 8-bit cache written and read back, attention over that cache.

Each case is one operator on one batch.  With `own` the calls go through the framework's entry points (arcinferzero_amd.Engine);
without it they are computed from elementary torch operations in 32 bits.

  rope   rows of f32 heads turned by their positions on one axis (text) or three (time, height, width: images and video)
  cache  the new rows of every sequence written into its pages, quantized, and the blocks that they touched read back
  attn   the rows of every sequence against the keys in its pages

listed() names twelve of them, draw() gives more of the same ranges.
"""
import math
import random

import numpy as np
import torch

own = False


def listed():
    return [
        # -- rotary positions
        # one token of a decode step, 32 query heads and 8 of keys: as short as a call gets
        dict(name="rope_1", op="rope", T=1, heads=40, hd=128, pairs=64, neighbours=False, axes=1, far=4000),
        # a prompt chunk of images among text: three axes dealt out over the pairs in turn
        dict(name="rope_3_axes_4096", op="rope", T=4096, heads=48, hd=128, pairs=64, neighbours=False, axes=3, far=4096),
        # an odd number of tokens far behind in a long context, half of each head turned, neighbouring values as pairs
        dict(name="rope_half_neighbours_777", op="rope", T=777, heads=36, hd=128, pairs=32, neighbours=True, axes=1, far=1000000),
        # -- the cache: written, the touched blocks read back
        # a decode step of 48 sequences: a token each, into blocks that hold older ones
        dict(name="cache_48_tokens", op="cache", seqs=48, rows=1, len=4000, kv=8, hd=128, page=64, block=64),
        # ragged prompts, a scale for every token
        dict(name="cache_ragged_prompts", op="cache", seqs=5, rows=1100, len=1700, kv=4, hd=256, page=32, block=1),
        # the largest chunk of a prompt, scales for blocks of 32 tokens
        dict(name="cache_chunk_8192", op="cache", seqs=1, rows=8192, len=12293, kv=8, hd=128, page=256, block=32),
        # -- attention
        # one token of a young conversation: latency alone
        dict(name="attn_1_token_at_517", op="attn", seqs=1, rows=1, len=517, heads=32, kv=8, hd=128, page=64, block=64, form="causal"),
        # one token behind a long document: the cache read once
        dict(name="attn_1_token_at_131072", op="attn", seqs=1, rows=1, len=131072, heads=40, kv=8, hd=128, page=64, block=64, form="causal"),
        # a batch of decoding sequences of every age
        dict(name="attn_64_tokens_ragged", op="attn", seqs=64, rows=1, len=8100, heads=32, kv=4, hd=128, page=32, block=16, form="causal"),
        # eight drafted tokens of four sequences, capped scores and a window, wide heads
        dict(name="attn_8_drafts_capped_window", op="attn", seqs=4, rows=8, len=6000, heads=16, kv=8, hd=256, page=16, block=16, form="cap_window"),
        # ragged prompts packed from several documents each
        dict(name="attn_documents_ragged", op="attn", seqs=3, rows=1333, len=1400, heads=40, kv=8, hd=128, page=128, block=128, form="documents"),
        # the largest prompt chunk, causal over itself and the context in front of it
        dict(name="attn_chunk_8192", op="attn", seqs=1, rows=8192, len=9000, heads=32, kv=8, hd=128, page=64, block=64, form="causal"),
    ]


FORMS = ("causal", "causal", "cap", "cap_window", "window", "distance", "documents", "prefix")
MOST = {"rope": 4096 * 48 * 128, "cache": 8192 * 8 * 128, "attn": 6e11}


def _log(rng, lo, hi):
    """Whole numbers between lo and hi, even over the logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    while True:
        op = rng.choice(("rope", "cache", "attn", "attn"))
        hd = rng.choice((64, 128, 128, 128, 256))
        if op == "rope":
            pairs = rng.choice((hd // 2, hd // 2, hd // 2, hd // 4, hd // 4 - 3))
            c = dict(op=op, T=_log(rng, 1, 8192), heads=rng.choice((5, 10, 12, 36, 40, 48)), hd=hd, pairs=pairs, neighbours=rng.random() < 0.3,
                     axes=rng.choice((1, 1, 3)), far=_log(rng, 100, 2000000))
            if c["T"] * c["heads"] * hd <= MOST["rope"]:
                return c
            continue
        page = rng.choice((16, 32, 64, 128, 256))
        block = rng.choice([b for b in (1, 16, 32, 64, 128, 256) if b <= page])
        kv = rng.choice((1, 2, 4, 8))
        if op == "cache":
            rows = 1 if rng.random() < 0.4 else _log(rng, 2, 8192)
            c = dict(op=op, seqs=_log(rng, 1, 128), rows=rows, len=rows + _log(rng, 1, 20000), kv=kv, hd=hd, page=page, block=block)
            # (the pages of every sequence are held: a few GB at most)
            if c["seqs"] * rows * kv * hd <= MOST["cache"] and c["seqs"] * c["len"] * kv * hd <= 5e8:
                return c
            continue
        group = rng.choice((1, 2, 4, 4, 5, 6, 7, 8, 8, 16))
        rows = rng.choice((1, 1, _log(rng, 2, 16), _log(rng, 16, 4096)))
        c = dict(op=op, seqs=_log(rng, 1, 96), rows=rows, len=rows + _log(rng, 1, 131072 if rows <= 16 else 16384), heads=kv * group, kv=kv, hd=hd, page=page,
                 block=block, form=rng.choice(FORMS))
        scores = c["seqs"] * rows * c["heads"] * c["len"]
        if work(c)["flops"] <= MOST["attn"] and scores <= 2.3e9 and c["seqs"] * c["len"] * kv * hd <= 3e8:
            return c


# ---------------------------------------------------------------- a batch's sequences
def _shape(case):
    """(rows, keys) of every sequence: the first one has the most, the others fewer in no order."""
    n, rng = [], random.Random(case["seqs"] * 1000003 + case["rows"] * 101 + case["len"])
    for s in range(case["seqs"]):
        f = 1.0 if s == 0 else rng.uniform(0.05, 1.0)
        r = case["rows"] if s == 0 or case["rows"] <= 16 else max(1, int(case["rows"] * rng.uniform(0.02, 1.0)))
        n.append((r, max(r, int(case["len"] * f))))
    return n


def _window(case):
    return 1024 if "window" in case["form"] else 0


def _prefix(case, n, l):
    return l // 2 if case["form"] == "prefix" else 0


def _documents(n, l):
    """The first position of the document of each of a sequence's last n of l positions: three documents of unlike lengths."""
    cuts = (0, l // 5, (3 * l) // 5)
    return [max(c for c in cuts if c <= p) for p in range(l - n, l)]


def _visible(case, n, l):
    """Visible (row, key) pairs of one sequence."""
    t = 0
    docs = _documents(n, l) if case["form"] == "documents" else None
    w, pre = _window(case), _prefix(case, n, l)
    for i, p in enumerate(range(l - n, l)):
        lo = max(docs[i] if docs else 0, p - w + 1 if w else 0)
        t += max(0, max(p + 1, pre) - lo)
    return t


def work(case):
    if case["op"] == "rope":
        v, p = case["T"] * case["heads"] * case["hd"], case["T"] * case["heads"] * case["pairs"]
        return {"bytes": 8 * v + 4 * case["axes"] * case["T"], "flops": 6.0 * p}
    seqs, kv, hd = _shape(case), case["kv"], case["hd"]
    if case["op"] == "cache":
        new = sum(n for n, _ in seqs)
        old = sum((l - n) % case["block"] for n, l in seqs)   # (older tokens of the blocks written)
        blocks = sum(-(-l // case["block"]) - (l - n) // case["block"] for n, l in seqs)
        # new rows read in f32 and stored in 8 bits, both kinds; all touched rows read back as f32, their scales read and written
        return {"bytes": 2 * kv * (hd * (4 * new + new + (new + old) * 5) + 12 * blocks), "flops": 2.0 * kv * hd * (3 * new + new + old)}
    rows, pairs = sum(n for n, _ in seqs), sum(_visible(case, n, l) for n, l in seqs)
    keys = sum(min(l, n + _window(case)) if _window(case) else l for n, l in seqs)
    return {"bytes": 2 * kv * (keys * hd + 4 * keys / case["block"]) + 8 * rows * case["heads"] * hd, "flops": 4.0 * hd * case["heads"] * pairs}


# ---------------------------------------------------------------- inputs
class _State:
    def __init__(self, case):
        self.case, self.held = case, []

    def __del__(self):
        for h in reversed(self.held):
            h.free()


def _quantized(x, block):
    """Rows [..., tokens, hd] in 8 bits with a scale for each block of tokens."""
    b = x.unflatten(-2, (-1, block))
    d = b.abs().amax((-1, -2)) / 127.0
    q = torch.round(b / d[..., None, None]).to(torch.int8).flatten(-3, -2)
    return q, d


def _frequencies(case):
    return [10000.0 ** (-i / case["pairs"]) for i in range(case["pairs"])]


def _axes(case):
    """The axis of each pair: one for all, or the three in turn for the fast ones and time for the slow rest."""
    p = case["pairs"]
    return [0] * p if case["axes"] == 1 else [i % 3 if i < 3 * (p // 4) else 0 for i in range(p)]


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    s = _State(case)

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda")

    if case["op"] == "rope":
        T, h, hd = case["T"], case["heads"], case["hd"]
        s.x = normal(T, h * hd)
        s.y = torch.empty_like(s.x)
        t = torch.arange(T, device="cuda") + int(case["far"]) + seed % 17
        if case["axes"] == 1:
            s.pos = t[None].int()
        else:   # text in front, then a picture of 64 patches a row: time stands still, height and width run
            i, text = torch.arange(T, device="cuda"), T // 8
            at = (i - text).clamp_min(0)
            s.pos = torch.stack([torch.where(i < text, t, t[text]), torch.where(i < text, t, t[text] + at // 64), torch.where(i < text, t, t[text] + at % 64)]).int()
    else:
        kv, hd, page, block = case["kv"], case["hd"], case["page"], case["block"]
        seqs = _shape(case)
        s.T = sum(n for n, _ in seqs)
        s.max_rows, s.max_len = max(n for n, _ in seqs), max(l for _, l in seqs)
        need = [-(-l // page) for _, l in seqs]
        pages = sum(need) + 3
        order = torch.randperm(pages, generator=g, device="cuda").int()
        table, at = torch.full((len(seqs), max(need)), -1, dtype=torch.int32), 0
        order = order.cpu()
        for i, n in enumerate(need):
            table[i, :n] = order[at:at + n]
            at += n
        s.table = table.cuda()
        s.rows = torch.tensor(np.cumsum([0] + [n for n, _ in seqs]), dtype=torch.int32, device="cuda")
        s.len = torch.tensor([l for _, l in seqs], dtype=torch.int32, device="cuda")
        # (keys have a few large columns)
        columns = 1.0 + 3.0 * (torch.rand((kv, 1, hd), generator=g, device="cuda") < 0.04)
        s.kq, s.ks = _quantized(normal(pages, kv, page, hd) * columns, block)
        s.vq, s.vs = _quantized(normal(pages, kv, page, hd), block)
        if case["op"] == "cache":
            # the k and v columns of rows [q | k | v], of a model with four query heads for each pair of the others
            s.ld = 6 * kv * hd
            s.x = normal(s.T, s.ld) * (1.0 + 0.3 * torch.rand((s.T, 1), generator=g, device="cuda"))
            back = [(n + (l - n) % block, l) for n, l in seqs]   # (what is read back: the blocks that are written, from their first tokens on)
            s.back_T, s.back_rows = sum(n for n, _ in back), max(n for n, _ in back)
            s.back = torch.tensor(np.cumsum([0] + [n for n, _ in back]), dtype=torch.int32, device="cuda")
            s.k, s.v = (torch.empty((s.back_T, kv * hd), device="cuda") for _ in range(2))
        else:
            h = case["heads"]
            s.ld = (h + 2 * kv) * hd
            s.x = normal(s.T, s.ld) * 1.3
            s.out = torch.empty((s.T, h * hd), device="cuda")
            s.scale, s.cap = hd ** -0.5, 30.0 if "cap" in case["form"] else 0.0
            s.slopes = s.prefix = s.first = None
            if case["form"] == "distance":
                s.slopes = torch.tensor([2.0 ** (-8.0 * (i + 1) / h) for i in range(h)], device="cuda")
            if case["form"] == "prefix":
                s.prefix = torch.tensor([_prefix(case, n, l) for n, l in seqs], dtype=torch.int32, device="cuda")
            if case["form"] == "documents":
                s.first = torch.tensor([f for n, l in seqs for f in _documents(n, l)], dtype=torch.int32, device="cuda")
    if own:
        _handles(s)
    torch.cuda.synchronize()
    return s


# ---------------------------------------------------------------- the framework's calls
_engine = None


def _handles(s):
    """What a program of the framework keeps: its engine, handles of the buffers, the cache, the batch, the rotation."""
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
    s.bx = wrap(s.x)
    if c["op"] == "rope":
        s.by, s.bpos = wrap(s.y), wrap(s.pos)
        s.rope = keep(_engine.make_rope(_frequencies(c), _axes(c), c["neighbours"]))
        return
    s.kvc = keep(_engine.make_kv(s.kq.shape[0], c["page"], c["block"], c["kv"], c["hd"], wrap(s.kq), wrap(s.vq), wrap(s.ks), wrap(s.vs)))
    table, lens = wrap(s.table), wrap(s.len)
    s.batch = az.KvBatch(wrap(s.rows), lens, table, c["seqs"], s.table.shape[1], s.T, s.max_rows, s.max_len)
    if c["op"] == "cache":
        s.back_batch = az.KvBatch(wrap(s.back), lens, table, c["seqs"], s.table.shape[1], s.back_T, s.back_rows, s.max_len)
        s.bk, s.bv = wrap(s.k), wrap(s.v)
    else:
        s.bout = wrap(s.out)
        s.form = az.Attention(s.scale, s.cap, _window(c), wrap(s.slopes), wrap(s.prefix), wrap(s.first))


def _run_own(s):
    c = s.case
    if c["op"] == "rope":
        w = c["heads"] * c["hd"]
        _engine.rope(s.rope, s.bx, w, 0, s.by, w, 0, c["T"], c["heads"], c["hd"], s.bpos)
        return s.y
    w = c["kv"] * c["hd"]
    if c["op"] == "cache":
        _engine.kv_write(s.kvc, s.batch, s.bx, s.ld, 4 * w, s.bx, s.ld, 5 * w)
        _engine.kv_read(s.kvc, s.back_batch, s.bk, w, 0, s.bv, w, 0)
        return s.k, s.v
    _engine.attention(s.kvc, s.batch, s.bx, s.ld, 0, c["heads"], s.bout, c["heads"] * c["hd"], 0, s.form)
    return s.out


# ---------------------------------------------------------------- the plain forms
def _where(s, rows, T):
    """Sequence, position, page and place in it of each of T rows, `rows` of them to each sequence."""
    n = (rows[1:] - rows[:-1]).long()
    seq = torch.repeat_interleave(torch.arange(n.numel(), device="cuda"), n, output_size=T)
    pos = s.len.long()[seq] - n[seq] + torch.arange(T, device="cuda") - rows.long()[seq]
    page = s.case["page"]
    return seq, pos, s.table[seq, pos // page].long(), pos % page


def _plain_rope(s):
    c = s.case
    T, h, hd, p = c["T"], c["heads"], c["hd"], c["pairs"]
    freq = torch.tensor(_frequencies(c), dtype=torch.float64, device="cuda")
    angle = s.pos[torch.tensor(_axes(c), device="cuda")].T.double() * freq   # (far positions: 64 bits)
    co, si = angle.cos().float()[:, None], angle.sin().float()[:, None]
    x = s.x.view(T, h, hd)
    y = x.clone()
    a, b = (x[..., 0:2 * p:2], x[..., 1:2 * p:2]) if c["neighbours"] else (x[..., :p], x[..., p:2 * p])
    u, v = a * co - b * si, a * si + b * co
    if c["neighbours"]:
        y[..., 0:2 * p:2], y[..., 1:2 * p:2] = u, v
    else:
        y[..., :p], y[..., p:2 * p] = u, v
    return y.view(T, h * hd)


def _plain_write(s, x, q, d):
    """Rows x [T, kv, hd] into the cache's values q and scales d, which change in place."""
    c = s.case
    block, per = c["block"], c["page"] // c["block"]
    seq, pos, page, off = _where(s, s.rows, s.T)
    new = x.abs().amax(-1)
    new = new / torch.full_like(new, 127.0)   # (a number's reciprocal would be multiplied with instead)
    flat = d.transpose(1, 2).reshape(-1, c["kv"]).clone()   # [page, block in it][kv]
    at = page * per + off // block
    # a block that holds older tokens keeps at least their scale
    begin = s.len.long() - (s.rows[1:] - s.rows[:-1]).long()
    older = begin % block != 0
    first = s.table.gather(1, (begin // c["page"]).clamp_max(s.table.shape[1] - 1)[:, None])[:, 0].long().clamp_min(0) * per + begin % c["page"] // block
    scale = torch.zeros_like(flat)
    was = flat[first]
    scale[first] = torch.where(older[:, None], was, scale[first])
    scale.index_reduce_(0, at, new, "amax")
    inverse = torch.where(scale >= 2.0 ** -120, 1.0 / scale, torch.zeros_like(scale))
    # the older tokens of the first blocks, on the new scale
    j = torch.arange(block, device="cuda")
    p = begin[:, None] // block * block + j
    real = (p < begin[:, None]) & older[:, None]
    rp = s.table.gather(1, (p // c["page"]).clamp_max(s.table.shape[1] - 1)).long().clamp_min(0)[real]
    ro, rf = (p % c["page"])[real], first[:, None].expand_as(p)[real]
    ratio = flat[rf] * inverse[rf]
    grown = scale[rf] > flat[rf]
    old = q[rp, :, ro]
    q[rp, :, ro] = torch.where(grown[..., None], torch.round(old.float() * ratio[..., None]), old.float()).to(torch.int8)
    q[page, :, off] = torch.round(x * inverse[at][..., None]).clamp(-127, 127).to(torch.int8)
    flat[at] = scale[at]
    d.copy_(flat.view(-1, per, c["kv"]).transpose(1, 2))


def _plain_cache(s):
    c = s.case
    w = c["kv"] * c["hd"]
    _plain_write(s, s.x[:, 4 * w:5 * w].unflatten(1, (c["kv"], c["hd"])), s.kq, s.ks)
    _plain_write(s, s.x[:, 5 * w:].unflatten(1, (c["kv"], c["hd"])), s.vq, s.vs)
    _, _, page, off = _where(s, s.back, s.back_T)
    return tuple((q[page, :, off].float() * d[page, :, off // c["block"]][..., None]).flatten(1) for q, d in ((s.kq, s.ks), (s.vq, s.vs)))


def _plain_attention(s):
    c = s.case
    kv, hd, h, S, R, L = c["kv"], c["hd"], c["heads"], c["seqs"], s.max_rows, s.max_len
    G = h // kv
    n, l = (s.rows[1:] - s.rows[:-1]).long()[:, None], s.len.long()[:, None]
    i, j = torch.arange(R, device="cuda")[None], torch.arange(L, device="cuda")
    row = (s.rows[:-1].long()[:, None] + i).clamp_max(s.T - 1)          # [S, R]
    q = s.x[row, :h * hd].view(S, R, kv, G, hd).permute(0, 2, 1, 3, 4).reshape(S, kv, R * G, hd)
    pages = s.table.long().clamp_min(0)
    k, v = ((a[pages].float().unflatten(3, (-1, c["block"])) * d[pages][..., None, None]).flatten(3, 4).transpose(1, 2).reshape(S, kv, -1, hd)[:, :, :L]
            for a, d in ((s.kq, s.ks), (s.vq, s.vs)))
    p = (l - n + i)[:, :, None]                                          # [S, R, 1]
    seen = (j < l[:, :, None]) & ((j <= p) if s.prefix is None else (j <= p) | (j < s.prefix.long()[:, None, None]))
    if _window(c):
        seen &= p - j < _window(c)
    if s.first is not None:
        seen &= j >= s.first.long()[row][:, :, None]
    a = (q * s.scale) @ k.transpose(-1, -2).contiguous()
    a = a.view(S, kv, R, G, L)
    if s.cap:
        a = s.cap * torch.tanh(a / s.cap)
    if s.slopes is not None:
        a = a - s.slopes.view(kv, 1, G, 1) * (p - j).abs().float()[:, None, :, None]
    a = a.masked_fill(~seen[:, None, :, None], -math.inf)
    a = (a - a.amax(-1, keepdim=True).clamp_min(-3e38)).exp()
    a = a / a.sum(-1, keepdim=True).clamp_min(1e-37)
    o = (a.view(S, kv, R * G, L) @ v).view(S, kv, R, G, hd).permute(0, 2, 1, 3, 4).reshape(S, R, h * hd)
    return o[i.expand(S, R) < n]


def run(state):
    if own:
        return _run_own(state)
    return {"rope": _plain_rope, "cache": _plain_cache, "attn": _plain_attention}[state.case["op"]](state)


# ---------------------------------------------------------------- the definitions in 64 bits
def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    return {"rope": _exact_rope, "cache": _exact_cache, "attn": _exact_attention}[case["op"]](s)


def _exact_rope(s):
    c = s.case
    T, hd, p = c["T"], c["hd"], c["pairs"]
    x = s.x.double().view(T, c["heads"], hd)
    y = x.clone()
    for i, (f, a) in enumerate(zip(_frequencies(c), _axes(c))):
        m, n = (2 * i, 2 * i + 1) if c["neighbours"] else (i, i + p)
        z = torch.polar(torch.ones(T, dtype=torch.float64, device="cuda"), s.pos[a].double() * f)[:, None] * torch.complex(x[..., m], x[..., n])
        y[..., m], y[..., n] = z.real, z.imag
    return y.view(T, -1)


def _f32(x):
    """A 64-bit value rounded as the 32-bit operation rounds it: the stored integers hang on it."""
    return x.float().double()


def _exact_cache(s):
    c = s.case
    kv, hd, page, block, w = c["kv"], c["hd"], c["page"], c["block"], c["kv"] * c["hd"]
    table, outs = s.table.cpu().tolist(), []
    if c["seqs"] * (c["rows"] // block + 2) > 6000:
        return None
    for q, d, col in ((s.kq, s.ks, 4 * w), (s.vq, s.vs, 5 * w)):
        parts, at = [], 0
        for i, (n, l) in enumerate(_shape(c)):
            new = s.x[at:at + n, col:col + w].double().view(n, kv, hd)
            at += n
            p = l - n
            while p < l:
                lo, hi = p // block * block, min(l, p // block * block + block)
                pg, o = table[i][lo // page], lo % page
                x = new[p - (l - n):hi - (l - n)]
                top = _f32(x.abs().amax((0, 2)) / 127.0)
                was = d[pg, :, o // block].double() if p > lo else torch.zeros_like(top)
                to = torch.maximum(top, was)
                inv = torch.where(to >= 2.0 ** -120, _f32(1.0 / to), torch.zeros_like(to))
                if p > lo:
                    old = q[pg, :, o:o + p - lo].double()
                    old = torch.where((to > was)[:, None, None], torch.round(_f32(old * _f32(was * inv)[:, None, None])), old)
                    parts.append((old * to[:, None, None]).transpose(0, 1))
                parts.append(torch.round(_f32(x * inv[:, None])).clamp(-127, 127) * to[:, None])
                p = hi
        outs.append(torch.cat(parts).reshape(-1, w))
    return tuple(outs)


def _exact_attention(s):
    c = s.case
    kv, hd, h, page, block = c["kv"], c["hd"], c["heads"], c["page"], c["block"]
    G, out, at = h // kv, torch.empty((s.T, h, hd), dtype=torch.float64, device="cuda"), 0
    for i, (n, l) in enumerate(_shape(c)):
        pages = s.table[i, :-(-l // page)].long()
        for g in range(kv):
            k, v = (a[pages, g].double().reshape(-1, hd)[:l] * d[pages, g].double().reshape(-1).repeat_interleave(block)[:l, None] for a, d in ((s.kq, s.ks), (s.vq, s.vs)))
            k = k.T.contiguous()
            step = max(1, int(2e8 // (l * G)))
            for r in range(0, n, step):
                m = min(step, n - r)
                q = s.x[at + r:at + r + m, g * G * hd:(g + 1) * G * hd].double().reshape(m * G, hd)
                a = (q @ k).view(m, G, l) * s.scale
                p, j = torch.arange(l - n + r, l - n + r + m, device="cuda")[:, None], torch.arange(l, device="cuda")
                if s.cap:
                    a = torch.tanh(a / s.cap) * s.cap
                if s.slopes is not None:
                    a = a - s.slopes[g * G:(g + 1) * G].double()[:, None] * (p - j).abs()[:, None]
                low = torch.zeros_like(p)
                if _window(c):
                    low = torch.maximum(low, p - _window(c) + 1)
                if s.first is not None:
                    low = torch.maximum(low, s.first[at + r:at + r + m].long()[:, None])
                end = p + 1 if s.prefix is None else torch.maximum(p + 1, s.prefix[i].long())
                a = a.masked_fill(((j < low) | (j >= end))[:, None], -math.inf)
                out[at + r:at + r + m, g * G:(g + 1) * G] = (torch.softmax(a, -1).view(m * G, l) @ v).view(m, G, hd)
        at += n
    return out.view(s.T, h * hd)
