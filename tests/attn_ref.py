"""The attention block's operators in numpy, in 64 bits (the stored bytes of the cache: in the 32-bit operations that define
them), and batches of sequences for the tests."""
import numpy as np

import arcinferzero_amd as az

F = np.float32


def rope(x, pos, freq, axis, neighbours, mscale=1.0):
    """x [T][heads][hd], pos [axes][T] -> the same, turned, in 64 bits."""
    x = x.astype(np.float64)
    y, p = x.copy(), len(freq)
    for i, (f, a) in enumerate(zip(freq, axis)):
        m, n = (2 * i, 2 * i + 1) if neighbours else (i, i + p)
        # (the angle modulo a turn from the position's product in more than 64 bits)
        t = pos[a].astype(np.longdouble) * np.longdouble(f)
        c, s = (np.asarray(g(t), np.float64)[:, None] * mscale for g in (np.cos, np.sin))
        y[..., m], y[..., n] = x[..., m] * c - x[..., n] * s, x[..., m] * s + x[..., n] * c
    return y


class Cache:
    """Pages of 8-bit values on the host: q int8 [2][pages][heads][page][hd], d f32 [2][pages][heads][page / block]."""

    def __init__(self, pages, page, block, heads, hd, seed=0, zeros=False):
        self.pages, self.page, self.block, self.heads, self.hd = pages, page, block, heads, hd
        rng = np.random.default_rng(seed)
        shape = (2, pages, heads, page, hd)
        self.q = np.zeros(shape, np.int8) if zeros else rng.integers(-127, 128, size=shape).astype(np.int8)
        self.d = (rng.uniform(0.5, 1.5, size=shape[:3] + (page // block,)) * 0.02).astype(F)

    def values(self, which, table, n):
        """f64 [n][heads][hd] of the first n positions of a sequence."""
        out = np.zeros((n, self.heads, self.hd))
        for p in range(n):
            pg = table[p // self.page]
            if 0 <= pg < self.pages:
                o = p % self.page
                out[p] = self.q[which, pg, :, o].astype(np.float64) * self.d[which, pg, :, o // self.block].astype(np.float64)[:, None]
        return out

    def scales(self, which, table, n):
        """f64 [n][heads]"""
        out = np.zeros((n, self.heads))
        for p in range(n):
            pg = table[p // self.page]
            if 0 <= pg < self.pages:
                out[p] = self.d[which, pg, :, p % self.page // self.block]
        return out

    def there(self, table, n):
        return np.array([0 <= table[p // self.page] < self.pages for p in range(n)], bool)

    def write(self, which, table, p0, rows):
        """rows f32 [n][heads][hd] at positions p0 ..., every operation in f32."""
        n, B = len(rows), self.block
        p = max(p0, 0)
        with np.errstate(all="ignore"):
            while p < p0 + n:
                b0 = p // B * B
                e = min(p0 + n, b0 + B)
                pg, o = table[b0 // self.page], b0 % self.page
                if 0 <= pg < self.pages:
                    for h in range(self.heads):
                        x = rows[p - p0:e - p0, h].astype(F)
                        top = F(np.nan) if not np.isfinite(x).all() else F(np.abs(x).max()) / F(127)
                        was = self.d[which, pg, h, o // B] if p > b0 else F(0)
                        s = F(np.nan) if np.isnan(was) or np.isnan(top) else max(was, top)
                        i = F(1) / s if s >= F(2.0 ** -120) else F(0)
                        if p > b0 and s > was:
                            old = self.q[which, pg, h, o:o + p - b0].astype(F)
                            self.q[which, pg, h, o:o + p - b0] = np.clip(np.rint(old * F(was * i)), -127, 127).astype(np.int8)
                        self.q[which, pg, h, o + p - b0:o + e - b0] = np.clip(np.rint(x * i), -127, 127).astype(np.int8) if i > 0 else 0
                        self.d[which, pg, h, o // B] = s
                p = e


def attention(cache, q, rows, lens, table, scale, cap=0.0, window=0, slopes=None, prefix=None, first=None, max_rows=1 << 30, only=None):
    """q [T][heads][hd] -> (out f64 [T][heads][hd], bound on each value's error, rows that were computed: all, or those of `only`).

    The bound counts the f32 steps behind the exact 8-bit values: a score's error is that of a sum of 2 hd products of f16 parts
    (22 bits of each row's value: 2^-22; the sum in f32: each of hd / 16 steps' result rounded, both parts, and inside a step
    the 16 products with the accumulator, taken as 2^-23 a step), of the multiplication with its scale, of the logarithm of the
    values' scale added to it (2^-23 of its size, 2^-22 with the logarithm's own) and of the difference with the reference, up
    to 24 octaves of range each rounded to 2^-24; with a cap, of 2^-21 of the cap (its exponential, sum, reciprocal, product).
    The exponential itself adds 2^-22, weight and sum parts of 22 bits 2^-21, the sums over keys 2^-23 a step of 16 keys where a
    part of the row lies in one accumulator (keys / 16 steps at most, their errors adding up as sqrt).

    A weight times its values' scale is held in two f16, whose last place ends at 2^-24; the row's largest is at least 2^8 there.  So
    every key adds its 8-bit value times up to 2^-32 of the row's largest weight times scale -- what is left of the error where the
    keys that count hold a zero in some column.  A block of zeros has a weight there too, its own times a scale of at most 2^-60:
    where such blocks have all of a row's weight, the f16 of the other keys, whose parts are then less than 2^-60 of it, end at that."""
    T, H, hd = q.shape
    G = H // cache.heads
    out, tol, done = np.zeros((T, H, hd)), np.zeros((T, H, hd)), np.zeros(T, bool)
    for s in range(len(lens)):
        n, l = rows[s + 1] - rows[s], lens[s]
        k, v = cache.values(0, table[s], l), cache.values(1, table[s], l)
        vs = cache.scales(1, table[s], l)
        there = cache.there(table[s], l)
        j = np.arange(l)
        for i in range(min(n, max_rows)):
            t, p = rows[s] + i, l - n + i
            if only is not None and t not in only:
                continue
            done[t] = True
            see = there & ((j <= p) | (j < (prefix[s] if prefix is not None else 0)))
            if window:
                see &= p - j < window
            if first is not None:
                see &= j >= first[t]
            if not see.any():
                continue
            kk, vv, jj = k[see], v[see], j[see]
            for h in range(H):
                g = h // G
                with np.errstate(all="ignore"):
                    prod = q[t, h].astype(np.float64) * kk[:, g]
                    a = scale * prod.sum(1)
                    size = abs(scale) * np.abs(prod).sum(1)
                    ds = size * (2.0 ** -22 + (hd / 16) * 2.0 ** -23) + np.abs(a) * 2.0 ** -22
                    if cap:
                        a = cap * np.tanh(a / cap)
                        ds = ds + cap * 2.0 ** -21
                    if slopes is not None:
                        b = float(slopes[h]) * np.abs(p - jj)
                        a = a - b
                        ds = ds + b * 2.0 ** -22
                    ds = ds + 24 * 2.0 ** -23 + np.abs(a) * 2.0 ** -23
                    e = np.exp(a - a.max())
                    e /= e.sum()
                    out[t, h] = e @ vv[:, g]
                    rel = ds + 2.0 ** -20 + np.sqrt(len(jj) / 16.0) * 2.0 ** -23
                    # (d out = sum p_j ds_j (v_j - out))
                    tol[t, h] = (e * rel) @ np.abs(vv[:, g] - out[t, h]) + np.abs(out[t, h]) * 2.0 ** -20 + (e @ np.abs(vv[:, g])) * 2.0 ** -21
                    d = vs[see, g]
                    ints = np.abs(np.divide(vv[:, g], d[:, None], out=np.zeros_like(vv[:, g]), where=d[:, None] > 0))
                    tol[t, h] += 2.0 ** -32 * np.max(e * np.where(d > 0, d, 2.0 ** -60)) * ints.sum(0)
    return out, tol, done


class Batch:
    """Sequences of (rows, keys) on the host and, as buffers, on the GPU; pages in no order."""

    def __init__(self, seqs, page, seed=0, spare_pages=2, ld_extra=1, T=None, max_rows=None, tail_page=-1):
        rng = np.random.default_rng(seed)
        self.seqs = seqs
        self.rows = np.cumsum([0] + [n for n, _ in seqs]).astype(np.int32)
        self.lens = np.array([l for _, l in seqs], np.int32)
        need = [max(1, -(-l // page)) for _, l in seqs]
        self.pages = sum(need) + spare_pages
        order = rng.permutation(self.pages).astype(np.int32)
        self.ldt = max(need) + ld_extra
        self.table = np.full((len(seqs), self.ldt), tail_page, np.int32)
        at = 0
        for s, n in enumerate(need):
            self.table[s, :n] = order[at:at + n]
            at += n
        self.T = int(self.rows[-1]) if T is None else T
        self.max_rows = max(n for n, _ in seqs) if max_rows is None else max_rows
        self.max_len = int(self.lens.max())

    def device(self, hold):
        b = [az.Runtime.from_numpy(a) for a in (self.rows, self.lens, self.table)]
        hold += b
        return az.KvBatch(*b, len(self.seqs), self.ldt, self.T, self.max_rows, self.max_len)


def device_cache(eng, c, hold):
    b = [az.Runtime.from_numpy(a) for a in (c.q[0], c.q[1], c.d[0], c.d[1])]
    kv = eng.make_kv(c.pages, c.page, c.block, c.heads, c.hd, *b)
    hold += b + [kv]
    return kv


def read_cache(kv, c):
    """(int8 [2][...], f32 [2][...]) as the GPU holds them."""
    q = [kv.buffer(i).read(np.int8, c.q[0].size).reshape(c.q[0].shape) for i in (0, 1)]
    d = [kv.buffer(i).read(np.float32, c.d[0].size).reshape(c.d[0].shape) for i in (2, 3)]
    return np.stack(q), np.stack(d)


def free(hold):
    for h in reversed(hold):
        h.free()
    hold.clear()
