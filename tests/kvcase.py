"""A small cache, drafted tokens and 64-bit results of the calls between the linears, in numpy, for their GPU tests."""
import numpy as np

import p8x

F16, BF16, F32 = p8x.F16, p8x.BF16, p8x.F32


def to_bits(a, dtype):
    """f32 values as the type's bits (16-bit types as uint16, to nearest even)"""
    a = np.ascontiguousarray(a, np.float32)
    if dtype == F32:
        return a
    if dtype == F16:
        with np.errstate(over="ignore"):
            return a.astype(np.float16).view(np.uint16)
    u = a.view(np.uint32).astype(np.uint64)
    out = ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(a), np.uint16(0x7FC0), out).astype(np.uint16)


def from_bits(b, dtype):
    """the values that the bits stand for, in 64 bits"""
    if dtype == F32:
        return b.astype(np.float64)
    if dtype == F16:
        return b.view(np.float16).astype(np.float64)
    return (b.astype(np.uint32) << 16).view(np.float32).astype(np.float64)


def half_ulp(dtype):
    """largest relative error of a rounding to the type"""
    return {F32: 2.0 ** -24, F16: 2.0 ** -11, BF16: 2.0 ** -8}[dtype]


class Case:
    """lens: slots in use; toks: drafted tokens of each sequence. Slots not in use, pages not in a table and rows not in
    a sequence hold NaN."""

    def __init__(self, lens, toks, heads=4, kv=2, D=128, page=16, cache=F16, q=F32, kv_in=None, layout="head", table=True, max_len=None, seed=0,
                 mask="tree", fused=True, extra=0):
        rng = self.rng = np.random.default_rng(seed)
        S = len(lens)
        self.S, self.lens, self.toks, self.H, self.kv, self.G, self.D, self.page = S, list(lens), list(toks), heads, kv, heads // kv, D, page
        self.cache, self.qt, self.kt = cache, q, q if kv_in is None else kv_in
        self.max_len = max_len or max(l + t for l, t in zip(lens, toks)) + 3
        self.layout = layout
        if table:
            per = -(-self.max_len // page)
            self.n_pages = S * per + 2
            self.pages = rng.permutation(self.n_pages)[:S * per].reshape(S, per).astype(np.int32)
        else:
            self.n_pages, page, self.pages = S, self.max_len + extra, None
            self.page = page
        shape = (self.n_pages, kv, page, D) if layout == "head" else (self.n_pages, page, kv, D)
        self.pool_shape = shape
        nan = to_bits(np.float32(np.nan), cache)
        self.kb, self.vb = np.full(shape, nan, np.uint16), np.full(shape, nan, np.uint16)
        for s in range(S):
            for j in range(lens[s]):
                for pool, scale in ((self.kb, 1.0), (self.vb, 1.0)):
                    self.row(pool, s, j)[:] = to_bits(rng.standard_normal((kv, D)) * scale, cache)
        n = self.n = sum(toks) + extra
        self.first = np.concatenate([[0], np.cumsum(toks)]).astype(np.int32)
        self.tk = max(toks) if toks else 0
        if fused:   # q, k and v side by side, with a few columns between rows
            self.ld = (heads + 2 * kv) * D + 8
            one = np.full((n, self.ld), np.nan, np.float32)
            one[:, :(heads + 2 * kv) * D] = rng.standard_normal((n, (heads + 2 * kv) * D))
            one[:, :heads * D] *= 1.5
            assert self.kt == self.qt
            self.buf = to_bits(one, q)
            self.at_k, self.at_v = heads * D, (heads + kv) * D
            self.qb = self.buf[:, :heads * D].reshape(n, heads, D)
            self.knb, self.vnb = (self.buf[:, a:a + kv * D].reshape(n, kv, D) for a in (self.at_k, self.at_v))
        else:
            self.buf = None
            self.qb = to_bits(1.5 * rng.standard_normal((n, heads, D)), q)
            self.knb, self.vnb = (to_bits(rng.standard_normal((n, kv, D)), self.kt) for _ in range(2))
        self.mask = np.zeros(n, np.uint64)
        for s in range(S):
            for i in range(toks[s]):
                if mask == "tree":
                    p = int(rng.integers(0, max(1, i)))
                    m = (int(self.mask[self.first[s] + p]) if i else 0) | 1 << i
                elif mask == "chain":
                    m = (1 << (i + 1)) - 1
                elif mask == "none":
                    m = 0
                else:
                    m = int(rng.integers(0, 1 << 63)) << 1 | int(rng.integers(0, 2))
                self.mask[self.first[s] + i] = m & ((1 << 64) - 1)
        self.scale = float(np.float32(D ** -0.5))
        self.accept = None
        self.keep = []

    def place(self, s, j):
        if self.pages is None:
            return s, j
        return int(self.pages[s, j // self.page]), j % self.page

    def row(self, pool, s, j):
        """[kv][D] of a slot in a host pool"""
        p, o = self.place(s, j)
        return pool[p, :, o] if self.layout == "head" else pool[p, o]

    def there(self, s, j):
        return self.pages is None or 0 <= self.pages[s, j // self.page] < self.n_pages

    # ---- device side
    def dev(self, a):
        b = p8x.DeviceBuffer.from_numpy(a)
        self.keep.append(b)
        return b

    def make_cache(self):
        self.kd, self.vd, self.lend = self.dev(self.kb), self.dev(self.vb), self.dev(np.asarray(self.lens, np.int32))
        P, page, kv, D = self.n_pages, self.page, self.kv, self.D
        hs, ss = (page * D, D) if self.layout == "head" else (D, kv * D)
        return p8x.KvCache(self.cache, self.S, kv, D, self.kd, self.vd, page_stride=page * kv * D, head_stride=hs, slot_stride=ss, page_size=page,
                           n_pages=P, len=self.lend, max_len=self.max_len, pages=None if self.pages is None else self.dev(self.pages),
                           ld_pages=0 if self.pages is None else self.pages.shape[1])

    def drafts(self, q=True, mask=True):
        d = dict(n_tokens=self.n, max_tokens=self.tk, first=self.dev(self.first), kv_dtype=self.kt, mask=self.dev(self.mask) if mask else None)
        size = 4 if self.qt == F32 else 2
        if self.buf is not None:
            b = self.dev(self.buf)
            d.update(k=b.addr + size * self.at_k, v=b.addr + size * self.at_v, ld_kv=self.ld)
            if q:
                d.update(q=b, ld_q=self.ld)
        else:
            d.update(k=self.dev(self.knb), v=self.dev(self.vnb))
            if q:
                d.update(q=self.dev(self.qb))
        if q:
            d.update(q_dtype=self.qt, n_heads=self.H, scale=self.scale)
        return d

    # ---- 64-bit results
    def kn(self, bits):
        """draft rows as the cache holds them"""
        return from_bits(to_bits(from_bits(bits, self.kt).astype(np.float32), self.cache), self.cache)

    def sees(self, s, i, mask=True):
        """[len + toks] whether token i of sequence s sees each slot and drafted token"""
        n, t = self.lens[s], self.toks[s]
        ctx = [self.there(s, j) for j in range(n)]
        m = int(self.mask[self.first[s] + i]) if mask else (2 << i) - 1
        return np.array(ctx + [bool(m >> j & 1) for j in range(t)], bool)

    def keys(self, pool, new, s, h):
        n = self.lens[s]
        k = np.zeros((n, self.D))
        for j in range(n):
            if self.there(s, j):
                k[j] = from_bits(self.row(pool, s, j)[h], self.cache)
        a, b = self.first[s], self.first[s] + self.toks[s]
        return np.concatenate([k, self.kn(new[a:b, h])])

    def attention(self, mask=True):
        out = np.zeros((self.n, self.H, self.D))
        lse = np.full((self.n, self.H), np.nan)
        for s in range(self.S):
            for h in range(self.kv):
                k, v = self.keys(self.kb, self.knb, s, h), self.keys(self.vb, self.vnb, s, h)
                for i in range(self.toks[s]):
                    tok, see = self.first[s] + i, self.sees(s, i, mask)
                    for g in range(self.G):
                        q = from_bits(self.qb[tok, h * self.G + g], self.qt)
                        x = self.scale * (k[see] @ q)
                        if x.size == 0:
                            lse[tok, h * self.G + g] = -np.inf
                            continue
                        m = x.max()
                        z = m + np.log(np.exp(x - m).sum())
                        lse[tok, h * self.G + g] = z
                        out[tok, h * self.G + g] = np.exp(x - z) @ v[see]
        return out, lse

    def accepted(self, s):
        t = range(self.toks[s])
        return list(t) if self.accept is None else [j for j in t if int(self.accept[s]) >> j & 1]

    def score(self, lse, score, out, decay, mask=True):
        out = out.astype(np.float64).copy()
        for s in range(self.S):
            n, acc = self.lens[s], self.accepted(s)
            for h in range(self.kv):
                k = self.keys(self.kb, self.knb, s, h)
                w = np.zeros(len(k))
                for i in acc:
                    see = self.sees(s, i, mask)
                    for g in range(self.G):
                        tok, hd = self.first[s] + i, h * self.G + g
                        x = self.scale * (k[see] @ from_bits(self.qb[tok, hd], self.qt))
                        w[see] += np.exp(x - float(lse[tok, hd]))
                out[s, h, :n] = decay * score[s, h, :n] + w[:n]
                new = w[n:][acc][:max(0, self.max_len - n)]
                out[s, h, n:n + len(new)] = new
        return out
