"""Plain forms of the paged cache's operators in numpy, for the tests: float32 step by step where the
library's bits are defined that way (append), float64 elsewhere.  Test infrastructure only."""
import ctypes as C

import numpy as np

import dfx

BLOCK = 16


def e4m3_table():
    """Value of every E4M3 code (OCP: 0x7f and 0xff are NaN, no infinities)."""
    c = np.arange(256)
    s, e, m = c >> 7, (c >> 3) & 15, c & 7
    v = np.where(e == 0, m * 2.0 ** -9, (8 + m) * 2.0 ** (e.astype(np.float64) - 10))
    v[(c & 127) == 127] = np.nan
    return np.where(s == 1, -v, v)


TABLE = e4m3_table()
_MID = (TABLE[:126] + TABLE[1:127]) / 2


def e4m3(x):
    """Codes of x rounded to nearest, ties to the even code; NaN where x is not finite.  |x| <= 448."""
    x = np.asarray(x, np.float64)
    a = np.abs(np.where(np.isfinite(x), x, 0.0))
    c = np.searchsorted(_MID, a, side="left")                # first code whose upper midpoint is >= a
    tie = (c < 126) & (a == _MID[np.minimum(c, 125)]) & (c % 2 == 1)
    c = np.minimum(c + tie, 126) | np.where(np.signbit(x), 128, 0)
    return np.where(np.isfinite(x), c, 127).astype(np.uint8)


def scale_of(a):
    """2^k of a block whose largest finite magnitude is a."""
    if not a > 0:
        return np.float32(2.0 ** -15)
    k = -15
    while k < 7 and a > 448.0 * 2.0 ** k:
        k += 1
    return np.float32(2.0 ** k)


def rope_table(n_pos, hd, base=500000.0):
    th = np.arange(n_pos, dtype=np.float64)[:, None] * base ** (-np.arange(hd // 2) * 2.0 / hd)
    return np.stack([np.cos(th), np.sin(th)], -1).astype(np.float32)


def rotate(x, tab, pos):
    """NEOX rotation, every product and sum rounded in x's type."""
    h = x.shape[-1] // 2
    cs = tab[pos].astype(x.dtype)[:, None]
    c, s = cs[..., 0], cs[..., 1]
    a, b = x[..., :h], x[..., h:]
    return np.concatenate([a * c - b * s, a * s + b * c], -1)


class Cache:
    """A paged cache in numpy and on the device."""

    def __init__(self, typ, page, Hkv, hd, n_pages, seed=0, fill=True):
        self.typ, self.page, self.Hkv, self.hd, self.n_pages = typ, page, Hkv, hd, n_pages
        self.f8 = typ == dfx.TYPE_F8
        B = page // BLOCK
        rng = np.random.default_rng(seed)
        ks, vs = (n_pages, Hkv, page, hd), (n_pages, Hkv, B, hd, BLOCK)
        if self.f8:
            # what lies in pages before they are written is anything, NaN codes included
            self.k = rng.integers(0, 256, ks, dtype=np.uint8)
            self.v = rng.integers(0, 256, vs, dtype=np.uint8)
            self.scale = (2.0 ** rng.integers(-6, 3, (n_pages, Hkv, B, 2))).astype(np.float32)
        else:
            self.k = rng.standard_normal(ks).astype(np.float16)
            self.v = rng.standard_normal(vs).astype(np.float16)
            self.k[rng.random(ks) < 0.01] = np.nan
            self.v[rng.random(vs) < 0.01] = np.inf
            self.scale = None
        self.dk, self.dv = dfx.Buf.of(self.k), dfx.Buf.of(self.v)
        self.ds = dfx.Buf.of(self.scale) if self.f8 else None

    def desc(self):
        return dfx.PagedCache(self.typ, self.page, self.Hkv, self.hd, self.n_pages, self.dk.ptr, self.dv.ptr,
                              self.ds.ptr if self.f8 else None)

    def upload(self):
        self.dk.upload(self.k)
        self.dv.upload(self.v)
        if self.f8:
            self.ds.upload(self.scale)

    def download(self):
        k, v = self.dk.download(self.k.dtype, shape=self.k.shape), self.dv.download(self.v.dtype, shape=self.v.shape)
        return k, v, self.ds.download(np.float32, shape=self.scale.shape) if self.f8 else None

    def values(self, page, h, pos):
        """(key, value) in float64 at position pos % page of a page."""
        t, b = pos % self.page, pos % self.page // BLOCK
        if self.f8:
            sk, sv = self.scale[page, h, b].astype(np.float64)
            return TABLE[self.k[page, h, t]] * sk, TABLE[self.v[page, h, b, :, t % 16]] * sv
        return self.k[page, h, t].astype(np.float64), self.v[page, h, b, :, t % 16].astype(np.float64)


class Batch:
    """Rows, key counts and page ids of the sequences, in numpy and on the device."""

    def __init__(self, n, keys, page, n_pages, seed=0, pad_rows=0, ld_extra=0, pages=None, max_keys=None):
        self.n, self.keys, self.page = list(n), list(keys), page
        self.rows = np.concatenate([[0], np.cumsum(n)]).astype(np.int32)
        self.M = int(self.rows[-1]) + pad_rows
        need = [-(-k // page) for k in keys]
        ld = max(max(need, default=0), 1) + ld_extra
        if pages is None:
            order = np.random.default_rng(seed).permutation(n_pages)
            pages = np.full((len(n), ld), -1, np.int32)
            at = 0
            for s, m in enumerate(need):
                pages[s, :m] = order[at:at + m]
                at += m
            assert at <= n_pages
        self.pages = pages.astype(np.int32)
        self.max_keys = max(keys, default=0) if max_keys is None else max_keys
        self.d = [dfx.Buf.of(self.rows), dfx.Buf.of(np.asarray(keys, np.int32)), dfx.Buf.of(self.pages)]

    def desc(self):
        return dfx.PagedBatch(len(self.n), self.M, self.d[0].ptr, self.d[1].ptr, self.d[2].ptr, self.pages.shape[1],
                              self.max_keys)

    def set(self, n=None, keys=None):
        """Other lengths in the same device arrays (as a serving loop writes them between replays)."""
        if n is not None:
            self.n, self.rows = list(n), np.concatenate([[0], np.cumsum(n)]).astype(np.int32)
            self.d[0].upload(self.rows)
        if keys is not None:
            self.keys = list(keys)
            self.d[1].upload(np.asarray(keys, np.int32))

    def page_of(self, s, pos, n_pages):
        """Page id of a position, or -1."""
        if pos < 0 or pos // self.page >= self.pages.shape[1]:
            return -1
        p = int(self.pages[s, pos // self.page])
        return p if 0 <= p < n_pages else -1


def ref_append(c, b, qkv, H, tab, q_out):
    """Appends to c's arrays and fills q_out: float32 steps, the bits that the library defines."""
    Hkv, hd = c.Hkv, c.hd
    cap = b.pages.shape[1] * b.page
    x = qkv.reshape(b.M, H + 2 * Hkv, hd)
    for s, m in enumerate(b.n):
        r0 = int(b.rows[s])
        keys = min(max(b.keys[s], 0), cap)
        pos = keys - m + np.arange(m)
        ok = (pos >= 0) & (pos < len(tab))
        if ok.any():
            rows = r0 + np.flatnonzero(ok)
            y = rotate(x[rows][:, :H + Hkv], tab, pos[ok])
            q_out[rows] = y[:, :H].astype(q_out.dtype)
        ok &= pos < cap
        blocks = sorted({int(p) // BLOCK for p in pos[ok]})
        for blk in blocks:
            new = [i for i in range(m) if ok[i] and pos[i] // BLOCK == blk]
            page = b.page_of(s, blk * BLOCK, c.n_pages)
            if page < 0:
                continue
            t0, nb = int(pos[new[0]]) % BLOCK, blk * BLOCK % b.page // BLOCK
            yk = rotate(x[[r0 + i for i in new]][:, H:H + Hkv], tab, pos[new])
            yv = x[[r0 + i for i in new]][:, H + Hkv:]
            for h in range(Hkv):
                kb = c.k[page, h, nb * BLOCK:(nb + 1) * BLOCK]           # [16][hd]
                vb = c.v[page, h, nb].T                                  # [16][hd] view
                for side, cells, y in ((0, kb, yk[:, h]), (1, vb, yv[:, h])):
                    if not c.f8:
                        with np.errstate(over="ignore"):
                            cells[t0:t0 + len(new)] = y.astype(np.float16)
                        continue
                    fin = np.abs(np.where(np.isfinite(y), y, 0.0))
                    sc, old = scale_of(fin.max()), c.scale[page, h, nb, side]
                    if t0 > 0 and old != sc:
                        if old > sc:
                            sc = old
                        else:
                            cells[:t0] = e4m3(TABLE[cells[:t0]] * np.float64(old / sc))
                    c.scale[page, h, nb, side] = sc
                    z = np.where(np.isfinite(y), np.clip(y / sc, np.float32(-448), np.float32(448)), np.nan)
                    cells[t0:t0 + len(new)] = e4m3(z)


def same_cells(c, got, want):
    """Codes equal, NaN codes of either sign alike."""
    if not c.f8:
        return np.array_equal(got.view(np.uint16) & 0x7fff == 0, want.view(np.uint16) & 0x7fff == 0) and \
            np.array_equal(got, want, equal_nan=True)
    nan = (got & 127) == 127
    return np.array_equal(nan, (want & 127) == 127) and np.array_equal(got[~nan], want[~nan])


def ref_attention(c, b, q, causal, window):
    """(out, tolerance base) in float64 from the cache's values: out[r][h], and what the error bound of
    each output is made of: A = sum p |v| (sum of absolute terms), E = the largest sum of |q k| / sqrt(hd)."""
    M, H, hd = q.shape
    G = H // c.Hkv
    cap = b.pages.shape[1] * b.page
    out, A, E = np.zeros((M, H, hd)), np.zeros((M, H, hd)), np.zeros((M, H))
    q = q.astype(np.float64)
    for s, m in enumerate(b.n):
        r0, keys = int(b.rows[s]), min(max(b.keys[s], 0), cap)
        at = np.array([p for p in range(keys) if b.page_of(s, p, c.n_pages) >= 0], np.int64)
        if not len(at) or not m:
            continue
        pos = (keys - m + np.arange(m))[:, None]
        see = np.ones((m, len(at)), bool)
        if causal:
            see &= at <= pos
            if window:
                see &= at > pos - window
        see = np.repeat(see, G, 0)                               # rows of (row, head of the group)
        some = see.any(1)
        for h in range(c.Hkv):
            kv = [c.values(b.page_of(s, int(p), c.n_pages), h, int(p)) for p in at]
            k, v = np.stack([x for x, _ in kv]), np.stack([x for _, x in kv])
            x = q[r0:r0 + m, h * G:(h + 1) * G].reshape(m * G, hd)
            with np.errstate(all="ignore"):
                # NaN of a hidden key must not reach a row: products only where it is seen
                sc = np.where(see, x @ np.where(np.isnan(k), 0.0, k).T / np.sqrt(hd), -np.inf)
                bad = np.isnan(k).any(1)
                sc = np.where(see & bad, np.nan, sc)
                top = np.max(np.where(np.isnan(sc), -np.inf, sc), 1, keepdims=True)
                e = np.where(see, np.exp(sc - np.where(np.isfinite(top), top, 0.0)), 0.0)
                e = e / e.sum(1, keepdims=True)
                fine = np.isfinite(v)
                o, a = e @ np.where(fine, v, 0.0), e @ np.abs(np.where(fine, v, 0.0))
                for j in np.flatnonzero(~fine.all(1)):           # what is not finite, to the rows that see it
                    o[see[:, j]] += np.where(fine[j], 0.0, v[j])
                ee = np.max(np.where(see, np.abs(x) @ np.abs(np.where(np.isnan(k), 0.0, k)).T, 0.0), 1) / np.sqrt(hd)
            o[~some], a[~some] = 0.0, 0.0
            out[r0:r0 + m, h * G:(h + 1) * G] = o.reshape(m, G, hd)
            A[r0:r0 + m, h * G:(h + 1) * G] = a.reshape(m, G, hd)
            E[r0:r0 + m, h * G:(h + 1) * G] = ee.reshape(m, G)
    return out, A, E


def attention_bound(out, A, E, hd, n, f32):
    """Largest error of the library's attention, from its arithmetic.
    Scores: f32 sums of hd exact products, (hd + 3) roundings of 2^-24 of at most E; an error d of a
    score is an error of 2 d (numerator and denominator) of a probability.  Probabilities: exp2 and its
    argument 2^-20 in all; rounded to f16 (2^-11) before P V, as two terms 2^-21.  Sums of n terms:
    n 2^-24 of A each for P V and l.  Terms below f16's range: 2^-39 each, of values up to 2^16 (f16
    results only; 2^-50 with two terms).  The result's rounding: 2^-11 or 2^-24 of it.  f32 queries: two
    f16 terms leave 2^-21 of |q|."""
    Ab = np.nan_to_num(A)
    rel = (2.0 ** -21 if f32 else 2.0 ** -11) + 2 * (hd + 3) * 2.0 ** -24 * E[..., None] + 2.0 ** -20 + 2 * n * 2.0 ** -24
    if f32:
        rel = rel + 2 * 2.0 ** -21 * E[..., None]
    return rel * Ab + (2.0 ** -24 if f32 else 2.0 ** -11) * np.abs(np.nan_to_num(out)) + n * 2.0 ** (-50 if f32 else -39) * 8 + 2.0 ** (-149 if f32 else -25)


def check_attention(got, c, b, q, causal, window, f32):
    out, A, E = ref_attention(c, b, q, causal, window)
    live = int(b.rows[-1])
    g, w = got[:live].astype(np.float64), out[:live]
    lim = np.finfo(np.float32 if f32 else np.float16).max
    with np.errstate(invalid="ignore"):
        w = np.where(np.abs(w) > lim, np.sign(w) * np.inf, w)
    assert np.array_equal(np.isnan(g), np.isnan(w))
    inf = np.isinf(w)
    assert np.array_equal(np.isinf(g), inf) and np.array_equal(g[inf], w[inf])
    n = max(b.keys, default=1)
    fin = np.isfinite(w)
    E = np.nan_to_num(E, nan=0.0, posinf=0.0)
    tol = attention_bound(out, A, E, c.hd, max(n, 1), f32)[:live]
    err = np.abs(g[fin] - w[fin])
    assert (err <= tol[fin]).all(), (float((err / tol[fin]).max()), float(err.max()))


def ref(x):
    return C.byref(x)
