"""The paged key and value cache in 64 bits: 8-bit codes, rotation, append and attention by their formulas."""
import numpy as np

F32, BF16, E4M3 = 0, 1, 2
U = 2.0 ** -24  # half a step of f32


def e4m3_values():
    i = np.arange(256)
    e, f = (i >> 3) & 15, i & 7
    v = np.where(e == 0, f / 8 * 2.0 ** -6, (1 + f / 8) * 2.0 ** (e - 7.0))
    v = np.where(i >= 128, -v, v)
    v[127] = v[255] = np.nan
    return v


VALUES = e4m3_values()
MAGS = VALUES[:127]


def e4m3_codes(x):
    """Codes of 64-bit values: the nearest, of two equally near the even one; what is not finite becomes NaN."""
    a = np.abs(np.where(np.isfinite(x), x, 0.0))
    hi = np.clip(np.searchsorted(MAGS, a), 0, 126)
    lo = np.maximum(hi - 1, 0)
    dl, dh = a - MAGS[lo], MAGS[hi] - a
    c = np.where((dh < dl) | ((dh == dl) & (hi % 2 == 0)), hi, lo)
    c = np.where(np.isfinite(x), c, 127)
    return (c | np.where(np.signbit(x), 128, 0)).astype(np.uint8)


def scale_byte(top):
    """The byte of the least power of two of which 448 times reach top."""
    s = -200.0
    if top > 0:
        s = np.ceil(np.log2(top / 448.0))
        while 448.0 * 2.0 ** (s - 1) >= top:
            s -= 1
        while 448.0 * 2.0 ** s < top:
            s += 1
    return int(max(s + 127, 10))


def rotate(x, pos, freq, amp, rot, inter):
    """x [..., dh] turned by pos * freq, in 64 bits."""
    y = np.array(x, np.float64)
    if not rot:
        return y
    w = pos * np.asarray(freq, np.float64)
    c, s = amp * np.cos(w), amp * np.sin(w)
    i = np.arange(rot // 2)
    a, b = (2 * i, 2 * i + 1) if inter else (i, i + rot // 2)
    y[..., a], y[..., b] = x[..., a] * c - x[..., b] * s, x[..., b] * c + x[..., a] * s
    return y


class Pages:
    """A cache's memory on the host: pages in mixed order, entries of -1 behind each sequence's last."""

    def __init__(self, rng, typ, heads, dh, page, tokens, drop=(), spare=2):
        """tokens: what every row of the table holds; drop: (row, page) that are taken out of the table."""
        self.typ, self.heads, self.dh, self.page = typ, heads, dh, page
        counts = [-(-t // page) for t in tokens]
        self.pages = sum(counts) + spare
        order = rng.permutation(self.pages)
        self.table = np.full((len(tokens), max(1, max(counts)) + 1), -1, np.int32)
        at = 0
        for r, c in enumerate(counts):
            self.table[r, :c] = order[at:at + c]
            at += c
        for r, j in drop:
            self.table[r, j] = -1
        shape = (self.pages, heads, page, dh)
        if typ == E4M3:
            self.k, self.v = (e4m3_codes(rng.standard_normal(shape) * 64) for _ in "kv")
            self.ks, self.vs = (rng.integers(119, 123, (self.pages, heads, page // 16)).astype(np.uint8) for _ in "kv")
        else:
            self.k, self.v = ((rng.standard_normal(shape).astype(np.float32).view(np.uint32) >> 16).astype(np.uint16) for _ in "kv")
            self.ks = self.vs = None

    def values(self, name):
        """All values in 64 bits, [pages][heads][page][dh]."""
        c = getattr(self, name)
        if self.typ == E4M3:
            s = getattr(self, name + "s").astype(np.float64) - 127
            return VALUES[c] * np.repeat(2.0 ** s, 16, 2)[..., None]
        return (c.astype(np.uint32) << 16).view(np.float32).astype(np.float64)

    def tokens(self, name, row, n):
        """(values [n][heads][dh], whether they are there) of a row's first n tokens."""
        j = np.arange(n)
        p = self.table[row][j // self.page]
        ok = (p >= 0) & (p < self.pages)
        v = self.values(name)[np.where(ok, p, 0), :, j % self.page]
        return np.where(ok[:, None, None], v, 0.0), ok


def attend(q, pages, seqs, window, sinks, scale, typ, out):
    """(rows, bounds) of q [M][heads][dh] in 64 bits over the sequences, into copies of out [M][heads][dh].  The bound of
    an element, with the formula's weights p_j: a logit is off by (dh + 16) roundings of the sum of its products'
    magnitudes and 4 of its own and the maximum's, the exponential adds 2 roundings; the sums add one rounding for every step of 32 tokens and 40 for the joining; bf16 rows round
    every probability and the output (2^-8 each)."""
    y, e = out.astype(np.float64), np.zeros_like(out, np.float64)
    heads, dh = q.shape[1:]
    group = heads // pages.heads
    for first, rows, start, row in seqs:
        if not rows:
            continue
        n = start + rows
        k, ok = pages.tokens("k", row, n)
        v, _ = pages.tokens("v", row, n)
        j = np.arange(n)
        for i in range(rows):
            p = start + i
            see = ok & (j <= p)
            if window:
                see &= (j > p - window) | (j < sinks)
            for h in range(heads):
                if not see.any():
                    y[first + i, h] = 0.0
                    continue
                kk, vv, qq = k[see, h // group], v[see, h // group], q[first + i, h]
                s = scale * (kk @ qq)
                w = np.exp(s - s.max())
                w /= w.sum()
                o = w @ vv
                d = U * ((dh + 16) * scale * (np.abs(kk) @ np.abs(qq)) + 4 * (np.abs(s) + np.abs(s).max()) + 2)
                a = w @ np.abs(vv)
                err = (w * d) @ (np.abs(vv) + np.abs(o)) + U * (n / 32 + 40) * a
                if typ == BF16:
                    err += 2.0 ** -8 * (a + np.abs(o) + err)
                y[first + i, h], e[first + i, h] = o, err + 1e-36
    return y, e
