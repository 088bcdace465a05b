"""The paged key and value cache on the GPU: rotated rows appended and read back, and attention over it, against the
formulas in 64 bits (kv_ref.py has the bounds of the attention).

A rotated value x c - y s is off by at most 8 roundings (u = 2^-24) of amp (|x| + |y|): cosine and sine 2 each with the factor
amp's, two products' and the difference's.  Values that are not rotated are exact in f32.  bf16 rounds once more (2^-8), 8
bits too: 2^-4 of the value, or half a step of the block's smallest codes (2^-10 of its scale).
"""
import copy
import ctypes as C

import numpy as np
import pytest

import nemoasr
import oracle
from kv_ref import BF16, E4M3, F32, U, VALUES, Pages, attend, e4m3_codes, rotate, scale_byte

pytestmark = pytest.mark.gpu


def bits(x, typ):
    return oracle.f32_to_bf16(np.asarray(x, np.float32)) if typ == BF16 else np.ascontiguousarray(x, np.float32)


def kept(x, typ):
    """What rows of the type hold of x, in 64 bits."""
    x = np.asarray(x, np.float32)
    return (oracle.bf16_to_f32(oracle.f32_to_bf16(x)) if typ == BF16 else x).astype(np.float64)


def back(b, typ):
    return (oracle.bf16_to_f32(b) if typ == BF16 else b).astype(np.float64)


class Rows:
    """Rows [M][n] of a type on the device inside a larger buffer: `off` values before, a stride of ld, `behind` rows behind."""

    def __init__(self, gpu, x, typ, ld=None, off=0, behind=2, fill=9):
        M, n = x.shape
        self.typ, self.M, self.n, self.ld, self.off = typ, M, n, ld or n, off
        dt = np.uint16 if typ == BF16 else np.float32
        self.a = np.full(off + (M + behind) * self.ld, fill, dt)
        self.a[off:off + M * self.ld].reshape(M, self.ld)[:, :n] = bits(x, typ)
        self.buf = gpu.put(self.a)

    @property
    def ptr(self):
        return self.buf.at(self.off * self.a.itemsize)

    def read(self):
        """([M][n] bits, whether all else is as it was)"""
        b = self.buf.read(self.a.shape, self.a.dtype)
        rest, was = b.copy(), self.a.copy()
        for r in (rest, was):
            r[self.off:self.off + self.M * self.ld].reshape(self.M, self.ld)[:, :self.n] = 0
        return b[self.off:self.off + self.M * self.ld].reshape(self.M, self.ld)[:, :self.n], np.array_equal(rest, was)


class Cache:
    """A Pages on the device."""

    def __init__(self, gpu, pages):
        self.pages = pages
        self.bufs = [gpu.put(x) if x is not None else None for x in (pages.k, pages.v, pages.ks, pages.vs, pages.table)]
        k, v, ks, vs, table = (b.ptr if b else None for b in self.bufs)
        self.kv = nemoasr.Kv(type=pages.typ, heads=pages.heads, dh=pages.dh, page=pages.page, pages=pages.pages, k=k, v=v, ks=ks, vs=vs,
                             table=table, ldt=pages.table.shape[1], tables=pages.table.shape[0])

    def pull(self):
        """The host's Pages with what the device has now."""
        p = self.pages
        for b, name in zip(self.bufs, ("k", "v", "ks", "vs")):
            if b:
                setattr(p, name, b.read(getattr(p, name).shape, getattr(p, name).dtype))
        return p

    def free(self):
        for b in self.bufs:
            if b:
                b.free()


def sequences(rows, starts, gap=0):
    """Table rows of sequences one after another; their rows of the page table in another order."""
    out, first, n = [], 0, len(rows)
    for i, (r, s) in enumerate(zip(rows, starts)):
        out.append((first, r, s, n - 1 - i))
        first += r + gap
    return np.array(out, np.int32).reshape(-1, 4), max(1, first)


def tokens_of(seqs):
    n = np.zeros(len(seqs), int)
    for _, rows, start, row in seqs:
        n[row] = rows + start
    return n


def close(got, ref, bound):
    bad = ~(np.abs(got - ref) <= bound)
    assert not bad.any(), (int(bad.sum()), np.argwhere(bad)[:3], got[bad][:3], ref[bad][:3], np.broadcast_to(bound, ref.shape)[bad][:3])


# ---- append ------------------------------------------------------------------------------------------

BATCHES = [  # rows and tokens before them
    ([1], [0]),
    ([1, 1, 1], [5, 16, 4095]),
    ([3, 0, 40, 17, 1], [13, 7, 0, 31, 100]),
    ([70, 16, 15], [0, 32, 1]),
]
FREQ = 10000.0


def freqs(rot, scaling=0, *more):
    f = np.zeros(max(1, rot // 2), np.float32)
    if rot:
        assert nemoasr.lib().nk_rope_freqs(f.ctypes.data, rot, FREQ, scaling, *(more or (1.0, 0.0, 0.0, 0.0))) == 0
    return f


def run_append(gpu, cache, typ, q, k, v, seqs, heads, rot, inter, freq, amp=1.0, max_rows=None, ld=None, off=0, inplace=False):
    M = (q if q is not None else k).shape[0]
    dq = Rows(gpu, q, typ, ld, off) if q is not None else None
    dk, dv = (Rows(gpu, x, typ, ld, off) if x is not None else None for x in (k, v))
    do = dq if inplace else Rows(gpu, np.zeros_like(q), typ, ld and ld + 8, off) if q is not None else None
    ds, df = gpu.put(seqs), gpu.put(freq)
    a = nemoasr.Append(type=typ, heads=heads, rot=rot, inter=int(inter), freq=df.ptr, amp=amp, seqs=ds.ptr, nseq=len(seqs),
                       max_rows=max_rows or int(seqs[:, 1].max()), M=M)
    if dq:
        a.q, a.ldq, a.qo, a.ldqo = dq.ptr, dq.ld, do.ptr, do.ld
    if dk:
        a.k, a.ldk, a.v, a.ldv = dk.ptr, dk.ld, dv.ptr, dv.ld
    gpu.begin()
    gpu.check(nemoasr.lib().nk_kv_append(gpu.h, C.byref(cache.kv), C.byref(a)))
    gpu.end()
    out = None
    if do:
        out, same = do.read()
        assert same
    for r in (dk, dv):
        if r:
            b, same = r.read()
            assert same and b.tobytes() == r.a[r.off:r.off + r.M * r.ld].reshape(r.M, r.ld)[:, :r.n].tobytes()  # NaN among them
    for b in [ds, df] + [r.buf for r in {id(x): x for x in (dq, dk, dv, do) if x}.values()]:
        b.free()
    return out


def check_append(before, after, seqs, k, v, typ, rot, inter, freq, amp):
    """The cache after an append against the one before; k, v [M][heads][dh] as the rows hold them."""
    ref = {n: getattr(before, n).copy() for n in ("k", "v")}
    want_s = {n: None if before.ks is None else getattr(before, n + "s").copy() for n in ("k", "v")}
    dh = before.dh
    for first, rows, start, row in seqs:
        for name, x in (("k", k), ("v", v)):
            new = np.array([rotate(x[first + i], start + i, freq, amp, rot, inter) for i in range(rows)]).reshape(rows, before.heads, dh) \
                if name == "k" else x[first:first + rows]
            turned = np.zeros(dh, bool)
            if name == "k":
                turned[:rot] = True
            cells = getattr(before, name)
            got = getattr(after, name)
            for b in range(start // 16, -(-(start + rows) // 16) if rows else start // 16):
                p = before.table[row][16 * b // before.page]
                if not 0 <= p < before.pages:
                    continue
                lo, hi, o = max(start, 16 * b), min(start + rows, 16 * b + 16), 16 * b % before.page
                fresh = new[lo - start:hi - start].transpose(1, 0, 2)  # [heads][tokens][dh]
                src = np.abs(x[first + lo - start:first + hi - start]).transpose(1, 0, 2)
                pair = np.zeros_like(src)
                if name == "k" and rot:
                    i = np.arange(rot // 2)
                    ia, ib = (2 * i, 2 * i + 1) if inter else (i, i + rot // 2)
                    pair[..., ia] = pair[..., ib] = abs(amp) * (src[..., ia] + src[..., ib])
                err = 8 * U * pair
                for h in range(before.heads):
                    cell = got[p, h, o + lo - 16 * b:o + hi - 16 * b]
                    if before.typ == BF16:
                        g = oracle.bf16_to_f32(cell).astype(np.float64)
                        close(g, fresh[h], err[h] + 2.0 ** -8 * (np.abs(fresh[h]) + err[h]))
                        assert np.array_equal(cell[:, ~turned], oracle.f32_to_bf16(fresh[h][:, ~turned].astype(np.float32)))
                        ref[name][p, h, o + lo - 16 * b:o + hi - 16 * b] = cell
                        continue
                    s_got = int(getattr(after, name + "s")[p, h, o // 16])
                    a = np.abs(fresh[h])[np.isfinite(fresh[h])]
                    top, e_top = (float(a.max()), float(err[h].max())) if a.size else (0.0, 0.0)
                    was = int(getattr(before, name + "s")[p, h, o // 16]) if lo > 16 * b else 0
                    assert s_got in {max(scale_byte(t), was) for t in (top - e_top, top, top + e_top)}, (s_got, top, was)
                    want_s[name][p, h, o // 16] = s_got
                    step = 2.0 ** (s_got - 127)
                    with np.errstate(invalid="ignore"):
                        close(VALUES[cell][np.isfinite(fresh[h])] * step, fresh[h][np.isfinite(fresh[h])],
                              (err[h] + 2.0 ** -4 * (np.abs(fresh[h]) + err[h]) + 2.0 ** -10 * step)[np.isfinite(fresh[h])])
                    assert np.array_equal(cell[:, ~turned] & 127 if not np.isfinite(fresh).all() else cell[:, ~turned],
                                          e4m3_codes(fresh[h][:, ~turned] / step) & (127 if not np.isfinite(fresh).all() else 255))
                    ref[name][p, h, o + lo - 16 * b:o + hi - 16 * b] = cell
                    if was and s_got > was:  # the older tokens' codes rounded again
                        old = cells[p, h, o:o + lo - 16 * b]
                        again = e4m3_codes(VALUES[old] * 2.0 ** (was - s_got))
                        assert np.array_equal(got[p, h, o:o + lo - 16 * b], again)
                        ref[name][p, h, o:o + lo - 16 * b] = again
    for name in ("k", "v"):  # and nothing else
        assert np.array_equal(getattr(after, name), ref[name])
        if want_s[name] is not None:
            assert np.array_equal(getattr(after, name + "s"), want_s[name])


HEADS = [  # heads, heads of the cache, dh, rotated, pairs side by side
    (8, 8, 128, 128, False), (4, 1, 64, 64, True), (6, 2, 96, 48, True), (3, 3, 80, 20, False), (5, 5, 16, 0, False), (8, 2, 256, 64, False),
    (2, 1, 48, 6, True), (2, 2, 112, 24, False),
]


@pytest.mark.parametrize("batch", range(len(BATCHES)))
@pytest.mark.parametrize("shape", range(len(HEADS)))
@pytest.mark.parametrize("cache_type", [BF16, E4M3])
@pytest.mark.parametrize("typ", [F32, BF16])
def test_append(gpu, batch, shape, cache_type, typ):
    heads, hk, dh, rot, inter = HEADS[shape]
    rng = np.random.default_rng([batch, shape, cache_type, typ])
    seqs, M = sequences(*BATCHES[batch], gap=batch % 2)
    page = (16, 64, 32)[(batch + shape) % 3]
    pages = Pages(rng, cache_type, hk, dh, page, tokens_of(seqs))
    before = copy.deepcopy(pages)
    q, k, v = (rng.standard_normal((M, n * dh)) * np.exp(rng.standard_normal((M, 1))) for n in (heads, hk, hk))
    # the rows as they are, strides of other rows between, rows off 16 bytes
    more = [dict(), dict(ld=max(heads, hk) * dh + 24), dict(ld=max(heads, hk) * dh + 3, off=1), dict(off=4)][(batch + shape) % 4]
    freq = freqs(rot)
    amp = 1.0 if shape % 2 else 1.25
    cache = Cache(gpu, pages)
    out = run_append(gpu, cache, typ, q, k, v, seqs, heads, rot, inter, freq, amp, max_rows=int(seqs[:, 1].max()) + 50 * (shape % 2), **more)
    after = cache.pull()
    cache.free()
    qk, kk, vk = (kept(x, typ).reshape(M, -1, dh) for x in (q, k, v))
    check_append(before, after, seqs, kk, vk, typ, rot, inter, freq, np.float32(amp))
    got = back(out, typ).reshape(M, heads, dh)
    mine = np.zeros(M, bool)
    for first, rows, start, _ in seqs:
        for i in range(first, first + rows):
            mine[i] = True
            ref = rotate(qk[i], start + i - first, freq, np.float32(amp), rot, inter)
            err = np.zeros_like(ref)
            if rot:
                j = np.arange(rot // 2)
                a, b = (2 * j, 2 * j + 1) if inter else (j, j + rot // 2)
                err[:, a] = err[:, b] = 8 * U * amp * (np.abs(qk[i][:, a]) + np.abs(qk[i][:, b]))
            close(got[i], ref, err + (2.0 ** -8 * (np.abs(ref) + err) if typ == BF16 else 0))
    assert (out[~mine] == 0).all()


@pytest.mark.parametrize("typ", [F32, BF16])
def test_append_far_positions(gpu, typ):
    """Angles of a million radians keep their turns; scaled frequencies."""
    rng = np.random.default_rng(3)
    heads, dh, rot = 2, 64, 64
    seqs = np.array([(0, 3, 1000003, 0), (3, 2, 2 ** 24 + 1, 1)], np.int32)
    page = 1 << 15
    table_len = (2 ** 24 + 3) // page + 1
    pages = Pages(rng, BF16, heads, dh, page, [1, 1])
    pages.table = np.full((2, table_len), -1, np.int32)
    pages.table[0, 1000003 // page] = 1
    pages.table[1, (2 ** 24 + 1) // page] = 0
    before = copy.deepcopy(pages)
    freq = freqs(rot, 3, 8.0, 8192.0, 1.0, 4.0)
    q, k, v = (rng.standard_normal((5, heads * dh)) for _ in "qkv")
    cache = Cache(gpu, pages)
    out = run_append(gpu, cache, typ, q, k, v, seqs, heads, rot, False, freq)
    after = cache.pull()
    cache.free()
    check_append(before, after, seqs, kept(k, typ).reshape(5, heads, dh), kept(v, typ).reshape(5, heads, dh), typ, rot, False, freq, 1.0)
    for first, rows, start, _ in seqs:
        for i in range(rows):
            x = kept(q, typ).reshape(5, heads, dh)[first + i]
            ref = rotate(x, start + i, freq, 1.0, rot, False)
            err = 8 * U * np.tile(np.abs(x[:, :32]) + np.abs(x[:, 32:]), 2)
            close(back(out, typ).reshape(5, heads, dh)[first + i], ref, err + (2.0 ** -8 * (np.abs(ref) + err) if typ == BF16 else 0))


def test_append_scales_of_far_apart_values(gpu):
    """Rows one at a time into a block: the scale grows with them and never falls, older codes become subnormal and zero;
    zeros, tiny and huge values, infinities and NaN."""
    rng = np.random.default_rng(4)
    hk, dh = 1, 32
    tops = [0.0, 1e-38, 1e-3, 1.0, 448.0, 449.0, 1e4, 3.0, 1e9, 3e38, 0.0, 1.0, np.inf, np.nan, 2.0, 5.0]
    pages = Pages(rng, E4M3, hk, dh, 16, [17])
    cache = Cache(gpu, pages)
    for t, top in enumerate(tops):
        before = copy.deepcopy(cache.pages)
        x = rng.uniform(-1, 1, (1, dh)).astype(np.float32)
        x[0, 5] = 1.0
        with np.errstate(invalid="ignore"):
            x *= np.float32(top) if np.isfinite(top) else np.float32(1.0)
        if not np.isfinite(top):
            x[0, 7] = top
            x[0, 8] = -top
        seqs = np.array([(0, 1, t, 0)], np.int32)
        run_append(gpu, cache, F32, None, x, -x[:, ::-1], seqs, 1, 0, False, freqs(0))
        after = cache.pull()
        check_append(before, after, seqs, kept(x, F32).reshape(1, hk, dh), kept(-x[:, ::-1], F32).reshape(1, hk, dh), F32, 0, False, None, 1.0)
    cache.free()


def test_append_parts(gpu):
    """Queries alone, in place; keys and values alone; entries that do not fit, pages that are not there."""
    rng = np.random.default_rng(5)
    heads, hk, dh = 4, 2, 32
    seqs = np.array([(0, 3, 14, 0), (3, 2, 40, 1), (5, 2, 0, 9), (-1, 2, 0, 0), (5, 3, 0, 1), (5, 2, 47, 1), (5, 1, -1, 1)], np.int32)
    M = 7
    q, k, v = (rng.standard_normal((M, n * dh)) for n in (heads, hk, hk))
    pages = Pages(rng, E4M3, hk, dh, 16, [17, 42])
    pages.table = np.ascontiguousarray(pages.table[:, :3])  # 48 tokens
    pages.table[0, 1] = pages.pages  # token 16 of the first is nowhere
    before = copy.deepcopy(pages)
    cache = Cache(gpu, pages)
    freq = freqs(32)
    out = run_append(gpu, cache, F32, q, None, None, seqs, heads, 32, False, freq, inplace=True, max_rows=3)
    after = cache.pull()
    assert np.array_equal(after.k, before.k) and np.array_equal(after.ks, before.ks)
    qk = kept(q, F32).reshape(M, heads, dh)
    for i, p in enumerate([14, 15, 16, 40, 41]):
        ref = rotate(qk[i], p, freq, 1.0, 32, False)
        close(out[i].reshape(heads, dh), ref, 8 * U * np.tile(np.abs(qk[i][:, :16]) + np.abs(qk[i][:, 16:]), 2))
    assert np.array_equal(out[5:], bits(q, F32)[5:])  # of sequences that are left out
    run_append(gpu, cache, F32, None, k, v, seqs, heads, 32, False, freq, max_rows=3)
    after = cache.pull()
    cache.free()
    check_append(before, after, seqs[:2], kept(k, F32).reshape(M, hk, dh), kept(v, F32).reshape(M, hk, dh), F32, 32, False, freq, 1.0)


def test_append_many_sequences(gpu):
    """More sequences than a wavefront has lanes, most of them with one row or none."""
    rng = np.random.default_rng(6)
    n, hk, dh = 700, 1, 16
    rows = rng.integers(0, 3, n)
    rows[[3, 500]] = 37, 60
    seqs, M = sequences(list(rows), list(rng.integers(0, 40, n)))
    pages = Pages(rng, E4M3, hk, dh, 16, tokens_of(seqs))
    before = copy.deepcopy(pages)
    k, v = (rng.standard_normal((M, dh)) for _ in "kv")
    cache = Cache(gpu, pages)
    run_append(gpu, cache, BF16, None, k, v, seqs, 1, 16, True, freqs(16))
    after = cache.pull()
    cache.free()
    check_append(before, after, seqs, kept(k, BF16).reshape(M, 1, dh), kept(v, BF16).reshape(M, 1, dh), BF16, 16, True, freqs(16), 1.0)


@pytest.mark.parametrize("typ", [F32, BF16])
@pytest.mark.parametrize("cache_type", [BF16, E4M3])
@pytest.mark.parametrize("dh,ld,off", [(128, None, 0), (80, 83, 1), (16, None, 0)])
def test_read(gpu, typ, cache_type, dh, ld, off):
    rng = np.random.default_rng([typ, cache_type, dh])
    hk = 3 if dh == 128 else 1
    seqs, M = sequences([1, 0, 40, 21], [7, 3, 0, 30], gap=1)
    pages = Pages(rng, cache_type, hk, dh, 32, tokens_of(seqs), drop=[(0, 1)])
    cache = Cache(gpu, pages)
    K, V = (Rows(gpu, np.zeros((M, hk * dh)), typ, ld, off) for _ in "kv")
    ds = gpu.put(seqs)
    gpu.begin()
    gpu.check(nemoasr.lib().nk_kv_read(gpu.h, C.byref(cache.kv), K.ptr, K.ld, V.ptr, V.ld, typ, ds.ptr, len(seqs), 99, M))
    gpu.check(nemoasr.lib().nk_kv_read(gpu.h, C.byref(cache.kv), None, 0, V.ptr, V.ld, typ, ds.ptr, len(seqs), 40, M))
    gpu.end()
    for name, r in (("k", K), ("v", V)):
        got, same = r.read()
        assert same
        ref = np.zeros((M, hk, dh))
        for first, rows, start, row in seqs:
            ref[first:first + rows] = pages.tokens(name, row, start + rows)[0][start:]
        assert np.array_equal(back(got, typ).reshape(M, hk, dh), ref)
        r.buf.free()
    ds.free()
    cache.free()


# ---- attention ---------------------------------------------------------------------------------------


def run_attend(gpu, cache, typ, q, seqs, heads, window=0, sinks=0, scale=None, max_rows=None, max_len=None, ld=None, off=0, fill=0.0):
    M = q.shape[0]
    dq = Rows(gpu, q, typ, ld, off)
    do = Rows(gpu, np.full_like(q, fill), typ, ld and ld + 4, off)
    ds = gpu.put(seqs)
    a = nemoasr.Attend(type=typ, q=dq.ptr, ldq=dq.ld, o=do.ptr, ldo=do.ld, heads=heads, window=window, sinks=sinks,
                       scale=scale or cache.pages.dh ** -0.5, seqs=ds.ptr, nseq=len(seqs), max_rows=max_rows or int(seqs[:, 1].max()),
                       max_len=max_len or int((seqs[:, 1] + seqs[:, 2]).max()), M=M)
    gpu.begin()
    gpu.check(nemoasr.lib().nk_attention_kv(gpu.h, C.byref(cache.kv), C.byref(a)))
    gpu.end()
    out, same = do.read()
    assert same
    for b in (dq.buf, do.buf, ds):
        b.free()
    return out


def check_attend(gpu, rng, typ, cache_type, heads, hk, dh, page, seqs, M, window=0, sinks=0, drop=(), scale=None, **more):
    pages = Pages(rng, cache_type, hk, dh, page, tokens_of(seqs), drop)
    cache = Cache(gpu, pages)
    q = rng.standard_normal((M, heads * dh)) * 2
    out = run_attend(gpu, cache, typ, q, seqs, heads, window, sinks, scale, fill=7.0, **more)
    cache.free()
    ref, bound = attend(kept(q, typ).reshape(M, heads, dh), pages, seqs, window, sinks, np.float32(scale or dh ** -0.5), typ,
                        np.full((M, heads, dh), 7.0))
    close(back(out, typ).reshape(M, heads, dh), ref, bound)


ATTEND_BATCHES = [
    ([1], [0]),
    ([1, 1, 1, 1], [0, 31, 32, 400]),
    ([7, 0, 1, 16], [50, 9, 700, 15]),
    ([70, 1, 33], [0, 300, 5]),
]
ATTEND_HEADS = [(8, 8, 128), (8, 2, 64), (3, 1, 80), (4, 4, 16), (6, 2, 256), (40, 2, 32), (2, 2, 192), (12, 4, 96)]


@pytest.mark.parametrize("batch", range(len(ATTEND_BATCHES)))
@pytest.mark.parametrize("shape", range(len(ATTEND_HEADS)))
@pytest.mark.parametrize("cache_type", [BF16, E4M3])
@pytest.mark.parametrize("typ", [F32, BF16])
def test_attend(gpu, batch, shape, cache_type, typ):
    heads, hk, dh = ATTEND_HEADS[shape]
    rng = np.random.default_rng([7, batch, shape, cache_type, typ])
    seqs, M = sequences(*ATTEND_BATCHES[batch], gap=shape % 2)
    more = [dict(), dict(ld=heads * dh + 8), dict(ld=heads * dh + 3, off=1), dict(max_rows=200, max_len=5000)][(batch + shape) % 4]
    check_attend(gpu, rng, typ, cache_type, heads, hk, dh, (16, 64, 32)[(batch + shape) % 3], seqs, M, **more)


@pytest.mark.parametrize("window,sinks", [(1, 0), (16, 4), (33, 40), (100, 1), (31, 64), (1000, 5)])
@pytest.mark.parametrize("batch", [1, 2, 3])
@pytest.mark.parametrize("cache_type", [BF16, E4M3])
def test_attend_window(gpu, window, sinks, batch, cache_type):
    rng = np.random.default_rng([8, window, sinks, batch])
    seqs, M = sequences(*ATTEND_BATCHES[batch])
    typ = (F32, BF16)[(window + batch) % 2]
    drop = []
    for _, rows, start, row in seqs:  # pages that no row sees are gone
        drop += [(row, j) for j in range((start + rows) // 16) if sinks <= 16 * j and 16 * j + 16 <= start + 1 - window]
    check_attend(gpu, rng, typ, cache_type, 4, 2, 64, 16, seqs, M, window, sinks, drop)


@pytest.mark.parametrize("typ", [F32, BF16])
@pytest.mark.parametrize("cache_type", [BF16, E4M3])
def test_attend_pages_not_there(gpu, typ, cache_type):
    """Tokens of such a page are not seen; a row that sees none gets zeros."""
    rng = np.random.default_rng([9, typ, cache_type])
    seqs, M = sequences([20, 3, 1], [20, 0, 600], gap=2)
    check_attend(gpu, rng, typ, cache_type, 4, 2, 48, 16, seqs, M, drop=[(2, 0), (2, 2), (1, 0)] + [(0, j) for j in range(38)])
    check_attend(gpu, rng, typ, cache_type, 4, 2, 48, 16, seqs, M, 16, 3, drop=[(0, j) for j in range(0, 38, 3)] + [(1, 0), (2, 1)])


@pytest.mark.parametrize("typ", [F32, BF16])
@pytest.mark.parametrize("cache_type", [BF16, E4M3])
@pytest.mark.parametrize("heads,hk,dh", [(4, 1, 128), (8, 8, 64), (2, 1, 256)])
def test_attend_long(gpu, typ, cache_type, heads, hk, dh):
    """Enough tokens to be split, with short sequences beside them."""
    rng = np.random.default_rng([10, typ, cache_type, heads])
    seqs, M = sequences([1, 1, 2, 0], [5000, 3, 2047, 77])
    check_attend(gpu, rng, typ, cache_type, heads, hk, dh, 64, seqs, M)
    check_attend(gpu, rng, typ, cache_type, heads, hk, dh, 64, seqs, M, 1500, 70)


def test_attend_many_sequences(gpu):
    rng = np.random.default_rng(11)
    n = 300
    rows = rng.integers(0, 3, n)
    rows[[7, 200]] = 30, 50
    seqs, M = sequences(list(rows), list(rng.integers(0, 90, n)))
    check_attend(gpu, rng, BF16, BF16, 2, 1, 32, 16, seqs, M)
    seqs[:, 2] += np.where(np.arange(n) % 50 == 9, 900, 0)
    check_attend(gpu, rng, BF16, E4M3, 2, 1, 32, 16, seqs, M)


def test_attend_entries_that_do_not_fit(gpu):
    rng = np.random.default_rng(12)
    seqs, M = sequences([2, 2, 2, 2, 2, 2], [30, 5, 40, 4, 9, 3])
    pages = Pages(rng, BF16, 2, 32, 16, tokens_of(seqs))
    cache = Cache(gpu, pages)
    q = rng.standard_normal((M, 128))
    bad = seqs.copy()
    bad[0, 3], bad[1, 2], bad[2, 1], bad[3, 0], bad[4, 3] = 6, 47, 9, M - 1, -1
    out = run_attend(gpu, cache, F32, q, bad, 4, max_rows=8, max_len=48, fill=7.0)
    cache.free()
    ref, bound = attend(kept(q, F32).reshape(M, 4, 32), pages, seqs[5:], 0, 0, np.float32(32 ** -0.5), F32, np.full((M, 4, 32), 7.0))
    close(out.reshape(M, 4, 32), ref, bound)


@pytest.mark.parametrize("typ", [F32, BF16])
@pytest.mark.parametrize("long", [0, 3000])
def test_attend_values_not_finite(gpu, typ, long):
    """Infinities and NaN of keys and values: in the rows that see them, as the formula has it, and in no other; tokens
    behind the last row may hold anything."""
    rng = np.random.default_rng([13, long])
    dh, rows = 64, 40
    seqs = np.array([(0, rows, long, 0), (rows, 1, 5, 1)], np.int32)
    n = long + rows
    pages = Pages(rng, BF16, 1, dh, 16, [n, 6])

    def put(name, j, d, value):
        getattr(pages, name)[pages.table[0, j // 16], 0, j % 16, d] = oracle.f32_to_bf16(np.array([value], np.float32))[0]

    put("v", long + 10, 3, np.inf)
    put("v", long + 10, 4, -np.inf)
    put("v", long + 20, 5, np.nan)
    put("v", long + 25, 3, -np.inf)
    put("k", long + 30, 7, np.nan)
    for name in ("k", "v"):  # behind the last row, and pages of no sequence
        c = getattr(pages, name)
        used = np.zeros(c.shape[:1] + c.shape[2:3], bool)
        for r, t in ((0, n), (1, 6)):
            j = np.arange(t)
            used[pages.table[r][j // 16], j % 16] = True
        c[~used[:, None, :]] = 0x7fc0
    q = kept(rng.standard_normal((rows + 1, dh)), typ)
    cache = Cache(gpu, pages)
    out = back(run_attend(gpu, cache, typ, q, seqs, 1), typ).reshape(rows + 1, 1, dh)
    cache.free()
    k, v = (pages.tokens(x, 0, n)[0][:, 0] for x in "kv")
    fin = np.where(np.isfinite(v), v, 0.0)
    for i in range(rows):
        p = long + i
        if i >= 30:
            assert np.isnan(out[i]).all()
            continue
        s = (k[:p + 1] @ q[i]) * dh ** -0.5
        w = np.exp(s - s.max())
        ref = w @ fin[:p + 1] / w.sum()
        for d in range(dh):
            if d == 3 and i >= 25:
                assert np.isnan(out[i, 0, d])
            elif d == 3 and i >= 10:
                assert out[i, 0, d] == np.inf
            elif d == 4 and i >= 10:
                assert out[i, 0, d] == -np.inf
            elif d == 5 and i >= 20:
                assert np.isnan(out[i, 0, d])
            else:
                assert abs(out[i, 0, d] - ref[d]) < 0.05, (i, d)  # values below 5, two roundings to bf16
    assert np.isfinite(out[rows]).all()


def test_attend_logits_far_apart(gpu):
    """Logits of +-1e4 and products past f32: the largest wins, and what overflows is what the formula gives in f32."""
    rng = np.random.default_rng(14)
    dh = 32
    seqs = np.array([(0, 40, 0, 0)], np.int32)
    pages = Pages(rng, BF16, 1, dh, 16, [40])
    cache = Cache(gpu, pages)
    for size in (1e3, 1e-30):
        q = kept(rng.standard_normal((40, dh)) * size, F32)
        out = run_attend(gpu, cache, F32, q, seqs, 1)
        ref, bound = attend(q.reshape(40, 1, dh), pages, seqs, 0, 0, np.float32(dh ** -0.5), F32, np.zeros((40, 1, dh)))
        close(out.reshape(40, 1, dh), ref, bound)
    cache.free()


def test_attend_largest_queries(gpu):
    """Queries up to the largest f32, which round to infinity in bf16, against keys that keep the products in range; where
    they are not, the formula's logits are infinite and the row NaN."""
    rng = np.random.default_rng(25)
    dh = 32
    seqs = np.array([(0, 3, 20, 0)], np.int32)
    pages = Pages(rng, BF16, 1, dh, 16, [23])
    pages.k = oracle.f32_to_bf16(oracle.bf16_to_f32(pages.k) * np.float32(2.0 ** -120))
    cache = Cache(gpu, pages)
    q = np.full((3, dh), np.finfo(np.float32).max, np.float64) * np.where(rng.random((3, dh)) < 0.5, -1, 1)
    out = run_attend(gpu, cache, F32, q, seqs, 1, scale=2.0 ** -8)
    ref, bound = attend(kept(q, F32).reshape(3, 1, dh), pages, seqs, 0, 0, np.float32(2.0 ** -8), F32, np.zeros((3, 1, dh)))
    close(out.reshape(3, 1, dh), ref, bound)
    cache.free()
    pages.k = oracle.f32_to_bf16(oracle.bf16_to_f32(pages.k) * np.float32(2.0 ** 120))
    cache = Cache(gpu, pages)
    assert np.isnan(run_attend(gpu, cache, F32, np.abs(q), seqs, 1)).all()
    cache.free()


@pytest.mark.parametrize("typ", [F32, BF16])
@pytest.mark.parametrize("rows,start", [(1, 700), (150, 0), (3, 5000)])
def test_attend_all_values_nan(gpu, typ, rows, start):
    """A cache that holds nothing but NaN, and queries that are NaN: NaN rows, and at once."""
    rng = np.random.default_rng(26)
    seqs = np.array([(0, rows, start, 0)], np.int32)
    pages = Pages(rng, E4M3, 2, 64, 16, [rows + start])
    q = rng.standard_normal((rows, 256))
    q[0, 64:128] = np.nan
    cache = Cache(gpu, pages)
    out = back(run_attend(gpu, cache, typ, q, seqs, 4), typ).reshape(rows, 4, 64)
    cache.free()
    assert np.isnan(out[0, 1]).all() and np.isfinite(out[0, [0, 2, 3]]).all() and np.isfinite(out[1:]).all()
    pages.k[:] = 0x7f
    pages.v[:] = 0xff
    cache = Cache(gpu, pages)
    assert np.isnan(back(run_attend(gpu, cache, typ, q, seqs, 4), typ)).all()
    cache.free()


def test_captured_steps(gpu):
    """Appends and attention of tokens one after another, captured once and replayed with other tables and rows, against
    eager calls, with other work between."""
    rng = np.random.default_rng(15)
    L = nemoasr.lib()
    heads, hk, dh, page, n = 8, 2, 64, 16, 5
    starts = np.array([0, 15, 300, 700, 31])
    steps = 6
    freq = freqs(dh)
    pages = Pages(rng, E4M3, hk, dh, page, starts + steps)
    ca, cb = Cache(gpu, copy.deepcopy(pages)), Cache(gpu, copy.deepcopy(pages))
    width = (heads + 2 * hk) * dh
    x = gpu.alloc(n * width * 4)
    seqs, df = gpu.alloc(n * 16), gpu.put(freq)
    qo, outs = gpu.alloc(n * heads * dh * 4), [gpu.alloc(n * heads * dh * 4) for _ in range(2)]

    def step(cache, out):
        a = nemoasr.Append(type=F32, q=x.ptr, ldq=width, k=x.at(4 * heads * dh), ldk=width, v=x.at(4 * (heads + hk) * dh), ldv=width, qo=qo.ptr,
                           ldqo=heads * dh, heads=heads, rot=dh, freq=df.ptr, amp=1.0, seqs=seqs.ptr, nseq=n, max_rows=4, M=n)
        gpu.check(L.nk_kv_append(gpu.h, C.byref(cache.kv), C.byref(a)))
        b = nemoasr.Attend(type=F32, q=qo.ptr, ldq=heads * dh, o=out.ptr, ldo=heads * dh, heads=heads, window=400, sinks=4, scale=dh ** -0.5,
                           seqs=seqs.ptr, nseq=n, max_rows=4, max_len=1 << 14, M=n)
        gpu.check(L.nk_attention_kv(gpu.h, C.byref(cache.kv), C.byref(b)))

    graph = None
    host = copy.deepcopy(pages)
    for t in range(steps):
        rows = rng.standard_normal((n, width)).astype(np.float32)
        here = [(i, 0 if (i + t) % 4 == 3 else 1, int(starts[i]), i) for i in range(n)]
        table = np.array(here, np.int32)
        x.write(rows)
        seqs.write(table)
        gpu.begin()
        step(ca, outs[0])
        gpu.end()
        if graph is None:
            gpu.begin()
            assert L.gpu_capture_begin(gpu.h) == 0
            step(cb, outs[1])
            graph = L.gpu_capture_end(gpu.h)
            assert graph
            gpu.end()
        gpu.begin()
        gpu.check(L.gpu_graph_launch(gpu.h, graph))
        gpu.end()
        a, b = (o.read((n, heads * dh)) for o in outs)
        live = table[:, 1] > 0
        np.testing.assert_array_equal(a[live].view(np.uint32), b[live].view(np.uint32))
        # against the formulas, from the cache as it stands
        host.k, host.v, host.ks, host.vs = (ca.bufs[i].read(getattr(host, m).shape, np.uint8) for i, m in enumerate(("k", "v", "ks", "vs")))
        q = qo.read((n, heads, dh)).astype(np.float64)
        ref, bound = attend(q, host, table, 400, 4, np.float32(dh ** -0.5), F32, np.zeros((n, heads, dh)))
        close(a.reshape(n, heads, dh)[live], ref[live], bound[live])
        starts = starts + table[:, 1]
    for i, m in enumerate(("k", "v", "ks", "vs")):
        assert np.array_equal(ca.bufs[i].read(getattr(host, m).shape, np.uint8), cb.bufs[i].read(getattr(host, m).shape, np.uint8))
    L.gpu_graph_free(graph)
    for b in [x, seqs, df, qo] + outs:
        b.free()
    ca.free()
    cb.free()


@pytest.mark.parametrize("cache_type", [BF16, E4M3])
def test_prompt_then_tokens(gpu, cache_type):
    """A prompt in two parts and tokens behind it, as a program runs them: append, attention, the cache carried on.
    Every output against attention over all keys and values kept on the host as the cache holds them."""
    rng = np.random.default_rng([16, cache_type])
    heads, hk, dh = 4, 2, 64
    total = [90, 41]
    pages = Pages(rng, cache_type, hk, dh, 32, total)
    cache = Cache(gpu, pages)
    freq = freqs(dh)
    done = [0, 0]
    for part in ([50, 17], [30, 20], [1, 1], [1, 1], [8, 2]):
        seqs = np.array([(0, part[0], done[0], 0), (part[0], part[1], done[1], 1)], np.int32)
        M = sum(part)
        x = rng.standard_normal((M, (heads + 2 * hk) * dh))
        before = copy.deepcopy(cache.pages)
        q = run_append(gpu, cache, BF16, x[:, :heads * dh], x[:, heads * dh:(heads + hk) * dh], x[:, (heads + hk) * dh:], seqs, heads, dh,
                       False, freq)
        after = cache.pull()
        check_append(before, after, seqs, kept(x[:, heads * dh:(heads + hk) * dh], BF16).reshape(M, hk, dh),
                     kept(x[:, (heads + hk) * dh:], BF16).reshape(M, hk, dh), BF16, dh, False, freq, 1.0)
        qv = back(q, BF16)
        out = run_attend(gpu, cache, BF16, qv, seqs, heads)
        ref, bound = attend(qv.reshape(M, heads, dh), after, seqs, 0, 0, np.float32(dh ** -0.5), BF16, np.zeros((M, heads, dh)))
        close(back(out, BF16).reshape(M, heads, dh), ref, bound)
        done = [d + p for d, p in zip(done, part)]
    cache.free()


# ---- many rows ---------------------------------------------------------------------------------------

PROMPT_HEADS = [(4, 4, 128), (2, 1, 96), (6, 2, 64), (2, 1, 256), (3, 3, 192), (4, 1, 80), (20, 1, 32)]


@pytest.mark.parametrize("window,sinks", [(0, 0), (70, 0), (100, 70)])
@pytest.mark.parametrize("shape", range(len(PROMPT_HEADS)))
@pytest.mark.parametrize("cache_type", [BF16, E4M3])
@pytest.mark.parametrize("typ", [F32, BF16])
def test_attend_prompts(gpu, window, sinks, shape, cache_type, typ):
    """Prompts over more than one tile of 128 packed rows, tokens and chunks beside them, an empty sequence."""
    heads, hk, dh = PROMPT_HEADS[shape]
    rng = np.random.default_rng([17, window, shape, cache_type, typ])
    seqs, M = sequences([150, 1, 0, 33, 4], [7 * shape, 300, 9, 100, 64], gap=shape % 2)
    more = [dict(), dict(ld=heads * dh + 3, off=1), dict(max_rows=1000, max_len=100000)][(shape + window) % 3]
    check_attend(gpu, rng, typ, cache_type, heads, hk, dh, (64, 16, 32)[shape % 3], seqs, M, window, sinks, **more)


@pytest.mark.parametrize("typ", [F32, BF16])
@pytest.mark.parametrize("cache_type", [BF16, E4M3])
@pytest.mark.parametrize("dh", [64, 128, 192, 256])
def test_attend_prompt_behind_many_tokens(gpu, typ, cache_type, dh):
    """Few tiles of many rows, split along their tokens; pages that are not there among them."""
    rng = np.random.default_rng([18, typ, cache_type, dh])
    seqs, M = sequences([130], [2900])
    check_attend(gpu, rng, typ, cache_type, 1, 1, dh, 16, seqs, M)
    check_attend(gpu, rng, typ, cache_type, 1, 1, dh, 16, seqs, M, 2000, 100, drop=[(0, 3), (0, 70), (0, 100), (0, 189)])


def test_attend_pairs_of_tiles(gpu):
    """Sizes at which tiles go two to a CU, the long ones beside the short ones."""
    rng = np.random.default_rng(19)
    seqs, M = sequences([1060], [3])
    check_attend(gpu, rng, BF16, BF16, 64, 32, 16, 64, seqs, M, 60)


@pytest.mark.parametrize("typ", [F32, BF16])
def test_attend_prompt_values_not_finite(gpu, typ):
    rng = np.random.default_rng(20)
    dh, rows = 64, 150
    seqs = np.array([(0, rows, 0, 0)], np.int32)
    pages = Pages(rng, BF16, 1, dh, 16, [rows])

    def put(name, j, d, value):
        getattr(pages, name)[pages.table[0, j // 16], 0, j % 16, d] = oracle.f32_to_bf16(np.array([value], np.float32))[0]

    put("v", 70, 3, np.inf)
    put("v", 75, 4, np.nan)
    put("k", 140, 0, -np.inf)
    q = kept(rng.standard_normal((rows, dh)), typ)
    q[:, 0] = np.abs(q[:, 0]) + 0.1  # the logit of token 140 is -inf: it has no weight
    q = kept(q, typ)
    cache = Cache(gpu, pages)
    out = back(run_attend(gpu, cache, typ, q, seqs, 1), typ)
    cache.free()
    k, v = (pages.tokens(x, 0, rows)[0][:, 0] for x in "kv")
    fin = np.where(np.isfinite(v), v, 0.0)
    for i in range(rows):
        s = (k[:i + 1] @ q[i]) * dh ** -0.5
        w = np.exp(s - s.max())
        ref = w @ fin[:i + 1] / w.sum()
        for d in range(dh):
            if d == 3 and i >= 70:
                assert out[i, d] == np.inf or i >= 140 and np.isinf(out[i, d])
            elif d == 4 and i >= 75:
                assert np.isnan(out[i, d])
            else:
                assert abs(out[i, d] - ref[d]) < 0.05, (i, d)  # values below 5, two roundings to bf16


def test_attend_4096_sequences(gpu):
    """As many sequences as a call takes, most of them one token long."""
    rng = np.random.default_rng(21)
    n = 4096
    rows = (rng.random(n) < 0.7).astype(int)
    rows[[100, 2000, 4095]] = 3, 20, 2
    seqs, M = sequences(list(rows), list(rng.integers(0, 40, n)))
    check_attend(gpu, rng, BF16, BF16, 1, 1, 16, 16, seqs, M)


def test_captured_mixed_batches(gpu):
    """A captured call replayed with other tables: prompts, steps, both, none; against the formulas and eager calls."""
    rng = np.random.default_rng(22)
    L = nemoasr.lib()
    heads, hk, dh, n, M = 4, 2, 32, 4, 300
    pages = Pages(rng, BF16, hk, dh, 16, [3000, 400, 300, 200])
    cache = Cache(gpu, pages)
    q = kept(rng.standard_normal((M, heads * dh)), F32)
    dq, seqs, outs = gpu.put(bits(q, F32)), gpu.alloc(n * 16), [gpu.alloc(M * heads * dh * 4) for _ in range(2)]

    def call(out):
        a = nemoasr.Attend(type=F32, q=dq.ptr, ldq=heads * dh, o=out.ptr, ldo=heads * dh, heads=heads, window=0, sinks=0, scale=dh ** -0.5,
                           seqs=seqs.ptr, nseq=n, max_rows=250, max_len=3000, M=M)
        gpu.check(L.nk_attention_kv(gpu.h, C.byref(cache.kv), C.byref(a)))

    graph = None
    for table in ([(0, 200, 100, 1), (200, 1, 2990, 0), (201, 90, 0, 2), (291, 0, 0, 3)], [(0, 1, 2999, 0), (1, 1, 7, 1), (2, 1, 255, 2), (3, 1, 0, 3)],
                  [(0, 0, 5, 0), (0, 0, 5, 1), (0, 0, 5, 2), (0, 0, 5, 3)], [(10, 250, 2750, 0), (260, 3, 100, 1), (263, 2, 9, 2), (299, 1, 199, 3)]):
        table = np.array(table, np.int32)
        seqs.write(table)
        for o in outs:
            o.write(np.full((M, heads * dh), 7.0, np.float32))
        gpu.begin()
        call(outs[0])
        gpu.end()
        if graph is None:
            gpu.begin()
            assert L.gpu_capture_begin(gpu.h) == 0
            call(outs[1])
            graph = L.gpu_capture_end(gpu.h)
            assert graph
            gpu.end()
        for _ in range(2):
            gpu.begin()
            gpu.check(L.gpu_graph_launch(gpu.h, graph))
            gpu.end()
        a, b = (o.read((M, heads, dh)) for o in outs)
        np.testing.assert_array_equal(a.view(np.uint32), b.view(np.uint32))
        ref, bound = attend(q.reshape(M, heads, dh), pages, table, 0, 0, np.float32(dh ** -0.5), F32, np.full((M, heads, dh), 7.0))
        close(a, ref, bound)
    L.gpu_graph_free(graph)
    for b in [dq, seqs] + outs:
        b.free()
    cache.free()


def test_capture_needs_the_scratch(gpu):
    """A call that is split refuses to be captured before one has sized the scratch, and is captured after it."""
    rng = np.random.default_rng(23)
    own = nemoasr.Gpu()
    L = nemoasr.lib()
    pages = Pages(rng, BF16, 8, 128, 64, [700, 700])
    cache = Cache(own, pages)
    q, o = own.put(np.zeros((2, 8 * 128), np.uint16)), own.alloc(2 * 8 * 128 * 2)
    seqs = own.put(np.array([(0, 1, 600, 0), (1, 1, 5, 1)], np.int32))
    a = nemoasr.Attend(type=BF16, q=q.ptr, ldq=1024, o=o.ptr, ldo=1024, heads=8, scale=0.1, seqs=seqs.ptr, nseq=2, max_rows=1, max_len=1 << 20, M=2)

    def call():
        return L.nk_attention_kv(own.h, C.byref(cache.kv), C.byref(a))

    own.begin()
    assert L.gpu_capture_begin(own.h) == 0
    assert call() == -1 and "scratch unavailable" in L.gpu_last_error(own.h).decode()
    graph = L.gpu_capture_end(own.h)
    if graph:
        L.gpu_graph_free(graph)
    err = C.create_string_buffer(512)
    L.gpu_end(own.h, err, 512)
    own.begin()
    own.check(call())
    own.end()
    own.begin()
    assert L.gpu_capture_begin(own.h) == 0
    own.check(call())
    graph = L.gpu_capture_end(own.h)
    assert graph
    own.check(L.gpu_graph_launch(own.h, graph))
    own.end()
    L.gpu_graph_free(graph)
    own.close()
