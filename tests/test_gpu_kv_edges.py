"""The paged cache and its attention at the edges of what a call may ask, on the GPU: caches whose pages lie behind 2^32 bytes and
values, pages that nothing was ever written to, graphs that outlive the scratch that they were captured with, two contexts on one
cache."""
import copy
import ctypes as C

import numpy as np
import pytest

import nemoasr
from kv_ref import BF16, E4M3, F32, Pages, attend
from test_gpu_kv import Cache, back, bits, check_append, close, freqs, kept, run_append, run_attend, sequences, tokens_of

pytestmark = pytest.mark.gpu


class FarCache:
    """A Pages whose pages lie at the places `at` of a far larger cache."""

    def __init__(self, gpu, pages, total, at):
        self.pages, self.at = pages, np.asarray(at)
        self.arrays = [x for x in ("k", "v", "ks", "vs") if getattr(pages, x) is not None]
        self.bufs = {x: gpu.alloc(total * getattr(pages, x)[0].nbytes) for x in self.arrays}
        for x in self.arrays:
            for i, a in enumerate(self.at):
                self.bufs[x].write(getattr(pages, x)[i], int(a) * getattr(pages, x)[0].nbytes)
        self.table = gpu.put(np.where(pages.table >= 0, self.at[pages.table], -1).astype(np.int32))
        self.kv = nemoasr.Kv(type=pages.typ, heads=pages.heads, dh=pages.dh, page=pages.page, pages=total, table=self.table.ptr,
                             ldt=pages.table.shape[1], tables=pages.table.shape[0], **{x: b.ptr for x, b in self.bufs.items()})

    def pull(self):
        for x, b in self.bufs.items():
            a = getattr(self.pages, x)
            setattr(self.pages, x, np.stack([b.read(a[0].shape, a.dtype, int(i) * a[0].nbytes) for i in self.at]))
        return self.pages

    def free(self):
        for b in [self.table, *self.bufs.values()]:
            b.free()


@pytest.mark.parametrize("cache_type", [BF16, E4M3])
def test_pages_behind_4_gib(gpu, cache_type):
    """140000 pages of 32768 values: appended to, read back and attended over where their offsets pass 2^31 and 2^32, by steps and
    a prompt."""
    rng = np.random.default_rng([30, cache_type])
    heads, hk, dh, total = 4, 2, 256, 140000
    seqs, M = sequences([1, 150, 3], [200, 60, 500])
    pages = Pages(rng, cache_type, hk, dh, 64, tokens_of(seqs))
    edge = (1 << 31) // (hk * 64 * dh * (1 if cache_type == E4M3 else 2))
    places = [x for e in (edge, 2 * edge, 1 << 16, 1 << 17) for x in (e - 1, e) if x < total] + [0, 1] + list(range(total - 40, total))
    at = rng.permutation(np.unique(places))[:pages.pages]
    cache = FarCache(gpu, pages, total, at)
    before = copy.deepcopy(pages)
    q, k, v = (rng.standard_normal((M, n * dh)) for n in (heads, hk, hk))
    qr = run_append(gpu, cache, BF16, q, k, v, seqs, heads, dh, False, freqs(dh))
    after = cache.pull()
    check_append(before, after, seqs, kept(k, BF16).reshape(M, hk, dh), kept(v, BF16).reshape(M, hk, dh), BF16, dh, False, freqs(dh), 1.0)
    out, ds = [gpu.alloc(M * hk * dh * 4) for _ in "kv"], gpu.put(seqs)
    gpu.begin()
    gpu.check(nemoasr.lib().nk_kv_read(gpu.h, C.byref(cache.kv), out[0].ptr, hk * dh, out[1].ptr, hk * dh, F32, ds.ptr, len(seqs), 150, M))
    gpu.end()
    for x, b in zip("kv", out):
        got = b.read((M, hk, dh))
        for first, rows, start, row in seqs:
            assert np.array_equal(got[first:first + rows], after.tokens(x, row, start + rows)[0][start:])
    qv = back(qr, BF16)
    for rows_of in (seqs, seqs[[0, 2]]):  # with the prompt, and few rows
        got = back(run_attend(gpu, cache, BF16, qv, rows_of, heads), BF16).reshape(M, heads, dh)
        ref, bound = attend(qv.reshape(M, heads, dh), after, rows_of, 0, 0, np.float32(dh ** -0.5), BF16, np.zeros((M, heads, dh)))
        close(got, ref, bound)
    for b in out + [ds]:
        b.free()
    cache.free()


@pytest.mark.parametrize("typ", [F32, BF16])
@pytest.mark.parametrize("cache_type", [BF16, E4M3])
@pytest.mark.parametrize("rows,start,window", [(1, 300, 0), (5, 300, 40), (130, 90, 0), (130, 90, 50), (2, 3000, 0)])
def test_pages_never_written(gpu, typ, cache_type, rows, start, window):
    """Pages that are not there, in a cache whose other pages hold NaN and scales of no meaning: nothing of it shows."""
    rng = np.random.default_rng([31, typ, cache_type, rows, start])
    seqs, M = sequences([rows, 1], [start, 20], gap=1)
    gone = [(1, j) for j in range((start + rows) // 16) if j % 3 == 1]
    pages = Pages(rng, cache_type, 2, 64, 16, tokens_of(seqs), gone)
    pages.table[pages.table == 0] = np.setdiff1d(np.arange(pages.pages), pages.table)[-1]
    free = np.setdiff1d(np.arange(pages.pages), pages.table)
    assert 0 in free
    for x in (pages.k, pages.v):
        x[free] = 0x7f if cache_type == E4M3 else 0x7fc0
    if cache_type == E4M3:
        pages.ks[free], pages.vs[free] = 255, 0
    cache = Cache(gpu, pages)
    q = rng.standard_normal((M, 4 * 64)) * 2
    out = back(run_attend(gpu, cache, typ, q, seqs, 4, window, 3 if window else 0, fill=7.0), typ).reshape(M, 4, 64)
    cache.free()
    ref, bound = attend(kept(q, typ).reshape(M, 4, 64), pages, seqs, window, 3 if window else 0, np.float32(0.125), typ, np.full((M, 4, 64), 7.0))
    close(out, ref, bound)


def attend_call(gpu, cache, q, o, seqs, n, heads, max_rows, max_len, M):
    dh = cache.pages.dh
    a = nemoasr.Attend(type=BF16, q=q.ptr, ldq=heads * dh, o=o.ptr, ldo=heads * dh, heads=heads, scale=dh ** -0.5, seqs=seqs.ptr, nseq=n,
                       max_rows=max_rows, max_len=max_len, M=M)
    gpu.check(nemoasr.lib().nk_attention_kv(gpu.h, C.byref(cache.kv), C.byref(a)))


def test_graphs_outlive_the_scratch(gpu):
    """A split call captured twice, the scratch outgrown between and behind them: the replays give what eager calls give."""
    rng = np.random.default_rng(32)
    own, L = nemoasr.Gpu(), nemoasr.lib()
    heads, hk, dh = 8, 8, 128
    pages = Pages(rng, BF16, hk, dh, 64, [3000, 700])
    cache = Cache(own, pages)
    table = np.array([(0, 1, 2990, 0), (1, 1, 650, 1)], np.int32)
    seqs, long = own.put(table), own.put(np.array([(0, 90, 2900, 0), (90, 1, 5, 1)], np.int32))
    x = rng.standard_normal((91, heads * dh))
    q, outs = own.put(bits(x, BF16)), [own.alloc(91 * heads * dh * 2) for _ in range(3)]

    def eager(o, what=seqs, max_rows=1, M=2):
        own.begin()
        attend_call(own, cache, q, o, what, 2, heads, max_rows, 3000, M)
        own.end()

    def captured(o):
        own.begin()
        assert L.gpu_capture_begin(own.h) == 0
        attend_call(own, cache, q, o, seqs, 2, heads, 1, 3000, 2)
        graph = L.gpu_capture_end(own.h)
        assert graph
        own.end()
        return graph

    eager(outs[0])
    graphs = [captured(outs[1])]
    eager(outs[2], long, 200, 91)  # more scratch than the first graph has
    graphs.append(captured(outs[2]))
    ref, bound = attend(kept(x[:2], BF16).reshape(2, heads, dh), pages, table, 0, 0, np.float32(dh ** -0.5), BF16, np.zeros((2, heads, dh)))
    close(back(outs[0].read((2, heads, dh), np.uint16), BF16), ref, bound)
    for _ in range(3):
        for o, g in zip(outs[1:], graphs):
            o.write(np.zeros((2, heads * dh), np.uint16))
            own.begin()
            own.check(L.gpu_graph_launch(own.h, g))
            own.end()
            assert np.array_equal(o.read((2, heads * dh), np.uint16), outs[0].read((2, heads * dh), np.uint16))
        eager(outs[0], long, 200, 91)
        eager(outs[0])
    for g in graphs:
        L.gpu_graph_free(g)
    own.close()


def test_two_contexts_on_one_cache(gpu):
    """Split calls of two contexts under way at once, each with a scratch of its own."""
    rng = np.random.default_rng(33)
    other, L = nemoasr.Gpu(), nemoasr.lib()
    heads, hk, dh = 8, 4, 64
    pages = Pages(rng, E4M3, hk, dh, 32, [4000, 3000])
    cache = Cache(gpu, pages)
    M = 3
    xs = [rng.standard_normal((M, heads * dh)) for _ in range(2)]
    tables = [np.array([(0, 1, 3990, 0), (1, 2, 2000, 1)], np.int32), np.array([(0, 2, 700, 0), (2, 1, 2900, 1)], np.int32)]
    ctx = [(g, g.put(bits(x, BF16)), g.alloc(M * heads * dh * 2), g.put(t)) for g, x, t in zip((gpu, other), xs, tables)]
    for _ in range(3):
        for g, q, o, s in ctx:
            g.begin()
        for _ in range(5):
            for g, q, o, s in ctx:
                attend_call(g, cache, q, o, s, 2, heads, 2, 4000, M)
        for g, q, o, s in ctx:
            g.end()
        for (g, q, o, s), x, t in zip(ctx, xs, tables):
            ref, bound = attend(kept(x, BF16).reshape(M, heads, dh), pages, t, 0, 0, np.float32(0.125), BF16, np.zeros((M, heads, dh)))
            close(back(o.read((M, heads, dh), np.uint16), BF16), ref, bound)
    for g, *bufs in ctx[:1]:
        for b in bufs:
            b.free()
    other.close()
    cache.free()
