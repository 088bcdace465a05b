"""What the launchers of the paged cache refuse and the rotation's frequencies, without a GPU: the checks come before
anything touches the device, so a zeroed block of memory stands for the context (its error text is read back)."""
import ctypes as C
import os
import subprocess

import numpy as np
import pytest

import nemoasr
from conftest import REPO
from kv_ref import VALUES, e4m3_codes, scale_byte


class Ctx:
    def __init__(self):
        self.mem = C.create_string_buffer(1 << 16)
        self.h = C.cast(self.mem, C.c_void_p)

    def refused(self, rc, word):
        msg = nemoasr.lib().gpu_last_error(self.h).decode()
        assert rc == -1 and word in msg, (rc, msg)
        C.memset(self.mem, 0, len(self.mem))


@pytest.fixture
def ctx():
    return Ctx()


P = 0x10000  # an aligned address that nothing reads
KV = dict(type=1, heads=2, dh=64, page=32, pages=9, k=P, v=P, ks=P, vs=P, table=P, ldt=4, tables=3)
BAD_KV = [dict(type=0), dict(type=3), dict(heads=0), dict(heads=65536), dict(dh=0), dict(dh=24), dict(dh=272), dict(page=8), dict(page=48),
          dict(page=1 << 21), dict(pages=0), dict(pages=1 << 31), dict(k=None), dict(v=None), dict(k=P + 8), dict(v=P + 2),
          dict(type=2, ks=None), dict(type=2, vs=None), dict(table=None), dict(table=P + 2), dict(ldt=0), dict(tables=0)]
BAD_BATCH = [dict(seqs=None), dict(seqs=P + 4), dict(nseq=4097), dict(max_rows=(1 << 30) + 1)]


def kv(**more):
    return C.byref(nemoasr.Kv(**dict(KV, **more)))


def test_append_refusals(ctx):
    L = nemoasr.lib()

    def call(cache={}, **more):
        a = dict(type=0, q=P, ldq=256, k=P, ldk=128, v=P, ldv=128, qo=P + 4096, ldqo=256, heads=4, rot=64, freq=P, amp=1.0, seqs=P, nseq=2,
                 max_rows=5, M=7)
        return L.nk_kv_append(ctx.h, kv(**cache), C.byref(nemoasr.Append(**dict(a, **more))))

    assert call(nseq=0) == 0 and call(M=0) == 0 and call(max_rows=0) == 0
    for bad in BAD_KV:
        ctx.refused(call(bad), "kv: ")
    for bad in BAD_BATCH:
        ctx.refused(call(**bad), "kv: ")
    for bad in (dict(type=2), dict(type=-1), dict(q=None), dict(qo=None), dict(k=None), dict(v=None), dict(q=None, qo=None, k=None, v=None),
                dict(q=P + 2), dict(type=1, k=P + 1), dict(v=P + 2), dict(qo=P + 2), dict(ldq=255), dict(ldqo=255), dict(ldk=127), dict(ldv=127),
                dict(heads=0), dict(heads=65536, ldq=1 << 23, ldqo=1 << 23), dict(qo=P, ldqo=320), dict(rot=63), dict(rot=66), dict(freq=None), dict(freq=P + 2),
                dict(M=1 << 30, max_rows=1 << 30)):
        ctx.refused(call(**bad), "kv_append")
    assert L.nk_kv_append(ctx.h, kv(), None) == -1 and L.nk_kv_append(ctx.h, None, None) == -1


def test_read_refusals(ctx):
    L = nemoasr.lib()

    def call(cache={}, K=P, ldk=128, V=P, ldv=128, typ=0, seqs=P, nseq=2, max_rows=5, M=7):
        return L.nk_kv_read(ctx.h, kv(**cache), K, ldk, V, ldv, typ, seqs, nseq, max_rows, M)

    assert call(nseq=0) == 0 and call(M=0) == 0 and call(max_rows=0) == 0 and call(K=None, V=None) == 0
    for bad in BAD_KV:
        ctx.refused(call(bad), "kv: ")
    for bad in BAD_BATCH:
        ctx.refused(call(**bad), "kv: ")
    for bad in (dict(typ=2), dict(K=P + 2), dict(V=P + 2), dict(typ=1, V=P + 1), dict(ldk=127), dict(ldv=127), dict(M=1 << 30, max_rows=1 << 30)):
        ctx.refused(call(**bad), "kv_read")
    assert L.nk_kv_read(ctx.h, None, P, 128, P, 128, 0, P, 2, 5, 7) == -1


def test_attention_refusals(ctx):
    L = nemoasr.lib()

    def call(cache={}, **more):
        a = dict(type=0, q=P, ldq=256, o=P + 65536, ldo=256, heads=4, scale=0.125, seqs=P, nseq=2, max_rows=5, max_len=100, M=7)
        return L.nk_attention_kv(ctx.h, kv(**cache), C.byref(nemoasr.Attend(**dict(a, **more))))

    assert call(nseq=0) == 0 and call(M=0) == 0 and call(max_rows=0) == 0
    for bad in BAD_KV:
        ctx.refused(call(bad), "kv: ")
    for bad in BAD_BATCH:
        ctx.refused(call(**bad), "kv: ")
    for bad in (dict(type=2), dict(heads=0), dict(heads=3), dict(heads=2050, ldq=1 << 20, ldo=1 << 20), dict(q=None), dict(o=None), dict(q=P + 2),
                dict(o=P + 2), dict(type=1, q=P + 1), dict(ldq=255), dict(ldo=255), dict(o=P), dict(scale=0.0), dict(scale=-1.0),
                dict(scale=float("nan")), dict(scale=float("inf")), dict(max_len=(1 << 30) + 1), dict(M=1 << 30, max_rows=1 << 30)):
        ctx.refused(call(**bad), "attention_kv")
    assert L.nk_attention_kv(ctx.h, kv(), None) == -1 and L.nk_attention_kv(ctx.h, None, None) == -1


def test_sequence_entries(tmp_path):
    """The check that the kernels make of a table entry, compiled for the host: every entry it accepts keeps to the
    buffers, and every entry that does is accepted."""
    src = tmp_path / "t.c"
    src.write_text('''
#include "kernel_params.h"
#include <limits.h>
#include <stdio.h>
int main(void) {
    const int v[] = { INT_MIN, -2, -1, 0, 1, 2, 5, 9, 10, 11, INT_MAX - 1, INT_MAX };
    const int n = sizeof v / sizeof *v;
    const unsigned Ms[] = { 0, 1, 10, 0x80000000u, 0xffffffffu }, mr[] = { 0, 1, 9, 1u << 30 }, ts[] = { 0, 1, 10, 0x7fffffffu };
    const unsigned long long rooms[] = { 0, 1, 10, 0x7fffffffull, 0xffffffffull << 20 };
    int bad = 0;
    for (int a = 0; a < n; ++a) for (int b = 0; b < n; ++b) for (int c = 0; c < n; ++c) for (int d = 0; d < n; ++d)
        for (int i = 0; i < 5; ++i) for (int j = 0; j < 4; ++j) for (int k = 0; k < 4; ++k) for (int l = 0; l < 5; ++l) {
            const long long f = v[a], r = v[b], p = v[c], q = v[d];
            const int want = f >= 0 && r >= 0 && f + r <= (long long)Ms[i] && r <= (long long)mr[j] && p >= 0 &&
                             q >= 0 && q < (long long)ts[k] && p + r <= (long long)rooms[l];
            bad += want != nk_kv_seq_ok(v[a], v[b], v[c], v[d], Ms[i], mr[j], ts[k], rooms[l]);
        }
    printf("%d\\n", bad);
    return bad != 0;
}
''')
    exe = tmp_path / "t"
    subprocess.run(["gcc", "-std=c11", "-O1", "-Wall", "-I" + os.path.join(REPO, "nemo-c_amd", "csrc"), str(src), "-o", str(exe)], check=True)
    assert subprocess.run([str(exe)], capture_output=True, text=True).stdout == "0\n"


def freqs(rot, base, scaling=0, factor=1.0, old=0.0, lo=0.0, hi=0.0):
    f = np.zeros(rot // 2, np.float32)
    assert nemoasr.lib().nk_rope_freqs(f.ctypes.data, rot, base, scaling, factor, old, lo, hi) == 0
    return f.astype(np.float64)


@pytest.mark.parametrize("rot", [2, 4, 6, 48, 64, 128, 256])
@pytest.mark.parametrize("base", [10000.0, 500000.0, 2.0])
def test_rope_freqs(rot, base):
    """f32 roundings of the formulas (half a step, and a little of the power's own)."""
    plain = base ** (-np.arange(0, rot, 2) / rot)
    near = dict(rtol=2.0 ** -23, atol=0)
    np.testing.assert_allclose(freqs(rot, base), plain, **near)
    np.testing.assert_allclose(freqs(rot, base, 1, 8.0), plain / 8, **near)
    if rot >= 4:
        f = freqs(rot, base, 2, 8.0)
        np.testing.assert_allclose(f, (base * 8.0 ** (rot / (rot - 2))) ** (-np.arange(0, rot, 2) / rot), **near)
        np.testing.assert_allclose(f[[0, -1]], [1.0, plain[-1] / 8], **near)  # the fastest as it was, the slowest by the factor
    f = freqs(rot, base, 3, 8.0, 4096.0, 1.0, 4.0)
    turns = 4096 * plain / (2 * np.pi)
    np.testing.assert_allclose(f[turns >= 4], plain[turns >= 4], **near)
    np.testing.assert_allclose(f[turns <= 1], plain[turns <= 1] / 8, **near)
    assert ((f <= plain * (1 + 2.0 ** -23)) & (f >= plain / 8 * (1 - 2.0 ** -23))).all()


def test_rope_freqs_refusals():
    L = nemoasr.lib()
    f = np.zeros(64, np.float32)

    def call(p=f.ctypes.data, rot=64, base=1e4, scaling=0, factor=8.0, old=4096.0, lo=1.0, hi=4.0):
        return L.nk_rope_freqs(p, rot, base, scaling, factor, old, lo, hi)

    assert call() == 0
    nan, inf = float("nan"), float("inf")
    for bad in (dict(p=None), dict(rot=0), dict(rot=7), dict(base=0.0), dict(base=-1.0), dict(base=nan), dict(base=inf), dict(scaling=-1),
                dict(scaling=4), dict(scaling=1, factor=0.0), dict(scaling=2, factor=nan), dict(scaling=2, rot=2), dict(scaling=3, factor=-1.0),
                dict(scaling=3, old=0.0), dict(scaling=3, old=inf), dict(scaling=3, lo=4.0), dict(scaling=3, hi=nan)):
        assert call(**bad) == -1, bad


def test_codes_of_the_reference():
    """The reference's own rounding: every code stands for itself, and what lies between goes to the nearer."""
    assert np.array_equal(e4m3_codes(VALUES[:127]), np.arange(127))
    assert np.array_equal(e4m3_codes(-VALUES[:127]), np.arange(128, 255))
    mid = (VALUES[:126] + VALUES[1:127]) / 2
    up = np.arange(126) % 2 == 1
    assert np.array_equal(e4m3_codes(mid), np.arange(126) + up)
    assert np.array_equal(e4m3_codes(mid * (1 + 1e-12)), np.arange(1, 127)) and np.array_equal(e4m3_codes(mid * (1 - 1e-12)), np.arange(126))
    assert e4m3_codes(np.array([500.0, 1e9])).tolist() == [126, 126] and (e4m3_codes(np.array([np.inf, np.nan])) & 127 == 127).all()
    assert [scale_byte(t) for t in (448.0, 448.1, 224.0, 0.0, 1e-40)] == [127, 128, 126, 10, 10]
