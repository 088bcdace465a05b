"""What the launchers of the 4-bit products and the selective scan refuse, without a GPU: the checks come before
anything touches the device, so a zeroed block of memory stands for the context (its error text is read back)."""
import ctypes as C
import os
import subprocess

import pytest

import nemoasr
from conftest import REPO


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


def test_quant_refusals(ctx):
    L = nemoasr.lib()

    def call(f, x=P, typ=0, ldx=256, q=P, ldq=128, s=P, lds=8, m=2, k=256):
        args = (x, typ, ldx, q, ldq, s, lds, m, k) if f == "nk_fp4_quant" else (q, ldq, s, lds, x, typ, ldx, m, k)
        return getattr(L, f)(ctx.h, *args)

    for f in ("nk_fp4_quant", "nk_fp4_dequant"):
        assert call(f, m=0) == 0 and call(f, k=0) == 0
        for bad in (dict(x=None), dict(x=P + 2), dict(typ=1, x=P + 1), dict(typ=2), dict(ldx=255), dict(q=None), dict(q=P + 8),
                    dict(ldq=112), dict(ldq=136), dict(s=None), dict(s=P + 1), dict(lds=4), dict(lds=10),
                    dict(m=1 << 31, k=64), dict(k=(1 << 30) + 1, ldx=(1 << 30) + 1, ldq=1 << 30, lds=1 << 26)):
            ctx.refused(call(f, **bad), "fp4")


def test_product_refusals(ctx):
    L = nemoasr.lib()

    def call(kind, a=P, lda=None, s=P, lds=16, wq=P, ldw=256, ws=P, ldws=16, bias=None, c=P, ldc=64, m=3, n=64, k=512, act=0):
        end = (wq, ldw, ws, ldws, bias, c, ldc, m, n, k, act, 0, 1.0)
        if kind == "fp4":
            return L.nk_gemm_fp4(ctx.h, a, 256 if lda is None else lda, s, lds, *end)
        return L.nk_gemm_w4(ctx.h, a, 512 if lda is None else lda, *end)

    for kind in ("fp4", "w4"):
        assert call(kind, m=0) == 0
        for bad in (dict(a=None), dict(a=P + 4), dict(lda=240 if kind == "fp4" else 508), dict(lda=264 if kind == "fp4" else 514),
                    dict(wq=None), dict(wq=P + 4), dict(ldw=240), dict(ldw=260), dict(ws=None), dict(ws=P + 2), dict(ldws=12),
                    dict(ldws=18), dict(c=None), dict(c=P + 2), dict(bias=P + 1), dict(ldc=63), dict(n=0), dict(n=(1 << 28) + 2, ldc=1 << 29),
                    dict(ldw=1 << 24), dict(ldws=1 << 24), dict(act=3, n=63), dict(act=4), dict(act=-1), dict(k=0), dict(m=1 << 23)):
            ctx.refused(call(kind, **bad), "gemm")
    for bad in (dict(s=None), dict(s=P + 2), dict(lds=12), dict(lds=18), dict(lda=1 << 24), dict(lds=1 << 24)):
        ctx.refused(call("fp4", **bad), "gemm_fp4")


def test_conv_refusals(ctx):
    L = nemoasr.lib()

    def call(x=P, typ=0, ldx=100, w=P, bias=None, state=P, slots=4, seqs=P, nseq=2, max_rows=10, y=P, ldy=100, m=20, d=100, taps=4,
             act=1):
        return L.nk_causal_conv(ctx.h, x, typ, ldx, w, bias, state, slots, seqs, nseq, max_rows, y, ldy, m, d, taps, act)

    assert call(nseq=0) == 0 and call(d=0) == 0
    ctx.refused(call(x=P, y=P), "Y must not overlap X")
    for bad in (dict(seqs=None), dict(seqs=P + 4), dict(nseq=65536), dict(state=None), dict(state=P + 2), dict(slots=1 << 31),
                dict(max_rows=(1 << 30) + 1), dict(d=(1 << 28) + 1, ldx=1 << 29, ldy=1 << 29)):
        ctx.refused(call(**bad), "sequences")
    for bad in (dict(x=None), dict(x=P + 2), dict(typ=1, y=P + 1), dict(typ=3), dict(w=None), dict(w=P + 2), dict(bias=P + 3), dict(ldx=99),
                dict(ldy=99), dict(taps=1), dict(taps=5), dict(act=3), dict(act=-1)):
        ctx.refused(call(**bad), "causal_conv")


def test_scan_refusals(ctx):
    L = nemoasr.lib()

    def call(**more):
        a = dict(type=0, ldx=100, lddt=100, ldbc=32, ldz=100, ldy=100, x=P, dt=P, B=P, C=P + 64, z=P, y=P, A=P, skip=P, dt_bias=P,
                 state=P, seqs=P, slots=4, nseq=2, max_rows=10, M=20, D=100, N=16, groups=2, softplus=1)
        return L.nk_ssm_scan(ctx.h, C.byref(nemoasr.Scan(**dict(a, **more))))

    assert call(nseq=0) == 0 and call(D=0) == 0
    for bad in (dict(seqs=None), dict(seqs=P + 4), dict(nseq=65536), dict(state=None), dict(slots=1 << 31), dict(max_rows=(1 << 30) + 1),
                dict(D=1 << 29, ldx=1 << 29, lddt=1 << 29, ldy=1 << 29, ldz=1 << 29)):
        ctx.refused(call(**bad), "sequences")
    for bad in ([{k: None} for k in ("x", "dt", "B", "C", "y", "A")] + [{k: P + 2} for k in ("x", "dt", "B", "C", "z", "y", "A", "skip", "dt_bias")] +
                [{k: 99} for k in ("ldx", "lddt", "ldz", "ldy")] +
                [dict(type=1, x=P + 1), dict(type=2), dict(ldbc=31), dict(N=0), dict(N=65, ldbc=200), dict(groups=0), dict(groups=3)]):
        ctx.refused(call(**bad), "ssm_scan")
    for k in ("x", "dt", "B", "C", "z"):
        far = dict(x=P + 4096, dt=P + 8192, B=P + 12288, C=P + 16384, z=P + 20480)
        ctx.refused(call(**dict(far, **{k: P})), "y must not overlap the inputs")
    assert L.nk_ssm_scan(ctx.h, None) == -1


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
    const unsigned Ms[] = { 0, 1, 10, 0x80000000u, 0xffffffffu }, mr[] = { 0, 1, 9, 1u << 30 }, sl[] = { 0, 1, 10, 0x7fffffffu };
    int bad = 0;
    for (int a = 0; a < n; ++a) for (int b = 0; b < n; ++b) for (int c = 0; c < n; ++c) for (int d = 0; d < n; ++d)
        for (int i = 0; i < 5; ++i) for (int j = 0; j < 4; ++j) for (int k = 0; k < 4; ++k) {
            const long long f = v[a], r = v[b], p = v[c], q = v[d];
            const int want = f >= 0 && r >= 0 && f + r <= (long long)Ms[i] && r <= (long long)mr[j] && p >= -1 && q >= -1 &&
                             p < (long long)sl[k] && q < (long long)sl[k];
            bad += want != nk_seq_ok(v[a], v[b], v[c], v[d], Ms[i], mr[j], sl[k]);
        }
    printf("%d\\n", bad);
    return bad != 0;
}
''')
    exe = tmp_path / "t"
    subprocess.run(["gcc", "-std=c11", "-Wall", "-I" + os.path.join(REPO, "nemo-c_amd", "csrc"), str(src), "-o", str(exe)], check=True)
    assert subprocess.run([str(exe)], capture_output=True, text=True).stdout == "0\n"
