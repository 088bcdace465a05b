"""The launches that the hosts of the 4-bit products and the selective-scan block choose, without a GPU: their sources
compiled against a device layer of stubs that records launches."""
import ctypes as C
import itertools
import os
import re
import shutil
import subprocess

import pytest

import nemoasr
import test_gpu_fp4 as fp4
import test_gpu_ssm as ssm
from conftest import REPO

HOST = os.path.join(REPO, "nemo-c_amd", "csrc", "host")

STUBS = r"""
#include "gpu.h"
#include <stdio.h>
#include <string.h>
char names[8][64], error[256];
uint32_t grids[8][4], launches;
static float scratch[64];
void gpu_next_bytes(gpu_t *g, double b) {}
void gpu_next_flops(gpu_t *g, double f) {}
int gpu_fail(gpu_t *g, const char *m) { snprintf(error, sizeof error, "%s", m); return -1; }
float *gpu_scratch_ws(gpu_t *g, size_t n) { return scratch; }
int gpu_launch(gpu_t *g, const char *k, const void *a, size_t n, uint32_t x, uint32_t y, uint32_t z, uint32_t u, uint32_t v,
               uint32_t w) {
    if (!x || !y || !z) return 0;
    if (launches == 8) return -1;
    snprintf(names[launches], sizeof names[0], "%s", k);
    memcpy(grids[launches++], (uint32_t[4]){ x, y, z, u }, 16);
    return 0;
}
"""


class Recorder:
    def __init__(self, d):
        (d / "stubs.c").write_text(STUBS)
        so = str(d / "launchers.so")
        subprocess.run(["gcc", "-std=c11", "-D_GNU_SOURCE", "-w", "-shared", "-fPIC", "-O1", f"-I{HOST}", f"-I{HOST}/..", f"-I{REPO}/include",
                        str(d / "stubs.c"), os.path.join(HOST, "nk_fp4.c"), os.path.join(HOST, "nk_ssm.c"), "-o", so], check=True)
        self.L = C.CDLL(so)
        for f in ("nk_fp4_quant", "nk_fp4_dequant", "nk_gemm_fp4", "nk_gemm_w4", "nk_causal_conv", "nk_ssm_scan"):
            getattr(self.L, f).restype, getattr(self.L, f).argtypes = nemoasr.API[f]
        self.n = C.c_uint32.in_dll(self.L, "launches")
        self.names = (C.c_char * 64 * 8).in_dll(self.L, "names")
        self.grids = (C.c_uint32 * 4 * 8).in_dll(self.L, "grids")

    def __call__(self, f, *args):
        """[(kernel, workgroups in x, y and z, threads)] of a call"""
        self.n.value = 0
        rc = getattr(self.L, f)(None, *args)
        assert rc == 0, (C.c_char * 256).in_dll(self.L, "error").value
        return [(bytes(self.names[i]).split(b"\0")[0].decode(), *self.grids[i]) for i in range(self.n.value)]


@pytest.fixture(scope="module")
def launches(tmp_path_factory):
    if not shutil.which("gcc"):
        pytest.skip("gcc not present")
    return Recorder(tmp_path_factory.mktemp("launchers"))


P = 0x10000  # an aligned address that nothing reads


@pytest.mark.parametrize("D", [64, 2048, 1 << 16])
@pytest.mark.parametrize("typ", [0, 1])
@pytest.mark.parametrize("nseq,rows", [(1, 0), (1, 1), (1, 8192), (64, 64), (256, 256), (64, 8255), (300, 40000), (5000, 50000), (65535, 65535),
                                       (65535, 1 << 22), (3, 1 << 31)])
def test_conv_grid_goes_by_the_rows(launches, D, typ, nseq, rows):
    """Workgroups by the rows that there are and the sequences, whatever max_rows allows: one of 2^30 rows, as a
    captured graph may have it, is no more than a few times what the rows need."""
    for max_rows in (1, 7, 64, 1500, 1 << 18, 1 << 30):
        got = launches("nk_causal_conv", P, typ, D, P, P, P, 8, P, nseq, max_rows, 2 * P, D, rows, D, 4, 1)
        assert len(got) == 1
        name, x, y, z, threads = got[0]
        two = "x2" in name
        assert x * threads * (2 if two else 1) >= D and z == nseq and threads == 256 and 1 <= y <= 65535
        there = min(rows, nseq * max_rows)
        assert x * y * z <= x * (4 * (there // 8 + nseq)) + 16384 + x * nseq


def test_grids_of_no_rows(launches):
    """Sequences that have no rows still hand their states on."""
    for M, max_rows in ((0, 0), (0, 9), (7, 0)):
        _, x, y, z, _ = launches("nk_causal_conv", P, 0, 64, P, None, P, 8, P, 5, max_rows, 2 * P, 64, M, 64, 4, 1)[0]
        assert x == 1 and y >= 1 and z == 5


def parameters(fn):
    """The parameter sets of a test function."""
    sets = []
    for mark in fn.pytestmark:
        if mark.name == "parametrize":
            names = [n.strip() for n in mark.args[0].split(",")]
            sets.append([dict(zip(names, v if len(names) > 1 else (v,))) for v in mark.args[1]])
    return [{k: v for d in c for k, v in d.items()} for c in itertools.product(*sets)]


def test_gpu_tests_launch_every_kernel(launches):
    """Every kernel of the 4-bit and selective-scan operators that the library holds is launched by a GPU test: the
    launchers asked with the sizes of those tests name them all, and no other."""
    seen = set()

    def note(f, *args):
        seen.update(k[0] for k in launches(f, *args))

    for name, fn in vars(fp4).items():
        if not name.startswith("test_") or not isinstance(getattr(fn, "pytestmark", None), list):
            continue
        for c in parameters(fn):
            if not {"m", "n", "k"} <= c.keys():
                continue
            m, k, act = c["m"], c["k"], c.get("act", 0)
            n = c["n"] - (act == 3 and c["n"] % 2)
            row = fp4.row_bytes(k)
            end = (P, row, P, row // 16, None, P, n // 2 if act == 3 else n, m, n, k, act, 0, 1.0)
            if c.get("kind") == "fp4":
                note("nk_gemm_fp4", P, row, P, row // 16, *end)
            else:
                note("nk_gemm_w4", P, -(-k // 4) * 4, *end)
    for typ in (0, 1):  # test_quant_and_back
        note("nk_fp4_quant", P, typ, 128, P, 64, P, 4, 1, 128)
        note("nk_fp4_dequant", P, 64, P, 4, P, typ, 128, 1, 128)

    def conv(typ, lens, D, taps, ldx=None):
        note("nk_causal_conv", P, typ, ldx or D, P, None, P, 8, P, len(lens), max(lens), 2 * P, D, sum(lens), D, taps, 1)

    for c in parameters(ssm.test_conv):
        conv(c["typ"], ssm.CONV_CASES[c["case"]][0], c["D"], c["taps"])
    for c in parameters(ssm.test_conv_long):
        conv(c["typ"], [8100, 37, 200], c["D"], 4, c["more"].get("ldx"))
    for c in parameters(ssm.test_conv_long_of_fewer_taps):
        conv(1, [8100, 1, 37, 200], 2050, c["taps"])

    def scan(typ, nseq, max_rows, M, D, N, G):
        a = nemoasr.Scan(type=typ, ldx=D, lddt=D, ldbc=G * N, ldz=D, ldy=D, x=P, dt=P, B=P, C=P, z=P, y=2 * P, A=P, state=P, seqs=P,
                         slots=9999, nseq=nseq, max_rows=max_rows, M=M, D=D, N=N, groups=G, softplus=1)
        note("nk_ssm_scan", C.byref(a))

    for fn in (ssm.test_scan, ssm.test_scan_more_states):
        for c in parameters(fn):
            lens, slots, gap = ssm.SCAN_CASES[c["case"]]
            _, M = ssm._seqs(lens, slots, gap)
            scan(c["typ"], len(lens), max(lens) + c["case"] % 2 * 40, M, c["D"], c["N"], c["G"])
    for fn in (ssm.test_scan_many_sequences, ssm.test_scan_many_sequences_of_more_states):
        for c in parameters(fn):
            scan(c["typ"], 4200, 130, 4196 * 2 + 300, c["D"], c["N"], c["G"])
    with open(os.path.join(REPO, "nemo-c_amd", "libnemoasr_hip.so"), "rb") as f:
        built = re.findall(rb"\0((?:gemm_fp4|gemm_w4|fp4_|cconv_|scan_)\w*)\.kd\0", f.read())
    assert seen == {b.decode() for b in built}
