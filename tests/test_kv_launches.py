"""The launches that the hosts of the paged cache and its attention choose, without a GPU: their source compiled against a
device layer of stubs that records launches."""
import ctypes as C
import os
import re
import shutil
import subprocess

import numpy as np
import pytest

import nemoasr
import test_gpu_kv as kv
from conftest import REPO
from test_ssm_launches import HOST, STUBS, parameters

P = 0x10000  # an aligned address that nothing reads


class Recorder:
    def __init__(self, d):
        (d / "stubs.c").write_text(STUBS)
        so = str(d / "launchers.so")
        subprocess.run(["gcc", "-std=c11", "-D_GNU_SOURCE", "-w", "-shared", "-fPIC", "-O1", f"-I{HOST}", f"-I{HOST}/..", f"-I{REPO}/include",
                        str(d / "stubs.c"), os.path.join(HOST, "nk_kv.c"), "-o", so, "-lm"], check=True)
        self.L = C.CDLL(so)
        for f in ("nk_kv_append", "nk_kv_read", "nk_attention_kv"):
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


def cache(typ, heads, dh):
    return C.byref(nemoasr.Kv(type=typ, heads=heads, dh=dh, page=64, pages=9, k=P, v=P, ks=P, vs=P, table=P, ldt=1 << 20, tables=1 << 16))


def attend(launches, cache_type, typ, heads, hk, dh, nseq, max_rows, M, max_len=4000, window=0, ld=None):
    a = nemoasr.Attend(type=typ, q=P, ldq=ld or heads * dh, o=2 * P, ldo=ld or heads * dh, heads=heads, window=window, sinks=4, scale=0.1, seqs=P,
                       nseq=nseq, max_rows=max_rows, max_len=max_len, M=M)
    return launches("nk_attention_kv", cache(cache_type, hk, dh), C.byref(a))


def append(launches, cache_type, typ, heads, hk, dh, rot, nseq, max_rows, M, ld, off=0):
    a = nemoasr.Append(type=typ, q=P + off, ldq=ld, k=P + off, ldk=ld, v=P + off, ldv=ld, qo=2 * P + off, ldqo=ld, heads=heads, rot=rot, freq=P, amp=1.0,
                       seqs=P, nseq=nseq, max_rows=max_rows, M=M)
    return launches("nk_kv_append", cache(cache_type, hk, dh), C.byref(a))


def test_gpu_tests_launch_every_kernel(launches):
    """Every kernel of the cache and its attention that the library holds is launched by a GPU test: the launchers asked with
    the sizes of those tests name them all, and no other."""
    seen = set()

    def note(got):
        seen.update(k[0] for k in got)

    for c in parameters(kv.test_append):
        heads, hk, dh, rot, _ = kv.HEADS[c["shape"]]
        rows, starts = kv.BATCHES[c["batch"]]
        ld, off = [(max(heads, hk) * dh, 0), (max(heads, hk) * dh + 24, 0), (max(heads, hk) * dh + 3, 1), (heads * dh, 4)][(c["batch"] + c["shape"]) % 4]
        size = 4 if c["typ"] == kv.F32 else 2
        note(append(launches, c["cache_type"], c["typ"], heads, hk, dh, rot, len(rows), max(rows), sum(rows), ld, off * size))
    for c in parameters(kv.test_read):
        size = 4 if c["typ"] == kv.F32 else 2
        ld = c["ld"] or 3 * c["dh"]
        note(launches("nk_kv_read", cache(c["cache_type"], 1, c["dh"]), P + c["off"] * size, ld, P + c["off"] * size, ld, c["typ"], P, 4, 99, 65))
    for c in parameters(kv.test_attend):
        heads, hk, dh = kv.ATTEND_HEADS[c["shape"]]
        rows, starts = kv.ATTEND_BATCHES[c["batch"]]
        note(attend(launches, c["cache_type"], c["typ"], heads, hk, dh, len(rows), max(rows), sum(rows),
                    max(r + s for r, s in zip(rows, starts))))
    for c in parameters(kv.test_attend_prompts):
        heads, hk, dh = kv.PROMPT_HEADS[c["shape"]]
        note(attend(launches, c["cache_type"], c["typ"], heads, hk, dh, 5, 150, 188, 301, c["window"]))
    for c in parameters(kv.test_attend_prompt_behind_many_tokens):
        note(attend(launches, c["cache_type"], c["typ"], 1, 1, c["dh"], 1, 130, 130, 3030))
    with open(os.path.join(REPO, "nemo-c_amd", "libnemoasr_hip.so"), "rb") as f:
        built = re.findall(rb"\0((?:kv_|attn_)\w*)\.kd\0", f.read())
    assert seen == {b.decode() for b in built}


@pytest.mark.parametrize("max_rows,M", [(1, 64), (1 << 20, 64), (1, 1), (500, 8000)])
def test_grids_go_by_the_rows(launches, max_rows, M):
    """Workgroups by the rows and sequences that there are, whatever max_rows and max_len allow."""
    for nseq in (1, 64, 4096):
        for got in (append(launches, 2, 1, 32, 8, 128, 128, nseq, max_rows, M, 32 * 128), ):
            (name, x, y, z, _), = got
            assert x <= M // 16 + 2 * nseq and x * y <= max(4096, 2 * x) * 2 and z == 1
        for max_len in (100, 1 << 30):
            for name, x, y, z, threads in attend(launches, 2, 1, 32, 8, 128, nseq, max_rows, M, max_len):
                assert threads == 256
                if "join" in name:
                    assert x * y * z <= 4096
                else:
                    assert x <= 8 * max(M * 4 // 16 + nseq, 2 * 192) and y == z == 1


def test_steps_of_a_mixed_batch(launches):
    """Beside prompts, sequences of up to 16 packed rows have a launch of their own; one sequence's rows, or few, have one."""
    names = [k[0] for k in attend(launches, 1, 1, 32, 8, 128, 64, 500, 8000)]
    assert [n for n in names if "join" not in n] == ["attn_few_bf16_bf16_128_1", "attn_many_bf16_bf16_128"]
    for more in (dict(max_len=2048), dict(window=2000)):  # or none where a step sees little
        assert [k[0] for k in attend(launches, 1, 1, 32, 8, 128, 64, 500, 8000, **more)] == ["attn_many_bf16_bf16_128"]
    assert [k[0] for k in attend(launches, 1, 1, 32, 8, 128, 1, 5000, 5000)] == ["attn_many_bf16_bf16_128"]
    assert [k[0] for k in attend(launches, 1, 1, 32, 8, 128, 64, 1, 64)] == ["attn_few_bf16_bf16_128_1", "attn_join_bf16"]
    assert np.all([k[0] == "attn_few_bf16_bf16_128_1" for k in attend(launches, 1, 1, 32, 8, 128, 64, 1, 64, 100)])
