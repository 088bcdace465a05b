"""The attention's plan against the launches, without a GPU: the launcher and the planning that the kernels do of the table
(kernel_params.h), compiled together for the host.  Of many prompts and batches every tile is planned once, every step of a
tile lies in one piece, no piece lies beyond the grid or the scratch, and the joining launch covers the tiles that are split."""
import ctypes as C
import os
import shutil
import subprocess

import pytest

import nemoasr
import test_kv_launches
from conftest import REPO

HOST = os.path.join(REPO, "nemo-c_amd", "csrc", "host")

SOURCE = r"""
#include "nemo_kernels.h"
#include "gpu.h"
#include "kernel_params.h"
#include <stdio.h>
#include <stdlib.h>
#include <string.h>

/* the device layer: launches as they are asked for */
static struct { NkAttnKvArgs a; uint32_t x, y, z; int join; size_t floats; } did[8];
static int launches;
static size_t floats_now;
static float scratch[1];
void gpu_next_bytes(gpu_t *g, double b) { (void)g, (void)b; }
static const char *error;
int gpu_fail(gpu_t *g, const char *m) { (void)g; error = m; return -1; }
float *gpu_scratch_ws(gpu_t *g, size_t n) { (void)g; floats_now = n; return scratch; }
int gpu_launch(gpu_t *g, const char *k, const void *a, size_t n, uint32_t x, uint32_t y, uint32_t z, uint32_t u, uint32_t v, uint32_t w) {
    (void)g, (void)u, (void)v, (void)w;
    if (n != sizeof(NkAttnKvArgs) || launches == 8) abort();
    memcpy(&did[launches].a, a, n);
    did[launches].x = x, did[launches].y = y, did[launches].z = z;
    did[launches].join = strstr(k, "join") != NULL;
    did[launches++].floats = floats_now;
    return 0;
}

typedef struct { uint32_t first, rows, len, row; } seq_t;
static unsigned char *seen; /* tiles of the sequence at hand */
static uint32_t seen_room;
static long refused, planned, split_calls, split_tiles, most_share;

#define MUST(c) do { if (!(c)) { printf("line %d: %s\n", __LINE__, #c); return 1; } } while (0)

/* one launch and the joining one behind it (or NULL), for sums of steps that are `off` from the exact one */
static int plan(const NkAttnKvArgs *a, uint32_t x, const NkAttnKvArgs *j, uint32_t jx, uint32_t jz, size_t floats, const seq_t *s, uint32_t n, float off) {
    const uint32_t heads = a->kv.heads, launched = x / heads;
    uint32_t tiles = 0, piece = 0;
    double steps = 0;
    MUST(x % heads == 0 && !j == !a->slots);
    for (uint32_t i = 0; i < n; ++i) {
        const uint32_t t = nk_attn_tiles(a, s[i].rows);
        tiles += t;
        steps += nk_attn_all_steps(a, t, s[i].len, s[i].rows);
    }
    if (a->slots) {
        MUST(j->slots == a->slots && j->items == a->items && j->ws == a->ws && j->ws);
        MUST(floats >= ((uint64_t)a->items * heads << a->tile) * (a->kv.dh + 2));
        piece = nk_attn_piece(a, tiles, (float)steps * off);
    }
    split_calls += piece != 0;
    uint32_t item = 0, joined = 0;
    for (uint32_t i = 0; i < n; ++i) {
        const uint32_t rows = s[i].rows, len = s[i].len, t = nk_attn_tiles(a, rows);
        if (!t) continue;
        MUST(t == (rows * a->group + (1u << a->tile) - 1) >> a->tile);
        if (t > seen_room) seen = realloc(seen, seen_room = t);
        memset(seen, 0, t);
        const uint32_t pieces = nk_attn_pieces(a, len, rows, piece);
        for (uint32_t k = 0; k < t; ++k, item += pieces, joined += pieces > 1) {
            const nk_attn_tile_t w = nk_attn_tile(a, len, rows, k);
            const uint32_t q = w.r0 >> a->tile;
            MUST(w.r0 == q << a->tile && q < t && !seen[q]++ && w.nr == (q + 1 < t ? 1u << a->tile : rows * a->group - w.r0));
            MUST(w.pos_lo == len + w.r0 / a->group && w.pos_hi == len + (w.r0 + w.nr - 1) / a->group);
            const uint32_t lo = a->window && w.pos_lo >= a->window ? w.pos_lo + 1 - a->window : 0, S = 1u << a->step;
            const uint32_t sinks = a->window ? (a->sinks + S - 1) / S : 0;
            MUST(w.lo_step == lo / S && w.sink_steps == (sinks < w.lo_step ? sinks : w.lo_step));
            MUST(w.steps == w.sink_steps + w.pos_hi / S - w.lo_step + 1 && w.steps <= nk_attn_most_steps(a, len, rows));
            MUST(item + pieces <= launched);
            ++planned;
            if (pieces == 1) continue;
            const uint32_t each = nk_attn_piece_of(a, len, rows, pieces), real = (w.steps - 1) / each + 1;
            MUST(each && real <= pieces && (uint64_t)real * each >= w.steps && (real - 1) * each < w.steps);
            if (real == 1) continue;
            ++split_tiles;
            MUST(joined < jx && jz && item + real <= a->items);
        }
    }
    if (a->slots && piece) {
        const long share = 100l * item / a->slots;
        if (share > most_share) most_share = share;
    }
    return 0;
}

static int call(int type, uint32_t heads, uint32_t group, uint32_t dh, uint32_t window, uint32_t sinks, uint32_t max_rows, uint32_t max_len,
                uint32_t M, const seq_t *s, uint32_t n) {
    void *P = (void *)0x10000;
    nk_kv_t kv = { .type = NK_BF16, .heads = heads, .dh = dh, .page = 64, .pages = 9, .k = P, .v = P, .table = P, .ldt = 1 << 25, .tables = 1 << 20 };
    nk_attend_t p = { .type = type, .ldq = heads * group * dh, .ldo = heads * group * dh, .q = P, .o = (char *)P + 4096, .heads = heads * group,
                      .window = window, .sinks = sinks, .scale = 1.0f, .seqs = P, .nseq = n, .max_rows = max_rows, .max_len = max_len, .M = M };
    launches = 0;
    if (nk_attention_kv(NULL, &kv, &p)) {
        MUST(!strcmp(error, "attention_kv: more rows than a launch covers"));
        ++refused;
        return 0;
    }
    for (uint32_t i = 0; i < n; ++i) { /* every sequence is one launch's */
        int of = 0;
        for (int l = 0; l < launches; ++l) of += !did[l].join && s[i].rows > did[l].a.over && s[i].rows <= did[l].a.upto;
        MUST(of == (s[i].rows > 0));
    }
    for (int l = 0; l < launches; ++l) {
        if (did[l].join) continue;
        const int j = l + 1 < launches && did[l + 1].join;
        MUST(!j || did[l + 1].y == heads);
        for (int e = -1; e <= 1; ++e)
            if (plan(&did[l].a, did[l].x, j ? &did[l + 1].a : NULL, did[l + 1].x, did[l + 1].z, did[l].floats, s, n, 1.0f + 1e-5f * (float)e)) {
                printf("type %d, %u heads, group %u, dh %u, window %u, sinks %u, max_rows %u, max_len %u, M %u, %u sequences, rows %u and %u behind %u\n", type,
                       heads, group, dh, window, sinks, max_rows, max_len, M, n, s[0].rows, s[n > 1].rows, s[0].len);
                return 1;
            }
    }
    return 0;
}

static uint64_t state = 1;
static uint32_t below(uint32_t n) { /* 0 .. n - 1 */
    state = state * 6364136223846793005ull + 1442695040888963407ull;
    return (uint32_t)((state >> 33) * (uint64_t)n >> 31);
}
static uint32_t spread(uint32_t n) { /* 0 .. n - 1, over its logarithm */
    uint32_t bits = 0;
    while (n >> bits) ++bits;
    const uint32_t top = 1u << below(bits + 1);
    return below(top < n ? top : n);
}

int main(int argc, char **argv) {
    const int batches = argc > 1 && !strcmp(argv[1], "batches");
    const uint32_t hs[] = { 1, 2, 3, 4, 8, 16, 32, 48 }, gs[] = { 1, 2, 3, 4, 5, 8, 20, 64, 130 }, ds[] = { 64, 256 };
    if (!batches) { /* one prompt: lengths to 16384, alone, behind a few tokens and many, with windows */
        for (uint32_t h = 0; h < 8; ++h)
            for (uint32_t g = 0; g < 9; ++g)
                for (int type = 0; type < 2; ++type)
                    for (uint32_t rows = 1; rows <= 16384; rows += rows < 64 ? 1 : 31 + h) {
                        const uint32_t starts[] = { 0, 40, rows, 3000 }, windows[] = { 0, rows > 9 ? rows - 9 : 0, rows / 2, 512 };
                        const uint32_t start = starts[below(4)], window = windows[below(2) ? 0 : below(4)], more = below(8) ? 0 : 1000;
                        const seq_t s[1] = { { 0, rows, start, 0 } };
                        if (call(type, hs[h], gs[g], ds[below(2)], window, below(2) ? 4 : 100, rows + more, start + rows + 3 * more, rows + more, s, 1)) return 1;
                        const seq_t s0[1] = { { 0, rows, 0, 0 } };
                        if (call(type, hs[h], gs[g], 128, 0, 0, rows, rows, rows, s0, 1)) return 1;
                    }
    } else
        for (int i = 0; i < 120000; ++i) { /* prompts, chunks and steps beside one another, a few long ones among many short */
            static seq_t s[300];
            const uint32_t n = 1 + spread(below(8) ? 24 : 300), h = hs[below(8)], g = gs[below(9)], longest = 1 + spread(6000), far = 1 + spread(below(4) ? 9000 : 200000);
            uint32_t M = below(3), rows = 0, len = 0;
            for (uint32_t k = 0; k < n; ++k) {
                s[k] = (seq_t){ M, below(3) ? spread(longest + 1) : longest - 1 + below(2), below(2) ? spread(far) : 0, 0 };
                M += s[k].rows;
                if (s[k].rows > rows) rows = s[k].rows;
                if (s[k].rows + s[k].len > len) len = s[k].rows + s[k].len;
            }
            if (!rows) continue;
            const uint32_t window = below(3) ? 0 : 1 + spread(len + 1);
            if (call(below(2), h, g, 16 * (1 + below(16)), window, spread(200), rows + (below(4) ? 0 : spread(5000)), len + (below(4) ? 0 : spread(100000)),
                     M + below(4), s, n)) return 1;
        }
    printf("%ld tiles, %ld of them split, in %ld split plans; at most %ld hundredths of a piece a slot; %ld calls refused\n", planned, split_tiles,
           split_calls, most_share, refused);
    return 0;
}
"""


@pytest.fixture(scope="module")
def program(tmp_path_factory):
    if not shutil.which("gcc"):
        pytest.skip("gcc not present")
    d = tmp_path_factory.mktemp("plan")
    (d / "plan.c").write_text(SOURCE)
    exe = str(d / "plan")
    subprocess.run(["gcc", "-std=c11", "-D_GNU_SOURCE", "-O2", "-Wall", "-Wno-unused-function", "-Wno-missing-field-initializers", f"-I{HOST}", f"-I{HOST}/..",
                    f"-I{REPO}/include", str(d / "plan.c"), os.path.join(HOST, "nk_kv.c"), "-o", exe, "-lm"], check=True)
    return exe


@pytest.mark.parametrize("what", ["prompts", "batches"])
def test_pieces_lie_in_the_grid_and_the_scratch(program, what):
    r = subprocess.run([program, what], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout
    tiles, split, plans, share, refused = (int(w) for w in r.stdout.split() if w.isdigit())
    assert split > 100000 and plans > 10000  # tiles that are split were among them
    assert tiles > 10 ** 7 and refused < 5000 and share > 200  # and calls of more than two pieces a slot


def test_refused_calls_launch_nothing(tmp_path, monkeypatch):
    """A mixed batch whose prompts are refused, for their number or for want of scratch, is refused as a whole: the launch of its
    few-row sequences does not come first."""
    if not shutil.which("gcc"):
        pytest.skip("gcc not present")
    stubs = test_kv_launches.STUBS.replace("{ return scratch; }", "{ return n < 1u << 21 ? scratch : 0; }").replace("error", "why")  # libc has an `error`
    monkeypatch.setattr(test_kv_launches, "STUBS", stubs)
    rec, P = test_kv_launches.Recorder(tmp_path), test_kv_launches.P

    def call(**more):
        rec.n.value = 0
        a = dict(type=1, q=P, ldq=1024, o=2 * P, ldo=1024, heads=8, scale=0.1, seqs=P, nseq=2, max_rows=130, max_len=40000, M=131)
        rc = rec.L.nk_attention_kv(None, test_kv_launches.cache(1, 8, 128), C.byref(nemoasr.Attend(**dict(a, **more))))
        return rc, rec.n.value, (C.c_char * 256).in_dll(rec.L, "why").value

    assert call(max_rows=100, M=101, max_len=2100)[:2] == (0, 4)  # steps and prompts, joined each
    rc, n, why = call(max_rows=1 << 30, M=(1 << 30) + 1)
    assert (rc, n) == (-1, 0) and b"more rows" in why
    rc, n, why = call()
    assert (rc, n) == (-1, 0) and b"scratch" in why
