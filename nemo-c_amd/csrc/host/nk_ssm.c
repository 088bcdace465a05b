/* Launchers of the selective-scan block's operators (include/nemo_kernels.h): arguments are checked before any
 * launch; the sequences' table lies on the device and is checked by the kernels. */
#include "nemo_kernels.h"
#include "gpu.h"
#include "../kernel_params.h"
#include <stdio.h>

static int bad(gpu_t *g, const char *what) { return gpu_fail(g, what); }
static int aligned(const void *p, uintptr_t n) { return ((uintptr_t)p & (n - 1)) == 0; }

/* what both operators ask of the batch */
static const char *batch_bad(const float *state, uint32_t slots, const int *seqs, uint32_t nseq, uint32_t max_rows, uint32_t D) {
    if (!seqs || !aligned(seqs, 16)) return "sequences: a 16-byte aligned table";
    if (nseq > 65535) return "sequences: at most 65535 in a call";
    if (D > 1u << 27) return "sequences: at most 2^27 channels";
    if (slots > 0x7fffffffu || (slots && (!state || !aligned(state, 4)))) return "sequences: slots without a state";
    if (max_rows > 1u << 30) return "sequences: at most 2^30 rows each";
    return NULL;
}

int nk_causal_conv(gpu_t *g, const void *X, int type, uint32_t ldx, const float *W, const float *bias, float *state,
                   uint32_t slots, const int *seqs, uint32_t nseq, uint32_t max_rows, void *Y, uint32_t ldy, uint32_t M,
                   uint32_t D, uint32_t taps, int act) {
    if (!nseq || !D) return 0;
    const char *why = batch_bad(state, slots, seqs, nseq, max_rows, D);
    if (why) return bad(g, why);
    if (type != NK_F32 && type != NK_BF16) return bad(g, "causal_conv: rows are f32 or bf16");
    const uintptr_t size = type == NK_F32 ? 4 : 2;
    if (taps < 2 || taps > 4 || act < NK_ACT_NONE || act > NK_ACT_RELU)
        return bad(g, "causal_conv: 2 to 4 taps, no activation, SiLU or ReLU");
    if (!X || !Y || !W || !aligned(X, size) || !aligned(Y, size) || !aligned(W, 4) || !aligned(bias, 4) || ldx < D || ldy < D)
        return bad(g, "causal_conv: aligned rows of at least D values");
    if (X == Y) return bad(g, "causal_conv: Y must not overlap X");
    const uint64_t rows = (uint64_t)nseq * max_rows < M ? (uint64_t)nseq * max_rows : M;
    /* bf16: two channels a thread from 16 Mi values on (17760 rows of 2048 channels 39.5 -> 33.8 us; 8192 rows 15.9 / 16.1,
     * 4096 rows of 512 5.8 / 6.3) */
    const int two = type == NK_BF16 && D % 2 == 0 && ldx % 2 == 0 && ldy % 2 == 0 && aligned(X, 4) && aligned(Y, 4) &&
                    rows * D >= 1u << 24;
    const uint32_t blocks = ((two ? D / 2 : D) + 255) / 256;
    /* tiles of 8 to 64 rows, some 4096 workgroups (17760 rows of 2048 bf16 channels with 1024, 2048 and 4096: 37.4, 37.2,
     * 33.8 us) */
    uint64_t tile = rows * blocks / 4096 / 8 * 8;
    tile = tile < 8 ? 8 : tile > 64 ? 64 : tile;
    /* Workgroups for the longest sequence that may be, all sequences alike, but no more than four times what the rows need or
     * 16384 in all: those with no rows cost 0.45 us a thousand, and a longer sequence goes round (64 tokens with max_rows
     * 2^12 or 2^18 7.6 us, by the longest alone 112 us and 16 million workgroups; a prompt of 8192 rows beside 63 tokens 55 /
     * 131, beside 255 132 / 462, with 65536 in all 41 and 62 but the tokens 31). */
    const uint64_t last = max_rows < M ? max_rows : M, longest = (last + tile - 1) / tile;
    const uint64_t share = 4 * (rows / tile / nseq + 1), room = 16384 / ((uint64_t)blocks * nseq);
    uint64_t tiles = share > room ? share : room;
    if (tiles > longest) tiles = longest;
    tiles = tiles < 1 ? 1 : tiles > 65535 ? 65535 : tiles;
    NkCconvArgs a = { X, W, bias, state, seqs, Y, ldx, ldy, slots, nseq, max_rows, M, D, taps, (u32)act, (u32)tile };
    char name[24];
    snprintf(name, sizeof name, "cconv_%s_%u", type == NK_F32 ? "f32" : two ? "bf16x2" : "bf16", taps);
    gpu_next_bytes(g, 2.0 * size * M * D + 8.0 * nseq * (taps - 1) * D + 4.0 * D * (taps + 1));
    return gpu_launch(g, name, &a, sizeof a, blocks, (uint32_t)tiles, nseq, 256, 1, 1);
}

int nk_ssm_scan(gpu_t *g, const nk_scan_t *p) {
    if (!p) return bad(g, "ssm_scan: no arguments");
    if (!p->nseq || !p->D) return 0;
    const char *why = batch_bad(p->state, p->slots, p->seqs, p->nseq, p->max_rows, p->D);
    if (why) return bad(g, why);
    if (p->type != NK_F32 && p->type != NK_BF16) return bad(g, "ssm_scan: rows are f32 or bf16");
    const uintptr_t size = p->type == NK_F32 ? 4 : 2;
    if (!p->N || p->N > 64 || !p->groups || p->D % p->groups) return bad(g, "ssm_scan: 1 to 64 states, groups that divide the channels");
    if (!p->x || !p->dt || !p->B || !p->C || !p->y || !p->A || !aligned(p->x, size) || !aligned(p->dt, size) ||
        !aligned(p->B, size) || !aligned(p->C, size) || !aligned(p->z, size) || !aligned(p->y, size) || !aligned(p->A, 4) ||
        !aligned(p->skip, 4) || !aligned(p->dt_bias, 4))
        return bad(g, "ssm_scan: x, dt, B, C, y and A aligned to their values");
    if (p->ldx < p->D || p->lddt < p->D || p->ldy < p->D || (p->z && p->ldz < p->D) || p->ldbc < (uint64_t)p->groups * p->N)
        return bad(g, "ssm_scan: rows of at least D values, B and C of groups * N");
    if (p->y == p->x || p->y == p->dt || p->y == p->B || p->y == p->C || p->y == p->z)
        return bad(g, "ssm_scan: y must not overlap the inputs");
    const uint32_t per = p->D / p->groups, block = per >= 256 ? 256 : (per + 63) / 64 * 64;
    const uint32_t tiles = p->groups * ((per + block - 1) / block);
    const uint64_t waves = (uint64_t)p->nseq * tiles * (block / 64);
    NkScanArgs a = { p->x, p->dt, p->B, p->C, p->z, p->y, p->A, p->skip, p->dt_bias, p->state, p->seqs, NULL, NULL,
                     p->ldx, p->lddt, p->ldbc, p->ldz, p->ldy, p->slots, p->nseq, p->max_rows, p->M, p->D, p->N,
                     p->groups, p->softplus != 0, 0, 0, 0,
                     p->N % 4 == 0 && aligned(p->A, 16) && aligned(p->state, 16) };
    const uint32_t ns = p->N <= 8 ? 8 : p->N <= 16 ? 16 : p->N <= 32 ? 32 : 64;
    if ((uint64_t)tiles * block > 1u << 31) return bad(g, "ssm_scan: more channels than a launch covers");
    const char *type = p->type == NK_F32 ? "f32" : "bf16";
    char name[32];
    gpu_next_bytes(g, (double)size * p->M * (4.0 * p->D + 2.0 * p->groups * p->N) + 8.0 * p->nseq * p->D * p->N);
    gpu_next_flops(g, (double)p->M * p->D * (7.0 * p->N + 12));
    /* Estimates in us by wavefronts w of 64 channels, rows r of the longest sequence and R there can be, fitted to graph
     * replays with 16 states: states over lanes (few rows), sequences whole with the states in one lane, split along
     * their rows (every exponential twice, three launches).  Few / whole: 32 w 16 r 14.1 / 17.0, 32 r 22.7 / 23.7; 1024 w
     * 8 r 14.6 / 16.6, 16 r 21.2 / 21.0; 8192 w 4 r 44.5 / 73, 8 r 79 / 78.  Whole / split: 32 w 48 r 31 / 20, 1024 r
     * 466 / 50; 512 w 64 r 39.8 / 51, 600 r 283 / 185; 768 w 256 r 127 / 143, 600 r 284 / 249; 1024 w 600 r 287 / 337, of
     * ragged sequences with half the rows 281 / 188; 2048 w 2000 r, ragged, 1158 / 923. */
    const uint64_t all = (uint64_t)p->nseq * p->max_rows, R = all < p->M ? all : p->M;
    const double w = (double)waves, r = p->max_rows, x = (double)R * (double)(waves / p->nseq);
    const double few = 4.0 + r * (w < 350.0 ? 0.42 : 0.0012 * w), whole = 10.0 + 0.0045 * w + r * (0.39 + 0.0001 * w);
    const double split = 24.0 + 0.0005 * x + 0.0003 * (x < 65536.0 ? x : 65536.0) + 0.03 * p->nseq;
    if (p->max_rows <= 32 && few < whole) {
        uint32_t q = 1;
        while (4 * q < p->N) q *= 2;
        snprintf(name, sizeof name, "scan_few_%s_%u", type, q);
        return gpu_launch(g, name, &a, sizeof a, (uint32_t)(((uint64_t)p->D * q + 255) / 256), p->nseq, 1, 256, 1, 1);
    }
    if (split < whole && p->nseq <= 4096) {
        /* about 4096 wavefronts (four per SIMD: 8192 rows of one stream 335 us with 1024, 210 with 2048, 168), twice that
         * where each has enough to do (32 ragged sequences of up to 600 rows 202 / 188, 2000 rows 1297 / 923; 24 of 64 rows
         * 64 / 79), and pieces of some sqrt(r / 2) rows, between the pieces' time and that of joining them (512 rows:
         * pieces of 4, 8, 16 and 32 rows 45, 34, 31 and 42 us; 32 rows: 17.8, 20.8, 27.4, 30.1).  By the rows there are, a
         * sequence's last piece being half one: beyond the aim the rest takes a round of its own (8 sequences of 0 to
         * 2000 rows 241 us without the halves, 186 with them; 5 of up to 4000 192 / 155, 12 of up to 1000 114 / 102). */
        const uint64_t aim = x < 250000.0 ? 4096 : 8192;
        const uint64_t fill = R * (waves / p->nseq) / ((aim < waves ? waves : aim) - waves / 2);
        uint32_t piece = (uint32_t)fill / 4 * 4 + 4;
        while (piece < 8 || 2ull * piece * piece < p->max_rows) piece += 4;
        const uint32_t pieces = (p->max_rows + piece - 1) / piece;
        /* places for all sequences' pieces, or, where that is fewer (one long sequence among many short ones, max_rows far
         * above the longest), for one of each `piece` rows */
        const uint64_t table = (uint64_t)p->nseq * pieces, byrow = ((uint64_t)p->M + piece - 1) / piece + 1;
        a.byrow = byrow < table;
        const uint64_t places = (a.byrow ? byrow : table) * (p->N + 1) * p->D;
        a.ws = gpu_scratch_ws(g, (size_t)(places + (uint64_t)p->nseq * p->N * p->D));
        if (!a.ws) return bad(g, "ssm_scan: scratch unavailable (size it before capture)");
        a.first = a.ws + places;
        /* workgroups for the pieces that there can be, numbered over all sequences (a sequence of no rows has one) */
        const uint64_t most = R / piece + p->nseq;
        const uint32_t all_pieces = (uint32_t)(most < table ? most : table);
        a.piece = piece;
        a.pieces = pieces;
        snprintf(name, sizeof name, "scan_ends_%s_%u", type, ns);
        if (gpu_launch(g, name, &a, sizeof a, tiles, all_pieces, 1, block, 1, 1)) return -1;
        if (gpu_launch(g, "scan_join", &a, sizeof a, (p->D + 255) / 256, p->N, p->nseq, 256, 1, 1)) return -1;
        snprintf(name, sizeof name, "scan_from_%s_%u", type, ns);
        return gpu_launch(g, name, &a, sizeof a, tiles, all_pieces, 1, block, 1, 1);
    }
    snprintf(name, sizeof name, "scan_%s_%u", type, ns);
    return gpu_launch(g, name, &a, sizeof a, tiles, p->nseq, 1, block, 1, 1);
}
