/* Launchers of the 4-bit rows and products (include/nemo_kernels.h): arguments are checked before any launch, so
 * a kernel never sees a shape its grid or indexing does not cover. */
#include "nemo_kernels.h"
#include "gpu.h"
#include "../kernel_params.h"
#include <stdio.h>
#include <string.h>

static int bad(gpu_t *g, const char *what) { return gpu_fail(g, what); }
static int aligned(const void *p, uintptr_t n) { return ((uintptr_t)p & (n - 1)) == 0; }
#define FP4_STRIDE (1u << 24) /* the products' strides in bytes are below it: 24-bit multiplications, tiles below 4 GB */
/* codes and scales of rows of K values */
static int rows_ok(const uint8_t *Q, uint32_t ldq, const uint8_t *S, uint32_t lds, uint32_t K) {
    return Q && S && aligned(Q, 16) && ldq % 16 == 0 && ldq >= NK_FP4_ROW(K) && aligned(S, 4) && lds % 4 == 0 &&
           lds >= NK_FP4_SCALES(K);
}

static int convert(gpu_t *g, const char *kernel, void *X, int type, uint32_t ldx, uint8_t *Q, uint32_t ldq, uint8_t *S,
                   uint32_t lds, uint32_t M, uint32_t K) {
    if (!M || !K) return 0;
    if (type != NK_F32 && type != NK_BF16) return bad(g, "fp4: rows are f32 or bf16");
    const uint32_t size = type == NK_F32 ? 4 : 2;
    if (K > 1u << 30 || !X || !aligned(X, size) || ldx < K) return bad(g, "fp4: rows of at least K (at most 2^30) aligned values");
    if (!rows_ok(Q, ldq, S, lds, K))
        return bad(g, "fp4: codes 16-byte aligned, ldq % 16 == 0, scales 4-byte aligned, lds % 4 == 0, rows padded to 128 values");
    const uint32_t g8 = NK_FP4_ROW(K) / 4;
    if ((uint64_t)M * g8 > 0xffffff00u) return bad(g, "fp4: more than 2^32 runs of 8 values");
    NkFp4Args a = { X, Q, S, ldx, ldq, lds, M, K, g8, aligned(X, 16) && ldx * (uint64_t)size % 16 == 0 };
    char name[24];
    snprintf(name, sizeof name, "%s_%s", kernel, type == NK_F32 ? "f32" : "bf16");
    gpu_next_bytes(g, (double)M * ((double)size * K + K * 17.0 / 32));
    return gpu_launch(g, name, &a, sizeof a, (uint32_t)(((uint64_t)M * g8 + 255) / 256), 1, 1, 256, 1, 1);
}

int nk_fp4_quant(gpu_t *g, const void *X, int type, uint32_t ldx, uint8_t *Q, uint32_t ldq, uint8_t *S, uint32_t lds,
                 uint32_t M, uint32_t K) {
    return convert(g, "fp4_quant", (void *)X, type, ldx, Q, ldq, S, lds, M, K);
}

int nk_fp4_dequant(gpu_t *g, const uint8_t *Q, uint32_t ldq, const uint8_t *S, uint32_t lds, void *X, int type,
                   uint32_t ldx, uint32_t M, uint32_t K) {
    return convert(g, "fp4_dequant", X, type, ldx, (uint8_t *)Q, ldq, (uint8_t *)S, lds, M, K);
}

/* The products' kernels.  With t workgroups on the fullest CU a launch takes about fix microseconds per `percu` of them
 * and per K step max(lat, thr x t), fitted to graph replays:
 *   fp4 (steps of 256) 3584 x 4096 x 8192 and x 4096, 2048 x 4096 x 4096, 1024 x 4096 x 2048, 448 x 4096 x 1024,
 *   448 x 1024 x 4096, 128 x 4096 x 4096: 128x256 80, 50, 28, 16.4, 11.1, 17.6, 17.9 us, 64x128 102, 60, 36, 14.0, 7.9,
 *   11.0, 11.3, 64x64 133, 70, 42, 15.3, 7.1, 8.7, 9.4: the least is picked each time; few rows against the tiles:
 *   16 x 8192 x 2048 6.1 us, 32 rows 8.1, 64 rows 11.9, 64 x 8192 x 4096 21.0 / 9.7;
 *   w4 (steps of 64) 2048 x 4096 x 8192 and x 2048, 1024 x 4096 x 2048, 448 x 4096 x 1024, 448 x 1024 x 4096: 128x256
 *   316, 87, 73, 38, 118, 64x256 342, 92, 50, 23, 67, 64x128 390, 103, 55, 19, 48, 32x64 565, 143, 76, 23, 31; few rows
 *   (16 to a workgroup, one launch of them for 17 and more) with 16 and 32 columns against 32x64: 32 x 4096 x 1024 9.7,
 *   6.7 / 10.2, 48 rows 13.0, 10.6 / 10.2, 32 x 4096 x 4096 19.6, 12.7 / 30.3, 32 x 16384 x 1024 33, 20 / 11.7, 128 x 1024
 *   x 4096 19.9, 12.9 / 30.8, 64 x 1024 x 4096 10.9, 11.9 / 29.1. */
typedef struct { const char *name; uint16_t bm, bn, threads, percu; float fix, lat, thr; } tile_t;
static const tile_t fp4_tiles[] = {
    { "128x256", 128, 256, 768, 1, 10.0f, 1.0f, 1.0f },
    { "64x128", 64, 128, 512, 2, 5.5f, 0.38f, 0.45f },
    { "64x64", 64, 64, 512, 3, 4.5f, 0.30f, 0.24f },
};
static const tile_t w4_tiles[] = {
    { "128x256", 128, 256, 768, 1, 8.0f, 2.3f, 2.3f },
    { "64x256", 64, 256, 768, 1, 5.0f, 1.35f, 1.34f },
    { "64x128", 64, 128, 512, 2, 4.5f, 0.65f, 0.76f },
    { "32x64", 32, 64, 256, 4, 3.0f, 0.43f, 0.29f },
};
static uint64_t tiles_of(const tile_t *t, uint32_t M, uint32_t nout, int glu) {
    const uint32_t co = glu ? t->bn / 2u : t->bn;
    return (uint64_t)((M + t->bm - 1) / t->bm) * ((nout + co - 1) / co);
}
/* the tile of the least estimate, and that in *us */
static const tile_t *tile_pick(const tile_t *list, int n, uint32_t M, uint32_t nout, uint32_t steps, int glu, float *us) {
    const tile_t *best = NULL;
    for (const tile_t *t = list; t < list + n; ++t) {
        if (glu && t->bn < 128) continue; /* a wavefront holds 32 value and 32 gate columns, a load of scales one half's */
        const uint64_t w = (tiles_of(t, M, nout, glu) + 255) / 256;
        const float step = t->thr * (float)w > t->lat ? t->thr * (float)w : t->lat;
        const float e = (float)((w + t->percu - 1) / t->percu) * t->fix + step * (float)steps;
        if (!best || e < *us) { best = t; *us = e; }
    }
    return best;
}

/* the checks that both products share, and their launch */
static int product(gpu_t *g, NkGemm4Args *a) {
    const int glu = a->act == NK_ACT_GLU;
    if (a->act > NK_ACT_GLU) return bad(g, "gemm 4-bit: unknown activation");
    if (!a->N || a->N > 1u << 26 || !a->K || (glu && (a->N & 1))) return bad(g, "gemm 4-bit: bad shape");
    if (a->M > 65535 * 16) return bad(g, "gemm 4-bit: too many rows");
    if (!rows_ok(a->Wq, a->ldw, a->Ws, a->ldws, a->K) || a->ldw >= FP4_STRIDE || a->ldws >= FP4_STRIDE)
        return bad(g, "gemm 4-bit: weight codes 16-byte and scales 4-byte aligned, rows padded to 128 values, strides below 2^24");
    const uint32_t nout = glu ? a->N / 2 : a->N;
    if (!a->C || !aligned(a->C, 4) || !aligned(a->bias, 4) || a->ldc < nout) return bad(g, "gemm 4-bit: ldc < output width");
    a->vec = aligned(a->C, 16) && a->ldc % 4 == 0;
    gpu_next_bytes(g, 17.0 / 32 * a->N * a->K + (a->A ? 4.0 : 17.0 / 32) * a->M * a->K +
                          4.0 * a->M * nout * (a->accumulate ? 2 : 1) + (a->bias ? 4.0 * a->N : 0.0));
    gpu_next_flops(g, 2.0 * a->M * a->N * a->K);
    char name[32];
    const char *kind = a->A ? "w4" : "fp4", *gl = glu ? "_glu" : "";
    float us = 0;
    const tile_t *t = NULL;
    if (a->A) t = tile_pick(w4_tiles, 4, a->M, nout, (a->K + 63) / 64, glu, &us);
    else if (a->K > 384) t = tile_pick(fp4_tiles, 3, a->M, nout, (a->K + 255) / 256, glu, &us); /* four scales a load */
    /* few rows, 16 output columns to a workgroup: 4-bit rows up to 64 at a time, f32 rows 16 (or 32 columns, where that
     * takes fewer rounds of workgroups; up to five rows share a CU, there from 4096 columns on).  GLU: 16 and their gates */
    const uint32_t G = (a->K + 127) / 128, ti = a->M <= 16 ? 1 : a->M <= 32 ? 2 : 4, rows = a->A ? (a->M + 15) / 16 : 1;
    const uint64_t wg16 = (uint64_t)rows * ((nout + 15) / 16), wg32 = (uint64_t)rows * ((nout + 31) / 32);
    const float one = a->A ? 2.3f + 0.215f * (float)G : 0.75f + (0.08f + 0.05f * (float)ti) * (float)G;
    const float two = 2.6f + 0.26f * (float)G;
    const float few16 = 1.5f + (float)((wg16 + 255) / 256) * (a->A && glu ? two : one);
    const float few32 = 1.8f + (float)((wg32 + 255) / 256) * two;
    const uint32_t wide = a->A && !glu && (a->M <= 5 ? nout > 4096 : few32 < few16), co = wide ? 32 : 16;
    const float few = wide ? few32 : few16;
    if ((a->A ? a->M <= 16 : a->M <= 64 && !t) || ((a->A || a->M <= 64) && few < us)) {
        snprintf(name, sizeof name, "gemm_%s_few%u%s", kind, a->A ? (a->M <= 5 ? 5u : 16u) : 16 * ti, glu ? gl : wide ? "x2" : "");
        return gpu_launch(g, name, a, sizeof *a, (nout + co - 1) / co, rows, 1, 512, 1, 1);
    }
    if (t) {
        const uint64_t tiles = (tiles_of(t, a->M, nout, glu) + 7) / 8 * 8;
        if (tiles * t->threads > 0xffffffffu) return bad(g, "gemm 4-bit: more outputs than a launch covers");
        snprintf(name, sizeof name, "gemm_%s_%s%s", kind, t->name, gl);
        return gpu_launch(g, name, a, sizeof *a, (uint32_t)tiles, 1, 1, t->threads, 1, 1);
    }
    const uint32_t cols = glu ? 32 : 64;
    snprintf(name, sizeof name, "gemm_fp4%s", gl);
    return gpu_launch(g, name, a, sizeof *a, (nout + cols - 1) / cols, (a->M + 63) / 64, 1, 256, 1, 1);
}

int nk_gemm_fp4(gpu_t *g, const uint8_t *Aq, uint32_t lda, const uint8_t *As, uint32_t ldas, const uint8_t *Wq,
                uint32_t ldw, const uint8_t *Ws, uint32_t ldws, const float *bias, float *C, uint32_t ldc, uint32_t M,
                uint32_t N, uint32_t K, int act, int accumulate, float alpha) {
    if (!M) return 0;
    if (!rows_ok(Aq, lda, As, ldas, K) || lda >= FP4_STRIDE || ldas >= FP4_STRIDE)
        return bad(g, "gemm_fp4: row codes 16-byte and scales 4-byte aligned, rows padded to 128 values, strides below 2^24");
    NkGemm4Args a = { NULL, Aq, As, Wq, Ws, bias, C, lda, ldas, ldw, ldws, ldc, M, N, K, (u32)act, accumulate != 0, 0, alpha };
    return product(g, &a);
}

int nk_gemm_w4(gpu_t *g, const float *A, uint32_t lda, const uint8_t *Wq, uint32_t ldw, const uint8_t *Ws,
               uint32_t ldws, const float *bias, float *C, uint32_t ldc, uint32_t M, uint32_t N, uint32_t K, int act,
               int accumulate, float alpha) {
    if (!M) return 0;
    if (!A || !aligned(A, 16) || lda % 4 || lda < K) return bad(g, "gemm_w4: A 16-byte aligned with lda % 4 == 0, K <= lda");
    NkGemm4Args a = { A, NULL, NULL, Wq, Ws, bias, C, lda, 0, ldw, ldws, ldc, M, N, K, (u32)act, accumulate != 0, 0, alpha };
    return product(g, &a);
}
