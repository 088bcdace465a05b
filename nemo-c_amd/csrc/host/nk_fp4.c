/* Launchers of the 4-bit rows and products (include/nemo_kernels.h): arguments are checked before any launch, so
 * a kernel never sees a shape its grid or indexing does not cover. */
#include "nemo_kernels.h"
#include "gpu.h"
#include "../kernel_params.h"
#include <stdio.h>
#include <string.h>

static int bad(gpu_t *g, const char *what) { return gpu_fail(g, what); }
static int aligned(const void *p, uintptr_t n) { return ((uintptr_t)p & (n - 1)) == 0; }
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

/* the checks that both products share, and their launch */
static int product(gpu_t *g, NkGemm4Args *a) {
    const int glu = a->act == NK_ACT_GLU;
    if (a->act > NK_ACT_GLU) return bad(g, "gemm 4-bit: unknown activation");
    if (!a->N || a->N > 1u << 28 || !a->K || a->K > 1u << 30 || (glu && (a->N & 1))) return bad(g, "gemm 4-bit: bad shape");
    if (a->M > 65535 * 64) return bad(g, "gemm 4-bit: too many rows");
    if (!rows_ok(a->Wq, a->ldw, a->Ws, a->ldws, a->K))
        return bad(g, "gemm 4-bit: weight codes 16-byte and scales 4-byte aligned, rows padded to 128 values");
    const uint32_t nout = glu ? a->N / 2 : a->N;
    if (!a->C || !aligned(a->C, 4) || !aligned(a->bias, 4) || a->ldc < nout) return bad(g, "gemm 4-bit: ldc < output width");
    a->vec = aligned(a->C, 16) && a->ldc % 4 == 0;
    gpu_next_bytes(g, 17.0 / 32 * a->N * a->K + (a->A ? 4.0 : 17.0 / 32) * a->M * a->K +
                          4.0 * a->M * nout * (a->accumulate ? 2 : 1) + (a->bias ? 4.0 * a->N : 0.0));
    gpu_next_flops(g, 2.0 * a->M * a->N * a->K);
    const uint32_t cols = glu ? 32 : 64;
    char name[24];
    snprintf(name, sizeof name, "gemm_%s%s", a->A ? "w4" : "fp4", glu ? "_glu" : "");
    return gpu_launch(g, name, a, sizeof *a, (nout + cols - 1) / cols, (a->M + 63) / 64, 1, 256, 1, 1);
}

int nk_gemm_fp4(gpu_t *g, const uint8_t *Aq, uint32_t lda, const uint8_t *As, uint32_t ldas, const uint8_t *Wq,
                uint32_t ldw, const uint8_t *Ws, uint32_t ldws, const float *bias, float *C, uint32_t ldc, uint32_t M,
                uint32_t N, uint32_t K, int act, int accumulate, float alpha) {
    if (!M) return 0;
    if (!rows_ok(Aq, lda, As, ldas, K)) return bad(g, "gemm_fp4: row codes 16-byte and scales 4-byte aligned, rows padded to 128 values");
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
