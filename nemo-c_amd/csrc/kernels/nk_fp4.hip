/* Microscaled 4-bit rows: quantisation, the way back, and the products with 4-bit weights.
 *
 * A block of 32 values shares the power of two 2^(s - 127); the codes are e2m1 (0, 0.5, 1, 1.5, 2, 3, 4,
 * 6 with a sign).  gfx950 converts them (v_cvt_scalef32_*, exact the other way) and multiplies them directly
 * (v_mfma_scale_f32_*_f8f6f4): a lane holds the 32 codes of one block of one row and that block's scale; the 16 x 16
 * form takes 128 values, its four lane groups of 16 the four blocks, the 32 x 32 form 64 in two halves. */
#include "nk_common.h"

typedef int intx8 __attribute__((ext_vector_type(8)));
typedef float floatx16 __attribute__((ext_vector_type(16)));

/* the factor of a scale byte as f32: 2^-127 is subnormal, 255 (a block of NaN) a quiet NaN */
__device__ __forceinline__ float fp4_scale(u32 s) {
    return __uint_as_float(s == 255 ? 0x7fc00000u : s ? s << 23 : 0x00400000u);
}

/* values k .. k + 7 of a row, zeros past its end */
__device__ __forceinline__ void fp4_load8(float (&v)[8], const float *row, u32 k, u32 K, bool vec) {
    if (vec && k + 8 <= K) {
        const floatx4 x = ((const floatx4 *)(row + k))[0], y = ((const floatx4 *)(row + k))[1];
        v[0] = x[0]; v[1] = x[1]; v[2] = x[2]; v[3] = x[3]; v[4] = y[0]; v[5] = y[1]; v[6] = y[2]; v[7] = y[3];
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = k + e < K ? row[k + e] : 0.0f;
    }
}
__device__ __forceinline__ void fp4_load8(float (&v)[8], const u16 *row, u32 k, u32 K, bool vec) {
    if (vec && k + 8 <= K) {
        const uint4 x = *(const uint4 *)(row + k);
        v[0] = bf_lo(x.x); v[1] = bf_hi(x.x); v[2] = bf_lo(x.y); v[3] = bf_hi(x.y);
        v[4] = bf_lo(x.z); v[5] = bf_hi(x.z); v[6] = bf_lo(x.w); v[7] = bf_hi(x.w);
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = k + e < K ? bf2f(row[k + e]) : 0.0f;
    }
}

template <int CTRL> __device__ __forceinline__ u32 quad_u(u32 v) {
    return (u32)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xF, 0xF, false);
}

/* A lane takes 8 values, the four lanes of a quad one block.  The block's largest magnitude is found on
 * the bit patterns (every number < infinity < NaN); its exponent field less 2 is the scale.  Bound by memory:
 * 8192 x 4096 bf16 21 us from HBM (4.0 TB/s). */
template <typename T> __device__ __forceinline__ void fp4_quant_impl(const NkFp4Args &a) {
    const u32 i = blockIdx.x * 256 + threadIdx.x, row = i / a.g8, c = i - row * a.g8;
    if (row >= a.M) return; /* by whole quads: g8 is a multiple of 16 */
    float v[8];
    fp4_load8(v, (const T *)a.X + (u64)row * a.ldx, 8 * c, a.K, a.vec);
    u32 m = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) m = max(m, __float_as_uint(v[e]) & 0x7fffffffu);
    m = max(m, quad_u<DPP_QUAD_1032>(m));
    m = max(m, quad_u<DPP_QUAD_2301>(m));
    const u32 e = m >> 23, s = e == 255 ? 255 : e > 2 ? e - 2 : 0;
    u32 q = 0;
    if (e != 255) {
        const float f = fp4_scale(s); /* the conversion divides by it, rounds to nearest even and saturates */
        q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[0], v[1], f, 0);
        q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[2], v[3], f, 1);
        q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[4], v[5], f, 2);
        q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[6], v[7], f, 3);
    }
    ((u32 *)(a.Q + (u64)row * a.ldq))[c] = q;
    if ((c & 3) == 0) a.S[(u64)row * a.lds + c / 4] = (unsigned char)s;
}
extern "C" __global__ __launch_bounds__(256) void fp4_quant_f32(const NkFp4Args a) { fp4_quant_impl<float>(a); }
extern "C" __global__ __launch_bounds__(256) void fp4_quant_bf16(const NkFp4Args a) { fp4_quant_impl<u16>(a); }

template <int SEL> __device__ __forceinline__ floatx2 fp4_f32(u32 q, float f) {
    return __builtin_bit_cast(floatx2, __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, f, SEL));
}
template <int SEL> __device__ __forceinline__ u32 fp4_bf16(u32 q, float f) {
    return __builtin_bit_cast(u32, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, f, SEL));
}

/* 8 values of a row per lane; 8192 x 4096 to bf16 13.5 us, 6.3 TB/s, the codes coming from the caches */
template <bool BF> __device__ __forceinline__ void fp4_dequant_impl(const NkFp4Args &a) {
    const u32 i = blockIdx.x * 256 + threadIdx.x, row = i / a.g8, k = 8 * (i - row * a.g8);
    if (row >= a.M || k >= a.K) return;
    const u32 q = *(const u32 *)(a.Q + (u64)row * a.ldq + k / 2);
    const float f = fp4_scale(a.S[(u64)row * a.lds + k / 32]);
    if constexpr (BF) {
        u16 *y = (u16 *)a.X + (u64)row * a.ldx + k;
        const u32 p[4] = { fp4_bf16<0>(q, f), fp4_bf16<1>(q, f), fp4_bf16<2>(q, f), fp4_bf16<3>(q, f) };
        if (a.vec && k + 8 <= a.K) *(uint4 *)y = make_uint4(p[0], p[1], p[2], p[3]);
        else
#pragma unroll
            for (u32 e = 0; e < 8; ++e)
                if (k + e < a.K) y[e] = (u16)(p[e / 2] >> (16 * (e & 1)));
    } else {
        float *y = (float *)a.X + (u64)row * a.ldx + k;
        const floatx2 p[4] = { fp4_f32<0>(q, f), fp4_f32<1>(q, f), fp4_f32<2>(q, f), fp4_f32<3>(q, f) };
        if (a.vec && k + 8 <= a.K) {
            ((floatx4 *)y)[0] = (floatx4){ p[0].x, p[0].y, p[1].x, p[1].y };
            ((floatx4 *)y)[1] = (floatx4){ p[2].x, p[2].y, p[3].x, p[3].y };
        } else
#pragma unroll
            for (u32 e = 0; e < 8; ++e)
                if (k + e < a.K) y[e] = p[e / 2][e & 1];
    }
}
extern "C" __global__ __launch_bounds__(256) void fp4_dequant_f32(const NkFp4Args a) { fp4_dequant_impl<false>(a); }
extern "C" __global__ __launch_bounds__(256) void fp4_dequant_bf16(const NkFp4Args a) { fp4_dequant_impl<true>(a); }

/* the bias of columns n .. n + 3 (zeros without one; a column past the end counts as the last) */
__device__ __forceinline__ floatx4 fp4_bias4(const NkGemm4Args &a, u32 n, u32 nout, u32 gate) {
    floatx4 b = { 0.f, 0.f, 0.f, 0.f };
    if (a.bias)
#pragma unroll
        for (int e = 0; e < 4; ++e) b[e] = a.bias[min(n + e, nout - 1) + gate];
    return b;
}
/* what C holds in columns n .. n + 3 of row m where the product is added to it (four at once; fp4_store4 reads the rest
 * itself): loaded for several stores ahead, which wait a memory round trip each otherwise */
__device__ __forceinline__ floatx4 fp4_old4(const NkGemm4Args &a, u32 m, u32 n, u32 nout) {
    if (a.accumulate && a.vec && m < a.M && n + 4 <= nout) return *(const floatx4 *)(a.C + (u64)m * a.ldc + n);
    return (floatx4){ 0.f, 0.f, 0.f, 0.f };
}
/* activation of the sums s (bias added; GLU: t the gates'), alpha, accumulation and store of columns n .. n + 3 of
 * row m; old from fp4_old4 */
template <bool GLU>
__device__ __forceinline__ void fp4_store4(const NkGemm4Args &a, u32 m, u32 n, u32 nout, floatx4 s, floatx4 t, floatx4 old) {
    if (GLU)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[e] *= sigmoid_f(t[e]);
    else if (a.act == NK_ACT_SILU)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[e] = silu_f(s[e]);
    else if (a.act == NK_ACT_RELU)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[e] = relu_nan(s[e]);
    if (m >= a.M || n >= nout) return;
    float *c = a.C + (u64)m * a.ldc + n;
    if (a.vec && n + 4 <= nout) {
        const floatx4 v = s * a.alpha;
        *(floatx4 *)c = a.accumulate ? old + v : v;
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (n + e < nout) c[e] = a.accumulate ? c[e] + s[e] * a.alpha : s[e] * a.alpha;
    }
}
/* A wavefront's TI x TJ tiles from row m0 and the columns col[j] on (GLU: the second half of the tiles are gates):
 * the lane holds row m0 + 16 i + lane % 16, columns col[j] + 4 (lane / 16) .. + 3 */
template <bool GLU, int TI, int TJ>
__device__ __forceinline__ void fp4_epilogue(const NkGemm4Args &a, u32 m0, const u32 (&col)[TJ], const floatx4 (&acc)[TI][TJ]) {
    const u32 lane = threadIdx.x & 63, m = m0 + (lane & 15), nout = GLU ? a.N / 2 : a.N;
    constexpr int TO = GLU ? TJ / 2 : TJ;
    floatx4 b[TJ];
#pragma unroll
    for (int j = 0; j < TJ; ++j) b[j] = fp4_bias4(a, col[j % TO] + 4 * (lane >> 4), nout, j < TO ? 0 : nout);
#pragma unroll
    for (int i = 0; i < TI; ++i)
#pragma unroll
        for (int j = 0; j < TO; ++j)
            fp4_store4<GLU>(a, m + 16 * i, col[j] + 4 * (lane >> 4), nout, acc[i][j] + b[j], acc[i][j + (GLU ? TO : 0)] + b[j + (GLU ? TO : 0)],
                            fp4_old4(a, m + 16 * i, col[j] + 4 * (lane >> 4), nout));
}

__device__ __forceinline__ intx8 fp4_op(uint4 q) {
    return (intx8){ (int)q.x, (int)q.y, (int)q.z, (int)q.w, 0, 0, 0, 0 };
}
/* acc += W A^T of 16 weight rows and 16 rows over 128 values; the scales are in the low bytes */
__device__ __forceinline__ floatx4 fp4_mfma(uint4 w, u32 ws, uint4 x, u32 xs, floatx4 acc) {
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(fp4_op(w), fp4_op(x), acc, 4, 4, 0, (int)ws, 0, (int)xs);
}

/* Rows of at most 384 values, which the tiles below do not take (their loads of scales are four groups long): a
 * wavefront computes 32 rows by 32 columns (GLU: 16 value and 16 gate columns) with every fragment straight from
 * global memory; rows past the end repeat the last one and are not stored.  Little but outputs: 3584 x 4096 x 384
 * 27 us, where a copy's rate would write them in 12. */
template <bool GLU> __device__ __forceinline__ void gemm_fp4_impl(const NkGemm4Args &a) {
    const u32 lane = threadIdx.x & 63, wv = threadIdx.x >> 6, r = lane & 15, f = lane >> 4;
    const u32 nout = GLU ? a.N / 2 : a.N, G = (a.K + 127) / 128;
    const u32 m0 = blockIdx.y * 64 + (wv & 1) * 32, n0 = (blockIdx.x * 2 + (wv >> 1)) * (GLU ? 16 : 32);
    const unsigned char *w[2], *ws[2], *x[2], *xs[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const u32 n = GLU ? min(n0 + r, nout - 1) + j * nout : min(n0 + 16 * j + r, nout - 1);
        w[j] = a.Wq + (u64)n * a.ldw + 16 * f;
        ws[j] = a.Ws + (u64)n * a.ldws + f;
        const u32 m = min(m0 + 16 * j + r, a.M - 1);
        x[j] = a.Aq + (u64)m * a.lda + 16 * f;
        xs[j] = a.As + (u64)m * a.ldas + f;
    }
    floatx4 acc[2][2] = {};
    for (u32 g = 0; g < G; ++g) {
        uint4 wq[2], xq[2];
        u32 we[2], xe[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            wq[j] = *(const uint4 *)(w[j] + 64 * (u64)g);
            xq[j] = *(const uint4 *)(x[j] + 64 * (u64)g);
            we[j] = ws[j][4 * (u64)g];
            xe[j] = xs[j][4 * (u64)g];
        }
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j) acc[i][j] = fp4_mfma(wq[j], we[j], xq[i], xe[i], acc[i][j]);
    }
    const u32 col[2] = { n0, n0 + (GLU ? 0 : 16) };
    fp4_epilogue<GLU, 2, 2>(a, m0, col, acc);
}
extern "C" __global__ __launch_bounds__(256) void gemm_fp4(const NkGemm4Args a) { gemm_fp4_impl<false>(a); }
extern "C" __global__ __launch_bounds__(256) void gemm_fp4_glu(const NkGemm4Args a) { gemm_fp4_impl<true>(a); }

/* 16 bytes per lane from global memory at base + off into LDS bytes [lds + 16 i, +16), as dma16 */
__device__ __forceinline__ void dma16_at(const unsigned char *base, u32 off, lds_char_t *lds) {
    const u32 m = __builtin_amdgcn_readfirstlane((u32)(size_t)lds);
    asm volatile("s_mov_b32 m0, %2\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(off), "s"(base), "s"(m) : "memory");
}
/* and 4 bytes per lane into [lds + 4 i, +4) */
__device__ __forceinline__ void dma4_at(const unsigned char *base, u32 off, lds_char_t *lds) {
    const u32 m = __builtin_amdgcn_readfirstlane((u32)(size_t)lds);
    asm volatile("s_mov_b32 m0, %2\n\tglobal_load_lds_dword %0, %1" ::"v"(off), "s"(base), "s"(m) : "memory");
}
__device__ __forceinline__ const unsigned char *uniform_ptr(const unsigned char *p) {
    const u32 lo = __builtin_amdgcn_readfirstlane((u32)(u64)p), hi = __builtin_amdgcn_readfirstlane((u32)((u64)p >> 32));
    return (const unsigned char *)((u64)hi << 32 | lo);
}

/* the same of 32 weight rows and 32 rows over 64 values: lane l holds the 32 codes of block l / 32 of row l % 32; the
 * scales are in bytes B */
template <int B> __device__ __forceinline__ floatx16 fp4_mfma32(uint4 w, u32 ws, uint4 x, u32 xs, floatx16 acc) {
    return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(fp4_op(w), fp4_op(x), acc, 4, 4, B, (int)ws, B, (int)xs);
}
template <int V> struct const_t { static constexpr int v = V; };

/* A wavefront's 32 x 32 tiles from row m0 and column c0 on (GLU: the second half of the tiles are gates): lane l holds row
 * 32 i + l % 32, columns 32 j + 8 q + 4 (l / 32) .. + 3 in its elements 4 q .. */
template <bool GLU, int TI, int TJ>
__device__ __forceinline__ void tile_out(const NkGemm4Args &a, u32 m0, u32 c0, const floatx16 (&acc)[TI][TJ]) {
    constexpr int TO = GLU ? TJ / 2 : TJ;
    const u32 r = threadIdx.x & 31, f = threadIdx.x >> 5 & 1, nout = GLU ? a.N / 2 : a.N;
#pragma unroll
    for (int h = 0; h < 2 * TO; ++h) { /* half a tile at a time: more is spilled */
        const u32 n = c0 + 16 * h + 4 * f;
        floatx4 old[2][TI], b[2], d[2];
#pragma unroll
        for (int q = 0; q < 2; ++q) {
#pragma unroll
            for (int i = 0; i < TI; ++i) old[q][i] = fp4_old4(a, m0 + 32 * i + r, n + 8 * q, nout);
            b[q] = fp4_bias4(a, n + 8 * q, nout, 0);
            d[q] = GLU ? fp4_bias4(a, n + 8 * q, nout, nout) : b[q];
        }
#pragma unroll
        for (int q = 0; q < 2; ++q)
#pragma unroll
            for (int i = 0; i < TI; ++i) {
                const int at = 8 * (h & 1) + 4 * q;
                floatx4 v, t;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    v[e] = acc[i][h / 2][at + e] + b[q][e];
                    t[e] = acc[i][h / 2 + (GLU ? TO : 0)][at + e] + d[q][e];
                }
                fp4_store4<GLU>(a, m0 + 32 * i + r, n + 8 * q, nout, v, t, old[q][i]);
            }
        __builtin_amdgcn_sched_barrier(0);
    }
}

/* The product by tiles of BM x BN outputs (K > 384), WGM x WGN wavefronts with (BM / WGM) x (BN / WGN) each and PW that
 * only load (a wavefront that issues a direct load is held for 70 to 120 cycles), on the 32 x 32 MFMA: from registers
 * it reaches 9.2 PFLOP/s (7.1 on random codes), the 16 x 16 one 4.8.
 *
 * A K step is 256 values, four MFMA groups: whole 128-byte lines of every row.  A ring of NS stages in LDS is filled
 * by direct loads.  A load takes 8 rows, 8 lanes a row (with the rows side by side over the lanes each lane is a line of
 * its own: 139 us for 3584 x 4096 x 8192 on 128 x 128 tiles where this took 88); granule g of row r lies in slot
 * g ^ (r / 2 % 8), so a fragment read (one granule of 32 rows per half of the wavefront) is free of bank conflicts.
 * Scales come by 16 bytes of a row for two steps, and are read by 8 for one (a byte per fragment: 88 us, 74 with
 * no scales at all; by two times 4, as groups at odd places would need: 5% more).  Those of an odd last group come by
 * themselves, 4 bytes of a row.
 *
 * Bound by the loads from L2 at many rows: 2048 x 4096 x 8192 38.4 us (3.6 PFLOP/s; its products alone 15, with the
 * fragment reads 29), 3584 x 4096 x 8192 74 to 80; tiles of 128 x 128, 256 x 128 and 256 x 256 in other splits over
 * wavefronts took 80 to 110. */
template <int BM, int BN, int WGM, int WGN, int PW, int NS, bool GLU>
__device__ __forceinline__ void gemm_fp4_tile(const NkGemm4Args &a, lds_char_t *const smem) {
    constexpr int NW = PW, WTM = BM / WGM, WTN = BN / WGN, TI = WTM / 32, TJ = WTN / 32;
    constexpr int NC = NS / 2 + 1;                     /* chunks of scales: a stage's and those ahead of it */
    constexpr u32 ROWS = BM + BN, STAGE = ROWS * 128, SCALES = NS * STAGE, CHUNK = ROWS * 16, LAST = SCALES + NC * CHUNK;
    constexpr int LI = ROWS / 8 / NW;                  /* loads of codes per wavefront and stage */
    constexpr int LS = (ROWS / 64 + NW - 1) / NW;      /* loads of scales, of 64 rows of one operand (the last may repeat one) */
    static_assert(LI * NW * 8 == ROWS && BM % 64 == 0 && (GLU ? BN / 2 : BN) % 64 == 0 && NS >= 2 && (NS - 1) * (LI + LS) + LS < 64, "tile shape");
    const u32 tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const bool loader = wave >= WGM * WGN;
    const u32 wv = loader ? wave - WGM * WGN : wave, wm = wv / WGN, wn = wv % WGN, r = lane & 31, f = lane >> 5;
    const u32 nout = GLU ? a.N / 2 : a.N, G = (a.K + 127) / 128, S = (G + 1) / 2;
    const u32 even = (G - 4) & ~1u; /* the last group that a load of four groups' scales begins at: reads of 8 are aligned */
    constexpr u32 CO = GLU ? BN / 2 : BN; /* output columns of a tile */
    const u32 tm = (a.M + BM - 1) / BM, tn = (nout + CO - 1) / CO;
    /* workgroup b runs on XCD b % 8: each XCD takes a run of tiles, by groups of 8 row tiles */
    const u32 per = gridDim.x / 8, t = (blockIdx.x % 8) * per + blockIdx.x / 8;
    if (t >= tm * tn) return;
    const u32 grp = t / (8 * tn), in = t - grp * 8 * tn, gh = min(tm - grp * 8, 8u);
    const u32 m0 = (grp * 8 + in % gh) * BM, c0 = in / gh * CO;

    /* At the barrier of step q the loaders have stage q behind them and the others their reads of stage q - 1: the
     * latter's place takes stage q + NS - 1. */
    if (loader) {
        /* Sources as a uniform base and a lane's offset in the load (strides are below 2^24 bytes).  The rows of a load
         * are of one operand; GLU: the second half of the tile's weight rows are the gates'.  Rows past the end repeat
         * the last. */
        const unsigned char *base[LI], *sbase[LS];
        u32 last[LI], ld[LI], slast[LS], sld[LS]; /* uniform: the last row behind the base, the stride */
        auto place = [&](u32 q, bool scales, const unsigned char *&b, u32 &end, u32 &stride) {
            /* q: first row of the load in the stage */
            const u32 lda = scales ? a.ldas : a.lda, ldw = scales ? a.ldws : a.ldw;
            if (q < BM) {
                const u32 m = min(m0 + q, a.M - 1);
                b = uniform_ptr((scales ? a.As : a.Aq) + (u64)m * lda);
                end = a.M - 1 - m;
                stride = lda;
            } else {
                const u32 n = q - BM, gate = GLU && n >= CO, c = min(c0 + n - (gate ? CO : 0), nout - 1);
                b = uniform_ptr((scales ? a.Ws : a.Wq) + (u64)(c + (gate ? nout : 0)) * ldw);
                end = nout - 1 - c;
                stride = ldw;
            }
        };
#pragma unroll
        for (int j = 0; j < LI; ++j) place((NW * j + wv) * 8, false, base[j], last[j], ld[j]);
#pragma unroll
        for (int j = 0; j < LS; ++j) place((NW * j + wv) % (ROWS / 64) * 64, true, sbase[j], slast[j], sld[j]);
        static_assert(NW % 2 == 0, "the swizzle of a wavefront's loads is the same");
        const u32 row = lane >> 3, gran = (lane & 7) ^ swz_h(wv * 8 + row);
        u32 slot = 0, chunk = 0; /* places of the stage and of the scales that are loaded next */
        auto issue = [&](u32 q) {
            const u32 g = ((G & 1) && q + 1 == S ? gran & 3 : gran) * 16; /* the last lines may have no second half */
#pragma unroll
            for (int j = 0; j < LI; ++j) {
                dma16_at(base[j], __umul24(min(row, last[j]), ld[j]) + g, smem + slot + (NW * j + wv) * 1024);
                base[j] += 128;
            }
            slot = slot + STAGE == NS * STAGE ? 0 : slot + STAGE;
            if ((G & 1) && q + 1 == S)
#pragma unroll
                for (int j = 0; j < LS; ++j)
                    dma4_at(sbase[j] + 4 * (G - 1), __umul24(min(lane, slast[j]), sld[j]), smem + LAST + (NW * j + wv) % (ROWS / 64) * 256);
            if (q & 1) return;
#pragma unroll
            for (int j = 0; j < LS; ++j) /* groups 2 q .. 2 q + 3 of 128, or the row's last four */
                dma16_at(sbase[j] + 4 * min(2 * q, even), __umul24(min(lane, slast[j]), sld[j]),
                         smem + SCALES + chunk * CHUNK + (NW * j + wv) % (ROWS / 64) * 1024);
            chunk = chunk + 1 == NC ? 0 : chunk + 1;
        };
        for (u32 u = 0; u < min(S, (u32)NS - 1); ++u) issue(u);
        for (u32 q = 0; q < S; ++q) {
            wait_steps<NS - 2, LI>(min(S, q + NS - 1) - q - 1);
            barrier_mem();
            if (q + NS - 1 < S) issue(q + NS - 1);
        }
        return;
    }
    typedef const __attribute__((address_space(3))) uint4 *lds4;
    typedef const __attribute__((address_space(3))) uint2 *lds2;
    typedef const __attribute__((address_space(3))) u32 *lds1;
    uint4 x[TI], w[TJ];
    uint2 xs[TI], ws[TJ]; /* a step's eight scales of the lane's row, its own in bytes 0 and 2 of each half */
    /* the lane's places in a stage, the tiles' at constant distances: codes and scales of A, and of W */
    const u32 n0 = GLU ? wn * WTN / 2 : wn * WTN, sw = swz_h(r);
    u32 lo[4]; /* granule 2 h + f of row r */
#pragma unroll
    for (u32 h = 0; h < 4; ++h) lo[h] = r * 128 + ((2 * h + f) ^ sw) * 16;
    const u32 ox = wm * WTM * 128, oxs = (wm * WTM + r) * 16, ow = (BM + n0) * 128, ows = (BM + n0 + r) * 16;
    auto scales = [&](const lds_char_t *p) {
        const uint2 v = *(lds2)p;
        return make_uint2(v.x >> (8 * f), v.y >> (8 * f));
    };
    /* GLU: the first half of a wavefront's tiles are value columns, the second their gates */
    auto wcol = [](int j) { return (u32)(GLU && j >= TJ / 2 ? BN / 2 + 32 * (j - TJ / 2) : 32 * j); };
    auto read_w = [&](const lds_char_t *p, const lds_char_t *ps, bool fresh) {
#pragma unroll
        for (int j = 0; j < TJ; ++j) {
            w[j] = *(lds4)(p + wcol(j) * 128);
            if (fresh) ws[j] = scales(ps + wcol(j) * 16);
        }
    };
    auto read_x = [&](int i, const lds_char_t *p, const lds_char_t *ps, bool fresh) {
        x[i] = *(lds4)(p + i * 4096);
        if (fresh) xs[i] = scales(ps + i * 512);
    };
    floatx16 acc[TI][TJ] = {};
    auto mma = [&](int i, auto group) {
        constexpr int H = decltype(group)::v;
#pragma unroll
        for (int j = 0; j < TJ; ++j)
            acc[i][j] = fp4_mfma32<2 * (H & 1)>(w[j], H < 2 ? ws[j].x : ws[j].y, x[i], H < 2 ? xs[i].x : xs[i].y, acc[i][j]);
    };
    const lds_char_t *st, *ss; /* codes and scales of the stage entered last */
    /* the products of the group before the stage's group H, each row tile's fragment replaced by that group's as soon
     * as it is used, the weights' behind them */
    auto group = [&](auto next, bool whole = true) {
        constexpr int H = decltype(next)::v;
        const lds_char_t *p = st + ox + lo[H], *ps = ss + oxs;
#pragma unroll
        for (int i = 0; i < TI; ++i) {
            mma(i, const_t<(H + 3) % 4>());
            __builtin_amdgcn_sched_barrier(0); /* else the reads move up, into registers that are not there */
            read_x(i, p, ps, H == 0);
            if (!whole) x[i] = make_uint4(0, 0, 0, 0);
        }
        read_w(st + ow + lo[H], ss + ows, H == 0);
    };
    auto rest = [&] {
        group(const_t<1>());
        group(const_t<2>());
        group(const_t<3>());
    };
    u32 cur = 0, chunk = 0;
    auto enter = [&](u32 q) {
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        barrier_mem();
        st = smem + cur;
        ss = smem + SCALES + chunk * CHUNK + min(4 * (2 * q - min(2 * (q & ~1u), even)), 8u); /* an odd last group's: not used */
        cur = cur + STAGE == NS * STAGE ? 0 : cur + STAGE;
        chunk = !(q & 1) ? chunk : chunk + 1 == NC ? 0 : chunk + 1;
    };
    enter(0);
    read_w(st + ow + lo[0], ss + ows, true);
#pragma unroll
    for (int i = 0; i < TI; ++i) read_x(i, st + ox + lo[0], ss + oxs, true);
    for (u32 q = 1; q < S; ++q) {
        rest();
        enter(q);
        group(const_t<0>());
    }
    /* the last step, whose second half may not exist: zeros then, under scales of one */
    const bool whole = !(G & 1);
    if (!whole) {
        auto one = [&](u32 row) { return make_uint2(*(lds1)(smem + LAST + row * 4) >> (8 * f), 0x007f007f); };
#pragma unroll
        for (int j = 0; j < TJ; ++j) ws[j] = one(BM + n0 + r + wcol(j));
#pragma unroll
        for (int i = 0; i < TI; ++i) xs[i] = one(wm * WTM + r + 32 * i);
    }
    group(const_t<1>());
    group(const_t<2>(), whole);
    group(const_t<3>(), whole);
#pragma unroll
    for (int i = 0; i < TI; ++i) mma(i, const_t<3>());
    tile_out<GLU, TI, TJ>(a, m0 + wm * WTM, c0 + n0, acc);
}
#define FP4_TILE(BM, BN, WGM, WGN, PW, NS, GLU, NAME)                                                          \
    extern "C" __global__ __launch_bounds__(64 * (WGM * WGN + PW)) void gemm_fp4_##NAME(const NkGemm4Args a) { \
        __shared__ __attribute__((aligned(1024))) char smem[(BM + BN) * (NS * 128 + (NS / 2 + 1) * 16 + 4)];    \
        gemm_fp4_tile<BM, BN, WGM, WGN, PW, NS, GLU>(a, (lds_char_t *)smem);                                    \
    }
FP4_TILE(128, 256, 2, 4, 4, 3, false, 128x256)
FP4_TILE(128, 256, 2, 4, 4, 3, true, 128x256_glu)
FP4_TILE(64, 128, 2, 2, 4, 3, false, 64x128)
FP4_TILE(64, 128, 2, 2, 4, 3, true, 64x128_glu)
FP4_TILE(64, 64, 2, 2, 4, 3, false, 64x64)

/* Two f32 values as three bf16 terms each, packed: the upper 16 bits of what is left, so that the terms add up to all 24
 * significant bits (what is below 2^-133, the least bf16, is dropped).  FINITE: neither is an infinity or NaN.  Else of an
 * infinity the first term is infinite and the others are zero: anything else times large weights could pass the type's
 * range with the other sign.  What is left of a NaN is a quiet NaN, also where its mark is in the lower half alone. */
template <bool FINITE> __device__ __forceinline__ void split3(float a, float b, u32 (&t)[3]) {
    if (!FINITE) asm("" : "+v"(a), "+v"(b)); /* else what both have in common moves ahead of the question, into registers */
    const bool ia = !FINITE && __builtin_isinf(a), ib = !FINITE && __builtin_isinf(b);
#pragma unroll
    for (int k = 0; k < 3; ++k) {
        t[k] = __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302);
        a -= __uint_as_float(__float_as_uint(a) & 0xffff0000u);
        b -= __uint_as_float(__float_as_uint(b) & 0xffff0000u);
        if (k == 0) {
            a = ia ? 0.0f : a;
            b = ib ? 0.0f : b;
        }
    }
}
/* Calls split(finite) for the values x[0 .. n - 1] of the wavefront's lanes, finite saying whether all are: half an
 * instruction a value to ask, where the care for the others takes two (448 x 1024 x 4096 on tiles of 32 x 64: 33.7 us, 35.5
 * with care in every split).  ASK: without the question, for the few values of up to five rows (8192 x 2048 of one
 * row 5.6 us, 5.7 with it). */
template <bool ASK, int N, typename F> __device__ __forceinline__ void split_rows(const floatx4 (&x)[N], u32 n, F split) {
    if constexpr (ASK) {
        float top = 0.0f; /* the maximum that NaN wins */
#pragma unroll
        for (int l = 0; l < N; ++l) {
            if ((u32)l >= n) break;
            top = __builtin_elementwise_maximum(__builtin_elementwise_maximum(top, fabsf(x[l][0])), fabsf(x[l][1]));
            top = __builtin_elementwise_maximum(__builtin_elementwise_maximum(top, fabsf(x[l][2])), fabsf(x[l][3]));
        }
        if (!__builtin_amdgcn_ballot_w64(!(top < __builtin_inff()))) return split(const_t<1>());
    }
    split(const_t<0>());
}
/* 8 codes as bf16 values, exact */
__device__ __forceinline__ uint4 fp4_bf16x8(u32 q, float f) {
    return make_uint4(fp4_bf16<0>(q, f), fp4_bf16<1>(q, f), fp4_bf16<2>(q, f), fp4_bf16<3>(q, f));
}

#define FEW_WAVES 8
/* The sums of a workgroup's wavefronts, added in their order, and the epilogue.  TERMS 3: the rows 5 k + m of a tile are
 * the k-th terms of row m. */
template <int TI, int TJ, bool GLU, int TERMS>
__device__ __forceinline__ void few_out(const NkGemm4Args &a, floatx4 (*part)[TI * TJ][64], u32 n0, const floatx4 (&acc)[TI][TJ]) {
    constexpr int TO = GLU ? TJ / 2 : TJ;
    const u32 lane = threadIdx.x & 63, wv = threadIdx.x >> 6, r = lane & 15, f = lane >> 4, nout = GLU ? a.N / 2 : a.N;
#pragma unroll
    for (int i = 0; i < TI; ++i)
#pragma unroll
        for (int j = 0; j < TJ; ++j) part[wv][i * TJ + j][lane] = acc[i][j];
    __syncthreads();
    for (u32 t = wv; t < TI * TO; t += FEW_WAVES) {
        const u32 i = t / TO, j = t % TO, n = n0 + 16 * j + 4 * f;
        const floatx4 old = fp4_old4(a, 16 * i + r, n, nout);
        auto sum = [&](u32 tile) {
            floatx4 s = { 0.f, 0.f, 0.f, 0.f };
#pragma unroll
            for (int k = 0; k < TERMS; ++k)
#pragma unroll
                for (int v = 0; v < FEW_WAVES; ++v) s += part[v][tile][TERMS == 1 ? lane : 16 * f + min(r, 5u) + 5 * k];
            return s;
        };
        const floatx4 s = sum(i * TJ + j), d = GLU ? sum(i * TJ + j + TO) : s;
        fp4_store4<GLU>(a, 16 * i + r, n, nout, s + fp4_bias4(a, n, nout, 0), GLU ? d + fp4_bias4(a, n, nout, nout) : s, old);
    }
}

/* Few rows: the weights are streamed once and everything else is small.  A workgroup takes 16 TO output columns; its
 * wavefronts take every eighth group of 128 values each, fragments straight from global memory into registers,
 * and their sums meet in LDS.  Lane l of a fragment holds the 32 codes of block l / 16 of row l % 16.  Bound by the
 * weights' round trip: 4096 x 1024 of 16 rows 4.0 us. */
template <int TI, int TJ, bool GLU> __device__ __forceinline__ void fp4_few(const NkGemm4Args &a) {
    constexpr int TO = GLU ? TJ / 2 : TJ;
    __shared__ floatx4 part[FEW_WAVES][TI * TJ][64];
    const u32 lane = threadIdx.x & 63, wv = threadIdx.x >> 6, r = lane & 15, f = lane >> 4;
    const u32 nout = GLU ? a.N / 2 : a.N, G = (a.K + 127) / 128, n0 = blockIdx.x * 16 * TO;
    const unsigned char *w[TJ], *ws[TJ], *x[TI], *xs[TI];
#pragma unroll
    for (int j = 0; j < TJ; ++j) {
        const u32 n = min(n0 + 16 * (j % TO) + r, nout - 1) + (j < TO ? 0 : nout);
        w[j] = a.Wq + (u64)n * a.ldw + 16 * f;
        ws[j] = a.Ws + (u64)n * a.ldws + f;
    }
#pragma unroll
    for (int i = 0; i < TI; ++i) {
        const u32 m = min(16 * i + r, a.M - 1);
        x[i] = a.Aq + (u64)m * a.lda + 16 * f;
        xs[i] = a.As + (u64)m * a.ldas + f;
    }
    floatx4 acc[TI][TJ] = {};
    constexpr int U = 2; /* groups in flight (the last again past the end, not used) */
    for (u32 g0 = wv; g0 < G; g0 += U * FEW_WAVES) {
        uint4 wq[U][TJ], xq[U][TI];
        u32 we[U][TJ], xe[U][TI];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const u32 g = min(g0 + u * FEW_WAVES, G - 1);
#pragma unroll
            for (int j = 0; j < TJ; ++j) {
                wq[u][j] = *(const uint4 *)(w[j] + 64 * (u64)g);
                we[u][j] = ws[j][4 * (u64)g];
            }
#pragma unroll
            for (int i = 0; i < TI; ++i) {
                xq[u][i] = *(const uint4 *)(x[i] + 64 * (u64)g);
                xe[u][i] = xs[i][4 * (u64)g];
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (u && g0 + u * FEW_WAVES >= G) break;
#pragma unroll
            for (int i = 0; i < TI; ++i)
#pragma unroll
                for (int j = 0; j < TJ; ++j) acc[i][j] = fp4_mfma(wq[u][j], we[u][j], xq[u][i], xe[u][i], acc[i][j]);
        }
    }
    few_out<TI, TJ, GLU, 1>(a, part, n0, acc);
}

/* The same with f32 rows, as three bf16 terms against the weights' values in bf16: MFMA s of a group of 128 takes every
 * block's eighth s, the K order being the same on both sides.  The rows of a group are read whole (32 lanes a
 * row), split, and put into the wavefront's part of LDS as fragments (read as fragments from global memory each lane is a
 * line of its own, and all 16 rows of a fragment are split: 8192 x 2048 of one row 6.2 us against 5.6; 5 rows now
 * take 6.2 us and 16 rows 8.6).
 * PACK: at most five rows, whose terms lie in rows m, 5 + m and 10 + m of one fragment.  Otherwise 16 rows a workgroup, two
 * column tiles where that saves a round of workgroups (32 x 4096 x 4096 13 us, 19.6 with one; 32 rows a workgroup on four
 * wavefronts 25). */
template <int TJ, bool GLU, bool PACK> __device__ __forceinline__ void w4_few(NkGemm4Args a) {
    if (!PACK) { /* 16 rows a workgroup */
        a.A += (u64)blockIdx.y * 16 * a.lda;
        a.C += (u64)blockIdx.y * 16 * a.ldc;
        a.M -= blockIdx.y * 16;
    }
    constexpr int TO = GLU ? TJ / 2 : TJ, T = PACK ? 1 : 3, RL = PACK ? 3 : 8; /* fragments; loads of two rows */
    constexpr u32 ROWS = FEW_WAVES * T * 4096, PART = FEW_WAVES * TJ * 1024;
    __shared__ __attribute__((aligned(16))) char mem[ROWS > PART ? ROWS : PART];
    const u32 lane = threadIdx.x & 63, wv = threadIdx.x >> 6, r = lane & 15, f = lane >> 4;
    const u32 nout = GLU ? a.N / 2 : a.N, G = (a.K + 127) / 128, n0 = blockIdx.x * 16 * TO;
    char *frag = mem + wv * T * 4096; /* granule g (8 values) of row r in slot g ^ r */
    const unsigned char *w[TJ], *ws[TJ];
#pragma unroll
    for (int j = 0; j < TJ; ++j) {
        const u32 n = min(n0 + 16 * (j % TO) + r, nout - 1) + (j < TO ? 0 : nout);
        w[j] = a.Wq + (u64)n * a.ldw + 16 * f;
        ws[j] = a.Ws + (u64)n * a.ldws + f;
    }
    uint4 wq[TJ];
    u32 we[TJ];
    floatx4 x[RL];
    const u32 i4 = lane & 31, half = lane >> 5;
    auto load = [&](u32 g) { /* a group; rows past the end repeat the last, their products are not stored */
#pragma unroll
        for (int j = 0; j < TJ; ++j) {
            wq[j] = *(const uint4 *)(w[j] + 64 * (u64)g);
            we[j] = ws[j][4 * (u64)g];
        }
        const u32 k = 128 * g + 4 * i4;
#pragma unroll
        for (int l = 0; l < RL; ++l) {
            if (2 * (u32)l >= a.M) break;
            const float *row = a.A + (u64)min(2 * l + half, a.M - 1) * a.lda;
            if (k + 4 <= a.K) x[l] = *(const floatx4 *)(row + k);
            else
#pragma unroll
                for (int e = 0; e < 4; ++e) x[l][e] = k + e < a.K ? row[k + e] : 0.0f;
        }
    };
    if (wv < G) load(wv);
    /* rows that no load writes: zeros (their products are not stored, or belong to no row) */
    for (u32 o = lane * 16; o < T * 4096; o += 1024) *(uint4 *)(frag + o) = make_uint4(0, 0, 0, 0);
    floatx4 acc[1][TJ] = {};
    for (u32 g = wv; g < G; g += FEW_WAVES) {
        __builtin_amdgcn_wave_barrier();
        split_rows<!PACK>(x, (a.M + 1) / 2, [&](auto finite) {
#pragma unroll
            for (int l = 0; l < RL; ++l) {
                if (2 * (u32)l >= a.M) break;
                u32 p[3], q[3];
                split3<decltype(finite)::v>(x[l][0], x[l][1], p);
                split3<decltype(finite)::v>(x[l][2], x[l][3], q);
                const u32 m = 2 * l + half;
#pragma unroll
                for (int k = 0; k < 3; ++k) {
                    const u32 row = PACK ? min(m, 5u) + 5 * k : m; /* PACK: row 5 of a load overwrites nothing it should not */
                    if (!PACK || m < 5) *(uint2 *)(frag + (PACK ? 0 : k * 4096) + row * 256 + ((i4 / 2) ^ row) * 16 + (i4 & 1) * 8) = make_uint2(p[k], q[k]);
                }
            }
        });
        uint4 b[TJ];
        u32 q[TJ][4];
        float s[TJ];
#pragma unroll
        for (int j = 0; j < TJ; ++j) {
            q[j][0] = wq[j].x; q[j][1] = wq[j].y; q[j][2] = wq[j].z; q[j][3] = wq[j].w;
            s[j] = fp4_scale(we[j]);
        }
        if (g + FEW_WAVES < G) load(g + FEW_WAVES);
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int e = 0; e < 4; ++e) {
#pragma unroll
            for (int j = 0; j < TJ; ++j) b[j] = fp4_bf16x8(q[j][e], s[j]);
#pragma unroll
            for (int k = 0; k < T; ++k) {
                const uint4 v = *(const uint4 *)(frag + k * 4096 + r * 256 + ((4 * f + e) ^ r) * 16);
#pragma unroll
                for (int j = 0; j < TJ; ++j) acc[0][j] = mfma_bf16(b[j], v, acc[0][j]);
            }
        }
    }
    __syncthreads(); /* the sums take the fragments' place */
    few_out<1, TJ, GLU, PACK ? 3 : 1>(a, (floatx4(*)[TJ][64])mem, n0, acc);
}
#define FP4_FEW(NAME, TI, TJ, GLU) \
    extern "C" __global__ __launch_bounds__(64 * FEW_WAVES) void gemm_fp4_##NAME(const NkGemm4Args a) { fp4_few<TI, TJ, GLU>(a); }
#define W4_FEW(NAME, TJ, GLU, PACK) \
    extern "C" __global__ __launch_bounds__(64 * FEW_WAVES) void gemm_w4_##NAME(const NkGemm4Args a) { w4_few<TJ, GLU, PACK>(a); }
FP4_FEW(few16, 1, 1, false) FP4_FEW(few16_glu, 1, 2, true)
FP4_FEW(few32, 2, 1, false) FP4_FEW(few32_glu, 2, 2, true)
FP4_FEW(few64, 4, 1, false) FP4_FEW(few64_glu, 4, 2, true)
W4_FEW(few5, 1, false, true) W4_FEW(few5x2, 2, false, true) W4_FEW(few5_glu, 2, true, true)
W4_FEW(few16, 1, false, false) W4_FEW(few16x2, 2, false, false) W4_FEW(few16_glu, 2, true, false)

/* f32 rows and 4-bit weights by tiles, K steps of 64 values, on the 32 x 32 x 16 bf16 MFMA (2.2 PFLOP/s from
 * registers, the 16 x 16 one 1.3).  PW wavefronts load: f32 rows come into registers two steps ahead, are split once into
 * three bf16 planes (24 bits, every product of a term and a weight exact) and put into one of two LDS stages with
 * the weights' codes and scales, while the others multiply the stage before.  Lane l of a weight fragment holds the 32
 * codes of block l / 32 of row l % 32, converted in registers; MFMA s of a step takes every block's eighth s, of A
 * too.  1024 x 4096 x 2048 49 us, 2048 x 4096 x 8192 331 us: 1.05 and 1.24 PFLOP/s in the three products, where a
 * library product of 8192 cubed in bf16 reaches 1.20. */
template <int BM, int BN, int WGM, int WGN, int PW, int AHEAD, bool GLU>
__device__ __forceinline__ void gemm_w4_tile(const NkGemm4Args &a, char *const smem) {
    constexpr int WTM = BM / WGM, WTN = BN / WGN, TI = WTM / 32, TJ = WTN / 32;
    constexpr u32 PLANE = BM * 128, CODES = 3 * PLANE, SCALES = CODES + BN * 32, STAGE = SCALES + BN * 4;
    constexpr int LA = BM * 16 / (PW * 64), LW = BN * 2 / (PW * 64), LS = (BN + PW * 64 - 1) / (PW * 64);
    static_assert(LA * PW * 64 == BM * 16 && LW * PW * 64 == BN * 2 && TI >= 1 && TJ >= (GLU ? 2 : 1), "tile shape");
    const u32 tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const u32 nout = GLU ? a.N / 2 : a.N, S = (a.K + 63) / 64;
    constexpr u32 CO = GLU ? BN / 2 : BN; /* output columns of a tile */
    const u32 tm = (a.M + BM - 1) / BM, tn = (nout + CO - 1) / CO;
    /* workgroup b runs on XCD b % 8: each XCD takes a run of tiles, by groups of 8 row tiles */
    const u32 per = gridDim.x / 8, t = (blockIdx.x % 8) * per + blockIdx.x / 8;
    if (t >= tm * tn) return;
    const u32 grp = t / (8 * tn), in = t - grp * 8 * tn, gh = min(tm - grp * 8, 8u);
    const u32 m0 = (grp * 8 + in % gh) * BM, c0 = in / gh * CO;

    if (wave >= WGM * WGN) {
        const u32 p = (wave - WGM * WGN) * 64 + lane;
        /* float4 p % 16 of row p / 16, half p % 2 of the codes of weight row p / 2, and PW * 4 or PW * 32 rows on */
        const float *ar[LA];
        const unsigned char *wr[LW], *sr[LS];
        auto wrow = [&](u32 n) { return min(c0 + (GLU && n >= CO ? n - CO : n), nout - 1) + (GLU && n >= CO ? nout : 0); };
#pragma unroll
        for (int j = 0; j < LA; ++j) ar[j] = a.A + (u64)min(m0 + p / 16 + j * PW * 4, a.M - 1) * a.lda + p % 16 * 4;
#pragma unroll
        for (int j = 0; j < LW; ++j) wr[j] = a.Wq + (u64)wrow(p / 2 + j * PW * 32) * a.ldw + p % 2 * 16;
#pragma unroll
        for (int j = 0; j < LS; ++j) sr[j] = a.Ws + (u64)wrow(min(p + j * PW * 64, (u32)BN - 1)) * a.ldws;
        struct regs { floatx4 x[LA]; uint4 w[LW]; u32 e[LS]; } R[AHEAD];
        auto load_w = [&](regs &g, u32 q) {
#pragma unroll
            for (int j = 0; j < LW; ++j) g.w[j] = *(const uint4 *)(wr[j] + 32 * (u64)q);
#pragma unroll
            for (int j = 0; j < LS; ++j) g.e[j] = *(const u32 *)(sr[j] + 4 * (u64)(q / 2));
        };
        auto load_whole = [&](regs &g, u32 q) {
#pragma unroll
            for (int j = 0; j < LA; ++j) g.x[j] = *(const floatx4 *)(ar[j] + 64 * (u64)q);
            load_w(g, q);
        };
        auto load = [&](regs &g, u32 q) { /* any step, zeros past the rows' ends; none behind the last */
            if (q >= S) return;
            if (64 * q + 64 <= a.K) return load_whole(g, q);
            const u32 k = 64 * q + p % 16 * 4;
#pragma unroll
            for (int j = 0; j < LA; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i) g.x[j][i] = k + i < a.K ? ar[j][64 * (u64)q + i] : 0.0f;
            load_w(g, q);
        };
        auto put = [&](const regs &g, u32 q) {
            char *st = smem + (q & 1) * STAGE;
            split_rows<true>(g.x, LA, [&](auto finite) {
#pragma unroll
                for (int j = 0; j < LA; ++j) {
                    u32 lo[3], hi[3];
                    split3<decltype(finite)::v>(g.x[j][0], g.x[j][1], lo);
                    split3<decltype(finite)::v>(g.x[j][2], g.x[j][3], hi);
                    const u32 row = p / 16 + j * PW * 4, i4 = p % 16, at = row * 128 + ((i4 / 2) ^ swz_h(row)) * 16 + (i4 & 1) * 8;
#pragma unroll
                    for (int k = 0; k < 3; ++k) *(uint2 *)(st + k * PLANE + at) = make_uint2(lo[k], hi[k]);
                }
            });
#pragma unroll
            for (int j = 0; j < LW; ++j) *(uint4 *)(st + CODES + (p + j * PW * 64) * 16) = g.w[j];
#pragma unroll
            for (int j = 0; j < LS; ++j) *(u32 *)(st + SCALES + min(p + j * PW * 64, (u32)BN - 1) * 4) = g.e[j];
        };
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) load(R[u], u);
        /* At a barrier stage q is there and stage q - 1 read.  Whole steps without a branch: the compiler waits for all
         * loads where paths join, not for the oldest step's. */
        u32 q = 0;
        for (; 64 * q + 128 * AHEAD <= a.K; q += AHEAD)
#pragma unroll
            for (int u = 0; u < AHEAD; ++u) {
                put(R[u], q + u);
                load_whole(R[u], q + u + AHEAD);
                lds_barrier();
            }
        for (; q < S; q += AHEAD)
#pragma unroll
            for (int u = 0; u < AHEAD; ++u) {
                if (q + u >= S) break;
                put(R[u], q + u);
                load(R[u], q + u + AHEAD);
                lds_barrier();
            }
        return;
    }
    const u32 wm = wave / WGN, wn = wave % WGN, r = lane & 31, f = lane >> 5, sw = swz_h(r);
    const u32 n0 = GLU ? wn * WTN / 2 : wn * WTN;
    floatx16 acc[TI][TJ] = {};
    u32 wq[TJ][4];
    float ws[TJ];
    uint4 v[2][3][TI];
    auto read_w = [&](const char *st, u32 q) {
#pragma unroll
        for (int j = 0; j < TJ; ++j) {
            /* GLU: the first half of a wavefront's tiles are value columns, the second their gates */
            const u32 n = n0 + r + (GLU && j >= TJ / 2 ? BN / 2 + 32 * (j - TJ / 2) : 32 * j);
            const uint4 c = *(const uint4 *)(st + CODES + n * 32 + f * 16);
            wq[j][0] = c.x; wq[j][1] = c.y; wq[j][2] = c.z; wq[j][3] = c.w;
            ws[j] = fp4_scale(*(const u32 *)(st + SCALES + n * 4) >> (16 * (q & 1) + 8 * f) & 255);
        }
    };
    auto read_x = [&](const char *st, int s) {
#pragma unroll
        for (int k = 0; k < 3; ++k)
#pragma unroll
            for (int i = 0; i < TI; ++i)
                v[s & 1][k][i] = *(const uint4 *)(st + k * PLANE + (wm * WTM + 32 * i + r) * 128 + ((4 * f + s) ^ sw) * 16);
    };
    /* the fragments of MFMA s + 1 are read while those of s multiply */
    for (u32 q = 0; q < S; ++q) {
        const char *st = smem + (q & 1) * STAGE;
        lds_barrier();
        read_w(st, q);
        read_x(st, 0);
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            uint4 b[TJ];
#pragma unroll
            for (int j = 0; j < TJ; ++j) b[j] = fp4_bf16x8(wq[j][s], ws[j]);
            if (s < 3) read_x(st, s + 1);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int k = 0; k < 3; ++k)
#pragma unroll
                for (int i = 0; i < TI; ++i)
#pragma unroll
                    for (int j = 0; j < TJ; ++j)
                        acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(as_bf16x8(b[j]), as_bf16x8(v[s & 1][k][i]), acc[i][j], 0, 0, 0);
            __builtin_amdgcn_sched_barrier(0);
        }
    }
    tile_out<GLU, TI, TJ>(a, m0 + wm * WTM, c0 + n0, acc);
}
/* SIMD: wavefronts on a SIMD with the workgroups that the LDS of a CU holds (the widest tiles: one; 32 x 64 keeps a few
 * registers in memory for it, outside its loops) */
#define W4_TILE(BM, BN, WGM, WGN, PW, AHEAD, SIMD, GLU, NAME)                                                       \
    extern "C" __global__ __launch_bounds__(64 * (WGM * WGN + PW), SIMD) void gemm_w4_##NAME(const NkGemm4Args a) { \
        __shared__ __attribute__((aligned(1024))) char smem[2 * (BM * 384 + BN * 36)];                              \
        gemm_w4_tile<BM, BN, WGM, WGN, PW, AHEAD, GLU>(a, smem);                                                    \
    }
W4_TILE(128, 256, 2, 4, 4, 2, 3, false, 128x256)
W4_TILE(128, 256, 2, 4, 4, 2, 3, true, 128x256_glu)
W4_TILE(64, 128, 2, 2, 4, 4, 4, false, 64x128)
W4_TILE(64, 128, 2, 2, 4, 4, 4, true, 64x128_glu)
W4_TILE(32, 64, 1, 2, 2, 4, 4, false, 32x64)
W4_TILE(64, 256, 2, 4, 4, 3, 3, false, 64x256)
W4_TILE(64, 256, 2, 4, 4, 3, 3, true, 64x256_glu)
