/* Microscaled 4-bit rows: quantisation, the way back, and the products with 4-bit weights.
 *
 * A block of 32 values shares the power of two 2^(s - 127); the codes are e2m1 (0, 0.5, 1, 1.5, 2, 3, 4,
 * 6 with a sign).  gfx950 converts (v_cvt_scalef32_*) and multiplies (v_mfma_scale_f32_16x16x128_f8f6f4)
 * them directly: a lane holds the 32 codes of one block of one row and that block's scale, the four lane
 * groups of 16 the four blocks of 128 values. */
#include "nk_common.h"

typedef int intx8 __attribute__((ext_vector_type(8)));

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
 * the bit patterns (every number < infinity < NaN); its exponent field less 2 is the scale. */
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

/* 8 values of a row per lane */
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

/* bias, activation, alpha and accumulation of four consecutive columns n.. of row m (GLU: gate sums in t) */
template <bool GLU> __device__ __forceinline__ void fp4_store4(const NkGemm4Args &a, u32 m, u32 n, floatx4 s, floatx4 t) {
    const u32 nout = GLU ? a.N / 2 : a.N;
    if (m >= a.M || n >= nout) return;
    float *c = a.C + (u64)m * a.ldc + n;
    const bool vec = a.vec && n + 4 <= nout;
    floatx4 old = { 0.f, 0.f, 0.f, 0.f }, b = old, d = old;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const u32 col = min(n + e, nout - 1);
        if (a.bias) {
            b[e] = a.bias[col];
            if (GLU) d[e] = a.bias[col + nout];
        }
        if (a.accumulate && !vec) old[e] = a.C[(u64)m * a.ldc + col];
    }
    if (a.accumulate && vec) old = *(const floatx4 *)c;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        float v = s[e] + b[e];
        if (GLU) v *= sigmoid_f(t[e] + d[e]);
        else if (a.act == NK_ACT_SILU) v = silu_f(v);
        else if (a.act == NK_ACT_RELU) v = fmaxf(v, 0.0f);
        v *= a.alpha;
        s[e] = a.accumulate ? old[e] + v : v;
    }
    if (vec) *(floatx4 *)c = s;
    else
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (n + e < nout) c[e] = s[e];
}

__device__ __forceinline__ intx8 fp4_op(uint4 q) {
    return (intx8){ (int)q.x, (int)q.y, (int)q.z, (int)q.w, 0, 0, 0, 0 };
}
/* acc += W A^T of 16 weight rows and 16 rows over 128 values; the scales are in the low bytes */
__device__ __forceinline__ floatx4 fp4_mfma(uint4 w, u32 ws, uint4 x, u32 xs, floatx4 acc) {
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(fp4_op(w), fp4_op(x), acc, 4, 4, 0, (int)ws, 0, (int)xs);
}

/* A wavefront computes 32 rows by 32 columns (GLU: 16 value and 16 gate columns) with every fragment
 * straight from global memory; rows past the end repeat the last one and are not stored. */
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
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        if constexpr (GLU) fp4_store4<true>(a, m0 + 16 * i + r, n0 + 4 * f, acc[i][0], acc[i][1]);
        else
#pragma unroll
            for (int j = 0; j < 2; ++j) fp4_store4<false>(a, m0 + 16 * i + r, n0 + 16 * j + 4 * f, acc[i][j], acc[i][j]);
    }
}
extern "C" __global__ __launch_bounds__(256) void gemm_fp4(const NkGemm4Args a) { gemm_fp4_impl<false>(a); }
extern "C" __global__ __launch_bounds__(256) void gemm_fp4_glu(const NkGemm4Args a) { gemm_fp4_impl<true>(a); }

/* f32 rows: A = hi + lo in bf16 (16 significant bits), the weights' values exact in bf16.  Lane group f holds
 * values 32 f .. 32 f + 31 of a group of 128 as in the 4-bit product; MFMA j takes their eighth j, the K order
 * being the same on both sides. */
template <bool GLU> __device__ __forceinline__ void gemm_w4_impl(const NkGemm4Args &a) {
    const u32 lane = threadIdx.x & 63, wv = threadIdx.x >> 6, r = lane & 15, f = lane >> 4;
    const u32 nout = GLU ? a.N / 2 : a.N, G = (a.K + 127) / 128;
    const u32 m0 = blockIdx.y * 64 + (wv & 1) * 32, n0 = (blockIdx.x * 2 + (wv >> 1)) * (GLU ? 16 : 32);
    const unsigned char *w[2], *ws[2];
    const float *x[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const u32 n = GLU ? min(n0 + r, nout - 1) + j * nout : min(n0 + 16 * j + r, nout - 1);
        w[j] = a.Wq + (u64)n * a.ldw + 16 * f;
        ws[j] = a.Ws + (u64)n * a.ldws + f;
        x[j] = a.A + (u64)min(m0 + 16 * j + r, a.M - 1) * a.lda;
    }
    floatx4 acc[2][2] = {};
    for (u32 g = 0; g < G; ++g) {
        u32 wq[2][4];
        float we[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const uint4 q = *(const uint4 *)(w[j] + 64 * (u64)g);
            wq[j][0] = q.x; wq[j][1] = q.y; wq[j][2] = q.z; wq[j][3] = q.w;
            we[j] = fp4_scale(ws[j][4 * (u64)g]);
        }
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            uint4 b[2];
#pragma unroll
            for (int j = 0; j < 2; ++j)
                b[j] = make_uint4(fp4_bf16<0>(wq[j][s], we[j]), fp4_bf16<1>(wq[j][s], we[j]), fp4_bf16<2>(wq[j][s], we[j]),
                                  fp4_bf16<3>(wq[j][s], we[j]));
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                float v[8];
                uint4 hi, lo;
                fp4_load8(v, x[i], 128 * g + 32 * f + 8 * s, a.K, true);
                split8(v, hi, lo);
#pragma unroll
                for (int j = 0; j < 2; ++j) acc[i][j] = mfma_bf16(b[j], lo, mfma_bf16(b[j], hi, acc[i][j]));
            }
        }
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        if constexpr (GLU) fp4_store4<true>(a, m0 + 16 * i + r, n0 + 4 * f, acc[i][0], acc[i][1]);
        else
#pragma unroll
            for (int j = 0; j < 2; ++j) fp4_store4<false>(a, m0 + 16 * i + r, n0 + 16 * j + 4 * f, acc[i][j], acc[i][j]);
    }
}
extern "C" __global__ __launch_bounds__(256) void gemm_w4(const NkGemm4Args a) { gemm_w4_impl<false>(a); }
extern "C" __global__ __launch_bounds__(256) void gemm_w4_glu(const NkGemm4Args a) { gemm_w4_impl<true>(a); }
