/* The selective-scan block's operators over the sequences of a batch: the short causal convolution and
 * the scan (see the argument structs for the tables).  Every sequence's table entry is checked here
 * against the buffers' sizes, and one that does not fit is left out. */
#include "nk_common.h"

typedef struct {
    u32 first, rows;
    int from, to;
    bool ok;
} seq_t;
__device__ __forceinline__ seq_t seq_load(const int *seqs, u32 i, u32 M, u32 max_rows, u32 slots) {
    const int4 q = ((const int4 *)seqs)[i];
    return (seq_t){ (u32)q.x, (u32)q.y, q.z, q.w, nk_seq_ok(q.x, q.y, q.z, q.w, M, max_rows, slots) != 0 };
}

__device__ __forceinline__ float ld_row(const float *p) { return *p; }
__device__ __forceinline__ float ld_row(const u16 *p) { return bf2f(*p); }
__device__ __forceinline__ void st_row(float *p, float v) { *p = v; }
/* to bf16, to nearest even; the conversion keeps infinities and NaN */
__device__ __forceinline__ void st_row(u16 *p, float v) { *p = __builtin_bit_cast(u16, (__bf16)v); }

#define CCONV_ROWS 32 /* rows of a workgroup's tile */

/* One thread per channel and tile of rows, the last inputs in registers: every row is read once (and the
 * taps - 1 before the tile).  The tile with the sequence's first row reads the slot's rows and then
 * writes the new ones: nothing else touches the slots. */
template <typename T, int TAPS> __device__ __forceinline__ void cconv_impl(const NkCconvArgs &a) {
    const seq_t s = seq_load(a.seqs, blockIdx.z, a.M, a.max_rows, a.slots);
    const u32 d = blockIdx.x * 256 + threadIdx.x, t0 = blockIdx.y * CCONV_ROWS;
    if (!s.ok || d >= a.D || (t0 && t0 >= s.rows)) return;
    const T *x = (const T *)a.X + (u64)s.first * a.ldx + d;
    T *y = (T *)a.Y + (u64)s.first * a.ldy + d;
    float w[TAPS], v[TAPS];
#pragma unroll
    for (int j = 0; j < TAPS; ++j) w[j] = a.W[(u64)d * TAPS + j];
    const float b = a.bias ? a.bias[d] : 0.0f;
#pragma unroll
    for (int j = 0; j < TAPS - 1; ++j) {
        if (t0) v[j] = ld_row(x + (u64)(t0 + j - (TAPS - 1)) * a.ldx);
        else v[j] = s.from < 0 ? 0.0f : a.state[((u64)s.from * (TAPS - 1) + j) * a.D + d];
    }
    if (!t0 && s.to >= 0) {
        float n[TAPS - 1];
#pragma unroll
        for (int j = 0; j < TAPS - 1; ++j) { /* input rows - (TAPS - 1) + j, from the slot where that is before the first */
            const int t = (int)s.rows - (TAPS - 1) + j;
            n[j] = 0.0f;
            if (t >= 0) n[j] = ld_row(x + (u64)t * a.ldx);
            else
#pragma unroll
                for (int q = 0; q < TAPS - 1; ++q)
                    if (q == t + TAPS - 1) n[j] = v[q];
        }
#pragma unroll
        for (int j = 0; j < TAPS - 1; ++j) a.state[((u64)s.to * (TAPS - 1) + j) * a.D + d] = n[j];
    }
    for (u32 t = t0; t < min(t0 + CCONV_ROWS, s.rows); ++t) {
        v[TAPS - 1] = ld_row(x + (u64)t * a.ldx);
        float o = b;
#pragma unroll
        for (int j = 0; j < TAPS; ++j) o = fmaf(w[j], v[j], o);
        if (a.act == NK_ACT_SILU) o = silu_f(o);
        else if (a.act == NK_ACT_RELU) o = fmaxf(o, 0.0f);
        st_row(y + (u64)t * a.ldy, o);
#pragma unroll
        for (int j = 0; j < TAPS - 1; ++j) v[j] = v[j + 1];
    }
}
#define CCONV(T, NAME, TAPS) \
    extern "C" __global__ __launch_bounds__(256) void cconv_##NAME##_##TAPS(const NkCconvArgs a) { cconv_impl<T, TAPS>(a); }
CCONV(float, f32, 2) CCONV(float, f32, 3) CCONV(float, f32, 4)
CCONV(u16, bf16, 2) CCONV(u16, bf16, 3) CCONV(u16, bf16, 4)

/* log(1 + e^v), without a threshold */
__device__ __forceinline__ float softplus_f(float v) { return fmaxf(v, 0.0f) + log1pf(expf(-fabsf(v))); }

/* One thread per channel with its NS >= N states in registers, row after row.  e^(s A) is 2^(s A log2 e) by
 * the hardware's exponential (results below 2^-126 come out as 0). */
template <typename T, int NS> __device__ __forceinline__ void scan_impl(const NkScanArgs &a) {
    const seq_t s = seq_load(a.seqs, blockIdx.y, a.M, a.max_rows, a.slots);
    const u32 d = blockIdx.x * 256 + threadIdx.x;
    if (!s.ok || d >= a.D) return;
    const u32 g = d / (a.D / a.groups);
    const T *x = (const T *)a.x + (u64)s.first * a.ldx + d, *dt = (const T *)a.dt + (u64)s.first * a.lddt + d;
    const T *B = (const T *)a.B + (u64)s.first * a.ldbc + (u64)g * a.N, *C = (const T *)a.C + (u64)s.first * a.ldbc + (u64)g * a.N;
    const T *z = a.z ? (const T *)a.z + (u64)s.first * a.ldz + d : nullptr;
    T *y = (T *)a.y + (u64)s.first * a.ldy + d;
    const float skip = a.skip ? a.skip[d] : 0.0f, db = a.dt_bias ? a.dt_bias[d] : 0.0f;
    float A[NS], h[NS];
#pragma unroll
    for (int n = 0; n < NS; ++n) {
        A[n] = (u32)n < a.N ? a.A[(u64)d * a.N + n] * 1.44269504f : 0.0f;
        h[n] = (u32)n < a.N && s.from >= 0 ? a.state[((u64)s.from * a.D + d) * a.N + n] : 0.0f;
    }
    for (u32 t = 0; t < s.rows; ++t) {
        const float v = ld_row(x + (u64)t * a.ldx);
        float p = ld_row(dt + (u64)t * a.lddt) + db;
        if (a.softplus) p = softplus_f(p);
        float o = 0.0f;
#pragma unroll
        for (int n = 0; n < NS; ++n) {
            if ((u32)n < a.N) {
                const float b = ld_row(B + (u64)t * a.ldbc + n), c = ld_row(C + (u64)t * a.ldbc + n);
                h[n] = fmaf(__builtin_amdgcn_exp2f(p * A[n]), h[n], p * v * b);
                o = fmaf(c, h[n], o);
            }
        }
        if (a.skip) o = fmaf(skip, v, o);
        if (z) o *= silu_f(ld_row(z + (u64)t * a.ldz));
        st_row(y + (u64)t * a.ldy, o);
    }
    if (s.to >= 0)
#pragma unroll
        for (int n = 0; n < NS; ++n)
            if ((u32)n < a.N) a.state[((u64)s.to * a.D + d) * a.N + n] = h[n];
}
#define SCAN(T, NAME, NS) \
    extern "C" __global__ __launch_bounds__(256) void scan_##NAME##_##NS(const NkScanArgs a) { scan_impl<T, NS>(a); }
SCAN(float, f32, 8) SCAN(float, f32, 16) SCAN(float, f32, 32) SCAN(float, f32, 64)
SCAN(u16, bf16, 8) SCAN(u16, bf16, 16) SCAN(u16, bf16, 32) SCAN(u16, bf16, 64)
