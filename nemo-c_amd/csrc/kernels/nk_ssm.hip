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

/* v / (1 + e^-v) to about four steps in 12 instructions (the IEEE exponential and division take 25, a third of what the
 * convolution does): 2^(-v log2 e) with the product's rounding put back, the hardware's reciprocal.  The exponent is
 * kept where its own arithmetic is finite; from 2^128 on the exponential is infinite and its reciprocal zero (what is
 * flushed below v = -87 is under 2e-36). */
__device__ __forceinline__ float silu_q(float v) {
    const float n = __builtin_amdgcn_fmed3f(-v, -104.0f, 104.0f), t = n * 1.44269504f;
    const float r = fmaf(n, 1.92596299e-8f, fmaf(n, 1.44269504f, -t)), e = __builtin_amdgcn_exp2f(t);
    return v * __builtin_amdgcn_rcpf(fmaf(e, fmaf(r, 0.693147181f, 1.0f), 1.0f));
}

/* V values of a row as they lie in memory */
template <typename T, int V> struct row_t;
template <> struct row_t<float, 1> { float v; };
template <> struct row_t<u16, 1> { u16 v; };
template <> struct row_t<u16, 2> { u32 v; };
__device__ __forceinline__ void widen(float (&o)[1], row_t<float, 1> r) { o[0] = r.v; }
__device__ __forceinline__ void widen(float (&o)[1], row_t<u16, 1> r) { o[0] = bf2f(r.v); }
__device__ __forceinline__ void widen(float (&o)[2], row_t<u16, 2> r) {
    o[0] = bf_lo(r.v);
    o[1] = bf_hi(r.v);
}
template <typename T> __device__ __forceinline__ void store_row(T *p, const float (&v)[1]) { st_row(p, v[0]); }
__device__ __forceinline__ void store_row(u16 *p, const float (&v)[2]) {
    *(u32 *)p = __builtin_bit_cast(u32, __builtin_convertvector((floatx2){ v[0], v[1] }, bf16x2));
}

/* One thread per channel (bf16: two where rows allow it) and tile of a.tile rows (where a sequence has more of them than the
 * grid, every gridDim.y-th), the last inputs in registers and eight rows' loads in flight: every row is read once (and the
 * taps - 1 before the tile).  Bound by memory: 8192 rows of 2048 channels f32 30 us, bf16 16.  More channels per thread are
 * slower (16 bytes each: 37 and 29 us), their taps being far apart and their threads few.  The tile with the sequence's
 * first row reads the slot's rows and then writes the new ones: nothing else touches the slots. */
template <typename T, int TAPS, int V> __device__ __forceinline__ void cconv_impl(const NkCconvArgs &a) {
    const seq_t s = seq_load(a.seqs, blockIdx.z, a.M, a.max_rows, a.slots);
    const u32 d = (blockIdx.x * 256 + threadIdx.x) * V, step = gridDim.y * a.tile;
    u32 t0 = blockIdx.y * a.tile, end;
    if (!s.ok || d >= a.D || (t0 && t0 >= s.rows)) return;
    typedef row_t<T, V> row;
    const T *x = (const T *)a.X + (u64)s.first * a.ldx;
    T *y = (T *)a.Y + (u64)s.first * a.ldy;
    auto load = [&](u32 t) { return *(const row *)(x + (u64)t * a.ldx + d); };
    constexpr int B = 8; /* rows in flight (the tile's last again past its end, not used) */
    row q[B];
    auto first = [&] {
        end = min(t0 + a.tile, s.rows);
        if (t0 < end)
#pragma unroll
            for (u32 k = 0; k < B; ++k) q[k] = load(min(t0 + k, end - 1));
    };
    first();
    float w[TAPS][V], b[V], v[TAPS - 1 + B][V]; /* v: the inputs before a batch of B rows, then its own */
#pragma unroll
    for (int j = 0; j < TAPS; ++j)
#pragma unroll
        for (int e = 0; e < V; ++e) w[j][e] = a.W[(u64)(d + e) * TAPS + j];
#pragma unroll
    for (int e = 0; e < V; ++e) b[e] = a.bias ? a.bias[d + e] : 0.0f;
    auto before = [&] {
#pragma unroll
        for (int j = 0; j < TAPS - 1; ++j) widen(v[j], load(t0 + j - (TAPS - 1)));
    };
    if (t0) before();
    else
#pragma unroll
        for (int j = 0; j < TAPS - 1; ++j)
#pragma unroll
            for (int e = 0; e < V; ++e) v[j][e] = s.from < 0 ? 0.0f : a.state[((u64)s.from * (TAPS - 1) + j) * a.D + d + e];
    if (!t0 && s.to >= 0) {
        float n[TAPS - 1][V];
#pragma unroll
        for (int j = 0; j < TAPS - 1; ++j) { /* input rows - (TAPS - 1) + j, from the slot where that is before the first */
            const int t = (int)s.rows - (TAPS - 1) + j;
            if (t >= 0) widen(n[j], load((u32)t));
            else
#pragma unroll
                for (int k = 0; k < TAPS - 1; ++k)
#pragma unroll
                    for (int e = 0; e < V; ++e) n[j][e] = k == t + TAPS - 1 ? v[k][e] : k ? n[j][e] : 0.0f;
        }
#pragma unroll
        for (int j = 0; j < TAPS - 1; ++j)
#pragma unroll
            for (int e = 0; e < V; ++e) a.state[((u64)s.to * (TAPS - 1) + j) * a.D + d + e] = n[j][e];
    }
    for (;;) {
        for (u32 t = t0; t < end; t += B) {
#pragma unroll
            for (int k = 0; k < B; ++k) widen(v[TAPS - 1 + k], q[k]);
            if (t + B < end)
#pragma unroll
                for (u32 k = 0; k < B; ++k) q[k] = load(min(t + B + k, end - 1));
#pragma unroll
            for (u32 k = 0; k < B; ++k) {
                float o[V];
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    o[e] = b[e];
#pragma unroll
                    for (int j = 0; j < TAPS; ++j) o[e] = fmaf(w[j][e], v[k + j][e], o[e]);
                    if (a.act == NK_ACT_SILU) o[e] = silu_q(o[e]);
                    else if (a.act == NK_ACT_RELU) o[e] = relu_nan(o[e]);
                }
                if (t + k < end) store_row(y + (u64)(t + k) * a.ldy + d, o);
            }
#pragma unroll
            for (int j = 0; j < TAPS - 1; ++j)
#pragma unroll
                for (int e = 0; e < V; ++e) v[j][e] = v[B + j][e];
        }
        t0 += step;
        if (t0 >= s.rows) return;
        first();
        before();
    }
}
#define CCONV(T, NAME, TAPS, V) \
    extern "C" __global__ __launch_bounds__(256) void cconv_##NAME##_##TAPS(const NkCconvArgs a) { cconv_impl<T, TAPS, V>(a); }
CCONV(float, f32, 2, 1) CCONV(float, f32, 3, 1) CCONV(float, f32, 4, 1)
CCONV(u16, bf16, 2, 1) CCONV(u16, bf16, 3, 1) CCONV(u16, bf16, 4, 1)
CCONV(u16, bf16x2, 2, 2) CCONV(u16, bf16x2, 3, 2) CCONV(u16, bf16x2, 4, 2)

/* e^v for v <= 0 to about two steps: 2^(v log2 e) with the product's rounding put back (the hardware's
 * exponential gives 0 below 2^-126) */
__device__ __forceinline__ float exp_neg(float v) {
    const float t = v * 1.44269504f, r = fmaf(v, 1.44269504f, -t) + v * 1.92596299e-8f;
    const float e = __builtin_amdgcn_exp2f(t);
    return v < -104.0f ? 0.0f : fmaf(e, r * 0.693147181f, e); /* r is NaN where v is infinite */
}
/* log(1 + e^v) = max(v, 0) + 2 atanh(q), q = e / (2 + e) <= 1/3 with e = e^-|v|; atanh(q) = q + q^3 f(q^2), f a cubic
 * fitted for the least relative error of the whole on q^2 <= 1/9: 4.5e-9 */
__device__ __forceinline__ float softplus_f(float v) {
    const float e = exp_neg(-fabsf(v)), q = e * __builtin_amdgcn_rcpf(2.0f + e), w = q * q;
    const float f = fmaf(fmaf(fmaf(0.140059963f, w, 0.140009016f), w, 0.200107634f), w, 0.333332092f);
    return fmaxf(v, 0.0f) + 2.0f * fmaf(f * w, q, q); /* NaN comes through q */
}

/* A log2 e, the factor of a step in the exponent.  An infinite one counts as the largest number: the steps of zero that
 * fill a tile up would make it NaN. */
__device__ __forceinline__ float scan_rate(float A) {
    const float v = A * 1.44269504f;
    return __builtin_isinf(v) ? copysignf(3.4028235e38f, v) : v;
}

template <bool V> struct flag_t { static constexpr bool v = V; };

#define SCAN_TILE 64 /* rows whose B and C are in LDS at a time */

/* Rows t0 .. t1 - 1 of a sequence, one thread per channel with its NS >= N states in registers.
 * e^(s A) is 2^(s A log2 e) by the hardware's exponential (results below 2^-126 come out as 0).  B and C are the
 * same for every channel of the workgroup's group: a tile of their rows lies in LDS as f32, padded
 * with zeros to NS, and is read by all lanes at one address.  ENDS: only the states (from zero) and the
 * sum of the steps are wanted, no rows are written.  CARE: the states that fill N up to NS, zero as long as the inputs are
 * finite and NaN after an infinite one, are left out of the outputs.
 *
 * Bound by the vector units: per state and row an exponential, which takes the time of 1.85 products, and four more
 * operations, three of them where only the ends are wanted.  8192 rows of 2048 channels of 16 states, bf16: ends 66
 * us, rows 85, the joining between them 13, where those operations alone are 43 and 52 us at the 30 T products/s that
 * this card reaches; the softplus, the gate and the conversions of every row are the rest. */
template <typename T, int NS, bool ENDS, bool WHOLE, bool CARE>
__device__ __forceinline__ void scan_rows(const NkScanArgs &a, const seq_t &s, u32 t0, u32 t1, u32 g, u32 d, bool live,
                                          float (&h)[NS], float &sum, float *lds) {
    const T *x = (const T *)a.x + (u64)s.first * a.ldx, *dt = (const T *)a.dt + (u64)s.first * a.lddt;
    const T *B = (const T *)a.B + (u64)s.first * a.ldbc + (u64)g * a.N, *C = (const T *)a.C + (u64)s.first * a.ldbc + (u64)g * a.N;
    const u32 ldz = a.z ? a.ldz : a.ldx; /* no gate: x is read in its place, and not used */
    const T *z = a.z ? (const T *)a.z + (u64)s.first * a.ldz : x;
    T *y = (T *)a.y + (u64)s.first * a.ldy;
    const float skip = a.skip ? a.skip[d] : 0.0f, db = a.dt_bias ? a.dt_bias[d] : 0.0f;
    constexpr u32 W = ENDS ? NS : 2 * NS;
    float A[NS];
#pragma unroll
    for (int n = 0; n < NS; ++n) {
        const float v = a.A[(u64)d * a.N + min((u32)n, a.N - 1)];
        A[n] = (u32)n < a.N ? scan_rate(v) : 0.0f;
    }
    for (u32 u = t0; u < t1; u += SCAN_TILE) {
        const u32 rows = min(t1 - u, (u32)SCAN_TILE);
        __syncthreads();
        constexpr int L = 8; /* loads in flight (from places past the end: of the last) */
        const u32 all = (rows + 3) / 4 * 4 * W;
        for (u32 i0 = threadIdx.x; i0 < all; i0 += L * blockDim.x) {
            float v[L];
#pragma unroll
            for (u32 k = 0; k < L; ++k) {
                if (!WHOLE && k && i0 - threadIdx.x + k * blockDim.x >= all) break; /* pieces of a few rows */
                const u32 i = i0 + k * blockDim.x, r = min(i / W, rows - 1), n = i % W;
                v[k] = ld_row((n < NS ? B : C) + (u64)(u + r) * a.ldbc + min(n % NS, a.N - 1));
            }
#pragma unroll
            for (u32 k = 0; k < L; ++k) {
                const u32 i = i0 + k * blockDim.x;
                if (i < all) lds[i] = i / W < rows && i % NS < a.N ? v[k] : 0.0f;
            }
        }
        __syncthreads();
        /* four rows at a time, the next four's loads in flight; past the end a step of zero, which leaves the states
         * as they are.  What is the same for all rows (softplus, the gate) is asked once for the four: a branch a row
         * keeps the rows' chains of instructions apart. */
        float xn[4], pn[4], zn[4];
        auto load = [&](u32 r0) {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const u64 t = u + min(r0 + k, rows - 1);
                xn[k] = ld_row(x + t * a.ldx + d);
                pn[k] = ld_row(dt + t * a.lddt + d);
                if constexpr (!ENDS) zn[k] = ld_row(z + t * ldz + d);
            }
        };
        load(0);
#pragma unroll 1
        for (u32 r0 = 0; r0 < rows; r0 += 4) {
            float xv[4], p[4], zv[4], o[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                xv[k] = xn[k];
                p[k] = pn[k] + db;
                if constexpr (!ENDS) zv[k] = zn[k];
            }
            load(r0 + 4);
            if (a.softplus)
#pragma unroll
                for (int k = 0; k < 4; ++k) p[k] = softplus_f(p[k]);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const bool in = r0 + k < rows;
                float v = p[k] * xv[k];
                p[k] = in ? p[k] : 0.0f;
                v = in ? v : 0.0f;
                if constexpr (ENDS) sum += p[k];
                o[k] = 0.0f;
                const floatx4 *bc = (const floatx4 *)(lds + (r0 + k) * W);
#pragma unroll
                for (int n = 0; n < NS; n += 4) {
                    const floatx4 b = bc[n / 4];
                    floatx4 c;
                    if constexpr (!ENDS) c = bc[(NS + n) / 4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        h[n + e] = fmaf(__builtin_amdgcn_exp2f(p[k] * A[n + e]), h[n + e], v * b[e]);
                        if constexpr (!ENDS) o[k] = !CARE || (u32)(n + e) < a.N ? fmaf(c[e], h[n + e], o[k]) : o[k];
                    }
                }
                if constexpr (!ENDS) o[k] = fmaf(skip, xv[k], o[k]);
            }
            if constexpr (!ENDS) {
                if (a.z)
#pragma unroll
                    for (int k = 0; k < 4; ++k) o[k] *= silu_q(zv[k]);
                if (live)
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        if (r0 + k < rows) st_row(y + (u64)(u + r0 + k) * a.ldy + d, o[k]);
            }
        }
    }
}

/* channel of this thread: workgroups of blockDim channels inside one group */
struct chan_t {
    u32 g, d;
    bool live;
};
__device__ __forceinline__ chan_t scan_channel(const NkScanArgs &a) {
    const u32 per = a.D / a.groups, tiles = (per + blockDim.x - 1) / blockDim.x, g = blockIdx.x / tiles;
    const u32 c = (blockIdx.x - g * tiles) * blockDim.x + threadIdx.x;
    return (chan_t){ g, g * per + min(c, per - 1), c < per };
}

/* A piece's place in the scratch: N states of D channels, then the sums.  Places are needed only by pieces that another
 * follows, which are whole.  Either all sequences have a.pieces of them, or a piece's place is that of the one
 * multiple of a.piece among its rows' numbers: no row is in two sequences, so no place is in two pieces. */
__device__ __forceinline__ float *scan_place(const NkScanArgs &a, u32 i, const seq_t &s, u32 piece) {
    const u64 at = a.byrow ? (s.first + a.piece - 1) / a.piece + piece : (u64)i * a.pieces + piece;
    return a.ws + at * (a.N + 1) * a.D;
}

/* Piece p of all sequences one after another: the sequence, its table entry, and the piece's number in it (every
 * sequence has one at least); false behind the last.  64 sequences at a time, one to a lane.  So the pieces that there are
 * follow each other over the card; a grid of sequences by the longest one's pieces, most of them empty, leaves its work
 * where the empty ones fall (3 sequences of 360 to 3000 rows 140 us, so 118; 32 of 0 to 600 139 and 108). */
__device__ __forceinline__ bool scan_find(const NkScanArgs &a, u32 p, seq_t &s, u32 &i, u32 &piece) {
    if (a.nseq == 1) {
        s = seq_load(a.seqs, 0, a.M, a.max_rows, a.slots);
        i = 0;
        piece = p;
        return s.ok && (!p || p * a.piece < s.rows);
    }
    const u32 lane = threadIdx.x & 63;
    u32 before = 0;
    for (u32 base = 0; base < a.nseq; base += 64) {
        const seq_t q = seq_load(a.seqs, min(base + lane, a.nseq - 1), a.M, a.max_rows, a.slots);
        const u32 n = q.ok && base + lane < a.nseq ? max((q.rows + a.piece - 1) / a.piece, 1u) : 0;
        u32 upto = n; /* pieces of the lanes up to this one */
#pragma unroll
        for (u32 w = 1; w < 64; w *= 2) {
            const u32 v = __shfl_up(upto, w, 64);
            upto += lane >= w ? v : 0;
        }
        const u64 here = __ballot(before + upto > p);
        if (here) {
            const int l = __builtin_ctzll(here);
            auto of = [&](u32 v) { return (u32)__builtin_amdgcn_readlane((int)v, l); };
            s = (seq_t){ of(q.first), of(q.rows), (int)of((u32)q.from), (int)of((u32)q.to), true };
            i = base + l;
            piece = p - before - (of(upto) - of(n));
            return true;
        }
        before += (u32)__builtin_amdgcn_readlane((int)upto, 63);
    }
    return false;
}

/* PART 0: whole sequences.  PART 1: the states that the pieces of a.piece rows end in from zero, and their
 * sums of steps (of all but a sequence's last, which nothing follows).  PART 2: the pieces again from the
 * states that scan_join has put in their predecessors' places, a sequence's first from the copy of its slot. */
template <typename T, int NS, int PART> __device__ __forceinline__ void scan_impl(const NkScanArgs &a) {
    __shared__ float lds[SCAN_TILE * NS * (PART == 1 ? 1 : 2)];
    seq_t s;
    u32 i = blockIdx.y, piece = 0;
    if (PART) {
        if (!scan_find(a, blockIdx.y, s, i, piece)) return;
    } else {
        s = seq_load(a.seqs, i, a.M, a.max_rows, a.slots);
        if (!s.ok) return;
    }
    const chan_t c = scan_channel(a);
    const u32 t0 = PART ? piece * a.piece : 0, t1 = PART ? min(t0 + a.piece, s.rows) : s.rows;
    if (PART == 1 && t0 + a.piece >= s.rows) return;
    float h[NS], sum = 0.0f;
    float *ws = PART ? scan_place(a, i, s, piece) + c.d : nullptr;
    /* the slot of a sequence of several pieces may be written by its last before its first reads it */
    const bool joined = PART == 2 && t0, kept = PART == 2 && !t0 && s.rows > a.piece;
#pragma unroll
    for (int n = 0; n < NS; ++n) h[n] = 0.0f;
    auto start = [&] {
        if (joined || (PART != 1 && !t0 && s.from >= 0)) {
            const float *from = joined ? ws - (u64)(a.N + 1) * a.D : kept ? a.first + (u64)i * a.N * a.D + c.d
                                                                           : a.state + ((u64)s.from * a.D + c.d) * a.N;
#pragma unroll
            for (int n = 0; n < NS; ++n) {
                const float v = from[min((u32)n, a.N - 1) * (joined || kept ? (u64)a.D : 1)];
                h[n] = (u32)n < a.N ? v : 0.0f;
            }
        }
    };
    if (PART != 1) start();
    scan_rows<T, NS, PART == 1, PART == 0, false>(a, s, t0, t1, c.g, c.d, c.live, h, sum, lds);
    /* An input that is not finite makes the filling states NaN, and they stay so: the rows again without them.  Asked once
     * behind the rows, which costs 0 to 2%; asked for every four rows it took up to 70 registers, and a wavefront less on
     * every SIMD. */
    if (PART != 1 && __builtin_expect(a.N < NS, 0) && __builtin_expect(__syncthreads_or(h[NS - 1] != h[NS - 1]), 0)) {
#pragma unroll
        for (int n = 0; n < NS; ++n) h[n] = 0.0f;
        start();
        scan_rows<T, NS, false, PART == 0, true>(a, s, t0, t1, c.g, c.d, c.live, h, sum, lds);
    }
    if (!c.live || (PART != 1 && (s.to < 0 || t1 < s.rows))) return;
    float *to = PART == 1 ? ws : a.state + ((u64)s.to * a.D + c.d) * a.N;
#pragma unroll
    for (int n = 0; n < NS; ++n)
        if ((u32)n < a.N) to[n * (PART == 1 ? (u64)a.D : 1)] = h[n];
    if (PART == 1) ws[(u64)a.N * a.D] = sum;
}
#define SCAN(T, NAME, NS)                                                                                              \
    extern "C" __global__ __launch_bounds__(256) void scan_##NAME##_##NS(const NkScanArgs a) { scan_impl<T, NS, 0>(a); } \
    extern "C" __global__ __launch_bounds__(256) void scan_ends_##NAME##_##NS(const NkScanArgs a) { scan_impl<T, NS, 1>(a); } \
    extern "C" __global__ __launch_bounds__(256) void scan_from_##NAME##_##NS(const NkScanArgs a) { scan_impl<T, NS, 2>(a); }
SCAN(float, f32, 8) SCAN(float, f32, 16) SCAN(float, f32, 32) SCAN(float, f32, 64)
SCAN(u16, bf16, 8) SCAN(u16, bf16, 16) SCAN(u16, bf16, 32) SCAN(u16, bf16, 64)

/* The pieces of a sequence one after another: H <- e^(A sum) H + end, the state that the next piece starts from,
 * takes the place of the piece's own end.  The factor by halves: a piece of growing steps may pass 2^128 by itself where
 * no state does, and one that is zero stays so whatever the factor.  An infinite state stays infinite: the factor may be
 * below the type's range where no row's is (but not where a step or the rate is infinite: zero times infinity there too);
 * only batches that end in one ask for that.
 * One thread per state; the loads of JOIN pieces are in flight at a time (one at a time 36 us for 128 pieces of 2048
 * channels, a memory round trip each). */
#define JOIN 16
extern "C" __global__ __launch_bounds__(256) void scan_join(const NkScanArgs a) {
    const seq_t s = seq_load(a.seqs, blockIdx.z, a.M, a.max_rows, a.slots);
    const u32 d = blockIdx.x * 256 + threadIdx.x, n = blockIdx.y;
    if (!s.ok || d >= a.D || s.rows <= a.piece) return;
    const float A = 0.5f * scan_rate(a.A[(u64)d * a.N + n]), RATE_MAX = 0.5f * 3.4028235e38f;
    float h = s.from >= 0 ? a.state[((u64)s.from * a.D + d) * a.N + n] : 0.0f;
    if (s.from >= 0) a.first[((u64)blockIdx.z * a.N + n) * a.D + d] = h;
    const u32 ends = (s.rows - 1) / a.piece; /* pieces that another follows */
    const u64 step = (u64)(a.N + 1) * a.D;
    float *w = scan_place(a, blockIdx.z, s, 0) + d;
    for (u32 i = 0; i < ends; i += JOIN) {
        float end[JOIN], sum[JOIN];
#pragma unroll
        for (u32 k = 0; k < JOIN; ++k) {
            const float *p = w + min(i + k, ends - 1) * step;
            end[k] = p[(u64)n * a.D];
            sum[k] = p[(u64)a.N * a.D];
        }
        auto join = [&](auto finite) {
#pragma unroll
            for (u32 k = 0; k < JOIN; ++k) {
                if (i + k >= ends) break;
                const float e = __builtin_amdgcn_exp2f(sum[k] * A);
                const bool keep = !decltype(finite)::v && __builtin_isinf(h) && fabsf(sum[k]) < __builtin_inff() && fabsf(A) < RATE_MAX;
                h = h == 0.0f ? end[k] : keep ? h + end[k] : fmaf(e, e * h, end[k]);
                w[(i + k) * step + (u64)n * a.D] = h;
            }
        };
        const float before = h;
        join(flag_t<true>());
        if (!(fabsf(h) < __builtin_inff())) { /* no state comes back from there: the batch again */
            h = before;
            join(flag_t<false>());
        }
    }
}

/* Few rows (tokens): every state row is read and written once and the rows are nothing beside them, so the
 * states are spread over lanes: Q lanes per channel with four consecutive states each, a row's output
 * summed over the Q lanes.  One token of 2048 channels of 16 states: 1 stream 3.9 us, 64 streams 8.3, 256 streams 20.3
 * (its states read and written at 3.3 TB/s). */
template <typename T, int Q> __device__ __forceinline__ void scan_few_impl(const NkScanArgs &a) {
    const seq_t s = seq_load(a.seqs, blockIdx.y, a.M, a.max_rows, a.slots);
    const u32 i = blockIdx.x * 256 + threadIdx.x, n0 = 4 * (i % Q);
    const bool live = i / Q < a.D;
    const u32 d = min(i / Q, a.D - 1), g = d / (a.D / a.groups);
    if (!s.ok) return;
    /* the four states' places in a row of N (a place past the end counts as the last and is masked) */
    u32 at[4];
    float A[4], h[4] = { 0.f, 0.f, 0.f, 0.f };
#pragma unroll
    for (int e = 0; e < 4; ++e) at[e] = min(n0 + e, a.N - 1);
    const float *ar = a.A + (u64)d * a.N, *hr = a.state + ((u64)max(s.from, 0) * a.D + d) * a.N;
    if (a.vec && n0 < a.N) {
        const floatx4 v = *(const floatx4 *)(ar + n0);
        A[0] = v[0]; A[1] = v[1]; A[2] = v[2]; A[3] = v[3];
    } else
#pragma unroll
        for (int e = 0; e < 4; ++e) A[e] = ar[at[e]];
    if (s.from >= 0) {
        if (a.vec && n0 < a.N) {
            const floatx4 v = *(const floatx4 *)(hr + n0);
            h[0] = v[0]; h[1] = v[1]; h[2] = v[2]; h[3] = v[3];
        } else
#pragma unroll
            for (int e = 0; e < 4; ++e) h[e] = hr[at[e]];
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        A[e] = n0 + e < a.N ? scan_rate(A[e]) : 0.0f;
        h[e] = n0 + e < a.N ? h[e] : 0.0f;
    }
    const float skip = a.skip ? a.skip[d] : 0.0f, db = a.dt_bias ? a.dt_bias[d] : 0.0f;
    for (u32 t = s.first; t < s.first + s.rows; ++t) {
        const float v = ld_row((const T *)a.x + (u64)t * a.ldx + d);
        float p = ld_row((const T *)a.dt + (u64)t * a.lddt + d) + db;
        const T *B = (const T *)a.B + (u64)t * a.ldbc + (u64)g * a.N, *C = (const T *)a.C + (u64)t * a.ldbc + (u64)g * a.N;
        float b[4], c[4], o = 0.0f;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            b[e] = ld_row(B + at[e]);
            c[e] = ld_row(C + at[e]);
        }
        const float z = a.z ? ld_row((const T *)a.z + (u64)t * a.ldz + d) : 0.0f;
        if (a.softplus) p = softplus_f(p);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const bool in = n0 + e < a.N;
            h[e] = fmaf(__builtin_amdgcn_exp2f(p * A[e]), h[e], p * v * b[e]);
            o = in ? fmaf(c[e], h[e], o) : o;
        }
#pragma unroll
        for (int w = Q / 2; w > 0; w >>= 1) o += __shfl_xor(o, w, 64);
        o = fmaf(skip, v, o);
        if (a.z) o *= silu_q(z);
        if (live && n0 == 0) st_row((T *)a.y + (u64)t * a.ldy + d, o);
    }
    if (s.to < 0 || !live) return;
    float *to = a.state + ((u64)s.to * a.D + d) * a.N;
    if (a.vec && n0 < a.N) *(floatx4 *)(to + n0) = (floatx4){ h[0], h[1], h[2], h[3] };
    else
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (n0 + e < a.N) to[n0 + e] = h[e];
}
#define SCAN_FEW(Q)                                                                                                    \
    extern "C" __global__ __launch_bounds__(256) void scan_few_f32_##Q(const NkScanArgs a) { scan_few_impl<float, Q>(a); } \
    extern "C" __global__ __launch_bounds__(256) void scan_few_bf16_##Q(const NkScanArgs a) { scan_few_impl<u16, Q>(a); }
SCAN_FEW(1) SCAN_FEW(2) SCAN_FEW(4) SCAN_FEW(8) SCAN_FEW(16)
