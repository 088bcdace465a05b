/* Attention over the paged key and value cache.  Row i of a sequence stands behind `len` tokens at position
 * p = len + i and sees token j where j <= p and (no window, or j > p - window, or j < sinks); tokens of a page that there
 * is none of are not seen.  The rows of the heads that share a head of the cache lie one behind another ("packed":
 * row * group + head of the group), so its keys and values are read once for all of them.
 *
 *   o = sum_j 2^(x_j - m) v_j / sum_j 2^(x_j - m),   x_j = scale log2(e) q.k_j,   m = max_j x_j
 *
 * in one pass over the tokens, with the running maximum, sum and sums of v in 32 bits.  The products are on the matrix
 * units: keys and values are exact in bf16 (8-bit codes with their power of two too); bf16 rows are, and their
 * probabilities are rounded to bf16 (at most a relative 2^-8 of each, as the output is too: with both the error is 1.3 times
 * that of the output's rounding alone, and a second term would be half as many products again); f32 rows and their
 * probabilities are three bf16 terms, 24 bits.
 *
 * A bf16 row whose sum of weights is NaN has a logit that is (or an infinite one): all NaN, as the formula has it, where its
 * head fills the fragments.  Where it does not (pad), their rest is keys' last values again, times zeros of the row: NaN
 * of an infinite one, whose logit may be -inf and have no weight.  Such rows, and those whose result is not finite
 * otherwise (an infinity or NaN was near among the values, also of a token that only some rows see: 0 times it is NaN in a
 * product; of an f32 row's terms the later ones are zero too), or whose sum is zero, are computed again by the formula, row
 * by row, as far as a NaN logit. */
#include "nk_common.h"

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));

/* a 16-lane group's 4 rows of 16 values from LDS, each lane with its column's four: lane i gives the address of row i / 4,
 * values 4 (i % 4) on */
__device__ __forceinline__ uint2 lds_column4(const u16 *p) {
    return __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4bf16((__attribute__((address_space(3))) bf16x4 *)p));
}
__device__ __forceinline__ void swap32(float &a, float &b) { /* b's lower half <-> a's upper half */
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(a), __float_as_uint(b), false, false);
    a = __uint_as_float(r[0]);
    b = __uint_as_float(r[1]);
}
__device__ __forceinline__ void swap16(float &a, float &b) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(a), __float_as_uint(b), false, false);
    a = __uint_as_float(r[0]);
    b = __uint_as_float(r[1]);
}
/* one instruction for three, NaN if any is (fmaxf takes another to quiet a product's) */
__device__ __forceinline__ float max3(float a, float b, float c) { return __builtin_elementwise_maximum(__builtin_elementwise_maximum(a, b), c); }
/* over the lanes that agree in their low four bits (16: five) */
__device__ __forceinline__ float max_over32(float a) { float b = a; swap32(a, b); return fmaxf(a, b); }
__device__ __forceinline__ float sum_over32(float a) { float b = a; swap32(a, b); return a + b; }
__device__ __forceinline__ float max_over16(float a) { float b = a; swap16(a, b); return max_over32(fmaxf(a, b)); }
__device__ __forceinline__ float sum_over16(float a) { float b = a; swap16(a, b); return sum_over32(a + b); }

/* 8 codes to bf16 with the power of two of their block */
__device__ __forceinline__ u32x4 e4m3_bf16(u32 a, u32 b, float s) {
    return (u32x4){ __builtin_bit_cast(u32, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, s, false)),
                    __builtin_bit_cast(u32, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, s, true)),
                    __builtin_bit_cast(u32, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, s, false)),
                    __builtin_bit_cast(u32, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, s, true)) };
}
__device__ __forceinline__ floatx4 attn_mfma(u32x4 a, u32x4 b, floatx4 acc) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), acc, 0, 0, 0);
}

/* 8 f32 values as TERMS bf16 fragments: to nearest each, the first of what the values are, the next of what is left.  BIG: also
 * values that round to infinity, whose first term is the largest number */
template <int TERMS, bool BIG = false> __device__ __forceinline__ void attn_terms(const float (&x)[8], u32x4 (&t)[TERMS]) {
    floatx2 r[4];
#pragma unroll
    for (int p = 0; p < 4; ++p) r[p] = (floatx2){ x[2 * p], x[2 * p + 1] };
#pragma unroll
    for (int k = 0; k < TERMS; ++k) {
        u32 w[4];
#pragma unroll
        for (int p = 0; p < 4; ++p) {
            w[p] = __builtin_bit_cast(u32, __builtin_convertvector(r[p], bf16x2));
            if (BIG && TERMS > 1 && !k) {
                if ((w[p] & 0x7fffu) == 0x7f80u && fabsf(r[p].x) < INFINITY) w[p] -= 1;
                if ((w[p] & 0x7fff0000u) == 0x7f800000u && fabsf(r[p].y) < INFINITY) w[p] -= 0x10000u;
            }
            if (k + 1 < TERMS) r[p] -= (floatx2){ bf_lo(w[p]), bf_hi(w[p]) };
        }
        t[k] = (u32x4){ w[0], w[1], w[2], w[3] };
    }
}

/* the sum of eight probabilities: of bf16 rows as they were rounded, so that their weights add up to one */
template <int TERMS> __device__ __forceinline__ float attn_sum(float l, const float (&p)[8], u32x4 t) {
    if constexpr (TERMS > 1) return l + (((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7])));
    else {
        const bf16x2 one = { (__bf16)1.0f, (__bf16)1.0f };
#pragma unroll
        for (int i = 0; i < 4; ++i) l = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, (u32)t[i]), one, l, false);
        return l;
    }
}

/* ---- who does what ------------------------------------------------------------------------------------
 * The plan (kernel_params.h) of the table: pieces of equal length, by all the work that there is (the lengths are known here
 * alone); a piece's sums go to the scratch, and attn_join adds them up.  Items are numbered over all sequences. */
typedef struct {
    u32 first, rows, len, row;  /* the sequence */
    u32 r0, nr, pos_lo, pos_hi, lo_step, sink_steps, steps; /* the tile, as nk_attn_tile_t */
    u32 from, to;               /* the piece's */
    u32 split, item;            /* whether it has other pieces; this one's number over all */
} attn_work_t;

__device__ __forceinline__ u32 attn_row(const NkAttnKvArgs &a, u32 r) { return nk_attn_row(&a, r); }
__device__ __forceinline__ u32 attn_tiles(const NkAttnKvArgs &a, const kvseq_t &s) { return s.ok ? nk_attn_tiles(&a, s.rows) : 0; }
__device__ __forceinline__ kvseq_t attn_seq(const NkAttnKvArgs &a, u32 i) {
    return kvseq_load(a.seqs, i, a.M, a.max_rows, a.kv.tables, min(kv_room(a.kv), (u64)a.max_len));
}
/* the sequence of this lane, of the first 64 */
__device__ __forceinline__ kvseq_t attn_mine(const NkAttnKvArgs &a) { return attn_seq(a, min(threadIdx.x & 63, a.nseq - 1)); }
/* steps of a piece; 0: nothing is split.  All wavefronts of all workgroups come to the same. */
__device__ __forceinline__ u32 attn_piece(const NkAttnKvArgs &a, kvseq_t s) {
    const u32 lane = threadIdx.x & 63;
    if (!a.slots) return 0;
    u32 tiles = 0;
    float steps = 0.0f;
#pragma unroll 4
    for (u32 i = lane; i < a.nseq; i += 64) {
        if (i != lane) s = attn_seq(a, i);
        const u32 n = attn_tiles(a, s);
        tiles += n;
        steps += nk_attn_all_steps(&a, n, s.len, s.rows);
    }
    tiles = lane_of(wave_scan(tiles), 63);
    return tiles < a.slots ? nk_attn_piece(&a, tiles, wsum(steps)) : 0;
}
__device__ __forceinline__ u32 attn_pieces(const NkAttnKvArgs &a, const kvseq_t &s, u32 piece) { return nk_attn_pieces(&a, s.len, s.rows, piece); }
/* a sequence's are all alike */
__device__ __forceinline__ u32 attn_piece_of(const NkAttnKvArgs &a, const kvseq_t &s, u32 pieces) { return nk_attn_piece_of(&a, s.len, s.rows, pieces); }
__device__ __forceinline__ void attn_tile(const NkAttnKvArgs &a, const kvseq_t &s, u32 tile, attn_work_t &w) {
    const nk_attn_tile_t t = nk_attn_tile(&a, s.len, s.rows, tile);
    w.first = s.first, w.rows = s.rows, w.len = s.len, w.row = s.row;
    w.r0 = t.r0, w.nr = t.nr, w.pos_lo = t.pos_lo, w.pos_hi = t.pos_hi;
    w.lo_step = t.lo_step, w.sink_steps = t.sink_steps, w.steps = t.steps;
}
__device__ __forceinline__ void attn_uniform(attn_work_t &w) {
    u32 *p = &w.first;
#pragma unroll
    for (u32 i = 0; i < sizeof w / 4; ++i) p[i] = (u32)__builtin_amdgcn_readfirstlane((int)p[i]);
}
__device__ __forceinline__ bool attn_find(const NkAttnKvArgs &a, u32 id, attn_work_t &w) {
    const kvseq_t mine = attn_mine(a);
    const u32 piece = attn_piece(a, mine);
    const kvitem_t it = kv_find(a.nseq, id, mine, [&](u32 i) { return attn_seq(a, i); }, [&](const kvseq_t &s) {
        const u32 n = attn_tiles(a, s);
        return n ? n * attn_pieces(a, s, piece) : 0;
    });
    if (!it.found) return false;
    const u32 pieces = attn_pieces(a, it.seq, piece);
    w.item = id;
    attn_tile(a, it.seq, it.local / pieces, w);
    const u32 len = pieces > 1 ? attn_piece_of(a, it.seq, pieces) : w.steps;
    w.from = it.local % pieces * len;
    w.to = min(w.steps, w.from + len);
    w.split = w.steps > w.to - w.from;
    attn_uniform(w); /* or the compiler keeps all that follows from it per lane */
    return true;
}
/* a piece's place in the scratch: m and l of its rows, then their sums */
__device__ __forceinline__ float *attn_part(const NkAttnKvArgs &a, u32 item, u32 h) {
    return a.ws + (((u64)item * a.kv.heads + h) << a.tile) * (a.kv.dh + 2);
}

/* the page of a token, the same for all lanes (nothing writes the table meanwhile) */
__device__ __forceinline__ int attn_page(const NkKv &kv, u32 row, u32 token) {
    return ((const __attribute__((address_space(4))) int *)kv.table)[(u64)row * kv.ldt + (token >> kv.shift)];
}

__device__ __forceinline__ float kv_value(const NkKv &kv, const void *c, const unsigned char *s, u64 slot, u32 d) {
    if (!s) return bf2f(((const u16 *)c)[slot * kv.dh + d]);
    return __builtin_amdgcn_cvt_f32_fp8(((const unsigned char *)c)[slot * kv.dh + d], 0) * scale8(s[slot / NK_KV_BLOCK]);
}
__device__ __forceinline__ float ld_q(const float *p) { return *p; }
__device__ __forceinline__ float ld_q(const u16 *p) { return bf2f(*p); }
__device__ __forceinline__ void st_o(float *p, float v) { *p = v; }
__device__ __forceinline__ void st_o(u16 *p, float v) { *p = (u16)pk_bf16(v, 0.0f); }

/* Packed row r of a sequence by the formula: one wavefront, first the maximum, then the sums; 64 tokens at a time, a token a
 * lane for the logits and a lane's dims d = lane, lane + 64, ... for the sums.  No token seen: zeros.  Some 0.1 us a token. */
template <typename T> __device__ __forceinline__ void attn_by_formula(const NkAttnKvArgs &a, u32 first, u32 len, u32 row, u32 r, u32 h) {
    const NkKv &kv = a.kv;
    const u32 lane = threadIdx.x & 63, i = attn_row(a, r), p = len + i;
    const u64 at = (u64)(h * a.group + r - i * a.group) * kv.dh;
    const T *q = (const T *)a.q + (u64)(first + i) * a.ldq + at;
    T *o = (T *)a.o + (u64)(first + i) * a.ldo + at;
    const u32 lo = a.window && p >= a.window ? p + 1 - a.window : 0, sinks = a.window ? min(a.sinks, lo) : 0, n = sinks + p + 1 - lo;
    float m = -INFINITY, l = 0.0f, acc[4] = { 0.0f, 0.0f, 0.0f, 0.0f };
    u64 any = 0;
    bool nan = false;
    for (int pass = 0; pass < 2 && !nan; ++pass)
        for (u32 k0 = 0; k0 < n; k0 += 64) {
            const u32 k = min(k0 + lane, n - 1), j = k < sinks ? k : lo + k - sinks;
            const int pe = kv.table[(u64)row * kv.ldt + (j >> kv.shift)];
            const bool see = k0 + lane < n && (u32)pe < kv.pages;
            const u64 seen = __ballot(see);
            if (!seen) continue;
            const u64 slot = (((u64)(u32)(see ? pe : 0) * kv.heads + h) << kv.shift) + (j & ((1u << kv.shift) - 1));
            float s = 0.0f;
            for (u32 d = 0; d < kv.dh; ++d) s = fmaf(ld_q(q + d), kv_value(kv, kv.k, kv.ks, slot, d), s);
            s *= a.scale;
            if (!pass) {
                any |= seen;
                nan |= __ballot(see && s != s) != 0;
                m = fmaxf(m, wmax(see && s == s ? s : -INFINITY));
                if (nan) break;
                continue;
            }
            const float e = see ? expf(s - m) : 0.0f;
            l += e;
            for (u32 t0 = 0; t0 < 64; t0 += 8) {
                float v[8][4];
#pragma unroll
                for (u32 t = 0; t < 8; ++t) {
                    const u64 st = (u64)lane_of((u32)(slot >> 32), (int)(t0 + t)) << 32 | lane_of((u32)slot, (int)(t0 + t));
#pragma unroll
                    for (int u = 0; u < 4; ++u) v[t][u] = 64 * u < (int)kv.dh ? kv_value(kv, kv.v, kv.vs, st, min(lane + 64 * u, kv.dh - 1)) : 0.0f;
                }
#pragma unroll
                for (u32 t = 0; t < 8; ++t)
                    if (seen >> (t0 + t) & 1) {
                        const float g = __uint_as_float(lane_of(__float_as_uint(e), (int)(t0 + t)));
#pragma unroll
                        for (int u = 0; u < 4; ++u) acc[u] = fmaf(g, v[t][u], acc[u]);
                    }
            }
        }
    l = wave_sum(l);
#pragma unroll
    for (int u = 0; u < 4; ++u)
        if (lane + 64 * u < kv.dh) st_o(o + lane + 64 * u, !any ? 0.0f : nan ? __builtin_nanf("") : acc[u] / l);
}

/* ---- few rows: wavefronts over the tokens --------------------------------------------------------------
 * A workgroup's 16 QT packed rows; its four wavefronts take every fourth step of 32 tokens, each with sums of its own that
 * are joined at the end.  Keys go from memory into fragments (a fragment's sum may take its values in any order: lane
 * group g of a chunk pair has the values 16 g on), values through the wavefront's own LDS for their columns;
 * the next step's loads are in flight.
 *
 * Bound by memory where there is much: 131071 tokens of 8 heads of 128 bf16 96 us (5.6 TB/s), 64 sequences of up to 16384
 * 8-bit tokens 203 us (5.4 TB/s).  By round trips where there is little: 1000 tokens 7.7 us, of which the table 1.6, the
 * rows' queries 0.5, page and first keys 1.5, two steps 2, joining the wavefronts and storing 1.7.  More wavefronts per SIMD
 * (registers held to 128: 8-bit steps 230 -> 300 us) or per workgroup (eight: 112 and 240) are not faster. */
#define ATTN_STEP 32
template <typename T, typename CT, int DH, int QT> __device__ __forceinline__ void attn_few(const NkAttnKvArgs &a) {
    constexpr bool E4M3 = sizeof(CT) == 1;
    constexpr int NC = DH / 32, ND = DH / 16, TERMS = sizeof(T) == 4 ? 3 : 1, ROWS = 16 * QT, NW = 4;
    constexpr int LDV = DH + 16; /* u16 of a token's row in LDS: 32 bytes more, so that four tokens' are in other banks */
    constexpr int NK = E4M3 ? DH / 64 : DH / 32, NV = E4M3 ? DH / 32 : DH / 16; /* 16-byte loads of a lane: per 16 tokens; per step */
    constexpr u32 VBYTES = NW * ATTN_STEP * LDV * 2, OBYTES = NW * 16 * DH * 4;
    __shared__ __align__(16) char lds[VBYTES > OBYTES ? VBYTES : OBYTES];
    __shared__ float wm[NW][ROWS], wl[NW][ROWS];
    __shared__ u32 wrong[ROWS];
    const NkKv &kv = a.kv;
    const u32 h = blockIdx.x % kv.heads, lane = threadIdx.x & 63, c16 = lane & 15, g4 = lane >> 4;
    const u32 wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), dh = kv.dh;
    attn_work_t w;
    if (!attn_find(a, blockIdx.x / kv.heads, w) || w.from >= w.to) return;
    if (threadIdx.x < ROWS) wrong[threadIdx.x] = 0;
    const u32 pos_lo = w.pos_lo, pos_hi = w.pos_hi;

    u32x4 qf[QT][NC][TERMS];
    u32 pos[QT];
#pragma unroll
    for (int t = 0; t < QT; ++t) {
        const u32 r = w.r0 + min(16 * t + c16, w.nr - 1), i = attn_row(a, r);
        pos[t] = w.len + i;
        const T *q = (const T *)a.q + (u64)(w.first + i) * a.ldq + (u64)(h * a.group + r - i * a.group) * dh;
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            const u32 d = 64 * (c / 2) + 16 * g4 + 8 * (c % 2);
            const T *p = q + min(d, dh - 8);
            float v[8];
            if (a.vec) kv_load<8>(v, p);
            else
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = ld_q(p + e);
            if (d >= dh)
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = 0.0f;
            attn_terms<TERMS, true>(v, qf[t][c]);
        }
    }

    u32x4 kr[2][NK], vr[NV];
    u32 ksb[2], vsb[2];
    int pe[2];
    auto token = [&](u32 u) { return (u < w.sink_steps ? u : w.lo_step + u - w.sink_steps) * ATTN_STEP; };
    auto lookup = [&](u32 u) {
#pragma unroll
        for (int b = 0; b < 2; ++b) pe[b] = attn_page(kv, w.row, min(token(u) + 16 * b, pos_hi));
    };
    bool there[2];
    auto load = [&](u32 u) { /* from the pages that pe has */
        const u32 t0 = token(u);
        u64 at[2];
        u32 last[2]; /* tokens behind the last row's are not read: that one again */
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            const u32 tb = min(t0 + 16 * b, pos_hi & ~15u);
            there[b] = (u32)pe[b] < kv.pages;
            const u64 slot = (((u64)(u32)(there[b] ? pe[b] : 0) * kv.heads + h) << kv.shift) + (tb & ((1u << kv.shift) - 1));
            at[b] = slot * dh;
            last[b] = min(pos_hi - tb, 15u);
            if constexpr (E4M3) {
                ksb[b] = kv.ks[slot / NK_KV_BLOCK];
                vsb[b] = kv.vs[slot / NK_KV_BLOCK];
            }
            const u32 tok = min(c16, last[b]);
#pragma unroll
            for (int c = 0; c < NK; ++c) {
                const u32 d = E4M3 ? min(64 * c + 16 * g4, dh - 16) : min(64 * (c / 2) + 16 * g4 + 8 * (c % 2), dh - 8);
                kr[b][c] = *(const u32x4 *)((const CT *)kv.k + at[b] + tok * dh + d);
            }
        }
        constexpr int PER = E4M3 ? DH / 16 : DH / 8; /* lanes of a token's row */
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            constexpr int each = 64 / PER;
            const int b = i * each / 16;
            const u32 tok = min(i * each % 16 + lane / PER, last[b]), d = min(lane % PER * (16 / (u32)sizeof(CT)), dh - 16 / (u32)sizeof(CT));
            vr[i] = *(const u32x4 *)((const CT *)kv.v + at[b] + tok * dh + d);
        }
    };

    floatx4 o[QT][ND];
    float m[QT], l[QT];
#pragma unroll
    for (int t = 0; t < QT; ++t) {
        m[t] = -1e30f, l[t] = 0.0f;
#pragma unroll
        for (int n = 0; n < ND; ++n) o[t][n] = (floatx4){ 0, 0, 0, 0 };
    }
    u16 *vl = (u16 *)lds + wave * ATTN_STEP * LDV;
    const float scale2 = a.scale * 1.44269504f;
    const u32 reach = a.window ? a.window : 1u << 31; /* tokens that a row sees back: what lies ahead of it is far above */

    u32 u = w.from + wave;
    if (u < w.to) {
        lookup(u);
        load(u);
        lookup(min(u + NW, w.steps - 1));
    }
#pragma unroll 1
    for (; u < w.to; u += NW) {
        const u32 t0 = token(u);
        floatx4 s[QT][2];
        const bool th[2] = { there[0], there[1] };
#pragma unroll
        for (int t = 0; t < QT; ++t) s[t][0] = s[t][1] = (floatx4){ 0, 0, 0, 0 };
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                u32x4 kf;
                if constexpr (E4M3) kf = c % 2 ? e4m3_bf16(kr[b][c / 2].z, kr[b][c / 2].w, scale8(ksb[b])) : e4m3_bf16(kr[b][c / 2].x, kr[b][c / 2].y, scale8(ksb[b]));
                else kf = kr[b][c];
#pragma unroll
                for (int t = 0; t < QT; ++t)
#pragma unroll
                    for (int k = TERMS - 1; k >= 0; --k) s[t][b] = attn_mfma(kf, qf[t][c][k], s[t][b]);
            }
        constexpr int PER = E4M3 ? DH / 16 : DH / 8, each = 64 / PER;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            u16 *p = vl + (i * each + lane / PER) * LDV + lane % PER * (16 / (u32)sizeof(CT));
            if constexpr (E4M3) {
                const float f = scale8(vsb[i * each / 16]);
                *(u32x4 *)p = e4m3_bf16(vr[i].x, vr[i].y, f);
                *(u32x4 *)(p + 8) = e4m3_bf16(vr[i].z, vr[i].w, f);
            } else *(u32x4 *)p = vr[i];
        }
        if (u + NW < w.to) {
            load(u + NW);
            lookup(min(u + 2 * NW, w.steps - 1));
        }
        const bool whole = t0 + ATTN_STEP - 1 <= pos_lo && th[0] && th[1] &&
                           (!a.window || t0 + a.window > pos_hi || t0 + ATTN_STEP <= a.sinks);
        u32x4 pf[QT][TERMS];
#pragma unroll
        for (int t = 0; t < QT; ++t) {
            if (!whole) {
#pragma unroll
                for (int b = 0; b < 2; ++b)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const u32 j = t0 + 16 * b + 4 * g4 + i;
                        const bool see = th[b] & ((pos[t] - j < reach) | ((j < a.sinks) & (j <= pos[t]) & (reach < 1u << 31)));
                        s[t][b][i] = see ? s[t][b][i] : -INFINITY;
                    }
            }
            float top = max3(max3(s[t][0][0], s[t][0][1], s[t][0][2]), max3(s[t][1][0], s[t][1][1], s[t][1][2]),
                             __builtin_elementwise_maximum(s[t][0][3], s[t][1][3]));
            top = fmaxf(m[t], max_over16(top) * scale2);
            const float old = __builtin_amdgcn_exp2f(m[t] - top);
            m[t] = top;
            float p[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) p[i] = __builtin_amdgcn_exp2f(fmaf(s[t][i / 4][i % 4], scale2, -top));
            attn_terms<TERMS>(p, pf[t]);
            l[t] = attn_sum<TERMS>(l[t] * old, p, pf[t][0]);
#pragma unroll
            for (int n = 0; n < ND; ++n) o[t][n] *= old;
        }
        asm volatile("" ::: "memory"); /* the wavefront's own LDS, in order */
#pragma unroll
        for (int n = 0; n < ND; ++n) {
            const u16 *p = vl + (4 * g4 + c16 / 4) * LDV + 16 * n + 4 * (c16 % 4);
            const uint2 x = lds_column4(p), y = lds_column4(p + 16 * LDV);
            const u32x4 vf = { x.x, x.y, y.x, y.y };
#pragma unroll
            for (int t = 0; t < QT; ++t)
#pragma unroll
                for (int k = TERMS - 1; k >= 0; --k) o[t][n] = attn_mfma(vf, pf[t][k], o[t][n]);
        }
        asm volatile("" ::: "memory");
    }

    float *part = w.split ? attn_part(a, w.item, h) : NULL;
    float *ol = (float *)lds;
#pragma unroll
    for (int t = 0; t < QT; ++t) {
        l[t] = sum_over16(l[t]);
        __syncthreads();
        if (lane < 16) wm[wave][16 * t + lane] = m[t], wl[wave][16 * t + lane] = l[t];
#pragma unroll
        for (int n = 0; n < ND; ++n) *(floatx4 *)(ol + (wave * 16 + c16) * DH + 16 * n + 4 * g4) = o[t][n];
        __syncthreads();
        for (u32 i = threadIdx.x; i < 16 * DH / 4; i += NW * 64) {
            const u32 r = i / (DH / 4), d = i % (DH / 4) * 4, rt = 16 * t + r;
            if (rt >= w.nr || d >= dh) continue;
            float top = wm[0][rt], sum = 0.0f;
#pragma unroll
            for (int k = 1; k < NW; ++k) top = fmaxf(top, wm[k][rt]);
            floatx4 v = { 0, 0, 0, 0 };
#pragma unroll
            for (int k = 0; k < NW; ++k) {
                const float f = __builtin_amdgcn_exp2f(wm[k][rt] - top);
                sum = fmaf(wl[k][rt], f, sum);
                v += f * *(const floatx4 *)(ol + (k * 16 + r) * DH + d);
            }
            if (part) {
                if (!d) part[2 * rt] = top, part[2 * rt + 1] = sum;
                *(floatx2 *)(part + (2u << a.tile) + (u64)rt * dh + d) = v.xy;
                *(floatx2 *)(part + (2u << a.tile) + (u64)rt * dh + d + 2) = v.zw;
                continue;
            }
            v /= sum;
            const u32 pr = w.r0 + rt, pi = attn_row(a, pr);
            T *out = (T *)a.o + (u64)(w.first + pi) * a.ldo + (u64)(h * a.group + pr - pi * a.group) * dh + d;
            if ((TERMS > 1 || a.pad || sum == sum) && !(fabsf(v.x) < INFINITY && fabsf(v.y) < INFINITY && fabsf(v.z) < INFINITY && fabsf(v.w) < INFINITY)) wrong[rt] = 1;
            const float e[4] = { v.x, v.y, v.z, v.w };
            if (a.vec) kv_store<4>(out, e);
            else
#pragma unroll
                for (int k = 0; k < 4; ++k) st_o(out + k, e[k]);
        }
    }
    if (part) return;
    __syncthreads();
    for (u32 r = wave; r < w.nr; r += NW)
        if (wrong[r]) attn_by_formula<T>(a, w.first, w.len, w.row, w.r0 + r, h);
}
#define ATTN_FEW(T, TN, CT, CN, DH, QT)                                                                                  \
    extern "C" __global__ __launch_bounds__(256) void attn_few_##TN##_##CN##_##DH##_##QT(const NkAttnKvArgs a) {         \
        attn_few<T, CT, DH, QT>(a);                                                                                      \
    }
#define ATTN_FEW_DH(DH, QT)                                                                                              \
    ATTN_FEW(u16, bf16, u16, bf16, DH, QT) ATTN_FEW(u16, bf16, unsigned char, e4m3, DH, QT)                              \
    ATTN_FEW(float, f32, u16, bf16, DH, QT) ATTN_FEW(float, f32, unsigned char, e4m3, DH, QT)
ATTN_FEW_DH(64, 1) ATTN_FEW_DH(128, 1) ATTN_FEW_DH(256, 1) ATTN_FEW_DH(64, 2) ATTN_FEW_DH(128, 2)
ATTN_FEW(u16, bf16, u16, bf16, 256, 2) ATTN_FEW(u16, bf16, unsigned char, e4m3, 256, 2)

/* ---- many rows: wavefronts over the rows ----------------------------------------------------------------
 * A workgroup's 128 packed rows, 32 to a wavefront, over steps of 64 tokens whose keys and values lie in LDS for all of
 * them, the next step's on the way meanwhile.  Products on 32x32x16: first S^T = K Q^T, so that a lane has one row's logits
 * (its maximum and sum are the lane's own and one swap), then O^T = V^T P^T with P straight from those registers: their
 * tokens 4 hh + (0..3) and 8 on of every 16 (hh: the lane's half) are the order in which the columns of V are read.
 * A row of LDS is DH values; its 16-byte chunks are mixed by the token so that the lanes of a read spread over all
 * banks.  The maximum follows only where a logit is 2^8 times above it: 2^(x - m) may exceed 1 as well as not, and the
 * sums are rescaled once or twice a row instead of every step.
 *
 * 8192 rows of 32 heads on 8 of 128: 561 to 575 us calls one behind another, 0.96 to 0.98 PFLOP/s of those that count, under the
 * profiler 608 in the median (0.90): 74 to 80 % of a large library product's rate.  The matrix units are busy 47 % of the
 * cycles, the vector units (206 instructions of a wavefront's step: 32 exponentials, 32 products, maxima, sums, conversions)
 * nearly as many, at the 1.8 to 2.0 GHz that the card's power leaves; what was tried beside: the next
 * step's K Q^T while this one's weights are computed (7 % fewer cycles at a lower clock, 573 us against 569), two
 * workgroups' wavefronts of different priority (no change), eight wavefronts that share rows and halve the
 * tokens (607), per-lane 64-bit addresses (610).  Heads of 64 keep three workgroups a CU. */
typedef float floatx16 __attribute__((ext_vector_type(16)));
__device__ __forceinline__ floatx16 attn_mfma32(u32x4 a, u32x4 b, floatx16 acc) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), acc, 0, 0, 0);
}
/* dma16 (see there) from a base that all lanes share and 32 bits of a lane's own, to an LDS address; it writes where nothing
 * is read before the next wait and barrier, so that the reads around it may move */
__device__ __forceinline__ void dma16_at(const char *base, u32 off, u32 to) {
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(off), "s"(base), "s"(to));
}
#define ATTN_MANY 64
template <typename T, typename CT, int DC> __device__ __forceinline__ void attn_many(const NkAttnKvArgs &a) {
    constexpr bool E4M3 = sizeof(CT) == 1;
    constexpr int DH = DC <= 64 ? 64 : DC <= 128 ? 128 : 256; /* values of a row in LDS, of which DC count */
    constexpr int NC = DC / 16, ND = DC / 32, TERMS = sizeof(T) == 4 ? 3 : 1, CH = DH / 8; /* 16-byte chunks of a row */
    constexpr int TOK = ATTN_MANY / 4;                                /* tokens that a wavefront brings: a block */
    constexpr int PER = E4M3 ? DH / 16 : DH / 8, NL = TOK * PER / 64; /* lanes to a token; loads a wavefront, of keys and of values */
    static_assert(NL >= 1 && TOK == NK_KV_BLOCK, "loads");
    constexpr u32 HALF = ATTN_MANY * DH * 2;
    __shared__ __align__(16) char lds[4 * HALF]; /* keys of two steps, values of two */
    __shared__ __align__(4) unsigned char page_of[2][4];
    const NkKv &kv = a.kv;
    const u32 h = blockIdx.x % kv.heads, lane = threadIdx.x & 63, c32 = lane & 31, hh = lane >> 5, dh = kv.dh;
    const u32 wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    attn_work_t w;
    if (!attn_find(a, blockIdx.x / kv.heads, w) || w.from >= w.to) return;
    const u32 pos_lo = w.pos_lo, pos_hi = w.pos_hi;
    const u32 row = 32 * wave + c32, pr = w.r0 + min(row, w.nr - 1), pi = attn_row(a, pr), pos = w.len + pi;
    const u64 at_head = (u64)(h * a.group + pr - pi * a.group) * dh;

    auto token = [&](u32 u) { return (u < w.sink_steps ? u : w.lo_step + u - w.sink_steps) * ATTN_MANY; };
    auto mixk = [](u32 t) { return DH == 64 ? (t >> 1) & 7 : t & 15; };
    auto mixv = [](u32 t) { return DH == 64 ? (t << 1) & 4 : (t << 2) & 12; };
    /* A wavefront brings a block of 16 tokens, from one page; whether there is one, all learn through LDS. */
    int pe;
    u64 slot;   /* of the block's first token, and the last one that is read: behind the last row, that one again */
    u32 last;
    auto lookup = [&](u32 u) { pe = attn_page(kv, w.row, min(token(min(u, w.to - 1)) + TOK * wave, pos_hi)); };
    u32x4 kr[E4M3 ? NL : 1], vr[E4M3 ? NL : 1];
    u32 ksb, vsb;
    const u32 lds0 = __builtin_amdgcn_readfirstlane((u32)(size_t)(lds_char_t *)lds) + TOK * wave * DH * 2;
    const u32 lt = lane / PER, bytes = dh * sizeof(CT), lc = lane % PER;
    auto place = [&](u32 u) { /* the block of step u, whose page pe has */
        const u32 tb = min(token(u) + TOK * wave, pos_hi & ~15u);
        const bool ok = (u32)pe < kv.pages;
        last = min(pos_hi - tb, 15u);
        slot = (((u64)(ok ? (u32)pe : 0) * kv.heads + h) << kv.shift) + (tb & ((1u << kv.shift) - 1));
        return ok;
    };
    auto load = [&](const void *from, u32 to, u32x4 &r, int i, bool v) { /* the i-th of NL loads */
        const u32 t = i * (64 / PER) + lt, at = __umul24(min(t, last), bytes);
        const char *base = (const char *)from + slot * bytes;
        if constexpr (E4M3) r = *(const u32x4 *)(base + (at + min(lc * 16, bytes - 16)));
        else dma16_at(base, at + min((lc ^ (v ? mixv(t) : mixk(t))) * 16, bytes - 16), to + i * (64 / PER) * DH * 2);
    };
    auto load_k = [&](u32 buf, int i) { load(kv.k, lds0 + buf * HALF, kr[E4M3 ? i : 0], i, false); };
    auto load_v = [&](u32 buf, int i) { load(kv.v, lds0 + (2 + buf) * HALF, vr[E4M3 ? i : 0], i, true); };
    auto put = [&](u32 to, u32 sb, u32x4 r, int i, bool v) { /* 8-bit codes from registers: two chunks a lane */
        const u32 t = TOK * wave + i * (64 / PER) + lt, x = v ? mixv(t) : mixk(t);
        const float f = scale8(sb);
        *(u32x4 *)(lds + to + t * DH * 2 + ((2 * lc) ^ x) * 16) = e4m3_bf16(r.x, r.y, f);
        *(u32x4 *)(lds + to + t * DH * 2 + ((2 * lc + 1) ^ x) * 16) = e4m3_bf16(r.z, r.w, f);
    };
    auto put_k = [&](u32 buf) {
        if constexpr (E4M3)
#pragma unroll
            for (int i = 0; i < NL; ++i) put(buf * HALF, ksb, kr[i], i, false);
    };
    auto put_v = [&](u32 buf) {
        if constexpr (E4M3)
#pragma unroll
            for (int i = 0; i < NL; ++i) put((2 + buf) * HALF, vsb, vr[i], i, true);
    };
    auto begin_k = [&](u32 u, u32 buf) {
        const bool ok = place(u);
        if (lane == 0) page_of[buf][wave] = ok;
        if constexpr (E4M3) ksb = kv.ks[slot / NK_KV_BLOCK];
    };
    auto begin_v = [&] {
        if constexpr (E4M3) vsb = kv.vs[slot / NK_KV_BLOCK];
    };

    lookup(w.from);
    begin_k(w.from, 0);
    begin_v();
#pragma unroll
    for (int i = 0; i < NL; ++i) load_k(0, i), load_v(0, i);
    lookup(w.from + 1);

    u32x4 qf[NC][TERMS];
    {
        const T *q = (const T *)a.q + (u64)(w.first + pi) * a.ldq + at_head;
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            const u32 d = 16 * c + 8 * hh;
            const T *p = q + min(d, dh - 8);
            float v[8];
            if (a.vec) kv_load<8>(v, p);
            else
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = ld_q(p + e);
            if (d >= dh)
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = 0.0f;
            attn_terms<TERMS, true>(v, qf[c]);
        }
    }
    floatx16 o[ND];
#pragma unroll
    for (int n = 0; n < ND; ++n)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[n][i] = 0.0f;
    float m = -1e30f, l = 0.0f;
    const float scale2 = a.scale * 1.44269504f;
    const u32 reach = a.window ? a.window : 1u << 31;
    /* where this lane's first reads lie; the others by xor and constant distances */
    const u32 kat = c32 * DH * 2 + ((hh ^ mixk(c32)) << 4);
    const u32 vt = 4 * hh + (lane & 15) / 4, vat = vt * DH * 2 + (((lane >> 4 & 1) * 2 + (lane & 3) / 2) ^ mixv(vt)) * 16 + (lane & 1) * 8;

    auto key = [&](u32 buf, int c, int b) { return *(const u32x4 *)(lds + buf * HALF + (kat ^ (c << 5)) + b * 32 * DH * 2); };
    auto value = [&](u32 buf, int g, int n) {
        const u16 *q = (const u16 *)(lds + (2 + buf) * HALF + (vat ^ (n << 6)) + g * 16 * DH * 2);
        const uint2 x = lds_column4(q), y = lds_column4(q + 8 * DH);
        return (u32x4){ x.x, x.y, y.x, y.y };
    };
    /* logits of tokens that a row does not see */
    auto hide = [&](floatx16 (&s)[2], u32 u, u32 buf) {
        const u32 t0 = token(u), there = (u32)__builtin_amdgcn_readfirstlane(*(const int *)page_of[buf]); /* a byte for every block */
        if (t0 + ATTN_MANY - 1 <= pos_lo && there == 0x01010101u && (t0 + reach > pos_hi || t0 + ATTN_MANY <= a.sinks)) return;
        const u32 back = pos - t0 - 4 * hh; /* how far back token t0 + 4 hh lies; what lies ahead is far above `reach` */
        if (!a.window || t0 >= a.sinks)
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
                for (int i = 0; i < 16; ++i) s[b][i] = back - (32 * b + 8 * (i / 4) + i % 4) < reach ? s[b][i] : -INFINITY;
        else {
            const u32 left = a.sinks - t0; /* > 0; and what is ahead is behind pos */
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const u32 j = 32 * b + 8 * (i / 4) + i % 4;
                    s[b][i] = (back - j < reach) | ((4 * hh + j < left) & ((int)(back - j) >= 0)) ? s[b][i] : -INFINITY;
                }
        }
        if (there != 0x01010101u)
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
                for (int i = 0; i < 16; ++i) s[b][i] = there >> (8 * (2 * b + i / 8)) & 1 ? s[b][i] : -INFINITY;
    };
    auto largest = [&](const floatx16 (&s)[2]) {
        float t[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            t[k] = __builtin_elementwise_maximum(s[0][4 * k], s[1][4 * k]);
#pragma unroll
            for (int i = 1; i < 4; ++i) t[k] = max3(t[k], s[0][4 * k + i], s[1][4 * k + i]);
        }
        return max3(t[0], t[1], __builtin_elementwise_maximum(t[2], t[3]));
    };
    auto follow = [&](float top) { /* the maximum, where it has to */
        top = max_over32(top) * scale2;
        if (__ballot(top > m + 8.0f)) {
            top = fmaxf(m, top);
            const float old = __builtin_amdgcn_exp2f(m - top);
            m = top;
            l *= old;
#pragma unroll
            for (int n = 0; n < ND; ++n) o[n] *= old;
        }
    };
    auto weights = [&](const floatx16 (&s)[2], int g, u32x4 (&pf)[TERMS]) { /* of 16 tokens */
        float p[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) p[i] = __builtin_amdgcn_exp2f(fmaf(s[g / 2][8 * (g % 2) + i], scale2, -m));
        attn_terms<TERMS>(p, pf);
        l = attn_sum<TERMS>(l, p, pf[0]);
    };

#pragma unroll 1
    for (u32 u = w.from, buf = 0; u < w.to; ++u, buf ^= 1) {
        put_k(buf);
        put_v(buf);
        wait_vm_lgkm<0>(); /* this step's keys and values, of all wavefronts; no one reads the other halves any more */
        barrier_mem();
        if (u + 1 < w.to) {
            begin_k(u + 1, buf ^ 1);
            begin_v();
#pragma unroll
            for (int i = 0; i < NL; ++i) load_k(buf ^ 1, i), load_v(buf ^ 1, i);
            lookup(u + 2);
        }
        floatx16 s[2];
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int i = 0; i < 16; ++i) s[b][i] = 0.0f;
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                const u32x4 kf = key(buf, c, b);
#pragma unroll
                for (int k = TERMS - 1; k >= 0; --k) s[b] = attn_mfma32(kf, qf[c][k], s[b]);
            }
        hide(s, u, buf);
        follow(largest(s));
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            u32x4 pf[TERMS];
            weights(s, g, pf);
#pragma unroll
            for (int n = 0; n < ND; ++n) {
                const u32x4 vf = value(buf, g, n);
#pragma unroll
                for (int k = TERMS - 1; k >= 0; --k) o[n] = attn_mfma32(vf, pf[k], o[n]);
            }
        }
    }

    l = sum_over32(l);
    if (w.split) {
        float *part = attn_part(a, w.item, h);
        if (row < w.nr) {
            if (!hh) part[2 * row] = m, part[2 * row + 1] = l;
#pragma unroll
            for (int n = 0; n < ND; ++n)
#pragma unroll
                for (int i = 0; i < 16; i += 4) {
                    const u32 d = 32 * n + 2 * i + 4 * hh;
                    if (d < dh) *(floatx4 *)(part + (2u << a.tile) + (u64)row * dh + d) = (floatx4){ o[n][i], o[n][i + 1], o[n][i + 2], o[n][i + 3] };
                }
        }
        return;
    }
    bool bad = false;
    if (row < w.nr) {
        T *out = (T *)a.o + (u64)(w.first + pi) * a.ldo + at_head;
#pragma unroll
        for (int n = 0; n < ND; ++n)
#pragma unroll
            for (int i = 0; i < 16; i += 4) {
                const u32 d = 32 * n + 2 * i + 4 * hh;
                if (d >= dh) continue;
                float e[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    e[k] = o[n][i + k] / l;
                    bad |= (TERMS > 1 || a.pad || l == l) && !(fabsf(e[k]) < INFINITY);
                }
                if (a.vec) kv_store<4>(out + d, e);
                else
#pragma unroll
                    for (int k = 0; k < 4; ++k) st_o(out + d + k, e[k]);
            }
    }
    u64 wrong = __ballot(bad);
    for (wrong = (wrong | wrong >> 32) & 0xffffffffu; wrong; wrong &= wrong - 1)
        attn_by_formula<T>(a, w.first, w.len, w.row, w.r0 + 32 * wave + (u32)__ffsll((unsigned long long)wrong) - 1, h);
}
#define ATTN_MANY_K(T, TN, CT, CN, DC, OCC)                                                                          \
    extern "C" __global__ __launch_bounds__(256, OCC) void attn_many_##TN##_##CN##_##DC(const NkAttnKvArgs a) {      \
        attn_many<T, CT, DC>(a);                                                                                     \
    }
#define ATTN_MANY_DC(DC, OCC)                                                                                        \
    ATTN_MANY_K(u16, bf16, u16, bf16, DC, OCC) ATTN_MANY_K(u16, bf16, unsigned char, e4m3, DC, OCC)                  \
    ATTN_MANY_K(float, f32, u16, bf16, DC, OCC) ATTN_MANY_K(float, f32, unsigned char, e4m3, DC, OCC)
ATTN_MANY_K(u16, bf16, u16, bf16, 64, 3) ATTN_MANY_K(u16, bf16, unsigned char, e4m3, 64, 3)
ATTN_MANY_K(float, f32, u16, bf16, 64, 2) ATTN_MANY_K(float, f32, unsigned char, e4m3, 64, 2)
ATTN_MANY_DC(96, 2) ATTN_MANY_DC(128, 2) ATTN_MANY_DC(192, 1) ATTN_MANY_DC(256, 1)

/* The pieces of split sequences added up: a wavefront per packed row, or (share) four; a lane has
 * two neighbouring sums (and two more 128 on), eight pieces' in flight. */
template <typename T> __device__ __forceinline__ void attn_join(const NkAttnKvArgs &a) {
    __shared__ float4 sums[3][64];
    __shared__ float total[3];
    const u32 lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), h = blockIdx.y, dh = a.kv.dh;
    const kvseq_t mine = attn_mine(a);
    const u32 piece = attn_piece(a, mine);
    if (!piece) return;
    auto load = [&](u32 i) { return attn_seq(a, i); };
    const kvitem_t it = kv_find(a.nseq, blockIdx.x, mine, load, [&](const kvseq_t &s) {
        const u32 n = attn_tiles(a, s);
        return n && attn_pieces(a, s, piece) > 1 ? n : 0;
    });
    if (!it.found) return;
    u32 before = 0; /* items of the sequences before this one */
#pragma unroll 4
    for (u32 i = lane; i < it.i; i += 64) {
        const kvseq_t s = i == lane ? mine : load(i);
        const u32 n = attn_tiles(a, s);
        before += n ? n * attn_pieces(a, s, piece) : 0;
    }
    before = lane_of(wave_scan(before), 63);
    attn_work_t w;
    attn_tile(a, it.seq, it.local, w);
    const u32 all = attn_pieces(a, it.seq, piece), pieces = (w.steps - 1) / attn_piece_of(a, it.seq, all) + 1, item = before + it.local * all;
    if (pieces == 1 || item + pieces > a.items) return; /* items: of a table that has a row twice, or the scratch holds them */
    const u64 stride = ((u64)a.kv.heads << a.tile) * (dh + 2);
    const bool shared = a.share;
    const u32 begin = shared ? wave : 0, by = shared ? 4 : 1, d0 = min(2 * lane, dh - 2), d1 = min(128 + 2 * lane, dh - 2);
    for (u32 r = shared ? blockIdx.z : blockIdx.z * 4 + wave; r < w.nr; r += gridDim.z * (shared ? 1 : 4)) {
        const float *part = attn_part(a, item, h), *rows = part + (2u << a.tile) + (u64)r * dh;
        float top = -1e30f;
        for (u32 k = lane; k < pieces; k += 64) top = fmaxf(top, part[k * stride + 2 * r]);
        top = wmax(top);
        float sum = 0.0f;
        floatx2 v = { 0, 0 }, v1 = { 0, 0 };
        for (u32 k0 = 0; k0 < pieces; k0 += 64) {
            const float *p = part + min(k0 + lane, pieces - 1) * stride + 2 * r;
            const float f = k0 + lane < pieces ? __builtin_amdgcn_exp2f(p[0] - top) : 0.0f, l = f * p[1];
            const u32 n = min(pieces - k0, 64u);
            for (u32 k = begin; k < n; k += 8 * by) {
                floatx2 x[8], y[8];
#pragma unroll
                for (u32 e = 0; e < 8; ++e) {
                    const float *q = rows + (u64)(k0 + min(k + e * by, n - 1)) * stride;
                    x[e] = *(const floatx2 *)(q + d0);
                    if (dh > 128) y[e] = *(const floatx2 *)(q + d1);
                }
#pragma unroll
                for (u32 e = 0; e < 8; ++e)
                    if (k + e * by < n) {
                        const float g = __uint_as_float(lane_of(__float_as_uint(f), (int)(k + e * by)));
                        v += g * x[e];
                        if (dh > 128) v1 += g * y[e];
                        sum += __uint_as_float(lane_of(__float_as_uint(l), (int)(k + e * by)));
                    }
            }
        }
        if (shared) {
            __syncthreads();
            if (wave) {
                sums[wave - 1][lane] = make_float4(v.x, v.y, v1.x, v1.y);
                total[wave - 1] = sum;
            }
            __syncthreads();
            if (wave) continue;
#pragma unroll
            for (int k = 0; k < 3; ++k) {
                const float4 q = sums[k][lane];
                v += (floatx2){ q.x, q.y };
                v1 += (floatx2){ q.z, q.w };
                sum += total[k];
            }
        }
        const u32 pr = w.r0 + r, pi = attn_row(a, pr);
        T *out = (T *)a.o + (u64)(w.first + pi) * a.ldo + (u64)(h * a.group + pr - pi * a.group) * dh;
        const float e[4] = { v.x / sum, v.y / sum, v1.x / sum, v1.y / sum };
        bool bad = false;
#pragma unroll
        for (u32 k = 0; k < 4; ++k) {
            const u32 d = 128 * (k / 2) + 2 * lane + k % 2;
            if (d < dh) {
                bad |= (sizeof(T) == 4 || a.pad || sum == sum) && !(fabsf(e[k]) < INFINITY);
                st_o(out + d, e[k]);
            }
        }
        if (__ballot(bad)) attn_by_formula<T>(a, w.first, w.len, w.row, pr, h);
    }
}
extern "C" __global__ __launch_bounds__(256) void attn_join_f32(const NkAttnKvArgs a) { attn_join<float>(a); }
extern "C" __global__ __launch_bounds__(256) void attn_join_bf16(const NkAttnKvArgs a) { attn_join<u16>(a); }
