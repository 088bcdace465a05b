/* The paged key and value cache: rows rotated by their positions and appended, and read back.  Every table entry is
 * checked here against the buffers' sizes, and a sequence or a page that does not fit is left out. */
#include "nk_common.h"

typedef struct {
    u32 first, rows, len, row;
    bool ok;
} kvseq_t;
__device__ __forceinline__ kvseq_t kvseq_load(const int *seqs, u32 i, u32 M, u32 max_rows, u32 tables, u64 room) {
    const int4 q = ((const int4 *)seqs)[i];
    return (kvseq_t){ (u32)q.x, (u32)q.y, (u32)q.z, (u32)q.w, nk_kv_seq_ok(q.x, q.y, q.z, q.w, M, max_rows, tables, room) != 0 };
}
__device__ __forceinline__ u64 kv_room(const NkKv &kv) { return (u64)kv.ldt << kv.shift; }

/* blocks of 16 tokens that a sequence's rows touch */
__device__ __forceinline__ u32 kv_blocks(const kvseq_t &s) {
    return s.ok && s.rows ? (s.len % NK_KV_BLOCK + s.rows - 1) / NK_KV_BLOCK + 1 : 0;
}

/* sums over the lanes up to this one (rows of 16, then what the rows before have) */
__device__ __forceinline__ u32 wave_scan(u32 v) {
#define SCAN_DPP(CTRL, ROWS) v += (u32)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xF, false)
    SCAN_DPP(0x111, 0xF); /* row_shr 1, 2, 4, 8 */
    SCAN_DPP(0x112, 0xF);
    SCAN_DPP(0x114, 0xF);
    SCAN_DPP(0x118, 0xF);
    SCAN_DPP(0x142, 0xA); /* the last of a row to the next one, of the second to the upper two */
    SCAN_DPP(0x143, 0xC);
#undef SCAN_DPP
    return v;
}
__device__ __forceinline__ u32 lane_of(u32 v, int lane) { return (u32)__builtin_amdgcn_readlane((int)v, lane); }

/* The sequence that has number `id` when every sequence has count(it) of them, and its number there.  Every wavefront
 * looks by itself: `mine` is this lane's of the first 64, or, of more, four to a lane and 256 at a time by load(i). */
typedef struct {
    kvseq_t seq;
    u32 i, local;
    bool found;
} kvitem_t;
__device__ __forceinline__ kvseq_t kvseq_of(const kvseq_t &s, int lane) {
    return (kvseq_t){ lane_of(s.first, lane), lane_of(s.rows, lane), lane_of(s.len, lane), lane_of(s.row, lane), true };
}
template <typename L, typename F> __device__ __forceinline__ kvitem_t kv_find(u32 nseq, u32 id, const kvseq_t &mine, L load, F count) {
    const u32 lane = threadIdx.x & 63;
    if (nseq <= 64) {
        const u32 n = lane < nseq ? count(mine) : 0, sum = wave_scan(n);
        const u64 past = __ballot(sum > id);
        const int at = past ? __ffsll((unsigned long long)past) - 1 : 63;
        return (kvitem_t){ kvseq_of(mine, at), (u32)at, id - lane_of(sum - n, at), past != 0 };
    }
    u32 before = 0;
    for (u32 i0 = 0; i0 < nseq; i0 += 256) {
        kvseq_t s[4];
        u32 n[4], all = 0;
#pragma unroll
        for (u32 k = 0; k < 4; ++k) s[k] = load(min(i0 + 4 * lane + k, nseq - 1));
#pragma unroll
        for (u32 k = 0; k < 4; ++k) all += n[k] = i0 + 4 * lane + k < nseq ? count(s[k]) : 0;
        const u32 sum = wave_scan(all);
        const u64 past = __ballot(before + sum > id);
        if (past) {
            const int at = __ffsll((unsigned long long)past) - 1;
            u32 local = id - before - lane_of(sum - all, at), k = 0;
            kvseq_t q = kvseq_of(s[0], at);
#pragma unroll
            for (u32 e = 0; e < 3; ++e) {
                const u32 here = lane_of(n[e], at);
                if (k == e && local >= here) {
                    local -= here;
                    k = e + 1;
                    q = kvseq_of(s[e + 1], at);
                }
            }
            return (kvitem_t){ q, i0 + 4 * (u32)at + k, local, true };
        }
        before += lane_of(sum, 63);
    }
    return (kvitem_t){ mine, 0, 0, false };
}

/* P values of a row as f32, and back */
template <int P> __device__ __forceinline__ void kv_load(float (&v)[P], const float *p) {
    if constexpr (P % 4 == 0)
#pragma unroll
        for (int i = 0; i < P; i += 4) {
            const float4 q = *(const float4 *)(p + i);
            v[i] = q.x, v[i + 1] = q.y, v[i + 2] = q.z, v[i + 3] = q.w;
        }
    else
#pragma unroll
        for (int i = 0; i < P; ++i) v[i] = p[i];
}
template <int P> __device__ __forceinline__ void kv_load(float (&v)[P], const u16 *p) {
    u32 w[(P + 1) / 2];
    if constexpr (P == 8) *(uint4 *)w = *(const uint4 *)p;
    else if constexpr (P == 4) *(uint2 *)w = *(const uint2 *)p;
    else {
        static_assert(P == 1, "P");
        w[0] = *p;
    }
#pragma unroll
    for (int i = 0; i < P; ++i) v[i] = i & 1 ? bf_hi(w[i / 2]) : bf_lo(w[i / 2]);
}
template <int P> __device__ __forceinline__ void kv_store(float *p, const float (&v)[P]) {
    if constexpr (P % 4 == 0)
#pragma unroll
        for (int i = 0; i < P; i += 4) *(float4 *)(p + i) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
    else
#pragma unroll
        for (int i = 0; i < P; ++i) p[i] = v[i];
}
__device__ __forceinline__ u32 pk_bf16(float a, float b) {
    return __builtin_bit_cast(u32, __builtin_convertvector((floatx2){ a, b }, bf16x2));
}
template <int P> __device__ __forceinline__ void kv_store(u16 *p, const float (&v)[P]) {
    if constexpr (P == 8) *(uint4 *)p = make_uint4(pk_bf16(v[0], v[1]), pk_bf16(v[2], v[3]), pk_bf16(v[4], v[5]), pk_bf16(v[6], v[7]));
    else if constexpr (P == 4) *(uint2 *)p = make_uint2(pk_bf16(v[0], v[1]), pk_bf16(v[2], v[3]));
    else *p = (u16)pk_bf16(v[0], 0.0f);
}
__device__ __forceinline__ u32 pk_e4m3(float a, float b, float c, float d) {
    const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return (u32)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, lo, true);
}
template <int P> __device__ __forceinline__ void kv_store8(unsigned char *p, const float (&v)[P], float s) {
    if constexpr (P == 8)
        *(uint2 *)p = make_uint2(pk_e4m3(v[0] * s, v[1] * s, v[2] * s, v[3] * s), pk_e4m3(v[4] * s, v[5] * s, v[6] * s, v[7] * s));
    else if constexpr (P == 4) *(u32 *)p = pk_e4m3(v[0] * s, v[1] * s, v[2] * s, v[3] * s);
    else *p = (unsigned char)pk_e4m3(v[0] * s, 0.0f, 0.0f, 0.0f);
}
__device__ __forceinline__ float4 e4m3_f32(u32 w) {
    return make_float4(__builtin_amdgcn_cvt_f32_fp8((int)w, 0), __builtin_amdgcn_cvt_f32_fp8((int)w, 1),
                       __builtin_amdgcn_cvt_f32_fp8((int)w, 2), __builtin_amdgcn_cvt_f32_fp8((int)w, 3));
}
/* 2^(b - 127) of a scale byte, and its reciprocal; bytes are 10 (whose least code is 2^-126) to 247 */
__device__ __forceinline__ float scale8(u32 b) { return __uint_as_float(b << 23); }

/* cos and sin of position * freq: the angle reaches 10^6 and more, so its turns are counted in 64 bits and only the
 * part within an eighth of a turn of a quarter goes on in 32. */
__device__ __forceinline__ float2 kv_turn(u32 pos, float freq, float amp) {
    const double q = (double)pos * ((double)freq * (4.0 / 6.283185307179586476925)), n = rint(q);
    float s, c;
    sincospif(0.5f * (float)(q - n), &s, &c);
    const u32 k = (u32)(int)fma(-4.0, floor(n * 0.25), n); /* n mod 4; of a freq that is not finite: anything, s and c are NaN */
    const float x = k & 1 ? -s : c, y = k & 1 ? c : s;
    return make_float2(amp * (k & 2 ? -x : x), amp * (k & 2 ? -y : y));
}

/* The same in 64 bits: the codes of 8-bit keys.  Half a step of theirs is 2^-4 of a value, so that a rounding on the way
 * (2^-24) next to a border between two codes would move the value by a whole step. */
__device__ __forceinline__ double2 kv_turn64(u32 pos, float freq, float amp) {
    const double q = (double)pos * ((double)freq * (2.0 / 6.283185307179586476925)), n = rint(q);
    double s, c;
    sincospi(q - n, &s, &c);
    const double f = fma(-2.0, floor(n * 0.5), n) != 0.0 ? -(double)amp : (double)amp;
    return make_double2(f * c, f * s);
}
/* to f32 with the last bit set where it is not exact: rounds on to fewer bits as the value itself does */
__device__ __forceinline__ float to_odd(double d) {
    const float f = (float)d;
    const double b = (double)f;
    u32 u = __float_as_uint(f);
    if (b != d) u = (u - (fabs(b) > fabs(d))) | 1u;
    return __uint_as_float(u);
}

#define KV_PAIRS 128 /* dh / 2 at most */

/* A workgroup takes the rows of a sequence that fall into one block of 16 tokens; its wavefronts take heads, one at a
 * time: of the queries, or (behind a.qgroups in y) of the keys and the values.  The block's cosines and sines are computed
 * once for all of them.
 * Values go in pairs of P at a time: pair (i, i + rot / 2), or interleaved (2 i, 2 i + 1), and as they are behind the
 * rotated part.  8 bits: the block's scale is the least power of two of which 448 times reach the largest new value
 * and at least that of the tokens that the block has; where it grows, their codes are rounded again (exactly, but for
 * those that become subnormal).
 *
 * Bound by memory: 17.8 thousand f32 rows of 20 heads of 96 into bf16 43 us (5.8 TB/s, part of it from the caches; 57 us, 4.3
 * TB/s, with rows from HBM).  8 bits: 8192 bf16 rows of 48 heads of 128 56 us, 3.3 TB/s: the keys' sums in 64 bits take
 * registers (three wavefronts a SIMD; in f32 38 us, with two or three of 8 million codes a step off).  Loading the rows twice
 * instead of keeping them is as fast with warm caches and 5 us slower without; four rounds in flight need 248
 * registers (70 us).  One token of 64 streams 8 us: the table, the page, the rows and the stores, each a round trip. */
template <typename T, int P, bool E4M3> __device__ __forceinline__ void kv_append(const NkAppendArgs &a) {
    __shared__ union {
        float2 f[NK_KV_BLOCK][KV_PAIRS];
        double2 d[E4M3 ? NK_KV_BLOCK : 1][E4M3 ? KV_PAIRS : 1];
    } turn;
    const bool queries = blockIdx.y < a.qgroups, wide = E4M3 && !queries;
    const NkKv &kv = a.kv;
    const u64 room = kv_room(kv);
    auto load = [&](u32 i) { return kvseq_load(a.seqs, i, a.M, a.max_rows, kv.tables, room); };
    const kvitem_t it = kv_find(a.nseq, blockIdx.x, load(min(threadIdx.x & 63, a.nseq - 1)), load, kv_blocks);
    if (!it.found) return;
    const kvseq_t s = it.seq;
    const u32 t0 = (s.len / NK_KV_BLOCK + it.local) * NK_KV_BLOCK;
    const u32 lo = max(s.len, t0) - t0, hi = min(s.len + s.rows - t0, (u32)NK_KV_BLOCK), half = a.rot / 2;
    for (u32 i = threadIdx.x; i < (hi - lo) * half; i += 256) {
        const u32 t = lo + i / half, j = i % half;
        if constexpr (E4M3)
            if (wide) turn.d[t][j] = kv_turn64(t0 + t, a.freq[j], a.amp);
        if (!wide) turn.f[t][j] = kv_turn(t0 + t, a.freq[j], a.amp);
    }
    __syncthreads();
    const int pe = kv.table[(u64)s.row * kv.ldt + (t0 >> kv.shift)];
    const bool there = (u32)pe < kv.pages;
    const u32 lane = threadIdx.x & 63, U = kv.dh / (2 * P), rp = half / P;
    const u32 tpp = U <= 64 ? 64 / U : 1, tk0 = U <= 64 ? lane / U : 0, u0 = U > 64 ? lane : tk0 < tpp ? lane % U : U;
    const u32 groups = queries ? a.qgroups : gridDim.y - a.qgroups, units = queries ? a.heads : there ? 2 * kv.heads : 0;
    for (u32 w = (queries ? blockIdx.y : blockIdx.y - a.qgroups) * 4 + threadIdx.x / 64; w < units; w += groups * 4) {
        const bool isq = queries, isv = !isq && w >= kv.heads;
        const u32 h = isv ? w - kv.heads : w, ld = isq ? a.ldq : isv ? a.ldv : a.ldk;
        const u64 row0 = (u64)s.first + t0 - s.len; /* of token t0, which may lie before the first row */
        const T *src = (const T *)(isq ? a.q : isv ? a.v : a.k) + (u64)h * kv.dh;
        auto places = [&](u32 u, u32 &oa, u32 &ob, u32 &j) {
            j = !isv && u < rp ? u * P : half; /* half: not rotated */
            const bool split = j < half && !a.inter;
            oa = split ? j : 2 * P * u;
            ob = split ? j + half : oa + P;
        };
        auto turned = [&](u32 t, u32 j, float (&x)[P], float (&y)[P]) {
            if (j >= half) return;
            auto pair = [&](int i, float &p, float &q) {
                if constexpr (E4M3)
                    if (!isq) {
                        const double2 c = turn.d[t][j + i];
                        const double v = fma((double)p, c.x, -((double)q * c.y));
                        q = to_odd(fma((double)q, c.x, (double)p * c.y));
                        p = to_odd(v);
                        if (i % 2) __builtin_amdgcn_sched_barrier(0); /* two pairs' operands at a time (f32 rows: 167 registers -> 108) */
                        return;
                    }
                const float2 c = turn.f[t][j + i];
                const float v = fmaf(p, c.x, -(q * c.y));
                q = fmaf(q, c.x, p * c.y);
                p = v;
            };
            if (P > 1 && a.inter)
#pragma unroll
                for (int i = 0; i < P / 2; ++i) {
                    pair(i, x[2 * i], x[2 * i + 1]);
                    pair(i + P / 2, y[2 * i], y[2 * i + 1]);
                }
            else
#pragma unroll
                for (int i = 0; i < P; ++i) pair(i, x[i], y[i]);
        };
        /* two rounds of the lanes at a time, their loads in flight together */
        constexpr int NB = 2;
        const u32 wraps = U <= 64 ? 1 : (U - 1) / 64 + 1, rounds = U <= 64 ? (hi - lo - 1) / tpp + 1 : (hi - lo) * wraps;
        float x[NB][P], y[NB][P];
        u32 tt[NB], oa[NB], ob[NB];
        bool in[NB];
        auto load = [&](u32 r0) {
            u32 j[NB];
#pragma unroll
            for (int i = 0; i < NB; ++i) {
                const u32 r = r0 + i, t = U <= 64 ? lo + tk0 + r * tpp : lo + r / wraps, u = U <= 64 ? u0 : u0 + 64 * (r % wraps);
                in[i] = t < hi && u < U;
                tt[i] = min(t, hi - 1);
                places(min(u, U - 1), oa[i], ob[i], j[i]);
                if (i && r >= rounds) continue; /* the same for all lanes */
                const T *row = src + (row0 + tt[i]) * ld;
                kv_load<P>(x[i], row + oa[i]);
                kv_load<P>(y[i], row + ob[i]);
            }
#pragma unroll
            for (int i = 0; i < NB; ++i)
                if (!i || r0 + i < rounds) turned(tt[i], j[i], x[i], y[i]);
        };
        auto each = [&](u32 r0, auto f) {
#pragma unroll
            for (int i = 0; i < NB; ++i)
                if (in[i] && (!i || r0 + i < rounds)) f(tt[i], oa[i], ob[i], x[i], y[i]);
        };
        if (isq) {
            T *dst = (T *)a.qo + (u64)h * kv.dh;
            for (u32 r0 = 0; r0 < rounds; r0 += NB) {
                load(r0);
                each(r0, [&](u32 t, u32 ia, u32 ib, const float(&p)[P], const float(&q)[P]) {
                    T *r = dst + (row0 + t) * a.ldqo;
                    kv_store<P>(r + ia, p);
                    kv_store<P>(r + ib, q);
                });
            }
            continue;
        }
        const u64 slot = (((u64)(u32)pe * kv.heads + h) << kv.shift) + (t0 & ((1u << kv.shift) - 1)); /* of the block's first token */
        if constexpr (!E4M3) {
            u16 *dst = (u16 *)(isv ? kv.v : kv.k) + slot * kv.dh;
            for (u32 r0 = 0; r0 < rounds; r0 += NB) {
                load(r0);
                each(r0, [&](u32 t, u32 ia, u32 ib, const float(&p)[P], const float(&q)[P]) {
                    kv_store<P>(dst + t * kv.dh + ia, p);
                    kv_store<P>(dst + t * kv.dh + ib, q);
                });
            }
        } else {
            unsigned char *sb = (isv ? kv.vs : kv.ks) + slot / NK_KV_BLOCK, *dst = (unsigned char *)(isv ? kv.v : kv.k) + slot * kv.dh;
            const u32 was = lo ? min((u32)*sb, 247u) : 0;
            float top = 0.0f;
            for (u32 r0 = 0; r0 < rounds; r0 += NB) {
                load(r0);
                each(r0, [&](u32 t, u32 ia, u32 ib, const float(&p)[P], const float(&q)[P]) {
#pragma unroll
                    for (int i = 0; i < P; ++i) {
                        top = fmaxf(top, __builtin_isinf(p[i]) ? 0.0f : fabsf(p[i]));
                        top = fmaxf(top, __builtin_isinf(q[i]) ? 0.0f : fabsf(q[i]));
                    }
                });
            }
            const u32 bits = __float_as_uint(wmax(top)), e = bits >> 23;
            const u32 now = max(max(e < 18 ? 10u : e - 8 + ((bits & 0x7fffffu) > 0x600000u), was), 10u);
            if (lo && now > was) {
                const float f = scale8(max((int)(was + 127 - now), 1)); /* below 2^-18 every code becomes 0 */
                for (u32 i = lane; i < lo * kv.dh / 4; i += 64) {
                    const float4 v = e4m3_f32(((const u32 *)dst)[i]);
                    ((u32 *)dst)[i] = pk_e4m3(v.x * f, v.y * f, v.z * f, v.w * f);
                }
            }
            if (now != was || !lo) *sb = (unsigned char)now;
            const float r = scale8(254 - now);
            for (u32 r0 = 0; r0 < rounds; r0 += NB) {
                if (rounds > NB) load(r0); /* or they are still there */
                each(r0, [&](u32 t, u32 ia, u32 ib, const float(&p)[P], const float(&q)[P]) {
                    kv_store8<P>(dst + t * kv.dh + ia, p, r);
                    kv_store8<P>(dst + t * kv.dh + ib, q, r);
                });
            }
        }
    }
}
#define KV_APPEND(T, NAME, P)                                                                                                          \
    extern "C" __global__ __launch_bounds__(256) void kv_append_##NAME##_bf16(const NkAppendArgs a) { kv_append<T, P, false>(a); }     \
    extern "C" __global__ __launch_bounds__(256) void kv_append_##NAME##_e4m3(const NkAppendArgs a) { kv_append<T, P, true>(a); }
KV_APPEND(float, f32x4, 4) KV_APPEND(float, f32x1, 1) KV_APPEND(u16, bf16x8, 8) KV_APPEND(u16, bf16x4, 4) KV_APPEND(u16, bf16x1, 1)

/* Tokens back to rows: a wavefront takes a head's keys or values of up to 16 tokens, P at a time.  Tokens of a page
 * that there is none of are zeros. */
template <typename T, int P, bool E4M3> __device__ __forceinline__ void kv_read(const NkKvReadArgs &a) {
    const NkKv &kv = a.kv;
    const u64 room = kv_room(kv);
    auto load = [&](u32 i) { return kvseq_load(a.seqs, i, a.M, a.max_rows, kv.tables, room); };
    const kvitem_t it = kv_find(a.nseq, blockIdx.x, load(min(threadIdx.x & 63, a.nseq - 1)), load, kv_blocks);
    if (!it.found) return;
    const kvseq_t s = it.seq;
    const u32 t0 = (s.len / NK_KV_BLOCK + it.local) * NK_KV_BLOCK;
    const u32 lo = max(s.len, t0) - t0, hi = min(s.len + s.rows - t0, (u32)NK_KV_BLOCK), n = kv.dh / P;
    const int pe = kv.table[(u64)s.row * kv.ldt + (t0 >> kv.shift)];
    const bool there = (u32)pe < kv.pages;
    const u32 lane = threadIdx.x & 63;
    for (u32 w = blockIdx.y * 4 + threadIdx.x / 64; w < 2 * kv.heads; w += gridDim.y * 4) {
        const bool isv = w >= kv.heads;
        const u32 h = isv ? w - kv.heads : w, ld = isv ? a.ldv : a.ldk;
        T *out = (T *)(isv ? a.v : a.k);
        if (!out) continue;
        out += ((u64)s.first + t0 - s.len) * ld + (u64)h * kv.dh;
        const u64 slot = (((u64)(u32)(there ? pe : 0) * kv.heads + h) << kv.shift) + (t0 & ((1u << kv.shift) - 1));
        float f = 1.0f;
        if constexpr (E4M3) f = there ? scale8((isv ? kv.vs : kv.ks)[slot / NK_KV_BLOCK]) : 0.0f;
        for (u32 i = lo * n + lane; i < hi * n; i += 64) {
            float v[P];
#pragma unroll
            for (int k = 0; k < P; ++k) v[k] = 0.0f;
            if (there) {
                if constexpr (!E4M3) kv_load<P>(v, (const u16 *)(isv ? kv.v : kv.k) + slot * kv.dh + (u64)i * P);
                else {
                    const unsigned char *c = (const unsigned char *)(isv ? kv.v : kv.k) + slot * kv.dh + (u64)i * P;
                    if constexpr (P == 1) v[0] = e4m3_f32(*c).x * f;
                    else
#pragma unroll
                        for (int k = 0; k < P; k += 4) {
                            const float4 q = e4m3_f32(*(const u32 *)(c + k));
                            v[k] = q.x * f, v[k + 1] = q.y * f, v[k + 2] = q.z * f, v[k + 3] = q.w * f;
                        }
                }
            }
            kv_store<P>(out + (u64)(i / n) * ld + (u64)(i % n) * P, v);
        }
    }
}
#define KV_READ(T, NAME, P)                                                                                                     \
    extern "C" __global__ __launch_bounds__(256) void kv_read_##NAME##_bf16(const NkKvReadArgs a) { kv_read<T, P, false>(a); }  \
    extern "C" __global__ __launch_bounds__(256) void kv_read_##NAME##_e4m3(const NkKvReadArgs a) { kv_read<T, P, true>(a); }
KV_READ(float, f32x4, 4) KV_READ(float, f32x1, 1) KV_READ(u16, bf16x8, 8) KV_READ(u16, bf16x1, 1)
