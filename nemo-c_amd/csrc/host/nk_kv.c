/* Launchers of the paged key and value cache and the attention over it (include/nemo_kernels.h): arguments are checked
 * before any launch; the tables lie on the device and are checked by the kernels. */
#include "nemo_kernels.h"
#include "gpu.h"
#include "../kernel_params.h"
#include <math.h>
#include <stdio.h>

static int bad(gpu_t *g, const char *what) { return gpu_fail(g, what); }
static int aligned(const void *p, uintptr_t n) { return ((uintptr_t)p & (n - 1)) == 0; }

int nk_rope_freqs(float *freq, uint32_t rot, double base, int scaling, double factor, double old_len, double lo, double hi) {
    if (!freq || !rot || rot % 2 || !(base > 0.0) || !isfinite(base) || scaling < NK_ROPE_PLAIN || scaling > NK_ROPE_TURNS) return -1;
    if (scaling != NK_ROPE_PLAIN && (!(factor > 0.0) || !isfinite(factor))) return -1;
    if (scaling == NK_ROPE_BASE && rot < 4) return -1;
    if (scaling == NK_ROPE_TURNS && (!(old_len > 0.0) || !(lo < hi) || !isfinite(old_len) || !isfinite(lo) || !isfinite(hi))) return -1;
    if (scaling == NK_ROPE_BASE) base *= pow(factor, rot / (rot - 2.0)); /* the last pair's exponent is (rot - 2) / rot */
    for (uint32_t i = 0; i < rot / 2; ++i) {
        double f = pow(base, -2.0 * i / rot);
        if (scaling == NK_ROPE_LINEAR) f /= factor;
        if (scaling == NK_ROPE_TURNS) {
            double keep = (old_len * f / 6.283185307179586476925 - lo) / (hi - lo);
            keep = keep < 0.0 ? 0.0 : keep > 1.0 ? 1.0 : keep;
            f *= keep + (1.0 - keep) / factor;
        }
        freq[i] = (float)f;
    }
    return 0;
}

#define NK_KV_SEQS 4096 /* every wavefront finds its work in the table: 16 steps of it at the most */
/* what all ask of the cache and the batch */
static const char *cache_bad(const nk_kv_t *c, NkKv *kv, const int *seqs, uint32_t nseq, uint32_t max_rows) {
    if (c->type != NK_BF16 && c->type != NK_E4M3) return "kv: a cache of bf16 or e4m3";
    if (!c->heads || c->heads > 65535 || !c->dh || c->dh % 16 || c->dh > 256) return "kv: heads of 16 to 256 values, a multiple of 16";
    if (c->page < NK_KV_BLOCK || c->page & (c->page - 1) || c->page > 1u << 20) return "kv: pages of 16 to 2^20 tokens, a power of two";
    if (!c->pages || c->pages > 0x7fffffffu || !c->k || !c->v || !aligned(c->k, 16) || !aligned(c->v, 16)) return "kv: pages, 16-byte aligned";
    if (c->type == NK_E4M3 && (!c->ks || !c->vs)) return "kv: scales of an 8-bit cache";
    if (!c->table || !aligned(c->table, 4) || !c->ldt || !c->tables || c->tables > 0x7fffffffu) return "kv: a table of pages";
    if (!seqs || !aligned(seqs, 16)) return "kv: a 16-byte aligned table of sequences";
    if (nseq > NK_KV_SEQS) return "kv: at most 4096 sequences in a call";
    if (max_rows > 1u << 30) return "kv: at most 2^30 rows a sequence";
    uint32_t shift = 0;
    while (1u << shift < c->page) ++shift;
    *kv = (NkKv){ c->k, c->v, c->type == NK_E4M3 ? c->ks : NULL, c->type == NK_E4M3 ? c->vs : NULL, c->table, c->heads, c->dh, shift,
                  c->pages, c->ldt, c->tables };
    return NULL;
}
/* the most blocks of 16 tokens that the rows of the sequences touch */
static uint64_t blocks_of(uint32_t nseq, uint32_t max_rows, uint32_t M) {
    const uint64_t by_rows = M / NK_KV_BLOCK + 2ull * nseq, by_seqs = (uint64_t)nseq * ((max_rows + NK_KV_BLOCK - 1) / NK_KV_BLOCK + 1);
    return by_rows < by_seqs ? by_rows : by_seqs;
}
static const char *cache_name(const NkKv *kv) { return kv->ks ? "e4m3" : "bf16"; }

int nk_kv_append(gpu_t *g, const nk_kv_t *c, const nk_append_t *p) {
    if (!c || !p) return bad(g, "kv_append: no arguments");
    if (!p->nseq || !p->max_rows || !p->M) return 0;
    NkKv kv;
    const char *why = cache_bad(c, &kv, p->seqs, p->nseq, p->max_rows);
    if (why) return bad(g, why);
    if (p->type != NK_F32 && p->type != NK_BF16) return bad(g, "kv_append: rows are f32 or bf16");
    const uintptr_t size = p->type == NK_F32 ? 4 : 2;
    if ((!p->q && !p->k) || !p->k != !p->v || !p->q != !p->qo) return bad(g, "kv_append: queries with a place for them, or keys and values");
    if (!aligned(p->q, size) || !aligned(p->k, size) || !aligned(p->v, size) || !aligned(p->qo, size))
        return bad(g, "kv_append: rows aligned to their values");
    const uint64_t nk = (uint64_t)kv.heads * kv.dh, nq = (uint64_t)p->heads * kv.dh;
    if ((p->q && (!p->heads || p->heads > 65535 || p->ldq < nq || p->ldqo < nq)) || (p->k && (p->ldk < nk || p->ldv < nk)))
        return bad(g, "kv_append: rows of at least all heads' values");
    if (p->q == p->qo && p->q && p->ldq != p->ldqo) return bad(g, "kv_append: queries in place keep their stride");
    if (p->rot % 2 || p->rot > kv.dh || (p->rot && (!p->freq || !aligned(p->freq, 4))))
        return bad(g, "kv_append: an even number of rotated values, at most a head's, and their frequencies");
    /* pairs at a time: as many as lie in 16 bytes, where the parts of a head and the rows allow it */
    uint32_t P = 16 / size;
    for (; P > 1; P = P == 8 ? 4 : 1) {
        const uintptr_t b = P * size;
        const uint32_t half = p->rot / 2, tail = kv.dh - p->rot;
        const int rows = (!p->q || (aligned(p->q, b) && aligned(p->qo, b) && p->ldq % P == 0 && p->ldqo % P == 0)) &&
                         (!p->k || (aligned(p->k, b) && aligned(p->v, b) && p->ldk % P == 0 && p->ldv % P == 0));
        if (half % P == 0 && tail % (2 * P) == 0 && rows) break;
    }
    const uint64_t blocks = blocks_of(p->nseq, p->max_rows, p->M);
    if (blocks > 1u << 23) return bad(g, "kv_append: more rows than a launch covers");
    uint32_t gq = p->q ? (p->heads + 3) / 4 : 0, gk = p->k ? (2 * kv.heads + 3) / 4 : 0;
    while (gq + gk > 2 && blocks * (gq + gk) > 4096) gq = (gq + 1) / 2, gk = (gk + 1) / 2;
    NkAppendArgs a = { kv, p->q, p->k, p->v, p->qo, p->freq, p->seqs, p->ldq, p->ldk, p->ldv, p->ldqo, p->heads, p->rot, p->inter != 0,
                       p->nseq, p->max_rows, p->M, gq, p->amp };
    char name[32];
    snprintf(name, sizeof name, "kv_append_%sx%u_%s", p->type == NK_F32 ? "f32" : "bf16", P, cache_name(&kv));
    gpu_next_bytes(g, (double)p->M * ((p->q ? 2.0 * size * nq : 0.0) + (p->k ? 2.0 * nk * (size + (kv.ks ? 1 : 2)) : 0.0)));
    return gpu_launch(g, name, &a, sizeof a, (uint32_t)blocks, gq + gk, 1, 256, 1, 1);
}

int nk_kv_read(gpu_t *g, const nk_kv_t *c, void *K, uint32_t ldk, void *V, uint32_t ldv, int type, const int *seqs, uint32_t nseq,
               uint32_t max_rows, uint32_t M) {
    if (!c) return bad(g, "kv_read: no cache");
    if (!nseq || !max_rows || !M || (!K && !V)) return 0;
    NkKv kv;
    const char *why = cache_bad(c, &kv, seqs, nseq, max_rows);
    if (why) return bad(g, why);
    if (type != NK_F32 && type != NK_BF16) return bad(g, "kv_read: rows are f32 or bf16");
    const uint32_t size = type == NK_F32 ? 4 : 2;
    const uint64_t nk = (uint64_t)kv.heads * kv.dh;
    if (!aligned(K, size) || !aligned(V, size) || (K && ldk < nk) || (V && ldv < nk))
        return bad(g, "kv_read: aligned rows of at least all heads' values");
    const uint32_t P = 16 / size;
    const int vec = aligned(K, 16) && aligned(V, 16) && (!K || ldk % P == 0) && (!V || ldv % P == 0);
    const uint64_t blocks = blocks_of(nseq, max_rows, M);
    if (blocks > 1u << 23) return bad(g, "kv_read: more rows than a launch covers");
    uint32_t gy = (2 * kv.heads + 3) / 4;
    while (gy > 1 && blocks * gy > 4096) gy = (gy + 1) / 2;
    NkKvReadArgs a = { kv, K, V, seqs, ldk, ldv, nseq, max_rows, M };
    char name[32];
    snprintf(name, sizeof name, "kv_read_%sx%u_%s", type == NK_F32 ? "f32" : "bf16", vec ? P : 1, cache_name(&kv));
    gpu_next_bytes(g, 2.0 * M * nk * (size + (kv.ks ? 1 : 2)));
    return gpu_launch(g, name, &a, sizeof a, (uint32_t)blocks, gy, 1, 256, 1, 1);
}

/* A launch over the sequences of more than `over` and at most `upto` rows, and the join behind it. */
typedef struct {
    NkAttnKvArgs a;
    char name[40];
    int f32;
    uint32_t x, join_x, join_z; /* workgroups; join_x 0: nothing is split */
    uint64_t floats;            /* of scratch */
} attend_t;
static const char *attend_plan(attend_t *l, NkAttnKvArgs a, int type, uint32_t over, uint32_t upto) {
    const uint32_t rows = upto < a.M ? upto : a.M, dh = a.kv.dh, heads = a.kv.heads;
    const uint64_t packed = (uint64_t)rows * a.group;
    /* Up to 64 packed rows go 16 or 32 to a workgroup whose wavefronts share the tokens, more 128 to one whose wavefronts share
     * the rows (8 heads of 128, groups of 4, 4000 tokens: 64 packed rows 18.4 us; 32000 tokens and 256 rows 67; 8192 rows 1299
     * and 566 us). */
    const int many = packed > 64, f32 = type == NK_F32;
    const uint32_t QT = packed > 16 && (dh <= 128 || !f32) ? 2 : 1, tile = many ? 128 : 16 * QT, step = many ? 64 : 32;
    const uint32_t DH = dh <= 64 ? 64 : many && dh <= 96 ? 96 : dh <= 128 ? 128 : many && dh <= 192 ? 192 : 256;
    a.over = over;
    a.upto = upto;
    a.tile = many ? 7 : 3 + QT;
    a.step = many ? 6 : 5;
    a.first = tile / a.group + 1;
    a.pad = dh < DH;
    if (a.window)
        a.reach = (uint32_t)(((uint64_t)a.window + tile / a.group + 1 + step) / step + 1 + ((uint64_t)a.sinks + step - 1) / step);
    /* tiles that there can be (and, if the rows are there, are), and the pieces that a tile can have */
    const uint64_t by_rows = (uint64_t)a.M * a.group / tile, by_seqs = a.nseq * ((packed + tile - 1) / tile);
    const uint64_t tiles = by_seqs < by_rows + a.nseq ? by_seqs : by_rows + a.nseq;
    /* Steps are split where tiles are fewer than the workgroups wanted.  Sums of few rows cost little to write and add up: three
     * rounds of workgroups, which evens out mixed lengths (64 sequences of up to 16384 tokens 241, 234 and 221 us with 512, 1024
     * and 1536), one sequence's a single round (131071 tokens 111, 117 and 124 us); 128 rows' (66 KB and as much again to
     * read) only below a workgroup per CU (1024 rows 32 us whole, 62 split for 1024; 2048 rows 65 and 114), of f32 rows, whose
     * steps are three times as long, two (1000 rows 47 and 52). */
    const uint32_t wanted = packed <= 16 ? a.nseq > 1 && upto == a.max_rows ? 1536 : 512 : many && f32 ? 512 : 256, slots = (wanted + heads - 1) / heads;
    a.least = packed <= 16 || (many && f32) ? 4 : 8;
    const uint64_t pieces = ((a.max_len + step - 1) / step + a.least - 1) / a.least;
    if (tiles > 1u << 23) return "attention_kv: more rows than a launch covers";
    uint64_t items = tiles;
    if (pieces > 1 && slots > 1 && (by_rows < by_seqs ? by_rows : by_seqs) < slots) {
        a.slots = slots;
        a.per_slot = 1.0f / (float)slots;
        a.per_cu = (float)heads / (many && f32 ? 512.0f : 256.0f);
        const uint64_t split = nk_attn_items_bound(tiles, pieces, slots, packed <= tile);
        a.items = (uint32_t)split;
        if (items < split) items = split;
    }
    if (items * heads > 1u << 23) return "attention_kv: more rows than a launch covers";
    /* two workgroups a CU from the start: long tiles beside short ones (2048 rows 63 -> 60 us) */
    a.pair = many && tiles * heads > 256 && tiles * heads <= 512;
    *l = (attend_t){ .f32 = f32, .x = (uint32_t)items * heads, .floats = (uint64_t)a.items * heads * tile * (dh + 2) };
    if (many) snprintf(l->name, sizeof l->name, "attn_many_%s_%s_%u", f32 ? "f32" : "bf16", cache_name(&a.kv), DH);
    else snprintf(l->name, sizeof l->name, "attn_few_%s_%s_%u_%u", f32 ? "f32" : "bf16", cache_name(&a.kv), DH, QT);
    if (a.slots) {
        /* a row to a workgroup, or its wavefronts a row each and going round: some 1024 workgroups, one round of them (58 x 8
         * heads x 4 rows a workgroup each 216 us with what they join, 207 so; 24 x 4 x 128 rows by 512, 1024 and 2048: 46.4,
         * 42.6, 44.1) */
        const uint64_t most = packed < tile ? packed : tile, some = tiles < slots ? tiles : slots;
        uint64_t z = 1024 / (some * heads);
        a.share = some * heads * most <= 256;
        if (a.share) z = most;
        else if (z > (most + 3) / 4) z = (most + 3) / 4;
        l->join_x = (uint32_t)some;
        l->join_z = z ? (uint32_t)z : 1;
    }
    l->a = a;
    return NULL;
}

static int attend(gpu_t *g, const attend_t *l) {
    const NkAttnKvArgs *a = &l->a;
    gpu_next_bytes(g, (l->f32 ? 8.0 : 4.0) * a->M * a->heads * a->kv.dh);
    if (gpu_launch(g, l->name, a, sizeof *a, l->x, 1, 1, 256, 1, 1)) return -1;
    if (!l->join_x) return 0;
    return gpu_launch(g, l->f32 ? "attn_join_f32" : "attn_join_bf16", a, sizeof *a, l->join_x, a->kv.heads, l->join_z, 256, 1, 1);
}

int nk_attention_kv(gpu_t *g, const nk_kv_t *c, const nk_attend_t *p) {
    if (!c || !p) return bad(g, "attention_kv: no arguments");
    if (!p->nseq || !p->max_rows || !p->M) return 0;
    NkKv kv;
    const char *why = cache_bad(c, &kv, p->seqs, p->nseq, p->max_rows);
    if (why) return bad(g, why);
    if (p->type != NK_F32 && p->type != NK_BF16) return bad(g, "attention_kv: rows are f32 or bf16");
    const uintptr_t size = p->type == NK_F32 ? 4 : 2;
    if (!p->heads || p->heads % kv.heads || p->heads / kv.heads > 1024) return bad(g, "attention_kv: heads a multiple of the cache's");
    const uint64_t nq = (uint64_t)p->heads * kv.dh;
    if (!p->q || !p->o || !aligned(p->q, size) || !aligned(p->o, size) || p->ldq < nq || p->ldo < nq)
        return bad(g, "attention_kv: aligned rows of at least all heads' values");
    if (p->q == p->o) return bad(g, "attention_kv: o must not overlap q");
    if (!(p->scale > 0.0f) || !isfinite(p->scale)) return bad(g, "attention_kv: a scale above zero");
    if (p->max_len > 1u << 30) return bad(g, "attention_kv: at most 2^30 tokens a sequence");
    const uint32_t group = p->heads / kv.heads;
    if ((uint64_t)(p->max_rows < p->M ? p->max_rows : p->M) * group > 1u << 30) return bad(g, "attention_kv: more rows than a launch covers");
    NkAttnKvArgs a = { .kv = kv, .q = p->q, .o = p->o, .seqs = p->seqs, .ldq = p->ldq, .ldo = p->ldo, .heads = p->heads, .group = group,
                       .window = p->window >= p->max_len ? 0 : p->window, .sinks = p->sinks < p->max_len ? p->sinks : p->max_len,
                       .nseq = p->nseq, .max_rows = p->max_rows, .max_len = p->max_len, .M = p->M, .inv_group = 0xffffffffu / group,
                       .scale = p->scale };
    a.vec = aligned(p->q, 16) && aligned(p->o, 4 * size) && p->ldq % (16 / size) == 0 && p->ldo % 4 == 0;
    /* Beside prompts, sequences of a few rows (the steps of a mixed batch) have a launch of their own, which splits them, where
     * a step may see more than 2048 tokens: a workgroup of many rows takes 1.2 us for 64 of them, the launches some 6 us (12
     * prompts with a window of 512 tokens 53 and 60). */
    const uint32_t few = group <= 16 ? 16 / group : 64 / group;
    const uint64_t sees = a.window && (uint64_t)a.window + a.sinks < a.max_len ? (uint64_t)a.window + a.sinks : a.max_len;
    const int mixed = p->nseq > 1 && few && sees > 2048 && (uint64_t)(p->max_rows < p->M ? p->max_rows : p->M) * group > 64;
    attend_t l[2];
    const int n = mixed ? 2 : 1;
    if (mixed && (why = attend_plan(&l[0], a, p->type, 0, few))) return bad(g, why);
    if ((why = attend_plan(&l[n - 1], a, p->type, mixed ? few : 0, p->max_rows))) return bad(g, why);
    /* one after the other on the context's stream, they share its scratch */
    const uint64_t floats = mixed && l[0].floats > l[1].floats ? l[0].floats : l[n - 1].floats;
    float *ws = floats ? gpu_scratch_ws(g, (size_t)floats) : NULL;
    if (floats && !ws) return bad(g, "attention_kv: scratch unavailable (size it before capture)");
    for (int i = 0; i < n; ++i) {
        l[i].a.ws = ws;
        if (attend(g, &l[i])) return -1;
    }
    return 0;
}
