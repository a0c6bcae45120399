/* tl_chunk.h — launch blocks and device helpers of the calls on batches of
 * chunks over a paged cache (include/tlkv.h, tl_chunk). */
#pragma once
#include "tl_common.h"
#include "tl_internal.h"

#define CK_MAX_SEQ 32          /* chunks of one launch; longer batches take several */
#define CK_MAX_CHUNKS 4096     /* chunks of one call */
#define CK_KEYS 32             /* keys of one tile */
#define CK_COLS 16             /* (row, head) columns of a narrow workgroup */
#define CK_WCOLS 128           /* ... of a wide one */

/* waves of a narrow workgroup: one workgroup to a CU; four in a launch of both kinds */
#define CK_WAVES(D) ((D) == 256 ? 4 : 8)

/* Split merge: arrival counters of the groups, zero between launches, at the
 * start of the workspace; (max, sum) pairs and partial rows follow. */
#define CK_MAX_GROUPS 4096
#define CK_CNT_PAD 4
#define CK_CNT_WORDS (CK_MAX_GROUPS * CK_CNT_PAD)
/* Counters of a group of ns splits of `cols` columns in workgroups of `waves`:
 * its own and, where one workgroup would wait for memory twice or more to read
 * them all (eight float4s of a thread at a time), one for each CK_JOIN splits that
 * are joined first.  One join / joins of eight, us: 16 columns of 256 at 30000 keys
 * 98.9 / 49.9, 14 of 128 at 16000 keys 32.0 / 17.0; where one wait suffices, 4 of 128
 * at 6000 keys, 13.1 / 13.8. */
#define CK_JOIN 8
static constexpr TL_HOSTDEV u32 ck_join_counters(u32 ns, u32 cols, u32 head_dim, u32 waves) {
    const u32 units = (cols < CK_COLS ? cols : CK_COLS) * (head_dim / 4);
    return ns > CK_JOIN && (u64)ns * units >= 2 * 8 * 64 * waves ? 1 + (ns + CK_JOIN - 1) / CK_JOIN : 1;
}
static_assert(CK_CNT_WORDS <= TL_MERGE_CNT_WORDS, "counters of a stream's workspace");

/* Keys of a wide workgroup of the attention weight: two blocks of 32 to a wave
 * halve the work on the columns per key, where they do not cost half of the
 * waves.  512 rows over 4608 keys, us with one block / two: 32/8/128 f16 91 / 63,
 * 32/8/64 Q8_0 79 / 53, but 32/8/64 f16 45 / 51 (four waves to a SIMD / two). */
static constexpr TL_HOSTDEV int ck_weight_keys(int head_dim, bool q8) {
    return head_dim == 64 ? (q8 ? 512 : 256) : head_dim == 128 && !q8 ? 512 : 256;
}

/* One chunk of a launch: its workgroups are [wg0, next wg0), ncb column blocks
 * x n_kv heads x ns key splits of them; part0 / grp0: its first partial row
 * and merge counter (ns > 1). */
struct CkSeq {
    const u32 *pages;
    float *weight;
    u32 pos, n, row, prefix, rope_skip;
    u32 wg0, ncb, ns, part0, grp0;   /* part0 counts columns */
    u32 wide;                        /* in a launch of both kinds: 128 columns to a workgroup */
    u32 cb0;                         /* wide: its first column block (a band of the chunk's) */
    u32 counters;                    /* narrow: of one group */
};

struct CkCache {
    const u16 *k, *v;          /* f16 rows, or int8 rows of a Q8_0 cache */
    const u16 *ks, *vs;        /* Q8_0 scales */
    u32 cap, n_kv, shift;      /* page_size = 1 << shift */
};

struct CkAttnParams {
    u32 wg0[CK_MAX_SEQ];       /* seq[].wg0 side by side, ~0 past n_seq */
    CkSeq seq[CK_MAX_SEQ];
    CkCache c;
    const float *q;
    float *dst, *lse;
    const u32 *first;
    const float *slopes;
    u32 n_seq, n_head, gqa, q_stride, window;
    u32 gqa_mul;               /* x / gqa = high word of x * gqa_mul (gqa 1: 0) */
    float scale, softcap, inv_cap;
    float *ws_acc;
    float2 *ws_ml;
    u32 *cnt;
};

/* host side (tl_chunk.hip) */
int tl_chunk_check(const LayerView &L, const tl_chunk *chunks, u32 n_chunk, u32 rows,
                   u32 page_size, u32 *shift);
int tl_check_layer(const tl_kv_layer *L);
int tl_check_layer_q8(const tl_kv_layer_q8 *L);
LayerView tl_view_q8(const tl_kv_layer_q8 *L);
bool tl_ranges_overlap(const void *a, u64 a_bytes, const void *b, u64 b_bytes);
/* Does one of the intervals that are written overlap another one?  Sorts them. */
struct TlSpan {
    u64 at, end;
    bool write;
};
bool tl_spans_clash(TlSpan *a, u32 n);

/* ---- device ---------------------------------------------------------------- */

typedef _Float16 h8_t __attribute__((ext_vector_type(8)));
typedef float f4_t __attribute__((ext_vector_type(4)));
typedef u32 u4_t __attribute__((ext_vector_type(4)));

#define CK_LOG2E 1.4426950408889634f
#define CK_LN2 0.6931471805599453f

/* row and head of a column; exact below 2^32 / gqa, which the host sees to */
TL_DEV u32 ck_row_of(const CkAttnParams &p, u32 col) { return p.gqa_mul ? __umulhi(col, p.gqa_mul) : col; }

/* pool row of a session's position; ~0 where its page lies outside the pool */
TL_DEV u32 ck_row(const CkCache &c, const u32 *pages, u32 p) {
    if (!pages) return p;
    const u32 pg = pages[p >> c.shift];
    return pg <= c.cap >> c.shift ? (pg << c.shift) + (p & ((1u << c.shift) - 1)) : ~0u;
}

/* index of the launch's chunk that workgroup b belongs to (wg0 rises): one
 * load of all the starts, one comparison each */
TL_DEV u32 ck_find(const u32 *wg0, u32 n_seq, u32 b) {
    if (n_seq == 1) return 0;
    const u32 lane = threadIdx.x & (CK_MAX_SEQ - 1);
    return (u32)__builtin_amdgcn_readfirstlane((int)__popc((u32)__ballot(wg0[lane] <= b)) - 1);
}

/* tanh of N scores x c.  Below 0.6 a polynomial (odd, five coefficients fitted
 * to a relative error of 3e-9): scores lie far below their cap as a rule, and
 * there the error of the capped score has to be relative to the score, not to
 * the cap.  Where one of the wave's is above, (e - 1) / (e + 1) from e = exp(2
 * x) for those (its error, 1e-7 of the cap, is relative there). */
template <int N, class T>
TL_DEV void ck_tanh(T &s, float c) {
    float top = 0.f;
#pragma unroll
    for (int e = 0; e < N; e++) {
        s[e] *= c;
        top = fmaxf(top, fabsf(s[e]));
    }
    const bool big = __any(top >= 0.6f);
    float t[N];
#pragma unroll
    for (int e = 0; e < N; e++) {
        const float x = s[e], z = x * x;
        float q = fmaf(z, -0.005895147565752268f, 0.02079596184194088f);
        q = fmaf(z, q, -0.053783826529979706f);
        q = fmaf(z, q, 0.13331924378871918f);
        q = fmaf(z, q, -0.33333298563957214f);
        t[e] = fmaf(x * z, q, x);
    }
    if (big) {
#pragma unroll
        for (int e = 0; e < N; e++) {
            const float x = s[e] > 20.f ? 20.f : s[e];
            const float y = __builtin_amdgcn_exp2f(x * (2.f * CK_LOG2E));
            const float u = (y - 1.f) * __builtin_amdgcn_rcpf(y + 1.f);
            t[e] = fabsf(x) < 0.6f ? t[e] : u;
        }
    }
#pragma unroll
    for (int e = 0; e < N; e++) s[e] = t[e];
}

/* two f32 as pairs of f16 whose sums have 22 bits of them (x - hi is exact, one
 * mixed-precision fma) */
TL_DEV void ck_split2(float x, float y, u32 &hi, u32 &lo) {
    const tl_f16x2_t h = __builtin_convertvector((tl_f32x2_t){x, y}, tl_f16x2_t);
    const tl_f32x2_t r = {fmaf((float)h.x, -1.f, x), fmaf((float)h.y, -1.f, y)};
    hi = __builtin_bit_cast(u32, h);
    lo = __builtin_bit_cast(u32, __builtin_convertvector(r, tl_f16x2_t));
}

/* power of two that brings a row's largest |x| to [2^14, 2^15), so that both
 * halves of every element that matters are normal f16 numbers: exponent of it
 * (rows of zeros, infinities or NaN: any) */
TL_DEV int ck_row_exp(float amax) {
    const int e = (int)((__float_as_uint(amax) >> 23) & 0xff) - 127;
    return 14 - (e < -100 ? -100 : e > 126 ? 126 : e);
}

/* Which keys a (row, head) column sees: [lo, lo + w) and [f, f + pw). */
struct CkSees {
    u32 lo, w, f, pw, hi, pre;
    TL_DEV void set(u32 p, u32 end, u32 window, u32 prefix, u32 first) {
        f = first;
        pre = prefix < end ? prefix : end;
        hi = p + 1;
        lo = window && hi > window ? hi - window : 0;
        lo = lo > f ? lo : f;
        w = hi > lo ? hi - lo : 0;
        pw = pre > f ? pre - f : 0;
    }
    TL_DEV bool sees(u32 key) const { return key - lo < w || key - f < pw; }
};

/* over N neighbouring lanes */
template <int N>
TL_DEV u32 group_umin(u32 x) {
#pragma unroll
    for (int o = 1; o < N; o <<= 1) {
        const u32 y = __shfl_xor(x, o);
        x = y < x ? y : x;
    }
    return x;
}
template <int N>
TL_DEV u32 group_umax(u32 x) {
#pragma unroll
    for (int o = 1; o < N; o <<= 1) {
        const u32 y = __shfl_xor(x, o);
        x = y > x ? y : x;
    }
    return x;
}
TL_DEV u32 ck_uniform(u32 x) { return (u32)__builtin_amdgcn_readfirstlane((int)x); }

/* What the columns of rows r0 .. r1 (positions p0 .. p1) see together: from the
 * positions alone, and from the range of their first positions where rows have
 * those. */
struct CkSpan {
    u32 fmin, lo, hi, max_lo, min_hi, max_f, pre;
    TL_DEV void set(u32 p0, u32 p1, u32 end, u32 window, u32 prefix, u32 first_min, u32 first_max) {
        fmin = first_min;
        max_f = first_max;
        pre = prefix < end ? prefix : end;
        lo = window && p0 + 1 > window ? p0 + 1 - window : 0;
        lo = lo > fmin ? lo : fmin;
        hi = p1 + 1;
        max_lo = window && p1 + 1 > window ? p1 + 1 - window : 0;
        max_lo = max_lo > max_f ? max_lo : max_f;
        min_hi = p0 + 1;
    }
    /* every column sees every one of the n keys from kb on */
    TL_DEV bool full(u32 kb, u32 n) const {
        return (kb >= max_lo && kb + n <= min_hi) || (kb >= max_f && kb + n <= pre);
    }
    /* some column may see one of them */
    TL_DEV bool any(u32 kb, u32 n) const {
        return (kb < hi && kb + n > lo) || (kb < pre && kb + n > fmin);
    }
};

/* The tiles of KT keys that they need: na from a0 on of the prefix, then nb
 * from b0 on. */
template <u32 KT>
struct CkTiles {
    u32 a0, na, b0, nb;
    TL_DEV void set(const CkSpan &s) {
        a0 = na = b0 = nb = 0;
        if (s.fmin < s.pre) {
            a0 = s.fmin / KT;
            na = (s.pre + KT - 1) / KT - a0;
        }
        if (s.lo < s.hi) {
            b0 = s.lo / KT;
            const u32 b1 = (s.hi + KT - 1) / KT;
            if (na && b0 < a0 + na) b0 = a0 + na;
            nb = b1 > b0 ? b1 - b0 : 0;
        }
    }
    TL_DEV u32 count() const { return na + nb; }
    TL_DEV u32 key(u32 t) const { return (t < na ? a0 + t : b0 + (t - na)) * KT; }
};

/* ---- one wave's tile of 32 keys x 16 columns, operands straight from memory --
 *
 * S^T[key][col] = K . Q^T and O^T[dim][col] += V^T . P^T run on
 * v_mfma_f32_16x16x32_f16.  Lane (i = lane & 15, g = lane >> 4):
 *   K  two sub-tiles a: row i of the matrix is key 8 * (i >> 2) + 4 * a + (i & 3),
 *      k-step s the dims 32 s + 8 g ..: one 16-byte load each;
 *   S  so the accumulators of sub-tile a hold keys 8 g + 4 a + r of column i:
 *      a lane's eight scores are keys 8 g .. 8 g + 7, which is the order in
 *      which the second product takes them (k index 8 g + e);
 *   V  the lane loads dims (D / 16) i .. of those eight keys, whole rows per 16
 *      lanes; matrix m takes the m-th of its dims: eight halves picked from
 *      eight registers, one v_perm per pair.  No transposing pass over LDS.
 * A Q8_0 element is int8 x f16, 18 bits: taken as a pair hi + lo of f16 (the
 * product's rounding and its exact remainder). */
template <int D>
struct CkTileF16 {
    static constexpr int KS = D / 32, DW = D / 32;   /* k-steps; V dwords per key and lane */
    u4_t kr[2][KS];
    u32 vr[8][DW];
    TL_DEV void load_k(const CkCache &c, u32 kvh, const u32 (&rk)[2], u32 g) {
        const char *base = (const char *)(c.k + (u64)kvh * c.cap * D);
#pragma unroll
        for (int a = 0; a < 2; a++)
#pragma unroll
            for (int s = 0; s < KS; s++)
                kr[a][s] = *(const u4_t *)(base + (u64)(rk[a] * (u32)(D * 2) + s * 64 + g * 16));
    }
    TL_DEV void load_v(const CkCache &c, u32 kvh, const u32 (&rv)[8], u32 i) {
        const char *base = (const char *)(c.v + (u64)kvh * c.cap * D);
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const char *r = base + (u64)(rv[e] * (u32)(D * 2) + i * (D / 8));
            if constexpr (DW == 2) {
                const uint2 x = *(const uint2 *)r;
                vr[e][0] = x.x;
                vr[e][1] = x.y;
            } else {
#pragma unroll
                for (int j = 0; j < DW / 4; j++) {
                    const u4_t x = *(const u4_t *)(r + 16 * j);
                    vr[e][4 * j] = x[0];
                    vr[e][4 * j + 1] = x[1];
                    vr[e][4 * j + 2] = x[2];
                    vr[e][4 * j + 3] = x[3];
                }
            }
        }
    }
    TL_DEV void take_k(const CkTileF16 &o) {
#pragma unroll
        for (int x = 0; x < 2 * KS; x++) kr[x / KS][x % KS] = o.kr[x / KS][x % KS];
    }
    TL_DEV void get_k(int a, int s, h8_t &hi, h8_t &) const { hi = __builtin_bit_cast(h8_t, kr[a][s]); }
    TL_DEV void get_v(int m, h8_t &hi, h8_t &) const {
        u4_t x;
#pragma unroll
        for (int j = 0; j < 4; j++)
            x[j] = __builtin_amdgcn_perm(vr[2 * j + 1][m >> 1], vr[2 * j][m >> 1],
                                         m & 1 ? 0x07060302u : 0x05040100u);
        hi = __builtin_bit_cast(h8_t, x);
    }
    TL_DEV void clear_v(int e) {
#pragma unroll
        for (int d = 0; d < DW; d++) vr[e][d] = 0;
    }
    TL_DEV bool odd_v(int e) const {      /* key e holds infinities or NaN */
        bool b = false;
#pragma unroll
        for (int d = 0; d < DW; d++)
            b |= (vr[e][d] & 0x7c00u) == 0x7c00u || (vr[e][d] & 0x7c000000u) == 0x7c000000u;
        return b;
    }
};

/* int8 pairs x scale as f16 pairs hi + lo */
TL_DEV void ck_q8_pair(tl_half2 v, tl_half2 d, u32 &hi, u32 &lo) {
    const tl_half2 h = v * d;
    const tl_half2 l = __builtin_elementwise_fma(v, d, -h);
    hi = __builtin_bit_cast(u32, h);
    lo = __builtin_bit_cast(u32, l);
}

template <int D>
struct CkTileQ8 {
    static constexpr int KS = D / 32, NB = D / 16;   /* k-steps; V bytes per key and lane */
    uint2 kr[2][KS];
    u32 sk[2][KS / 2];
    u32 vr[8][NB / 4];
    u16 sv[8];
    TL_DEV void load_k(const CkCache &c, u32 kvh, const u32 (&rk)[2], u32 g) {
        const char *base = (const char *)c.k + (u64)kvh * c.cap * D;
        const char *sb = (const char *)(c.ks + (u64)kvh * c.cap * KS);
#pragma unroll
        for (int a = 0; a < 2; a++) {
#pragma unroll
            for (int s = 0; s < KS; s++)
                kr[a][s] = *(const uint2 *)(base + (u64)(rk[a] * (u32)D + s * 32 + g * 8));
#pragma unroll
            for (int s = 0; s < KS / 2; s++)
                sk[a][s] = *(const u32 *)(sb + (u64)(rk[a] * (u32)(KS * 2) + s * 4));
        }
    }
    TL_DEV void load_v(const CkCache &c, u32 kvh, const u32 (&rv)[8], u32 i) {
        const char *base = (const char *)c.v + (u64)kvh * c.cap * D;
        const char *sb = (const char *)(c.vs + (u64)kvh * c.cap * KS);
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const char *r = base + (u64)(rv[e] * (u32)D + i * NB);
            if constexpr (NB == 4) {
                vr[e][0] = *(const u32 *)r;
            } else if constexpr (NB == 8) {
                const uint2 x = *(const uint2 *)r;
                vr[e][0] = x.x;
                vr[e][1] = x.y;
            } else {
                const u4_t x = *(const u4_t *)r;
#pragma unroll
                for (int j = 0; j < 4; j++) vr[e][j] = x[j];
            }
            sv[e] = *(const u16 *)(sb + (u64)(rv[e] * (u32)(KS * 2) + i * NB / 32 * 2));
        }
    }
    TL_DEV void take_k(const CkTileQ8 &o) {
#pragma unroll
        for (int x = 0; x < 2 * KS; x++) kr[x / KS][x % KS] = o.kr[x / KS][x % KS];
#pragma unroll
        for (int x = 0; x < KS; x++) sk[x / (KS / 2)][x % (KS / 2)] = o.sk[x / (KS / 2)][x % (KS / 2)];
    }
    TL_DEV void get_k(int a, int s, h8_t &hi, h8_t &lo) const {
        const u32 d = (sk[a][s >> 1] >> (16 * (s & 1))) & 0xffffu;
        const tl_half2 d2 = __builtin_bit_cast(tl_half2, d * 0x10001u);
        tl_half2 v[4];
        i8x4_to_f16(kr[a][s].x, v[0], v[1]);
        i8x4_to_f16(kr[a][s].y, v[2], v[3]);
        u4_t h, l;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            u32 x, y;
            ck_q8_pair(v[j], d2, x, y);
            h[j] = x;
            l[j] = y;
        }
        hi = __builtin_bit_cast(h8_t, h);
        lo = __builtin_bit_cast(h8_t, l);
    }
    TL_DEV void get_v(int m, h8_t &hi, h8_t &lo) const {
        u4_t h, l;
        const u32 sel = 0x0c000c00u | (u32)(m & 3) | ((u32)(4 + (m & 3)) << 16);
        const tl_half2 bias = {(_Float16)1152.0f, (_Float16)1152.0f};
#pragma unroll
        for (int j = 0; j < 4; j++) {
            /* byte m of keys 2j and 2j + 1: q + 128 under the exponent of 1024 */
            const u32 b = __builtin_amdgcn_perm(vr[2 * j + 1][m >> 2], vr[2 * j][m >> 2], sel);
            const tl_half2 v = __builtin_bit_cast(tl_half2, (b ^ 0x00800080u) | 0x64006400u) - bias;
            u32 x, y;
            ck_q8_pair(v, __builtin_bit_cast(tl_half2, (u32)sv[2 * j] | ((u32)sv[2 * j + 1] << 16)), x, y);
            h[j] = x;
            l[j] = y;
        }
        hi = __builtin_bit_cast(h8_t, h);
        lo = __builtin_bit_cast(h8_t, l);
    }
    TL_DEV void clear_v(int e) { sv[e] = 0; }
    TL_DEV bool odd_v(int e) const { return (sv[e] & 0x7fffu) > 0x6006u; }   /* 127 d past f16 */
};

template <int D, bool Q8>
struct CkTile;
template <int D>
struct CkTile<D, false> : CkTileF16<D> {};
template <int D>
struct CkTile<D, true> : CkTileQ8<D> {};

/* q of a column as f16 pairs, scaled by its row's power of two; returns the
 * factor that takes the products back to scale * q.k.  The column's row lies
 * over G lanes, 64 / G apart: lane g of them holds dims 8 (G s + g) .. of step s.
 * load and split apart, so that other loads can be requested in between. */
template <int D, int G>
TL_DEV void ck_load_q(const float *qrow, u32 g, float4 (&x)[D / (8 * G)][2]) {
#pragma unroll
    for (int s = 0; s < D / (8 * G); s++)
#pragma unroll
        for (int j = 0; j < 2; j++) x[s][j] = *(const float4 *)(qrow + 8 * (G * s + g) + 4 * j);
}
template <int D, int G>
TL_DEV float ck_split_q(const float4 (&x)[D / (8 * G)][2], float scale, h8_t (&hi)[D / (8 * G)],
                        h8_t (&lo)[D / (8 * G)]) {
    constexpr int N = D / (8 * G);
    float m = 0.f;
#pragma unroll
    for (int s = 0; s < N; s++)
#pragma unroll
        for (int j = 0; j < 2; j++)
            m = fmaxf(fmaxf(m, fmaxf(fabsf(x[s][j].x), fabsf(x[s][j].y))), fmaxf(fabsf(x[s][j].z), fabsf(x[s][j].w)));
    if constexpr (G == 4) m = fmaxf(m, __shfl_xor(m, 16));
    m = fmaxf(m, __shfl_xor(m, 32));
    const int e = ck_row_exp(m);
    const float up = __uint_as_float((u32)(e + 127) << 23);
    const float down = __uint_as_float((u32)(127 - e) << 23);
#pragma unroll
    for (int s = 0; s < N; s++) {
        u4_t hw, lw;
#pragma unroll
        for (int j = 0; j < 2; j++) {
            u32 h[2], l[2];
            ck_split2(x[s][j].x * up, x[s][j].y * up, h[0], l[0]);
            ck_split2(x[s][j].z * up, x[s][j].w * up, h[1], l[1]);
            hw[2 * j] = h[0];
            hw[2 * j + 1] = h[1];
            lw[2 * j] = l[0];
            lw[2 * j + 1] = l[1];
        }
        hi[s] = __builtin_bit_cast(h8_t, hw);
        lo[s] = __builtin_bit_cast(h8_t, lw);
    }
    return down * scale;
}

/* How products become scores in units of log2: s * mul after apply(). */
template <bool BIAS>
struct CkScore {
    float mul, cap_in, slope;
    bool capped, sloped;
    /* cs: factor from the products to scale * q.k */
    TL_DEV void set(const CkAttnParams &p, float cs, u32 head) {
        mul = fmaxf(cs * CK_LOG2E, 1.1754944e-38f);      /* not zero: hidden scores are -infinity x mul */
        if constexpr (BIAS) {
            capped = p.softcap > 0.f;
            sloped = p.slopes != nullptr;
            slope = sloped ? p.slopes[head] * CK_LOG2E : 0.f;
            if (capped) mul = p.softcap * CK_LOG2E;
            cap_in = capped ? cs * p.inv_cap : 0.f;
        }
    }
    /* far0: position minus the key of element 0; off(e): how far key e lies behind that */
    template <int N, class T, class F>
    TL_DEV void apply(T &s, int far0, F off) const {
        if constexpr (BIAS) {
            if (capped) ck_tanh<N>(s, cap_in);
            if (sloped) {
                const float f = (float)far0;
#pragma unroll
                for (int e = 0; e < N; e++) s[e] = fmaf(s[e], mul, -slope * fabsf(f - (float)off(e)));
            }
        }
    }
    TL_DEV float factor() const { return BIAS && sloped ? 1.f : mul; }
};
