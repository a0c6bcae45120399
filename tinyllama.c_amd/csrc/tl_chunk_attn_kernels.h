/* tl_chunk_attn_kernels.h — attention of a batch of chunks over a paged cache.
 *
 * Columns: a chunk's rows x the q heads of one kv head (column = row * gqa +
 * head); a column's softmax runs in one pass over the keys with a running
 * maximum and sum.  f32 accuracy on f16 matrix instructions: q, scaled by a power
 * of two of its row, and the probabilities are pairs hi + lo of f16 (22 bits), K
 * and V exact; a Q8_0 element, int8 x f16 scale, is a pair too (K = kh + kl; the
 * product of the two low halves is below 2^-22 and left out).
 *
 * Few columns (narrow): 16 to a workgroup, whose waves take the tiles of 32 keys
 * in turn, K and V straight from memory into the matrix operands' layout.  Bound
 * by the read of K and V at long contexts (one session of 32782 keys at 32/8/128
 * 30.6 us, 4.4 TB/s, with capped scores; 16 sessions of 512 to 8192 keys at 28/4/128
 * 21.6 us), below some 5 us of work by the chain of look-up, tile, join: 4 sessions
 * of 5 rows, 32/8/64, 10.8 us. */
#pragma once
#include "tl_chunk.h"

/* the maximum moves only when a score passes it by more than 2^CK_LAZY, and
 * probabilities are taken against 2^CK_UP below it: they reach 2^15 at most, so
 * that the low halves of the small ones stay normal f16 numbers too */
#define CK_LAZY 8.f
#define CK_UP 7.f

template <int D, int NW>
struct CkNarrowShared {
    __align__(16) float o[NW * CK_COLS * (D + 4)];
    float m[NW][CK_COLS], l[NW][CK_COLS];
    u32 last;
};

template <int D, bool Q8, bool BIAS, int NW>
TL_DEV void ck_narrow(const CkAttnParams &p, const CkSeq &sq, CkNarrowShared<D, NW> &sh) {
    constexpr int KS = D / 32, NM = D / 16, NT = 64 * NW;
    constexpr int ROWF = D + 4;
    float *const s_o = sh.o;
    float (&s_m)[NW][CK_COLS] = sh.m, (&s_l)[NW][CK_COLS] = sh.l;
    const u32 lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const u32 i = lane & 15, g = lane >> 4;
    const u32 local = blockIdx.x - sq.wg0;
    const u32 kvh = local % p.c.n_kv, rest = local / p.c.n_kv;
    const u32 cb = rest % sq.ncb, split = rest / sq.ncb;
    const u32 c0 = cb * CK_COLS;
    const u32 ncol = min((u32)CK_COLS, sq.n * p.gqa - c0);
    /* columns past the last one repeat it and are not written */
    const u32 col = c0 + min(i, ncol - 1);
    const u32 r = ck_row_of(p, col), head = kvh * p.gqa + col - r * p.gqa;
    const u32 pq = sq.pos + r, end = sq.pos + sq.n;
    const u64 brow = (u64)sq.row + r;

    CkSees see;
    const u32 first = p.first ? p.first[brow] : 0;
    see.set(pq, end, p.window, sq.prefix, first);
    CkSpan span;
    span.set(sq.pos + ck_row_of(p, c0), sq.pos + ck_row_of(p, c0 + ncol - 1), end, p.window, sq.prefix,
             p.first ? ck_uniform(group_umin<16>(first)) : 0, p.first ? ck_uniform(group_umax<16>(first)) : 0);
    CkTiles<CK_KEYS> tiles;
    tiles.set(span);
    const u32 n_tiles = tiles.count();
    const u32 t0 = (u32)((u64)n_tiles * split / sq.ns), t1 = (u32)((u64)n_tiles * (split + 1) / sq.ns);

    CkTile<D, Q8> tile, ahead;               /* of `ahead` only K: one tile further where registers allow */
    constexpr bool TWO = D < 256;
    /* lane's key of a tile (the upper half of the wave repeats the lower) */
    auto look = [&](u32 t) -> u32 {
        const u32 key = tiles.key(t) + (lane & 31);
        return key < end ? ck_row(p.c, sq.pages, key) : ~0u;
    };
    auto rows_k = [&](u32 row, u32 (&rk)[2]) {
#pragma unroll
        for (int a = 0; a < 2; a++) rk[a] = __shfl(row, 8 * (i >> 2) + 4 * a + (i & 3));
    };
    auto rows_v = [&](u32 row, u32 (&rv)[8]) {
#pragma unroll
        for (int e = 0; e < 8; e++) rv[e] = __shfl(row, 8 * g + e);
    };
    /* the first tile's rows, q, then the tile itself are requested before q is used */
    u32 t = t0 + wave;
    u32 row = 0, next = 0;
    if (t < t1) row = look(t);
    float4 qx[KS][2];
    ck_load_q<D, 4>(p.q + brow * p.q_stride + (u64)head * D, g, qx);
    if (t < t1) {
        const u32 rc = row < p.c.cap ? row : 0;
        u32 rk[2], rv[8];
        rows_k(rc, rk);
        tile.load_k(p.c, kvh, rk, g);
        rows_v(rc, rv);
        tile.load_v(p.c, kvh, rv, i);
        if (t + NW < t1) next = look(t + NW);
    }
    h8_t qh[KS], ql[KS];
    CkScore<BIAS> score;
    score.set(p, ck_split_q<D, 4>(qx, p.scale, qh, ql), head);
    const float mul = score.factor();
    float m = -INFINITY, l = 0.f;
    f4_t o[NM];
#pragma unroll
    for (int j = 0; j < NM; j++) o[j] = (f4_t){0.f, 0.f, 0.f, 0.f};
    for (; t < t1; t += NW) {
        const u32 kb = tiles.key(t);
        const u64 bad = __ballot(row >= p.c.cap);
        const bool more = t + NW < t1;
        u32 rn = 0;
        if (TWO && more) {
            rn = next < p.c.cap ? next : 0;
            u32 rk[2];
            rows_k(rn, rk);
            ahead.load_k(p.c, kvh, rk, g);
        }
        float x[8];
#pragma unroll
        for (int a = 0; a < 2; a++) {
            f4_t acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int s = 0; s < KS; s++) {
                h8_t kh, kl;
                tile.get_k(a, s, kh, kl);
                acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(kh, qh[s], acc, 0, 0, 0);
                acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(kh, ql[s], acc, 0, 0, 0);
                if constexpr (Q8) acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(kl, qh[s], acc, 0, 0, 0);
            }
#pragma unroll
            for (int e = 0; e < 4; e++) x[4 * a + e] = acc[e];
        }
        score.template apply<8>(x, (int)(pq - kb - 8 * g), [](int e) { return e; });
        if (!TWO && more) {
            rn = next < p.c.cap ? next : 0;
            u32 rk[2];
            rows_k(rn, rk);
            tile.load_k(p.c, kvh, rk, g);
        }
        if (!span.full(kb, CK_KEYS) || bad) {
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const bool vis = see.sees(kb + 8 * g + e) && !((bad >> (8 * g + e)) & 1);
                x[e] = vis ? x[e] : -INFINITY;
                const u32 mine = (u32)(__ballot(vis) >> (16 * g)) & 0xffffu;
                if (mine == 0) {
                    tile.clear_v(e);
                } else if (__any(mine != 0xffffu)) {
                    /* seen by some columns: infinities and NaN go to those alone */
                    const bool odd = mine != 0xffffu && tile.odd_v(e);
                    const u64 ob = __ballot(odd);
                    if (ob) {
                        if (odd) tile.clear_v(e);
                        if (vis && ((ob >> (16 * g)) & 0xffffu)) l = NAN;
                    }
                }
            }
        }
        /* running maximum */
        float top = x[0];
#pragma unroll
        for (int e = 1; e < 8; e++) top = fmaxf(top, x[e]);
        top *= mul;
        const float thr = m == -INFINITY ? -INFINITY : m + CK_LAZY;
        if (__any(top > thr)) {
            top = fmaxf(top, __shfl_xor(top, 16));
            top = fmaxf(top, __shfl_xor(top, 32));
            const float mn = top > thr ? top : m;
            const float al = m == -INFINITY ? (mn == m ? 1.f : 0.f) : __builtin_amdgcn_exp2f(m - mn);
            l *= al;
#pragma unroll
            for (int j = 0; j < NM; j++) o[j] *= al;
            m = mn;
        }
        const float mref = m == -INFINITY ? 0.f : m - CK_UP;
        u4_t pw, qw;
        float l1 = 0.f;
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
            const float a = __builtin_amdgcn_exp2f(fmaf(x[e], mul, -mref)), b = __builtin_amdgcn_exp2f(fmaf(x[e + 1], mul, -mref));
            l += a;
            l1 += b;
            u32 hi, lo;
            ck_split2(a, b, hi, lo);
            pw[e >> 1] = hi;
            qw[e >> 1] = lo;
        }
        l += l1;
        const h8_t ph = __builtin_bit_cast(h8_t, pw), pl = __builtin_bit_cast(h8_t, qw);
#pragma unroll
        for (int j = 0; j < NM; j++) {
            h8_t vh, vl;
            tile.get_v(j, vh, vl);
            o[j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vh, ph, o[j], 0, 0, 0);
            o[j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vh, pl, o[j], 0, 0, 0);
            if constexpr (Q8) o[j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vl, ph, o[j], 0, 0, 0);
        }
        if (more) {
            u32 rv[8];
            rows_v(rn, rv);
            tile.load_v(p.c, kvh, rv, i);
            if constexpr (TWO) tile.take_k(ahead);
            row = next;
            if (t + 2 * NW < t1) next = look(t + 2 * NW);
        }
    }
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);

    /* the waves' states joined through LDS */
    if (g == 0) {
        s_m[wave][i] = m;
        s_l[wave][i] = l;
    }
#pragma unroll
    for (int e = 0; e < 4; e++)
#pragma unroll
        for (int j = 0; j < NM; j += 4)
            *(float4 *)&s_o[(wave * CK_COLS + i) * ROWF + NM * (4 * g + e) + j] =
                make_float4(o[j][e], o[j + 1][e], o[j + 2][e], o[j + 3][e]);
    __syncthreads();
    constexpr u32 V4 = D / 4;
    const u32 units = ncol * V4;
    const u32 group = kvh * sq.ncb + cb;
    const u64 part = (u64)sq.part0 + (u64)group * sq.ns * CK_COLS;      /* the group's first partial row */
    const __amdgpu_buffer_rsrc_t ra = buf_rsrc(p.ws_acc + part * D);
    const __amdgpu_buffer_rsrc_t rm = buf_rsrc(p.ws_ml + part);
    auto write = [&](u32 c, u32 d, float4 a, float sum, float M) {
        const u32 cc = c0 + c, rr = ck_row_of(p, cc), hh = kvh * p.gqa + cc - rr * p.gqa;
        const u64 br = (u64)sq.row + rr;
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
        *(float4 *)(p.dst + br * p.q_stride + (u64)hh * D + 4 * d) =
            make_float4(a.x * inv, a.y * inv, a.z * inv, a.w * inv);
        if (p.lse && d == 0)
            p.lse[br * p.n_head + hh] = sum == 0.f ? -INFINITY
                : ((M == -INFINITY ? 0.f : M) - CK_UP + __builtin_amdgcn_logf(sum)) * CK_LN2;
    };
    auto keep = [&](u32 s, u32 c, u32 d, float4 a, float sum, float M) {
        const u32x4v_t v = {__float_as_uint(a.x), __float_as_uint(a.y), __float_as_uint(a.z), __float_as_uint(a.w)};
        __builtin_amdgcn_raw_buffer_store_b128(v, ra, ((s * CK_COLS + c) * D + 4 * d) * 4, 0, TL_SC1);
        if (d == 0) {
            const u32x2v_t ml = {__float_as_uint(M), __float_as_uint(sum)};
            __builtin_amdgcn_raw_buffer_store_b64(ml, rm, (s * CK_COLS + c) * 8, 0, TL_SC1);
        }
    };
    for (u32 u = threadIdx.x; u < units; u += NT) {
        const u32 c = u / V4, d = u % V4;
        float M = -INFINITY;
#pragma unroll
        for (int w = 0; w < NW; w++) M = fmaxf(M, s_m[w][c]);
        const float M0 = M == -INFINITY ? 0.f : M;
        float sum = 0.f;
        float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < NW; w++) {
            const float f = __builtin_amdgcn_exp2f(s_m[w][c] - M0);
            const float4 v = *(const float4 *)&s_o[(w * CK_COLS + c) * ROWF + 4 * d];
            sum = fmaf(f, s_l[w][c], sum);
            a.x = fmaf(f, v.x, a.x);
            a.y = fmaf(f, v.y, a.y);
            a.z = fmaf(f, v.z, a.z);
            a.w = fmaf(f, v.w, a.w);
        }
        if (sq.ns == 1) write(c, d, a, sum, M);
        else keep(split, c, d, a, sum, M);
    }
    if (sq.ns == 1) return;
    /* The last split of the group to arrive joins them all.  One workgroup reads
     * some 0.1 MB in the time of a wait for memory: of many splits' rows, eight
     * splits at a time are joined first, by the last of the eight to arrive, and
     * the last of the last ones joins those.  The order of the sums is the splits',
     * whoever comes last. */
    auto arrive = [&](u32 *cnt, u32 of) -> bool {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        if (threadIdx.x == 0) {
            sh.last = __hip_atomic_fetch_add(cnt, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == of - 1;
            if (sh.last) __hip_atomic_store(cnt, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
        __syncthreads();
        return sh.last;
    };
    /* splits first, first + step, ... joined: `parts` threads to a float4 of the
     * output, each with a run of the splits, eight of them requested at a time; then
     * the parts through LDS, in order */
    auto join = [&](u32 first, u32 step, u32 count, auto to) {
        u32 parts = 1;
        while (parts < NW && parts * 2 * units <= NT && parts * 8 < count) parts *= 2;
        const u32 run = (count + parts - 1) / parts;
        const u32 lanes = parts == 1 ? NT : NT / parts;
        const u32 pi = threadIdx.x / lanes;
        for (u32 u = threadIdx.x % lanes; u < units; u += lanes) {
            const u32 c = u / V4, d = u % V4;
            float M = -INFINITY, sum = 0.f;
            float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
            const u32 s1 = min((pi + 1) * run, count);
            for (u32 s0 = pi * run; s0 < s1; s0 += 8) {
                u32x2v_t ml[8];
                u32x4v_t v[8];
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const u32 s = first + step * min(s0 + j, count - 1);
                    ml[j] = __builtin_amdgcn_raw_buffer_load_b64(rm, (s * CK_COLS + c) * 8, 0, TL_SC1);
                    v[j] = __builtin_amdgcn_raw_buffer_load_b128(ra, ((s * CK_COLS + c) * D + 4 * d) * 4, 0, TL_SC1);
                }
                float Mn = M;
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const u32 mb = ml[j][0];
                    Mn = fmaxf(Mn, s0 + j < s1 ? __uint_as_float(mb) : -INFINITY);
                }
                const float M0 = Mn == -INFINITY ? 0.f : Mn;
                const float f0 = __builtin_amdgcn_exp2f(M - M0);
                sum *= f0;
                a.x *= f0; a.y *= f0; a.z *= f0; a.w *= f0;
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    if (s0 + j >= s1) break;
                    const u32 mb = ml[j][0], lb = ml[j][1];
                    const u32 v0 = v[j][0], v1 = v[j][1], v2 = v[j][2], v3 = v[j][3];
                    const float f = __builtin_amdgcn_exp2f(__uint_as_float(mb) - M0);
                    sum = fmaf(f, __uint_as_float(lb), sum);
                    a.x = fmaf(f, __uint_as_float(v0), a.x);
                    a.y = fmaf(f, __uint_as_float(v1), a.y);
                    a.z = fmaf(f, __uint_as_float(v2), a.z);
                    a.w = fmaf(f, __uint_as_float(v3), a.w);
                }
                M = Mn;
            }
            if (parts == 1) {
                to(c, d, a, sum, M);
            } else {
                *(float4 *)&s_o[(pi * CK_COLS + c) * ROWF + 4 * d] = a;
                if (d == 0) {
                    s_m[pi][c] = M;
                    s_l[pi][c] = sum;
                }
            }
        }
        if (parts == 1) return;
        __syncthreads();
        for (u32 u = threadIdx.x; u < units; u += NT) {
            const u32 c = u / V4, d = u % V4;
            float M = -INFINITY, sum = 0.f;
            for (u32 w = 0; w < parts; w++) M = fmaxf(M, s_m[w][c]);
            const float M0 = M == -INFINITY ? 0.f : M;
            float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
            for (u32 w = 0; w < parts; w++) {
                const float f = __builtin_amdgcn_exp2f(s_m[w][c] - M0);
                const float4 v = *(const float4 *)&s_o[(w * CK_COLS + c) * ROWF + 4 * d];
                sum = fmaf(f, s_l[w][c], sum);
                a.x = fmaf(f, v.x, a.x);
                a.y = fmaf(f, v.y, a.y);
                a.z = fmaf(f, v.z, a.z);
                a.w = fmaf(f, v.w, a.w);
            }
            to(c, d, a, sum, M);
        }
    };
    const u32 n_cnt = sq.counters;
    u32 *cnt = p.cnt + ((u64)sq.grp0 + (u64)group * n_cnt) * CK_CNT_PAD;
    if (n_cnt > 1) {
        const u32 s0 = split / CK_JOIN * CK_JOIN, of = min((u32)CK_JOIN, sq.ns - s0);
        if (!arrive(cnt + (1 + split / CK_JOIN) * CK_CNT_PAD, of)) return;
        /* a column's threads are of one wave, which has read its row before it writes it */
        join(s0, 1, of, [&](u32 c, u32 d, float4 a, float sum, float M) { keep(s0, c, d, a, sum, M); });
        if (!arrive(cnt, n_cnt - 1)) return;
        join(0, CK_JOIN, n_cnt - 1, write);
    } else {
        if (!arrive(cnt, sq.ns)) return;
        join(0, 1, sq.ns, write);
    }
}

/* ---- many columns: 128 to a workgroup, K and V tiles shared through LDS ------
 *
 * A wave has 32 columns and runs S^T = K . Q^T and O^T += V^T . P^T on
 * v_mfma_f32_32x32x16_f16 (A rows: lane & 31, eight k's of half h = lane >> 5).
 * A lane's sixteen scores of a 32-key block are rows (r & 3) + 8 (r >> 2) + 4 h;
 * matrix row rho is fed key rho with bits 2 and 3 exchanged, so they are keys 16
 * u + 8 h + j (r = 8 u + j), the k order of step u of the second product.  At
 * head_dim 256 q and O of 32 columns would take all registers of a SIMD (the
 * compiler moved 370 accumulation registers per tile): there eight waves of 16
 * columns on v_mfma_f32_16x16x32_f16, keys 8 h + e with h = lane >> 4.
 *
 * Tiles of KT keys, two buffers, one barrier each.  The pool rows of a tile are
 * looked up by one wave three tiles ahead and handed on through LDS; K rows go
 * straight to LDS (LDS-direct loads, one tile ahead); V goes through registers,
 * eight keys to a lane, which transposes them on the way to LDS (v_perm on
 * pairs), so that both operands are 16-byte reads, four requested ahead of the
 * matrix instructions.  16-byte units are permuted within a row so that 16
 * lanes' reads cover all banks.  A Q8_0 tile is kept as two planes, hi and lo,
 * both through registers (waves 0 and 1 K, waves 2 and 3 V).
 *
 * Bound by the matrix instructions (four products for two, because of the pairs)
 * together with the seven vector ones that go with each of them: 512 rows of
 * documents of up to 9000 tokens at 16384 keys, 32/8/128, 141-148 us with the join
 * (8), 0.9 PFLOP/s of matrix work, matrix pipe busy half of the time.  A workgroup
 * by itself needs 0.43 us of it per tile and takes 1.16 (head_dim 256: 0.85 and
 * 1.62, its LDS reads as long as its matrix work), after some 8 us for the chain of
 * arguments, look-ups, first tiles and the last stores. */
typedef float f16_t __attribute__((ext_vector_type(16)));
template <int MC>
struct CkAcc {
    typedef f16_t type;
};
template <>
struct CkAcc<16> {
    typedef f4_t type;
};
TL_DEV void ck_mfma(f16_t &c, h8_t a, h8_t b) { c = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
TL_DEV void ck_mfma(f4_t &c, h8_t a, h8_t b) { c = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
/* key of a lane's score e within 32 */
template <int MC>
TL_DEV constexpr int ck_key(int e) {
    return MC == 32 ? 16 * (e >> 3) + (e & 7) : e;
}


template <int D, bool Q8>
struct CkWide {
    static constexpr int MC = D == 256 ? 16 : 32;    /* columns of a wave */
    static constexpr int NW = CK_WCOLS / MC, NT = 64 * NW;
    static constexpr int G = 64 / MC;                /* lanes of a column */
    static constexpr int KT = Q8 ? (D == 64 ? 64 : 32) : (D == 256 ? 32 : 64);
    static constexpr int U = D / 8;                  /* 16-byte units of a K row in LDS */
    static constexpr int VU = KT / 8;                /* ... of a V^T row */
    static constexpr int PL = Q8 ? 2 : 1;
    static constexpr int VL = Q8 ? NT / 2 : NT;      /* lanes that stage V */
    static constexpr int DPL = KT * D / 8 / VL;      /* dims of V of one of them */
    static constexpr int RU = Q8 ? D / 16 : D / 8;   /* 16-byte units of a K row in memory */
    static constexpr int KL = Q8 ? KT * RU / VL : KT * RU / NT;   /* ... of a staging lane */
    static constexpr int VD = Q8 ? DPL / 4 : DPL / 2;   /* dwords of V of a key and lane */
    static constexpr int ST = Q8 && KL * 4 > 8 * VD ? KL * 4 : 8 * VD;
    static constexpr int SC = Q8 ? 8 : 1;            /* scales of a staging lane */
    static_assert(Q8 ? DPL == 4 || DPL == 8 : DPL == 2 || DPL == 4, "staging");
    static constexpr int KP = KT * U * 16, VP = D * VU * 16;   /* bytes of a plane */
    /* byte offsets of units; exclusive-or linear in the bits of their arguments, so
     * an offset is the lane's part with a constant part put in (put) */
    static constexpr TL_HOSTDEV u32 kswz(u32 key) {
        return U == 8 ? (key >> 1) & 7 : MC == 16 ? (key & 3) | ((key >> 1) & 12) : key & 15;
    }
    static constexpr TL_HOSTDEV u32 kat(u32 key, u32 unit) { return (key * U + (unit ^ kswz(key))) * 16; }
    static constexpr TL_HOSTDEV u32 vat(u32 dim, u32 unit) {
        return (dim * VU + (unit ^ (VU == 8 ? ((dim >> 1) ^ (dim >> 3)) & 7 : (dim >> 2) & 3))) * 16;
    }
    static TL_DEV u32 kput(u32 lane_part, u32 c) {
        return (lane_part ^ (c & (U * 16 - 1))) + (c & ~(u32)(U * 16 - 1));
    }
    static TL_DEV u32 vput(u32 lane_part, u32 c) {
        return (lane_part ^ (c & (VU * 16 - 1))) + (c & ~(u32)(VU * 16 - 1));
    }
};

/* 64 lanes' 16 bytes at base + off straight to LDS at `to` (wave-uniform) + 16
 * lane; the caller waits (vmcnt) before the barrier that hands them on */
TL_DEV void ck_lds_load16(void *to, const void *base, u32 off) {
    const u64 g = (u64)base;
    const void *sb = (const void *)(((u64)ck_uniform((u32)(g >> 32)) << 32) | ck_uniform((u32)g));
    const u32 m0 = ck_uniform((u32)(u64)(__attribute__((address_space(3))) char *)to);
    asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(off), "s"(sb), "{m0}"(m0) : "memory");
}

#define CK_AHEAD 4   /* LDS operand reads in flight ahead of the matrix instructions */

template <int D, bool Q8>
struct CkWideShared {
    typedef CkWide<D, Q8> W;
    /* buffer b, plane l of K: k + (b * PL + l) * KP; of V the same */
    __align__(16) char k[2 * W::PL * W::KP];
    __align__(16) char v[2 * W::PL * W::VP];
    __align__(16) u32 row[2][W::KT];   /* pool rows of a tile's keys, 0 for the bad ones */
    u64 bad[4];                        /* keys of a tile without a row */
    u64 odd[2][W::NW];                 /* keys of a tile whose V is not all finite */
    u32 first[2][W::NW];
};

template <int D, bool Q8, bool BIAS>
TL_DEV void ck_wide(const CkAttnParams &p, const CkSeq &sq, CkWideShared<D, Q8> &sh) {
    typedef CkWide<D, Q8> W;
    typedef typename CkAcc<W::MC>::type acc_t;
    constexpr int KT = W::KT, MC = W::MC, G = W::G, NW = W::NW;
    constexpr int SN = MC / 2;                       /* scores of a lane and 32 keys */
    constexpr int NS = D / (8 * G);                  /* k-steps of the first product */
    constexpr int NO = D / MC;                       /* blocks of O^T */
    constexpr int VK = MC == 32 ? 2 : 1;             /* k-steps of the second product */
    char *const s_k = sh.k, *const s_v = sh.v;
    u32 (&s_row)[2][KT] = sh.row;
    u64 (&s_bad)[4] = sh.bad;
    u64 (&s_odd)[2][NW] = sh.odd;
    u32 (&s_first)[2][NW] = sh.first;
    const u32 lane = threadIdx.x & 63, wave = ck_uniform(threadIdx.x >> 6);
    const u32 i = lane & (MC - 1), h = lane / MC;
    const u32 local = blockIdx.x - sq.wg0;
    const u32 kvh = local % p.c.n_kv, rest = local / p.c.n_kv;
    const u32 cb = rest % sq.ncb, split = rest / sq.ncb;
    const u32 cols = sq.n * p.gqa, c0 = (sq.cb0 + cb) * CK_WCOLS, cw = c0 + wave * MC;
    const bool live = cw < cols;
    const u32 col = min(cw + i, cols - 1);
    const u32 end = sq.pos + sq.n;
    const u32 r = ck_row_of(p, col), head = kvh * p.gqa + col - r * p.gqa;
    const u32 pq = sq.pos + r;
    const u64 brow = (u64)sq.row + r;
    CkSees see;
    CkSpan span;
    const u32 first = p.first ? p.first[brow] : 0;
    see.set(pq, end, p.window, sq.prefix, first);
    span.set(sq.pos + ck_row_of(p, min(cw, cols - 1)), sq.pos + ck_row_of(p, min(cw + MC - 1, cols - 1)), end, p.window, sq.prefix,
             p.first ? ck_uniform(group_umin<MC>(first)) : 0, p.first ? ck_uniform(group_umax<MC>(first)) : 0);
    u32 fmin = span.fmin, fmax = span.max_f;
    if (p.first) {
        if (lane == 0) {
            s_first[0][wave] = fmin;
            s_first[1][wave] = fmax;
        }
        __syncthreads();
#pragma unroll
        for (int w = 0; w < NW; w++) {
            fmin = min(fmin, s_first[0][w]);
            fmax = max(fmax, s_first[1][w]);
        }
        fmin = ck_uniform(fmin);
        fmax = ck_uniform(fmax);
    }
    CkSpan all;
    all.set(sq.pos + ck_row_of(p, c0), sq.pos + ck_row_of(p, min(c0 + CK_WCOLS - 1, cols - 1)), end, p.window,
            sq.prefix, fmin, fmax);
    CkTiles<KT> tiles;
    tiles.set(all);
    const u32 n_tiles = tiles.count();
    const u32 t0 = (u32)((u64)n_tiles * split / sq.ns), t1 = (u32)((u64)n_tiles * (split + 1) / sq.ns);

    /* staging */
    u32 st[W::ST];
    u32 sc[W::SC];
    const char *kbase = (const char *)p.c.k + (u64)kvh * p.c.cap * (Q8 ? D : 2 * D);
    const char *vbase = (const char *)p.c.v + (u64)kvh * p.c.cap * (Q8 ? D : 2 * D);
    const u16 *ksb = p.c.ks + (u64)kvh * p.c.cap * (D / 32);
    const u16 *vsb = p.c.vs + (u64)kvh * p.c.cap * (D / 32);
    /* lane's pool row of a tile (KT = 32: the upper half repeats the lower) */
    auto look = [&](u32 t) -> u32 {
        const u32 key = tiles.key(t) + (lane & (KT - 1));
        return key < end ? ck_row(p.c, sq.pages, key) : ~0u;
    };
    auto hand_on = [&](u32 t, u32 row) {     /* by one wave */
        const u64 bad = __ballot(row >= p.c.cap);
        if (lane < KT) s_row[(t - t0) & 1][lane] = row < p.c.cap ? row : 0;
        if (lane == 0) s_bad[(t - t0) & 3] = bad;
    };
    /* the places of a staging lane, kept out of registers across the tile loop */
    auto place = [&](u32 &sl) {
        sl = Q8 ? threadIdx.x % W::VL : threadIdx.x;
        asm volatile("" : "+v"(sl));
    };
    auto fetch = [&](u32 t) {
        const u32 *rows = s_row[(t - t0) & 1];
        u32 sl;
        place(sl);
        const u32 dg = sl % (D / W::DPL), kg = sl / (D / W::DPL);      /* V: dims and keys of the lane */
        if constexpr (!Q8) {
            char *to = s_k + ((t - t0) & 1) * W::KP;
            const u32 ln = sl & 63;
#pragma unroll
            for (int j = 0; j < W::KL; j++) {
                const u32 c = wave * W::KL + j, key = c * (64 / W::U) + ln / W::U;
                ck_lds_load16(to + c * 1024, kbase, rows[key] * (u32)(2 * D) + ((ln % W::U) ^ W::kswz(key)) * 16);
            }
        } else if (wave < NW / 2) {
#pragma unroll
            for (int j = 0; j < W::KL; j++) {
                const u32 u = sl % W::RU, row = rows[j * (W::VL / W::RU) + sl / W::RU];
                const u4_t v = *(const u4_t *)(kbase + (u64)(row * (u32)(W::RU * 16) + u * 16));
#pragma unroll
                for (int d = 0; d < 4; d++) st[4 * j + d] = v[d];
                sc[j] = ksb[(u64)(row * (u32)(D / 32) + (u >> 1))];
            }
            return;
        }
        const u4_t ra = *(const u4_t *)(rows + 8 * kg), rb = *(const u4_t *)(rows + 8 * kg + 4);
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const u32 row = e < 4 ? ra[e & 3] : rb[e & 3];
            const char *a = vbase + (u64)(row * (u32)(Q8 ? D : 2 * D) + dg * (Q8 ? W::DPL : 2 * W::DPL));
            if constexpr (W::VD == 1) {
                st[e] = *(const u32 *)a;
            } else {
                const uint2 v = *(const uint2 *)a;
                st[2 * e] = v.x;
                st[2 * e + 1] = v.y;
            }
            if constexpr (Q8) sc[e] = vsb[(u64)(row * (u32)(D / 32) + dg * W::DPL / 32)];
        }
    };
    auto store = [&](u32 t) {
        const u32 buf = (t - t0) & 1;
        u32 sl;
        place(sl);
        const u32 dg = sl % (D / W::DPL), kg = sl / (D / W::DPL);
        if constexpr (Q8)
            if (wave < NW / 2) {
                const u32 kst = W::kat(sl / W::RU, 2 * (sl % W::RU));
                char *to = s_k + buf * (W::PL * W::KP);
#pragma unroll
                for (int j = 0; j < W::KL; j++) {
                    const u32 c = W::kat(j * (W::VL / W::RU), 0);
                    const tl_half2 d2 = __builtin_bit_cast(tl_half2, sc[j] * 0x10001u);
                    u32 hi[8], lo[8];
#pragma unroll
                    for (int d = 0; d < 4; d++) {
                        tl_half2 a, b;
                        i8x4_to_f16(st[4 * j + d], a, b);
                        ck_q8_pair(a, d2, hi[2 * d], lo[2 * d]);
                        ck_q8_pair(b, d2, hi[2 * d + 1], lo[2 * d + 1]);
                    }
#pragma unroll
                    for (int z = 0; z < 2; z++) {
                        char *at = to + W::kput(kst, c ^ (z * 16));
                        *(u4_t *)at = (u4_t){hi[4 * z], hi[4 * z + 1], hi[4 * z + 2], hi[4 * z + 3]};
                        *(u4_t *)(at + W::KP) = (u4_t){lo[4 * z], lo[4 * z + 1], lo[4 * z + 2], lo[4 * z + 3]};
                    }
                }
                return;
            }
        const u64 bad = s_bad[(t - t0) & 3];
        if (bad || !all.full(tiles.key(t), KT)) {
            /* keys without a row are zeros; infinities and NaN, which only some
             * columns may see, are zeros in the product, and the columns that do
             * see the key are told */
            u32 odd = 0;
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const bool none = (bad >> (8 * kg + e)) & 1;
                bool x = false;
                if constexpr (Q8) {
                    x = (sc[e] & 0x7fffu) > 0x6006u;
                    sc[e] = x || none ? 0 : sc[e];
                } else {
#pragma unroll
                    for (int d = 0; d < W::VD; d++)
                        x |= (st[W::VD * e + d] & 0x7c00u) == 0x7c00u || (st[W::VD * e + d] & 0x7c000000u) == 0x7c000000u;
                }
#pragma unroll
                for (int d = 0; d < W::VD; d++) st[W::VD * e + d] = x || none ? 0 : st[W::VD * e + d];
                odd |= (u32)(x && !none) << e;
            }
            u64 keys = 0;
            if (__any(odd)) {
                keys = (u64)odd << (8 * kg);
#pragma unroll
                for (int x = 1; x < 64; x <<= 1) keys |= __shfl_xor(keys, x);
            }
            if (lane == 0) s_odd[buf][wave] = keys;
        }
        const u32 vst = W::vat(dg * W::DPL, kg);
#pragma unroll
        for (int x = 0; x < W::DPL; x++) {
            u4_t hi, lo;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                if constexpr (!Q8) {
                    hi[j] = __builtin_amdgcn_perm(st[W::VD * (2 * j + 1) + (x >> 1)], st[W::VD * 2 * j + (x >> 1)],
                                                  x & 1 ? 0x07060302u : 0x05040100u);
                } else {
                    const u32 sel = 0x0c000c00u | (u32)(x & 3) | ((u32)(4 + (x & 3)) << 16);
                    const tl_half2 bias = {(_Float16)1152.0f, (_Float16)1152.0f};
                    const u32 b = __builtin_amdgcn_perm(st[W::VD * (2 * j + 1) + (x >> 2)], st[W::VD * 2 * j + (x >> 2)], sel);
                    const tl_half2 v = __builtin_bit_cast(tl_half2, (b ^ 0x00800080u) | 0x64006400u) - bias;
                    u32 a, c;
                    ck_q8_pair(v, __builtin_bit_cast(tl_half2, sc[2 * j] | (sc[2 * j + 1] << 16)), a, c);
                    hi[j] = a;
                    lo[j] = c;
                }
            }
            char *at = s_v + buf * (W::PL * W::VP) + W::vput(vst, W::vat(x, 0));
            *(u4_t *)at = hi;
            if constexpr (Q8) *(u4_t *)(at + W::VP) = lo;
        }
    };

    /* the first tiles' rows, q and the first tile are requested one after another
     * and waited for together */
    u32 next = 0, ra = 0, rb = 0;
    if (wave == 0 && t0 < t1) {
        ra = look(t0);
        if (t0 + 1 < t1) rb = look(t0 + 1);
        if (t0 + 2 < t1) next = look(t0 + 2);
    }
    float4 qx[NS][2];
    ck_load_q<D, G>(p.q + brow * p.q_stride + (u64)head * D, h, qx);
    if (t0 < t1) {
        if (wave == 0) {
            hand_on(t0, ra);
            if (t0 + 1 < t1) hand_on(t0 + 1, rb);
        }
        __syncthreads();
        fetch(t0);
    }
    h8_t qh[NS], ql[NS];
    CkScore<BIAS> score;
    score.set(p, ck_split_q<D, G>(qx, p.scale, qh, ql), head);
    const float mul = score.factor();
    float m = -INFINITY, l = 0.f;
    acc_t o[NO];
#pragma unroll
    for (int b = 0; b < NO; b++) o[b] = (acc_t)(0.f);
    if (t0 < t1) store(t0);
#pragma unroll 1
    for (u32 t = t0; t < t1; t++) {
        const u32 kt = tiles.key(t);
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        if (t + 1 < t1) fetch(t + 1);
        if (wave == 0 && t + 2 < t1) {
            hand_on(t + 2, next);
            if (t + 3 < t1) next = look(t + 3);
        }
        if (live && span.any(kt, KT)) {
            const u32 buf = (t - t0) & 1;
            u32 ii = i;
            asm volatile("" : "+v"(ii));
            const char *const kp = s_k + buf * (W::PL * W::KP), *const vp = s_v + buf * (W::PL * W::VP);
            const u32 krd = W::kat(MC == 32 ? (ii & 19) | ((ii & 4) << 1) | ((ii & 8) >> 1) : (ii & 3) | ((ii & 12) << 1), h);
            const u32 vrd = W::vat(ii, h);
#pragma unroll
            for (int sub = 0; sub < KT / 32; sub++) {
                const u32 kb = kt + 32 * sub;
                float s[SN];
                {
                    /* MC = 16: two blocks of 16 keys, one after the other */
                    constexpr int NR = MC == 32 ? NS : 2 * NS;
                    acc_t acc[MC == 32 ? 1 : 2];
                    h8_t a[CK_AHEAD], b[CK_AHEAD];
                    auto read = [&](int j) {
                        const char *at = kp + W::kput(krd, MC == 32 ? W::kat(32 * sub, 2 * j) : W::kat(32 * sub + 4 * (j & 1), 4 * (j >> 1)));
                        a[j % CK_AHEAD] = *(const h8_t *)at;
                        if constexpr (Q8) b[j % CK_AHEAD] = *(const h8_t *)(at + W::KP);
                    };
                    acc[0] = (acc_t)(0.f);
                    if constexpr (MC == 16) acc[1] = (acc_t)(0.f);
#pragma unroll
                    for (int j = 0; j < CK_AHEAD; j++) read(j);
#pragma unroll
                    for (int j = 0; j < NR; j++) {
                        const int k = MC == 32 ? j : j >> 1, c = MC == 32 ? 0 : j & 1;
                        __builtin_amdgcn_sched_barrier(0);
                        ck_mfma(acc[c], a[j % CK_AHEAD], qh[k]);
                        ck_mfma(acc[c], a[j % CK_AHEAD], ql[k]);
                        if constexpr (Q8) ck_mfma(acc[c], b[j % CK_AHEAD], qh[k]);
                        if (j + CK_AHEAD < NR) read(j + CK_AHEAD);
                    }
                    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                    for (int e = 0; e < SN; e++) s[e] = MC == 32 ? acc[0][e % (MC == 32 ? 16 : 4)] : acc[(e >> 2) & 1 & (MC == 32 ? 0 : 1)][e & 3];
                }
                score.template apply<SN>(s, (int)(pq - kb - 8 * h), [](int e) { return ck_key<MC>(e); });
                const u32 bad = (u32)(s_bad[(t - t0) & 3] >> (32 * sub));
                if (__builtin_expect(!span.full(kb, 32) || bad, 0)) {
                    asm volatile("");      /* stays a branch: made into selects it cost every tile 18% */
                    u64 keys = 0;
#pragma unroll
                    for (int w = Q8 ? NW / 2 : 0; w < NW; w++) keys |= s_odd[buf][w];
                    const u32 odd = (u32)(keys >> (32 * sub));
#pragma unroll
                    for (int e = 0; e < SN; e++) {
                        const u32 k = ck_key<MC>(e) + 8 * h;
                        const bool v = see.sees(kb + k) && !((bad >> k) & 1);
                        s[e] = v ? s[e] : -INFINITY;
                        if (v && ((odd >> k) & 1)) l = NAN;
                    }
                }
                float top = s[0];
#pragma unroll
                for (int e = 1; e < SN; e++) top = fmaxf(top, s[e]);
                top *= mul;
                const float thr = m == -INFINITY ? -INFINITY : m + CK_LAZY;
                if (__builtin_expect(__any(top > thr), 0)) {
                    if constexpr (MC == 16) top = fmaxf(top, __shfl_xor(top, 16));
                    top = fmaxf(top, __shfl_xor(top, 32));
                    const float mn = top > thr ? top : m;
                    const float al = m == -INFINITY ? (mn == m ? 1.f : 0.f) : __builtin_amdgcn_exp2f(m - mn);
                    l *= al;
#pragma unroll
                    for (int b = 0; b < NO; b++) o[b] *= al;
                    m = mn;
                }
                const float mref = m == -INFINITY ? 0.f : m - CK_UP;
                h8_t v[CK_AHEAD], w[CK_AHEAD];
                auto read = [&](int j) {
                    const char *at = vp + W::vput(vrd, W::vat(MC * (j % NO), 4 * sub + 2 * (j / NO)));
                    v[j % CK_AHEAD] = *(const h8_t *)at;
                    if constexpr (Q8) w[j % CK_AHEAD] = *(const h8_t *)(at + W::VP);
                };
#pragma unroll
                for (int j = 0; j < CK_AHEAD; j++) read(j);
                __builtin_amdgcn_sched_barrier(0);
                u4_t ph[VK], pl[VK];
                float l1 = 0.f;
#pragma unroll
                for (int e = 0; e < SN; e += 2) {
                    const float a = __builtin_amdgcn_exp2f(fmaf(s[e], mul, -mref));
                    const float b = __builtin_amdgcn_exp2f(fmaf(s[e + 1], mul, -mref));
                    l += a;
                    l1 += b;
                    u32 hi, lo;
                    ck_split2(a, b, hi, lo);
                    ph[e >> 3][(e & 7) >> 1] = hi;
                    pl[e >> 3][(e & 7) >> 1] = lo;
                }
                l += l1;
#pragma unroll
                for (int j = 0; j < VK * NO; j++) {
                    __builtin_amdgcn_sched_barrier(0);
                    const int b = j % NO, u = j / NO;
                    const h8_t x = __builtin_bit_cast(h8_t, ph[u]), y = __builtin_bit_cast(h8_t, pl[u]);
                    ck_mfma(o[b], v[j % CK_AHEAD], x);
                    ck_mfma(o[b], v[j % CK_AHEAD], y);
                    if constexpr (Q8) ck_mfma(o[b], w[j % CK_AHEAD], x);
                    if (j + CK_AHEAD < VK * NO) read(j + CK_AHEAD);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        if (t + 1 < t1) store(t + 1);
    }
    if constexpr (MC == 16) l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    if (!live || cw + i >= cols) return;
    /* block b, registers 4 e ..: dims MC b + 8 e + 4 h (MC = 16: 4 h) */
    if (sq.ns == 1) {
        const float inv = l == 0.f ? 0.f : 1.f / l;
        float *d = p.dst + brow * p.q_stride + (u64)head * D + 4 * h;
#pragma unroll
        for (int b = 0; b < NO; b++)
#pragma unroll
            for (int e = 0; e < MC / 8 * MC / 32; e++)
                *(float4 *)(d + MC * b + 8 * e) = make_float4(o[b][4 * e] * inv, o[b][4 * e + 1] * inv,
                                                             o[b][4 * e + 2] * inv, o[b][4 * e + 3] * inv);
        if (p.lse && h == 0)
            p.lse[brow * p.n_head + head] = l == 0.f ? -INFINITY
                : ((m == -INFINITY ? 0.f : m) - CK_UP + __builtin_amdgcn_logf(l)) * CK_LN2;
        return;
    }
    const u64 part = (u64)sq.part0 + ((u64)(kvh * sq.ncb + cb) * sq.ns + split) * CK_WCOLS + wave * MC + i;
    float *d = p.ws_acc + part * D + 4 * h;
#pragma unroll
    for (int b = 0; b < NO; b++)
#pragma unroll
        for (int e = 0; e < MC / 8 * MC / 32; e++)
            *(float4 *)(d + MC * b + 8 * e) = make_float4(o[b][4 * e], o[b][4 * e + 1], o[b][4 * e + 2], o[b][4 * e + 3]);
    if (h == 0) p.ws_ml[part] = make_float2(m, l);
}

template <int D, bool Q8, bool BIAS>
__global__ __launch_bounds__(64 * CK_WAVES(D), 1) void chunk_attn_kernel(const CkAttnParams p) {
    __shared__ CkNarrowShared<D, CK_WAVES(D)> sh;
    ck_narrow<D, Q8, BIAS, CK_WAVES(D)>(p, p.seq[ck_find(p.wg0, p.n_seq, blockIdx.x)], sh);
}

template <int D, bool Q8, bool BIAS>
__global__ __launch_bounds__((CkWide<D, Q8>::NT), 2) void chunk_attn_wide_kernel(const CkAttnParams p) {
    __shared__ CkWideShared<D, Q8> sh;
    ck_wide<D, Q8, BIAS>(p, p.seq[ck_find(p.wg0, p.n_seq, blockIdx.x)], sh);
}

/* A batch of both kinds, head_dim 64 and 128: prompts' chunks and single tokens
 * side by side in one launch, narrow workgroups of four waves.  (6 sessions of 1
 * to 200 rows over a Q8_0 cache at 32/8/128: 28.1 us, of which the join 5; 39.7
 * one after the other.) */
template <int D, bool Q8, bool BIAS>
__global__ __launch_bounds__(256, 2) void chunk_attn_both_kernel(const CkAttnParams p) {
    static_assert(CkWide<D, Q8>::NT == 256, "one workgroup size");
    __shared__ union {
        char any[1];
        CkWideShared<D, Q8> w;
        CkNarrowShared<D, 4> n;
    } sh;
    const CkSeq &sq = p.seq[ck_find(p.wg0, p.n_seq, blockIdx.x)];
    if (sq.wide) ck_wide<D, Q8, BIAS>(p, sq, sh.w);
    else ck_narrow<D, Q8, BIAS, 4>(p, sq, sh.n);
}

/* The splits of the wide columns joined: D / 4 threads to a column, a float4
 * each, eight splits' loads in flight. */
template <int D>
__global__ __launch_bounds__(256) void chunk_merge_kernel(const CkAttnParams p) {
    constexpr u32 V4 = D / 4, CPB = 256 / V4;
    const CkSeq &sq = p.seq[ck_find(p.wg0, p.n_seq, blockIdx.x)];
    const u32 at = (blockIdx.x - sq.wg0) * CPB + threadIdx.x / V4, d = threadIdx.x % V4;
    const u32 c0 = sq.cb0 * CK_WCOLS, cols = min(sq.n * p.gqa - c0, sq.ncb * CK_WCOLS);
    const u32 kvh = at / cols;
    if (kvh >= p.c.n_kv) return;
    const u32 cb = at % cols / CK_WCOLS, col = c0 + at % cols;
    const u64 part = (u64)sq.part0 + (u64)(kvh * sq.ncb + cb) * sq.ns * CK_WCOLS + col % CK_WCOLS;
    float M = -INFINITY, sum = 0.f;
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
    for (u32 s0 = 0; s0 < sq.ns; s0 += 8) {
        float2 ml[8];
        float4 v[8];
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const u64 x = part + (u64)min(s0 + j, sq.ns - 1) * CK_WCOLS;
            ml[j] = p.ws_ml[x];
            v[j] = *(const float4 *)(p.ws_acc + x * D + 4 * d);
        }
        float Mn = M;
#pragma unroll
        for (int j = 0; j < 8; j++) Mn = fmaxf(Mn, s0 + j < sq.ns ? ml[j].x : -INFINITY);
        const float M0 = Mn == -INFINITY ? 0.f : Mn;
        const float f0 = __builtin_amdgcn_exp2f(M - M0);
        sum *= f0;
        a.x *= f0; a.y *= f0; a.z *= f0; a.w *= f0;
#pragma unroll
        for (int j = 0; j < 8; j++) {
            if (s0 + j >= sq.ns) break;
            const float f = __builtin_amdgcn_exp2f(ml[j].x - M0);
            sum = fmaf(f, ml[j].y, sum);
            a.x = fmaf(f, v[j].x, a.x);
            a.y = fmaf(f, v[j].y, a.y);
            a.z = fmaf(f, v[j].z, a.z);
            a.w = fmaf(f, v[j].w, a.w);
        }
        M = Mn;
    }
    const u32 r = ck_row_of(p, col), head = kvh * p.gqa + col - r * p.gqa;
    const u64 brow = (u64)sq.row + r;
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    *(float4 *)(p.dst + brow * p.q_stride + (u64)head * D + 4 * d) = make_float4(a.x * inv, a.y * inv, a.z * inv, a.w * inv);
    if (p.lse && d == 0)
        p.lse[brow * p.n_head + head] = sum == 0.f ? -INFINITY
            : ((M == -INFINITY ? 0.f : M) - CK_UP + __builtin_amdgcn_logf(sum)) * CK_LN2;
}
