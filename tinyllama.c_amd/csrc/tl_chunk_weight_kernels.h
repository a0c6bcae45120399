/* tl_chunk_weight_kernels.h — the attention weight that every cached position
 * received from a batch of chunks: column sums of the probabilities, from the
 * row sums (lse) that the attention wrote. */
#pragma once
#include "tl_chunk.h"

/* ---- few columns (at most 16) --------------------------------------------------
 *
 * Bound by the read of K.  A workgroup has a run of 32-key tiles of a chunk; each
 * of its eight waves has one kv head (with fewer heads several waves share one
 * and take its tiles in turn; with more, the heads come in groups of eight) and
 * keeps that head's q in registers while K comes straight into the matrix operand
 * layout, one tile ahead.  A lane sums its eight keys' probabilities; the 16
 * columns are joined by DPP, the waves through LDS in order.  8 sessions of 3000 to
 * 12000 keys at 32/8/128: 22.4 us, 4.9 TB/s. */
#define CK_WTILES 32   /* tiles of a workgroup between two joins */

template <int D, bool Q8, bool BIAS>
__global__ __launch_bounds__(512, D == 64 ? 4 : 2) void chunk_weight_kernel(const CkAttnParams p) {
    constexpr int KS = D / 32;
    constexpr bool TWO = D < 256 || Q8;      /* room for two tiles' K */
    __shared__ float s_sum[8][CK_WTILES][CK_KEYS];
    const u32 lane = threadIdx.x & 63, wave = ck_uniform(threadIdx.x >> 6);
    const u32 i = lane & 15, g = lane >> 4;
    const CkSeq &sq = p.seq[ck_find(p.wg0, p.n_seq, blockIdx.x)];
    /* ncb: tiles of a workgroup; part0: the chunk's first key */
    const u32 end = sq.pos + sq.n, cols = sq.n * p.gqa;
    const u32 k0 = sq.part0 + (blockIdx.x - sq.wg0) * sq.ncb * CK_KEYS;
    const u32 tiles = min(sq.ncb, (end - k0 + CK_KEYS - 1) / CK_KEYS);
    const u32 share = p.c.n_kv >= 8 ? 1 : 8 / p.c.n_kv;       /* waves of a head */
    const u32 groups = (p.c.n_kv + 7) / 8;
    const u32 turn = wave / (8 / share);
    const bool real = i < cols;
    const u32 col = real ? i : cols - 1;
    const u32 r = ck_row_of(p, col);
    const u32 pq = sq.pos + r;
    const u64 brow = (u64)sq.row + r;
    const u32 first = p.first ? p.first[brow] : 0;
    CkSees see;
    see.set(pq, end, p.window, sq.prefix, first);
    CkSpan span;
    span.set(sq.pos, sq.pos + sq.n - 1, end, p.window, sq.prefix,
             p.first ? ck_uniform(group_umin<16>(first)) : 0, p.first ? ck_uniform(group_umax<16>(first)) : 0);
    auto look = [&](u32 t) -> u32 {
        const u32 key = k0 + t * CK_KEYS + (lane & 31);
        return key < end ? ck_row(p.c, sq.pages, key) : ~0u;
    };
    for (u32 b0 = 0; b0 < tiles; b0 += CK_WTILES) {
        const u32 b1 = min(b0 + CK_WTILES, tiles);
        for (u32 x = lane; x < CK_WTILES * CK_KEYS; x += 64) s_sum[wave][0][x] = 0.f;
        for (u32 hg = 0; hg < groups; hg++) {
            const u32 kvh = p.c.n_kv >= 8 ? hg * 8 + wave : wave % (8 / share);
            if (kvh >= p.c.n_kv || turn >= share) continue;
            const u32 head = kvh * p.gqa + col - r * p.gqa;
            CkTile<D, Q8> tile, ahead;
            auto load = [&](CkTile<D, Q8> &to, u32 row) {
                const u32 rc = row < p.c.cap ? row : 0;
                u32 rk[2];
#pragma unroll
                for (int a = 0; a < 2; a++) rk[a] = __shfl(rc, 8 * (i >> 2) + 4 * a + (i & 3));
                to.load_k(p.c, kvh, rk, g);
            };
            u32 t = b0 + turn;
            u32 row = t < b1 ? look(t) : 0, next = t + share < b1 ? look(t + share) : 0;
            float4 qx[KS][2];
            ck_load_q<D, 4>(p.q + brow * p.q_stride + (u64)head * D, g, qx);
            float lse = p.lse[brow * p.n_head + head] * CK_LOG2E;
            if (t < b1) load(tile, row);
            h8_t qh[KS], ql[KS];
            CkScore<BIAS> score;
            score.set(p, ck_split_q<D, 4>(qx, p.scale, qh, ql), head);
            const float mul = score.factor();
            lse = real ? lse : INFINITY;       /* columns past the last one count nothing */
            for (; t < b1; t += share) {
                const u32 kb = k0 + t * CK_KEYS;
                const u64 bad = __ballot(row >= p.c.cap);
                const u32 coming = next;
                if (TWO && t + share < b1) load(ahead, coming);
                row = next;
                if (TWO && t + 2 * share < b1) next = look(t + 2 * share);
                const bool any = span.any(kb, CK_KEYS);
                float x[8];
                if (any) {
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
                }
                if constexpr (!TWO) {
                    if (t + share < b1) load(tile, coming);
                    if (t + 2 * share < b1) next = look(t + 2 * share);
                }
                if (any) {
                    score.template apply<8>(x, (int)(pq - kb - 8 * g), [](int e) { return e; });
                    const bool full = span.full(kb, CK_KEYS) && !bad;
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        float pe = __builtin_amdgcn_exp2f(fmaf(x[e], mul, -lse));
                        if (!full) pe = see.sees(kb + 8 * g + e) && !((bad >> (8 * g + e)) & 1) ? pe : 0.f;
                        pe = group_sum<16>(pe);
                        if (i == 0) s_sum[wave][t - b0][8 * g + e] += pe;
                    }
                }
                if constexpr (TWO) tile = ahead;
            }
        }
        __syncthreads();
        for (u32 x = threadIdx.x; x < (b1 - b0) * CK_KEYS; x += 512) {
            const u32 key = k0 + b0 * CK_KEYS + x;
            float sum = 0.f;
#pragma unroll
            for (int w = 0; w < 8; w++) sum += s_sum[w][0][x];
            if (key < end) sq.weight[key] += sum;
        }
        __syncthreads();
    }
}

/* ---- many columns ------------------------------------------------------------
 *
 * A workgroup keeps 512 keys of one kv head in registers (256 where K takes too
 * many), 64 to a wave, as the A operands of v_mfma_f32_32x32x16_f16, and goes
 * through a share of the head's columns: CT at a time are fetched, split into
 * pairs of f16 and put to LDS by all 512 threads (two buffers, one barrier each),
 * and every wave multiplies its keys with them.  A lane sums 16 keys over one column of 32; the lanes are
 * joined at the end and the workgroup's sums go to its place in the workspace,
 * which chunk_weight_sum_kernel adds up in order.  Bound by the vector
 * instructions on the scores, with a cap 17 (nine of them its tanh): some 80
 * cycles for 64 scores beside 16 of matrix work.  512 rows over 4608 keys at
 * 32/8/64 with a cap 60.5 us, of which the sums of the shares 5. */
typedef float f16w_t __attribute__((ext_vector_type(16)));

template <int D, bool Q8>
struct CkWeight {
    static constexpr int KB = ck_weight_keys(D, Q8) / 256;   /* blocks of 32 keys of a wave */
    static constexpr int CT = D == 256 ? 32 : 64;     /* columns of a buffer */
    static constexpr int TPC = 512 / CT;              /* threads of a column */
    static constexpr int QV = D / 4 / TPC;            /* float4s of one of them */
    static constexpr int U = D / 8;                   /* 16-byte units of a column's row */
    static constexpr int PLANE = CT * U * 16;
    static TL_DEV u32 at(u32 col, u32 unit) {
        return (col * U + (unit ^ (U == 8 ? (col >> 1) & 7 : col & 15))) * 16;
    }
};

template <int D, bool Q8, bool BIAS>
__global__ __launch_bounds__(512, D == 64 && !Q8 ? 4 : 2) void chunk_weight_wide_kernel(const CkAttnParams p) {
    typedef CkWeight<D, Q8> W;
    constexpr int NS = D / 16, CT = W::CT, KB = W::KB, WKEYS = 256 * KB;
    __shared__ __align__(16) char s_q[2][2][W::PLANE];    /* buffer, hi / lo */
    __shared__ CkScore<BIAS> s_score[2][CT];
    __shared__ CkSees s_see[2][CT];
    __shared__ u32 s_pos[2][CT], s_first[2][CT];
    __shared__ float s_lse[2][CT];
    const u32 lane = threadIdx.x & 63, wave = ck_uniform(threadIdx.x >> 6);
    const u32 i = lane & 31, h = lane >> 5;
    const CkSeq &sq = p.seq[ck_find(p.wg0, p.n_seq, blockIdx.x)];
    /* ncb: key blocks from key part0 on; ns: shares of the columns; grp0: first set of sums */
    const u32 local = blockIdx.x - sq.wg0;
    const u32 kvh = local % p.c.n_kv, rest = local / p.c.n_kv;
    const u32 kblk = rest % sq.ncb, share = rest / sq.ncb;
    const u32 end = sq.pos + sq.n, cols = sq.n * p.gqa;
    const u32 k0 = sq.part0 + kblk * WKEYS + wave * (32 * KB);
    const u32 tiles = (cols + CT - 1) / CT;
    const u32 t0 = (u32)((u64)tiles * share / sq.ns), t1 = (u32)((u64)tiles * (share + 1) / sq.ns);

    /* matrix row rho is key rho with bits 2 and 3 exchanged (any order would do) */
    u32 row[KB];
#pragma unroll
    for (int x = 0; x < KB; x++) {
        const u32 key = k0 + 32 * x + ((i & 19) | ((i & 4) << 1) | ((i & 8) >> 1));
        row[x] = key < end ? ck_row(p.c, sq.pages, key) : ~0u;
    }
    h8_t kh[KB][NS], kl[Q8 ? KB : 1][Q8 ? NS : 1];
#pragma unroll
    for (int x = 0; x < KB; x++) {
        const u32 rc = row[x] < p.c.cap ? row[x] : 0;
        if constexpr (!Q8) {
            const char *base = (const char *)(p.c.k + (u64)kvh * p.c.cap * D);
#pragma unroll
            for (int s = 0; s < NS; s++) kh[x][s] = *(const h8_t *)(base + (u64)(rc * (u32)(2 * D) + s * 32 + h * 16));
        } else {
            const char *base = (const char *)p.c.k + (u64)kvh * p.c.cap * D;
            const u16 *sb = p.c.ks + (u64)kvh * p.c.cap * (D / 32);
#pragma unroll
            for (int s = 0; s < NS; s++) {
                const uint2 v = *(const uint2 *)(base + (u64)(rc * (u32)D + s * 16 + h * 8));
                const tl_half2 d2 = __builtin_bit_cast(tl_half2, (u32)sb[(u64)(rc * (u32)(D / 32) + (s >> 1))] * 0x10001u);
                tl_half2 w[4];
                i8x4_to_f16(v.x, w[0], w[1]);
                i8x4_to_f16(v.y, w[2], w[3]);
                u4_t a, b;
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    u32 y, z;
                    ck_q8_pair(w[j], d2, y, z);
                    a[j] = y;
                    b[j] = z;
                }
                kh[x][s] = __builtin_bit_cast(h8_t, a);
                kl[x][s] = __builtin_bit_cast(h8_t, b);
            }
        }
    }

    const u32 tc = threadIdx.x / W::TPC, tt = threadIdx.x % W::TPC;
    float4 qx[W::QV];
    auto fetch = [&](u32 t) {
        const u32 c = min(t * CT + tc, cols - 1);
        const u32 r = ck_row_of(p, c), head = kvh * p.gqa + c - r * p.gqa;
        const float *q = p.q + ((u64)sq.row + r) * p.q_stride + (u64)head * D + 4 * tt;
#pragma unroll
        for (int j = 0; j < W::QV; j++) qx[j] = *(const float4 *)(q + 4 * W::TPC * j);
    };
    auto store = [&](u32 t) {
        const u32 buf = (t - t0) & 1, cg = t * CT + tc, c = min(cg, cols - 1);
        float m = 0.f;
#pragma unroll
        for (int j = 0; j < W::QV; j++)
            m = fmaxf(fmaxf(m, fmaxf(fabsf(qx[j].x), fabsf(qx[j].y))), fmaxf(fabsf(qx[j].z), fabsf(qx[j].w)));
        m = group_max<W::TPC>(m);
        const int e = ck_row_exp(m);
        const float up = __uint_as_float((u32)(e + 127) << 23);
#pragma unroll
        for (int j = 0; j < W::QV; j++) {
            uint2 hi, lo;
            ck_split2(qx[j].x * up, qx[j].y * up, hi.x, lo.x);
            ck_split2(qx[j].z * up, qx[j].w * up, hi.y, lo.y);
            const u32 f = W::TPC * j + tt;      /* float4 of the row */
            const u32 at = W::at(tc, f >> 1) + (f & 1) * 8;
            *(uint2 *)(s_q[buf][0] + at) = hi;
            *(uint2 *)(s_q[buf][1] + at) = lo;
        }
        if (tt == 0) {
            const u32 r = ck_row_of(p, c), head = kvh * p.gqa + c - r * p.gqa, pq = sq.pos + r;
            const u64 brow = (u64)sq.row + r;
            const u32 first = p.first ? p.first[brow] : 0;
            CkSees see;
            see.set(pq, end, p.window, sq.prefix, first);
            CkScore<BIAS> score;
            score.set(p, __uint_as_float((u32)(127 - e) << 23) * p.scale, head);
            s_see[buf][tc] = see;
            s_score[buf][tc] = score;
            s_pos[buf][tc] = pq;
            s_first[buf][tc] = first;
            /* columns past the last one count nothing */
            s_lse[buf][tc] = cg < cols ? p.lse[brow * p.n_head + head] * CK_LOG2E : INFINITY;
        }
    };

    float sum[KB][16] = {};
    if (t0 < t1) {
        fetch(t0);
        store(t0);
    }
#pragma unroll 1
    for (u32 t = t0; t < t1; t++) {
        __syncthreads();
        if (t + 1 < t1) fetch(t + 1);
        const u32 buf = (t - t0) & 1;
#pragma unroll 1
        for (u32 sub = 0; sub < CT / 32; sub++) {
            const u32 cb = t * CT + 32 * sub;
            if (cb >= cols) break;
            u32 fmin = 0, fmax = 0;
            if (p.first) {
                const u32 f = s_first[buf][32 * sub + i];
                fmin = ck_uniform(group_umin<32>(f));
                fmax = ck_uniform(group_umax<32>(f));
            }
            CkSpan span;
            span.set(sq.pos + ck_row_of(p, cb), sq.pos + ck_row_of(p, min(cb + 31, cols - 1)), end, p.window, sq.prefix, fmin, fmax);
            if (!span.any(k0, 32 * KB)) continue;
            const u32 cl = 32 * sub + i;
            u32 rd = W::at(cl, h);
            asm volatile("" : "+v"(rd));
            const char *qp = s_q[buf][0];
            f16w_t s[KB];
#pragma unroll
            for (int x = 0; x < KB; x++) s[x] = (f16w_t)(0.f);
            constexpr int AHEAD = 4;
            h8_t a[AHEAD], b[AHEAD];
            auto read = [&](int j) {
                const char *at = qp + (rd ^ (j * 32));
                a[j % AHEAD] = *(const h8_t *)at;
                b[j % AHEAD] = *(const h8_t *)(at + W::PLANE);
            };
#pragma unroll
            for (int j = 0; j < AHEAD; j++) read(j);
#pragma unroll
            for (int j = 0; j < NS; j++) {
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int x = 0; x < KB; x++) {
                    s[x] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kh[x][j], a[j % AHEAD], s[x], 0, 0, 0);
                    s[x] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kh[x][j], b[j % AHEAD], s[x], 0, 0, 0);
                    if constexpr (Q8) s[x] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kl[x][j], a[j % AHEAD], s[x], 0, 0, 0);
                }
                if (j + AHEAD < NS) read(j + AHEAD);
            }
            __builtin_amdgcn_sched_barrier(0);
            const CkScore<BIAS> score = s_score[buf][cl];
            const float mul = score.factor(), lse = s_lse[buf][cl];
            const u32 pq = s_pos[buf][cl];
#pragma unroll
            for (int x = 0; x < KB; x++) {
                const u32 kb = k0 + 32 * x;
                score.template apply<16>(s[x], (int)(pq - kb - 8 * h), [](int e) { return 16 * (e >> 3) + (e & 7); });
                if (span.full(kb, 32)) {
#pragma unroll
                    for (int e = 0; e < 16; e++) sum[x][e] += __builtin_amdgcn_exp2f(fmaf(s[x][e], mul, -lse));
                } else {
                    asm volatile("");      /* stays a branch */
                    const CkSees see = s_see[buf][cl];
#pragma unroll
                    for (int e = 0; e < 16; e++) {
                        const bool v = see.sees(kb + 16 * (e >> 3) + 8 * h + (e & 7));
                        sum[x][e] += v ? __builtin_amdgcn_exp2f(fmaf(s[x][e], mul, -lse)) : 0.f;
                    }
                }
            }
        }
        if (t + 1 < t1) store(t + 1);
    }
    /* the columns' lanes joined; keys without a row count nothing */
    float *out = p.ws_acc + ((u64)sq.grp0 + (u64)(share * p.c.n_kv + kvh) * sq.ncb + kblk) * WKEYS + wave * (32 * KB);
#pragma unroll
    for (int x = 0; x < KB; x++) {
        const u64 bad = __ballot(row[x] >= p.c.cap);
#pragma unroll
        for (int e = 0; e < 16; e++) {
            const float y = group_sum<32>(sum[x][e]);
            const u32 k = 16 * (e >> 3) + 8 * h + (e & 7);
            const u32 rho = (k & 19) | ((k & 4) << 1) | ((k & 8) >> 1);      /* the lane that holds key k's row */
            if (i == 0) out[32 * x + k] = (bad >> rho) & 1 ? 0.f : y;
        }
    }
}
