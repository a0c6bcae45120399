/* tl_chunk_attn_kernels.h — attention of a batch of chunks over a paged cache.
 *
 * Columns: a chunk's rows x the q heads of one kv head (column = row * gqa +
 * head), 16 to a workgroup; a column's softmax runs in one pass over the keys
 * with a running maximum and sum. */
#pragma once
#include "tl_chunk.h"

#define CK_WAVES 4

/* the maximum moves only when a score passes it by more than 2^CK_LAZY, and
 * probabilities are taken against 2^CK_UP below it: they reach 2^15 at most, so
 * that the low halves of the small ones stay normal f16 numbers too */
#define CK_LAZY 8.f
#define CK_UP 7.f

template <int D, bool Q8, bool BIAS>
__global__ __launch_bounds__(64 * CK_WAVES, D == 256 ? 1 : 2) void chunk_attn_kernel(const CkAttnParams p) {
    constexpr int KS = D / 32, NM = D / 16;
    constexpr int ROWF = D + 4;
    __shared__ float s_o[CK_WAVES][CK_COLS][ROWF];
    __shared__ float s_m[CK_WAVES][CK_COLS], s_l[CK_WAVES][CK_COLS];
    __shared__ u32 s_last;
    const u32 lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const u32 i = lane & 15, g = lane >> 4;
    const CkSeq &sq = p.seq[ck_find(p.seq, p.n_seq, blockIdx.x)];
    const u32 local = blockIdx.x - sq.wg0;
    const u32 kvh = local % p.c.n_kv, rest = local / p.c.n_kv;
    const u32 cb = rest % sq.ncb, split = rest / sq.ncb;
    const u32 c0 = cb * CK_COLS;
    const u32 ncol = min((u32)CK_COLS, sq.n * p.gqa - c0);
    /* columns past the last one repeat it and are not written */
    const u32 col = c0 + min(i, ncol - 1);
    const u32 r = col / p.gqa, head = kvh * p.gqa + col % p.gqa;
    const u32 pq = sq.pos + r, end = sq.pos + sq.n;
    const u64 brow = (u64)sq.row + r;

    h8_t qh[KS], ql[KS];
    float cs = ck_load_q<D>(p.q + brow * p.q_stride + (u64)head * D, g, p.scale, qh, ql);
    if constexpr (!BIAS) cs *= CK_LOG2E;
    const float slope = BIAS && p.slopes ? p.slopes[head] : 0.f;
    const float icap = p.softcap > 0.f ? 1.f / p.softcap : 0.f;

    CkSees see;
    see.set(pq, end, p.window, sq.prefix, p.first ? p.first[brow] : 0);
    CkTiles tiles;
    tiles.set<16>(see);
    const u32 n_tiles = tiles.count();
    const u32 t0 = (u32)((u64)n_tiles * split / sq.ns), t1 = (u32)((u64)n_tiles * (split + 1) / sq.ns);

    float m = -INFINITY, l = 0.f;
    f4_t o[NM];
#pragma unroll
    for (int j = 0; j < NM; j++) o[j] = (f4_t){0.f, 0.f, 0.f, 0.f};

    CkTile<D, Q8> tile;
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
    u32 t = t0 + wave;
    u32 row = 0, next = 0;
    if (t < t1) {
        row = look(t);
        const u32 rc = row < p.c.cap ? row : 0;
        u32 rk[2], rv[8];
        rows_k(rc, rk);
        tile.load_k(p.c, kvh, rk, g);
        rows_v(rc, rv);
        tile.load_v(p.c, kvh, rv, i);
        if (t + CK_WAVES < t1) next = look(t + CK_WAVES);
    }
    for (; t < t1; t += CK_WAVES) {
        const u32 kb = tiles.key(t);
        const u64 bad = __ballot(row >= p.c.cap);
        const bool more = t + CK_WAVES < t1;
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
            for (int e = 0; e < 4; e++)
                x[4 * a + e] = ck_score<BIAS>(acc[e], cs, p.softcap, icap, slope, pq, kb + 8 * g + 4 * a + e);
        }
        u32 rn = 0;
        if (more) {
            rn = next < p.c.cap ? next : 0;
            u32 rk[2];
            rows_k(rn, rk);
            tile.load_k(p.c, kvh, rk, g);
        }
        u64 seen[8];
        bool slow = false;
        const bool full = tiles.full(kb) && !bad;
        if (!full) {
            bool odd = false;
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const bool vis = see.sees(kb + 8 * g + e) && !((bad >> (8 * g + e)) & 1);
                x[e] = vis ? x[e] : -INFINITY;
                seen[e] = __ballot(vis);
                const u32 mine = (u32)(seen[e] >> (16 * g)) & 0xffffu;
                if (mine == 0) tile.clear_v(e);
                else if (mine != 0xffffu) odd |= tile.odd_v(e);
            }
            slow = __any(odd);
        }
        /* running maximum */
        float top = x[0];
#pragma unroll
        for (int e = 1; e < 8; e++) top = fmaxf(top, x[e]);
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
        h8_t ph, pl;
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const float pe = __builtin_amdgcn_exp2f(x[e] - mref);
            l += pe;
            _Float16 a, b;
            ck_split(pe, a, b);
            ph[e] = a;
            pl[e] = b;
        }
        if (!slow) {
#pragma unroll
            for (int j = 0; j < NM; j++) {
                h8_t vh, vl;
                tile.get_v(j, vh, vl);
                o[j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vh, ph, o[j], 0, 0, 0);
                o[j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vh, pl, o[j], 0, 0, 0);
                if constexpr (Q8) o[j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vl, ph, o[j], 0, 0, 0);
            }
        } else {
            /* a key that only some columns see holds infinities or NaN: column
             * by column, the others' keys as zeros */
            for (u32 c = 0; c < CK_COLS; c++) {
                CkTile<D, Q8> tc = tile;
#pragma unroll
                for (int e = 0; e < 8; e++)
                    if (!((seen[e] >> (16 * g + c)) & 1)) tc.clear_v(e);
#pragma unroll
                for (int j = 0; j < NM; j++) {
                    h8_t vh, vl;
                    tc.get_v(j, vh, vl);
                    f4_t s = __builtin_amdgcn_mfma_f32_16x16x32_f16(vh, ph, o[j], 0, 0, 0);
                    s = __builtin_amdgcn_mfma_f32_16x16x32_f16(vh, pl, s, 0, 0, 0);
                    if constexpr (Q8) s = __builtin_amdgcn_mfma_f32_16x16x32_f16(vl, ph, s, 0, 0, 0);
                    if (i == c) o[j] = s;
                }
            }
        }
        if (more) {
            u32 rv[8];
            rows_v(rn, rv);
            tile.load_v(p.c, kvh, rv, i);
            row = next;
            if (t + 2 * CK_WAVES < t1) next = look(t + 2 * CK_WAVES);
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
            *(float4 *)&s_o[wave][i][NM * (4 * g + e) + j] =
                make_float4(o[j][e], o[j + 1][e], o[j + 2][e], o[j + 3][e]);
    __syncthreads();
    constexpr u32 V4 = D / 4;
    const u32 units = ncol * V4;
    const u32 group = kvh * sq.ncb + cb;
    const u64 set0 = (u64)sq.part0 + (u64)group * sq.ns;      /* the group's first partial set */
    const __amdgpu_buffer_rsrc_t ra = buf_rsrc(p.ws_acc + set0 * CK_COLS * D);
    const __amdgpu_buffer_rsrc_t rm = buf_rsrc(p.ws_ml + set0 * CK_COLS);
    for (u32 u = threadIdx.x; u < units; u += 64 * CK_WAVES) {
        const u32 c = u / V4, d = u % V4;
        float M = -INFINITY;
#pragma unroll
        for (int w = 0; w < CK_WAVES; w++) M = fmaxf(M, s_m[w][c]);
        const float M0 = M == -INFINITY ? 0.f : M;
        float sum = 0.f;
        float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < CK_WAVES; w++) {
            const float f = __builtin_amdgcn_exp2f(s_m[w][c] - M0);
            const float4 v = *(const float4 *)&s_o[w][c][4 * d];
            sum = fmaf(f, s_l[w][c], sum);
            a.x = fmaf(f, v.x, a.x);
            a.y = fmaf(f, v.y, a.y);
            a.z = fmaf(f, v.z, a.z);
            a.w = fmaf(f, v.w, a.w);
        }
        if (sq.ns == 1) {
            const u32 cc = c0 + c, rr = cc / p.gqa, hh = kvh * p.gqa + cc % p.gqa;
            const u64 br = (u64)sq.row + rr;
            const float inv = sum == 0.f ? 0.f : 1.f / sum;
            *(float4 *)(p.dst + br * p.q_stride + (u64)hh * D + 4 * d) =
                make_float4(a.x * inv, a.y * inv, a.z * inv, a.w * inv);
            if (p.lse && d == 0)
                p.lse[br * p.n_head + hh] = sum == 0.f ? -INFINITY : (M0 - CK_UP + __log2f(sum)) * CK_LN2;
        } else {
            const u32x4v_t v = {__float_as_uint(a.x), __float_as_uint(a.y), __float_as_uint(a.z), __float_as_uint(a.w)};
            __builtin_amdgcn_raw_buffer_store_b128(v, ra, ((split * CK_COLS + c) * D + 4 * d) * 4, 0, TL_SC1);
            if (d == 0) {
                const u32x2v_t ml = {__float_as_uint(M), __float_as_uint(sum)};
                __builtin_amdgcn_raw_buffer_store_b64(ml, rm, (split * CK_COLS + c) * 8, 0, TL_SC1);
            }
        }
    }
    if (sq.ns == 1) return;
    /* the last split of the group to arrive joins them all */
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    u32 *cnt = p.cnt + (u64)(sq.grp0 + group) * CK_CNT_PAD;
    if (threadIdx.x == 0)
        s_last = __hip_atomic_fetch_add(cnt, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == sq.ns - 1;
    __syncthreads();
    if (!s_last) return;
    for (u32 u = threadIdx.x; u < units; u += 64 * CK_WAVES) {
        const u32 c = u / V4, d = u % V4;
        float M = -INFINITY, sum = 0.f;
        float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
        for (u32 s0 = 0; s0 < sq.ns; s0 += 8) {
            u32x2v_t ml[8];
            u32x4v_t v[8];
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const u32 s = min(s0 + j, sq.ns - 1);
                ml[j] = __builtin_amdgcn_raw_buffer_load_b64(rm, (s * CK_COLS + c) * 8, 0, TL_SC1);
                v[j] = __builtin_amdgcn_raw_buffer_load_b128(ra, ((s * CK_COLS + c) * D + 4 * d) * 4, 0, TL_SC1);
            }
            float Mn = M;
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const u32 mb = ml[j][0];
                Mn = fmaxf(Mn, s0 + j < sq.ns ? __uint_as_float(mb) : -INFINITY);
            }
            const float M0 = Mn == -INFINITY ? 0.f : Mn;
            const float f0 = __builtin_amdgcn_exp2f(M - M0);
            sum *= f0;
            a.x *= f0; a.y *= f0; a.z *= f0; a.w *= f0;
#pragma unroll
            for (int j = 0; j < 8; j++) {
                if (s0 + j >= sq.ns) break;
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
        const u32 cc = c0 + c, rr = cc / p.gqa, hh = kvh * p.gqa + cc % p.gqa;
        const u64 br = (u64)sq.row + rr;
        const float M0 = M == -INFINITY ? 0.f : M;
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
        *(float4 *)(p.dst + br * p.q_stride + (u64)hh * D + 4 * d) =
            make_float4(a.x * inv, a.y * inv, a.z * inv, a.w * inv);
        if (p.lse && d == 0)
            p.lse[br * p.n_head + hh] = sum == 0.f ? -INFINITY : (M0 - CK_UP + __log2f(sum)) * CK_LN2;
    }
    if (threadIdx.x == 0)
        __hip_atomic_store(cnt, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
