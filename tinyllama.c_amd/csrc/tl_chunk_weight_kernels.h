/* tl_chunk_weight_kernels.h — the attention weight that every cached position
 * received from a batch of chunks: column sums of the probabilities, from the
 * row sums (lse) that the attention wrote. */
#pragma once
#include "tl_chunk.h"

/* One workgroup per tile of 32 keys of a chunk; its waves take the kv heads in
 * turn, each with the tile's K as the matrix operand in registers against all
 * column blocks of the head.  A lane sums its eight keys over its columns; the
 * 16 lanes of a key and then the waves are joined in a fixed order. */
template <int D, bool Q8, bool BIAS>
__global__ __launch_bounds__(256) void chunk_weight_kernel(const CkAttnParams p) {
    constexpr int KS = D / 32;
    __shared__ float s_sum[4][CK_KEYS];
    const u32 lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const u32 i = lane & 15, g = lane >> 4;
    const CkSeq &sq = p.seq[ck_find(p.wg0, p.n_seq, blockIdx.x)];
    const u32 kb = (blockIdx.x - sq.wg0) * CK_KEYS;
    const u32 end = sq.pos + sq.n, cols = sq.n * p.gqa;
    const u32 key = kb + (lane & 31);
    const u32 row = key < end ? ck_row(p.c, sq.pages, key) : ~0u;
    const u64 bad = __ballot(row >= p.c.cap);
    const u32 rc = row < p.c.cap ? row : 0;
    u32 rk[2];
#pragma unroll
    for (int a = 0; a < 2; a++) rk[a] = __shfl(rc, 8 * (i >> 2) + 4 * a + (i & 3));
    const float icap = p.softcap > 0.f ? 1.f / p.softcap : 0.f;
    float sum[8] = {};
    for (u32 kvh = wave; kvh < p.c.n_kv; kvh += 4) {
        CkTile<D, Q8> tile;
        tile.load_k(p.c, kvh, rk, g);
        for (u32 cb = 0; cb < sq.ncb; cb++) {
            const u32 c = cb * CK_COLS + i;
            const bool real = c < cols;
            const u32 col = real ? c : cols - 1;
            const u32 r = col / p.gqa, head = kvh * p.gqa + col % p.gqa;
            const u32 pq = sq.pos + r;
            const u64 brow = (u64)sq.row + r;
            CkSees see;
            see.set(pq, end, p.window, sq.prefix, p.first ? p.first[brow] : 0);
            bool any = false;
#pragma unroll
            for (int e = 0; e < 8; e++) any |= see.sees(kb + 8 * g + e);
            if (!__any(any && real)) continue;
            h8_t qh[KS], ql[KS];
            float4 qx[KS][2];
            ck_load_q<D, 4>(p.q + brow * p.q_stride + (u64)head * D, g, qx);
            float cs = ck_split_q<D, 4>(qx, p.scale, qh, ql);
            if constexpr (!BIAS) cs *= CK_LOG2E;
            const float slope = BIAS && p.slopes ? p.slopes[head] : 0.f;
            const float lse = p.lse[brow * p.n_head + head] * CK_LOG2E;
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
                for (int e = 0; e < 4; e++) {
                    const u32 k = kb + 8 * g + 4 * a + e;
                    const float x = ck_score<BIAS>(acc[e], cs, p.softcap, icap, slope, pq, k);
                    const bool vis = real && see.sees(k) && !((bad >> (8 * g + 4 * a + e)) & 1);
                    sum[4 * a + e] += vis ? __builtin_amdgcn_exp2f(x - lse) : 0.f;
                }
            }
        }
    }
#pragma unroll
    for (int e = 0; e < 8; e++) {
        const float s = group_sum<16>(sum[e]);
        if (i == 0) s_sum[wave][8 * g + e] = s;
    }
    __syncthreads();
    if (threadIdx.x < CK_KEYS && kb + threadIdx.x < end) {
        const u32 k = threadIdx.x;
        sq.weight[kb + k] += (s_sum[0][k] + s_sum[1][k]) + (s_sum[2][k] + s_sum[3][k]);
    }
}
