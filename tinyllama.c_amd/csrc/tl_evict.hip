/*
 * tl_evict.hip — which positions of a session stay in the cache, by the
 * attention weight that they have received (tl_kv_evict).
 */
#include "tl_chunk.h"

#include <string.h>

#define EV_MAX_SEQ 16
#define EV_THREADS 1024
#define EV_WAVES (EV_THREADS / 64)

struct EvSeq {
    const float *w;
    const u32 *pages;
    u32 *kept, *rows, *freed;
    float *w_out;
    u32 len, keep, sink, recent, shift;
};
struct EvParams {
    EvSeq seq[EV_MAX_SEQ];
};

/* order of the weights as unsigned numbers: NaN lowest, -0 as 0; positions
 * that stay in any case highest */
TL_DEV u32 ev_key(const EvSeq &s, u32 j) {
    if (j < s.sink || j >= s.len - s.recent) return 0xffffffffu;
    const float w = s.w[j];
    if (w != w) return 0;
    const u32 b = __float_as_uint(w + 0.f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

/* One workgroup per session.  Radix select of the keep-th largest key (four
 * passes of 8 bits, histograms in LDS), then one pass in position order that
 * ranks the kept and the evicted positions: of the keys equal to the
 * threshold the first ones stay. */
__global__ __launch_bounds__(EV_THREADS) void evict_kernel(const EvParams p) {
    __shared__ u32 s_hist[256];
    __shared__ u32 s_want, s_pref;
    __shared__ u32 s_eq[EV_WAVES], s_keep[EV_WAVES];
    const EvSeq &s = p.seq[blockIdx.x];
    const u32 tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    u32 pref = 0, want = s.keep;       /* the want-th largest among the keys that begin with pref */
    for (int sh = 24; sh >= 0; sh -= 8) {
        if (tid < 256) s_hist[tid] = 0;
        __syncthreads();
        for (u32 j = tid; j < s.len; j += EV_THREADS) {
            const u32 k = ev_key(s, j);
            if (sh == 24 || (k >> (sh + 8)) == pref) atomicAdd(&s_hist[(k >> sh) & 255], 1u);
        }
        __syncthreads();
        if (tid == 0) {
            u32 left = want, b = 255;
            while (s_hist[b] < left) left -= s_hist[b--];
            s_want = left;
            s_pref = (pref << 8) | b;
        }
        __syncthreads();
        want = s_want;
        pref = s_pref;
    }
    /* keys above pref stay, and the first `want` equal to it */
    u32 eq_base = 0, keep_base = 0;
    for (u32 j0 = 0; j0 < s.len; j0 += EV_THREADS) {
        const u32 j = j0 + tid;
        const bool in = j < s.len;
        const u32 k = in ? ev_key(s, j) : 0;
        const bool eq = in && k == pref;
        const u64 beq = __ballot(eq);
        const u64 below = (1ull << lane) - 1;
        if (lane == 0) s_eq[wave] = (u32)__popcll(beq);
        __syncthreads();
        u32 e = eq_base + (u32)__popcll(beq & below);
        for (u32 w = 0; w < EV_WAVES; w++) {
            if (w < wave) e += s_eq[w];
            eq_base += s_eq[w];
        }
        const bool stay = in && (k > pref || (eq && e < want));
        const u64 bk = __ballot(stay);
        if (lane == 0) s_keep[wave] = (u32)__popcll(bk);
        __syncthreads();
        u32 at = keep_base + (u32)__popcll(bk & below);
        for (u32 w = 0; w < EV_WAVES; w++) {
            if (w < wave) at += s_keep[w];
            keep_base += s_keep[w];
        }
        if (in) {
            const u32 row = s.pages ? (s.pages[j >> s.shift] << s.shift) + (j & ((1u << s.shift) - 1)) : j;
            if (stay) {
                if (s.kept) s.kept[at] = j;
                if (s.rows) s.rows[at] = row;
                if (s.w_out) s.w_out[at] = s.w[j];
            } else if (s.freed) {
                s.freed[j - at] = row;
            }
        }
        __syncthreads();
    }
}

extern "C" int tl_kv_evict(const tl_evict_seq *seqs, uint32_t n_seq, void *stream) {
    if (!n_seq) return TL_OK;
    if (!seqs) return tl_fail(TL_EINVAL, "evict: null sessions");
    for (u32 i = 0; i < n_seq; i++) {
        const tl_evict_seq &q = seqs[i];
        if (!q.weight || !q.len || !q.keep || q.keep > q.len || (u64)q.sink + q.recent > q.keep ||
            q.len > 0x7fffffffu)
            return tl_fail(TL_EINVAL, "evict: session %u: len %u keep %u sink %u recent %u", i, q.len,
                           q.keep, q.sink, q.recent);
        if (!q.page_size || (q.page_size & (q.page_size - 1)) || q.page_size > TL_MAX_PAGE)
            return tl_fail(TL_EINVAL, "evict: page size %u is no power of two up to %d", q.page_size, TL_MAX_PAGE);
        const void *in[2] = {q.weight, q.pages};
        const u64 in_n[2] = {q.len, ((u64)q.len + q.page_size - 1) / q.page_size};
        const void *out[4] = {q.kept, q.rows, q.freed, q.weight_out};
        const u64 out_n[4] = {q.keep, q.keep, (u64)q.len - q.keep, q.keep};
        for (int a = 0; a < 4; a++) {
            if (((uintptr_t)out[a] | (uintptr_t)in[a & 1]) & 3) return tl_fail(TL_EINVAL, "evict: session %u: alignment", i);
            for (int b = 0; b < 2; b++)
                if (tl_ranges_overlap(out[a], out_n[a] * 4, in[b], in_n[b] * 4))
                    return tl_fail(TL_EINVAL, "evict: session %u: an output overlaps an input", i);
            for (int b = 0; b < a; b++)
                if (tl_ranges_overlap(out[a], out_n[a] * 4, out[b], out_n[b] * 4))
                    return tl_fail(TL_EINVAL, "evict: session %u: outputs overlap", i);
        }
    }
    for (u32 i = 0; i < n_seq; i += EV_MAX_SEQ) {
        const u32 m = n_seq - i < EV_MAX_SEQ ? n_seq - i : EV_MAX_SEQ;
        EvParams p;
        memset(&p, 0, sizeof(p));
        for (u32 j = 0; j < m; j++) {
            const tl_evict_seq &q = seqs[i + j];
            EvSeq &s = p.seq[j];
            s.w = q.weight;
            s.pages = q.pages;
            s.kept = q.kept;
            s.rows = q.rows;
            s.freed = q.freed;
            s.w_out = q.weight_out;
            s.len = q.len;
            s.keep = q.keep;
            s.sink = q.sink;
            s.recent = q.recent;
            s.shift = (u32)__builtin_ctz(q.page_size);
        }
        hipLaunchKernelGGL(evict_kernel, dim3(m), dim3(EV_THREADS), 0, (hipStream_t)stream, p);
        HIP_TRY(hipGetLastError());
    }
    return TL_OK;
}
