/*
 * tl_evict.hip — which positions of a session stay in the cache, by the
 * attention weight that they have received (tl_kv_evict).
 */
#include "tl_chunk.h"

#include <stdlib.h>
#include <string.h>

#define EV_MAX_SEQ 16
#define EV_THREADS 1024
#define EV_WAVES (EV_THREADS / 64)
#define EV_ONE 8                            /* keys of a thread where one workgroup has a session */
#define EV_PER 2                            /* ... where several share it: more of them run at once */
#define EV_SEG (EV_THREADS * EV_PER)        /* positions of one of these */
#define EV_BINS 2048                        /* digits of 11, 11 and 10 bits */
#define EV_LOW 1024
#define EV_MAX_SEG EV_THREADS               /* segments of a session that several workgroups share */
#define EV_SEGW (EV_LOW + 8)                /* scratch words of a segment: counts by the last digit */
#define EV_AUX (EV_BINS + EV_LOW + 8)       /* of a session: histograms of digits 1 and 2, (prefix, want) of 0 and 1 */
static_assert(EV_MAX_SEQ * EV_BINS <= TL_MERGE_MAX_GROUPS * TL_MERGE_PAD, "counters of a stream's workspace");

struct EvSeq {
    const float *w;
    const u32 *pages;
    u32 *kept, *rows, *freed;
    float *w_out;
    u32 *cnt;                               /* histogram of digit 0, zero between calls */
    u32 *seg;                               /* EV_SEGW words per segment */
    u32 *aux;                               /* EV_AUX words */
    u32 len, keep, sink, recent, shift, wg0;
};
struct EvParams {
    u32 wg0[CK_MAX_SEQ];                    /* seq[].wg0 side by side */
    EvSeq seq[EV_MAX_SEQ];
    u32 n_seq;
};

/* order of the weights as unsigned numbers: NaN lowest, -0 as 0; positions
 * that stay in any case highest */
TL_DEV u32 ev_order(const EvSeq &s, u32 j, float w) {
    if (j < s.sink || j >= s.len - s.recent) return 0xffffffffu;
    if (w != w) return 0;
    const u32 b = __float_as_uint(w + 0.f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
TL_DEV u32 ev_key(const EvSeq &s, u32 j) { return ev_order(s, j, s.w[j]); }

/* inclusive sum over the wave's lanes: DPP moves within rows of 16, then the
 * rows' last lanes broadcast */
TL_DEV u32 ev_wave_scan(u32 x) {
#define EV_STEP(ctrl, rows) x += (u32)__builtin_amdgcn_update_dpp(0, (int)x, ctrl, rows, 0xf, false)
    EV_STEP(0x111, 0xf);
    EV_STEP(0x112, 0xf);
    EV_STEP(0x114, 0xf);
    EV_STEP(0x118, 0xf);
    EV_STEP(0x142, 0xa);
    EV_STEP(0x143, 0xc);
#undef EV_STEP
    return x;
}

/* Exclusive sum over the workgroup's threads, and the total.  One barrier: the
 * caller has one of its own between a scan and the next use of s_w. */
TL_DEV u32 ev_scan(u32 x, u32 *s_w, u32 &total) {
    const u32 lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const u32 y = ev_wave_scan(x);
    if (lane == 63) s_w[wave] = y;
    __syncthreads();
    u32 base = 0;
    total = 0;
#pragma unroll
    for (u32 w = 0; w < EV_WAVES; w++) {
        base += w < wave ? s_w[w] : 0;
        total += s_w[w];
    }
    return base + y - x;
}

/* The bin that holds the want-th key from the top, its rank in there and the
 * bin's keys; h: the thread's bins, 2047 - 2 tid downwards (a histogram of 1024
 * bins: the lowest of them).  Two barriers. */
TL_DEV void ev_pick(u32 h0, u32 h1, u32 &want, u32 &bin, u32 &held, u32 *s_w, u32 *s_pick) {
    u32 total;
    const u32 at = ev_scan(h0 + h1, s_w, total), tid = threadIdx.x;
    if (at < want && want <= at + h0) {
        s_pick[0] = EV_BINS - 1 - 2 * tid;
        s_pick[1] = want - at;
        s_pick[2] = h0;
    } else if (at + h0 < want && want <= at + h0 + h1) {
        s_pick[0] = EV_BINS - 2 - 2 * tid;
        s_pick[1] = want - at - h0;
        s_pick[2] = h1;
    }
    __syncthreads();
    bin = s_pick[0];
    want = s_pick[1];
    held = s_pick[2];
}
/* the thread's two bins of a histogram of n (2048 or 1024) */
template <u32 N>
TL_DEV uint2 ev_bins(const u32 *h) {
    if (2 * threadIdx.x < EV_BINS - N) return make_uint2(0, 0);
    const uint2 v = *(const uint2 *)&h[EV_BINS - 2 - 2 * threadIdx.x];
    return make_uint2(v.y, v.x);
}

/* Writes the workgroup's positions j0 .. (the thread has PER of them, keys k):
 * keys above `top` stay, and of those equal to it the first `want` of the
 * session (all of them if `all`); kept / equal: how many the positions before
 * the workgroup's have of them.  The order goes through LDS, so that
 * neighbouring threads write neighbouring words. */
template <u32 PER>
TL_DEV void ev_write(const EvSeq &s, u32 j0, const u32 (&k)[PER], u32 top, u32 want, bool all, u32 kept, u32 equal,
                     u32 *s_w, u16 *s_at) {
    const u32 n = min(s.len - j0, PER * EV_THREADS), p0 = threadIdx.x * PER;
    u32 total;
    if (!all) {
        u32 eq = 0;
#pragma unroll
        for (u32 e = 0; e < PER; e++) eq += p0 + e < n && k[e] == top;
        equal += ev_scan(eq, s_w, total);
        __syncthreads();
    }
    u32 stay = 0;
#pragma unroll
    for (u32 e = 0; e < PER; e++) {
        const bool is = p0 + e < n && k[e] == top;
        stay |= (u32)(p0 + e < n && (k[e] > top || (is && (all || equal < want)))) << e;
        equal += is;
    }
    u32 at = ev_scan((u32)__popc(stay), s_w, total);
#pragma unroll
    for (u32 e = 0; e < PER; e++) {
        const bool is = (stay >> e) & 1;
        if (p0 + e < n) s_at[is ? at : total + (p0 + e - at)] = (u16)(p0 + e);
        at += is;
    }
    __syncthreads();
    /* all the look-ups requested before the first is used */
    u32 j[PER], row[PER];
    float w[PER];
#pragma unroll
    for (u32 e = 0; e < PER; e++) {
        const u32 x = min(threadIdx.x + e * EV_THREADS, n - 1);
        j[e] = j0 + s_at[x];
        row[e] = s.pages ? s.pages[j[e] >> s.shift] : j[e] >> s.shift;
        w[e] = s.w_out ? s.w[j[e]] : 0.f;
    }
#pragma unroll
    for (u32 e = 0; e < PER; e++) {
        const u32 x = threadIdx.x + e * EV_THREADS;
        const u32 r = (row[e] << s.shift) + (j[e] & ((1u << s.shift) - 1));
        if (x >= n) break;
        if (x < total) {
            if (s.kept) s.kept[kept + x] = j[e];
            if (s.rows) s.rows[kept + x] = r;
            if (s.w_out) s.w_out[kept + x] = w[e];
        } else if (s.freed) {
            s.freed[j0 - kept + (x - total)] = r;
        }
    }
}

/* digit d of a key, and whether the digits before it are `pref` */
TL_DEV u32 ev_digit(u32 k, int d) { return d == 0 ? k >> 21 : d == 1 ? (k >> 10) & (EV_BINS - 1) : k & (EV_LOW - 1); }
TL_DEV bool ev_under(u32 k, int d, u32 pref) { return d == 0 || k >> (d == 1 ? 21 : 10) == pref; }
TL_DEV u32 ev_join(u32 pref, int d, u32 bin) { return d == 0 ? bin : (pref << (d == 1 ? 11 : 10)) | bin; }

/* A session of at most 8192 positions: one workgroup, the keys in registers,
 * the keep-th largest by three digits whose histograms lie in LDS.  Bound by
 * the chain of barriers and round trips: 8 sessions of up to 8192 12.7 us. */
__global__ __launch_bounds__(EV_THREADS) void evict_one_kernel(const EvParams p) {
    __shared__ __align__(8) u32 s_hist[EV_BINS];
    __shared__ u32 s_w[EV_WAVES], s_pick[3];
    __shared__ u16 s_at[EV_ONE * EV_THREADS];
    const EvSeq &s = p.seq[blockIdx.x];
    const u32 tid = threadIdx.x, j0 = tid * EV_ONE;
    float w[EV_ONE];
    u32 k[EV_ONE];
#pragma unroll
    for (u32 e = 0; e < EV_ONE; e++) w[e] = s.w[min(j0 + e, s.len - 1)];    /* all requested at once */
    *(uint2 *)&s_hist[2 * tid] = make_uint2(0, 0);
#pragma unroll
    for (u32 e = 0; e < EV_ONE; e++) k[e] = ev_order(s, j0 + e, w[e]);
    __syncthreads();
    u32 want = s.keep, pref = 0, held = 0;
#pragma unroll
    for (int d = 0; d < 3; d++) {
#pragma unroll
        for (u32 e = 0; e < EV_ONE; e++)
            if (j0 + e < s.len && ev_under(k[e], d, pref)) atomicAdd(&s_hist[ev_digit(k[e], d)], 1u);
        __syncthreads();
        const uint2 h = ev_bins<EV_BINS>(s_hist);
        *(uint2 *)&s_hist[EV_BINS - 2 - 2 * tid] = make_uint2(0, 0);
        u32 bin;
        ev_pick(h.x, h.y, want, bin, held, s_w, s_pick);
        pref = ev_join(pref, d, bin);
    }
    ev_write(s, 0, k, pref, want, want == held, 0, 0, s_w, s_at);
}

/* histogram of digit d */
TL_DEV u32 *ev_hist(const EvSeq &s, int d) { return d == 0 ? s.cnt : s.aux + (d == 1 ? 0 : EV_BINS); }

/* The digits before DIGIT: the last one from its histogram, by every workgroup
 * for itself, those before it as the session's first workgroup left them in the
 * launch before. */
template <int DIGIT>
TL_DEV u32 ev_prefix(const EvSeq &s, u32 seg, u32 &want, u32 &held, u32 *s_w, u32 *s_pick) {
    want = s.keep;
    if constexpr (DIGIT == 0) return 0;
    else {
        u32 pref = 0, bin, *left = s.aux + EV_BINS + EV_LOW + 2 * (DIGIT - 1);
        const uint2 h = ev_bins<(DIGIT == 3 ? EV_LOW : EV_BINS)>(ev_hist(s, DIGIT - 1));
        if constexpr (DIGIT > 1) {
            pref = left[-2];
            want = left[-1];
        }
        ev_pick(h.x, h.y, want, bin, held, s_w, s_pick);
        pref = ev_join(pref, DIGIT - 1, bin);
        if (DIGIT < 3 && seg == 0 && threadIdx.x == 0) {
            left[0] = pref;
            left[1] = want;
        }
        return pref;
    }
}

/* Longer sessions: a workgroup per EV_SEG positions, one launch per digit.  A
 * workgroup adds its LDS histogram to the session's (integer atomics); those of
 * the next launch find the digit from it, each for itself (one round trip with
 * their keys'; a last workgroup that did it for all cost three more: 43 us for
 * 131072 positions, so 17; four empty launches are 10).  The last digit's counts
 * are also kept by segment. */
template <int DIGIT>
__global__ __launch_bounds__(EV_THREADS) void evict_digit_kernel(const EvParams p) {
    constexpr u32 NB = DIGIT == 2 ? EV_LOW : EV_BINS;
    __shared__ __align__(8) u32 s_hist[EV_BINS];
    __shared__ u32 s_w[EV_WAVES], s_pick[3];
    const EvSeq &s = p.seq[ck_find(p.wg0, p.n_seq, blockIdx.x)];
    const u32 seg = blockIdx.x - s.wg0, tid = threadIdx.x;
    float w[EV_PER];
    u32 k[EV_PER];
#pragma unroll
    for (u32 e = 0; e < EV_PER; e++) w[e] = s.w[min(seg * EV_SEG + e * EV_THREADS + tid, s.len - 1)];
    *(uint2 *)&s_hist[2 * tid] = make_uint2(0, 0);
    u32 want, held;
    const u32 pref = ev_prefix<DIGIT>(s, seg, want, held, s_w, s_pick);
    /* the next launches' histograms to zero, and the first one for the next call */
    if (DIGIT == 0 && seg == 0)
        for (u32 x = tid; x < EV_BINS + EV_LOW; x += EV_THREADS) s.aux[x] = 0;
    if (DIGIT == 2 && seg == 0) *(uint2 *)&s.cnt[2 * tid] = make_uint2(0, 0);
    __syncthreads();
    u32 above = 0;
#pragma unroll
    for (u32 e = 0; e < EV_PER; e++) {
        const u32 j = seg * EV_SEG + e * EV_THREADS + tid;
        k[e] = ev_order(s, j, w[e]);
        if (j >= s.len) continue;
        if (ev_under(k[e], DIGIT, pref)) atomicAdd(&s_hist[ev_digit(k[e], DIGIT)], 1u);
        above += DIGIT == 2 && k[e] >> 10 > pref;
    }
    __syncthreads();
    u32 *hist = ev_hist(s, DIGIT);
#pragma unroll
    for (u32 e = 0; e < NB / EV_THREADS; e++) {
        const u32 n = s_hist[e * EV_THREADS + tid];
        if (n) __hip_atomic_fetch_add(&hist[e * EV_THREADS + tid], n, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    if constexpr (DIGIT == 2) {
        /* word d: the segment's keys with a digit of d or more, or above pref (1024: these alone) */
        u32 *sw = s.seg + (u64)seg * EV_SEGW;
        u32 total, all;
        ev_scan(above, s_w, total);
        __syncthreads();
        const u32 n = s_hist[NB - 1 - tid];
        const u32 over = total + ev_scan(n, s_w, all);
        sw[NB - 1 - tid] = over + n;
        if (tid == 0) sw[NB] = total;
    }
}

__global__ __launch_bounds__(EV_THREADS) void evict_write_kernel(const EvParams p) {
    __shared__ u32 s_w[EV_WAVES], s_pick[3], s_base[2];
    __shared__ u16 s_at[EV_SEG];
    const EvSeq &s = p.seq[ck_find(p.wg0, p.n_seq, blockIdx.x)];
    const u32 tid = threadIdx.x, seg = blockIdx.x - s.wg0, j0 = seg * EV_SEG, p0 = j0 + tid * EV_PER;
    u32 k[EV_PER];
    float w[EV_PER];
#pragma unroll
    for (u32 e = 0; e < EV_PER; e++) w[e] = s.w[min(p0 + e, s.len - 1)];
#pragma unroll
    for (u32 e = 0; e < EV_PER; e++) k[e] = ev_order(s, p0 + e, w[e]);
    u32 want, held, total;
    const u32 top = ev_prefix<3>(s, seg, want, held, s_w, s_pick);
    /* what the segments before this one hold: a thread each (at most EV_MAX_SEG) */
    const u32 bin = top & (EV_LOW - 1);
    const u32 *sw = s.seg + (u64)tid * EV_SEGW + bin;
    const u32 more = tid < seg ? sw[1] : 0, eq = tid < seg ? sw[0] - more : 0;
    __syncthreads();
    const u32 eq0 = ev_scan(eq, s_w, total);
    if (tid == 0) s_base[0] = total;
    const u32 stay = more + (eq0 < want ? min(eq, want - eq0) : 0);
    __syncthreads();
    ev_scan(stay, s_w, total);
    if (tid == 0) s_base[1] = total;
    __syncthreads();
    ev_write(s, j0, k, top, want, want == held, s_base[1], s_base[0], s_w, s_at);
}

/* Any length without a workspace (captured calls, sessions past EV_MAX_SEG
 * segments): one workgroup per session.  Radix select of the keep-th largest
 * key (four passes of 8 bits, histograms in LDS), then one pass in position
 * order that ranks the kept and the evicted positions: of the keys equal to
 * the threshold the first ones stay. */
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
    if (!seqs || n_seq > CK_MAX_CHUNKS) return tl_fail(TL_EINVAL, "evict: 1..%d sessions", CK_MAX_CHUNKS);
    for (u32 i = 0; i < n_seq; i++) {
        const tl_evict_seq &q = seqs[i];
        if (!q.weight || !q.len || !q.keep || q.keep > q.len || (u64)q.sink + q.recent > q.keep ||
            q.len > 0x7fffffffu)
            return tl_fail(TL_EINVAL, "evict: session %u: len %u keep %u sink %u recent %u", i, q.len,
                           q.keep, q.sink, q.recent);
        if (!q.page_size || (q.page_size & (q.page_size - 1)) || q.page_size > TL_MAX_PAGE)
            return tl_fail(TL_EINVAL, "evict: page size %u is no power of two up to %d", q.page_size, TL_MAX_PAGE);
        if (((uintptr_t)q.weight | (uintptr_t)q.pages | (uintptr_t)q.kept | (uintptr_t)q.rows |
             (uintptr_t)q.freed | (uintptr_t)q.weight_out) & 3)
            return tl_fail(TL_EINVAL, "evict: session %u: alignment", i);
    }
    /* no output over an input or another output, of any session */
    TlSpan few[6 * EV_MAX_SEQ], *spans = n_seq > EV_MAX_SEQ ? (TlSpan *)malloc(6 * sizeof(TlSpan) * (size_t)n_seq) : few;
    if (!spans) return tl_fail(TL_ENOMEM, "evict: %u sessions", n_seq);
    u32 n = 0;
    for (u32 i = 0; i < n_seq; i++) {
        const tl_evict_seq &q = seqs[i];
        auto add = [&](const void *at, u64 words, bool write) {
            if (at && words) spans[n++] = {(u64)(uintptr_t)at, (u64)(uintptr_t)at + 4 * words, write};
        };
        add(q.weight, q.len, false);
        add(q.pages, ((u64)q.len + q.page_size - 1) / q.page_size, false);
        add(q.kept, q.keep, true);
        add(q.rows, q.keep, true);
        add(q.freed, (u64)q.len - q.keep, true);
        add(q.weight_out, q.keep, true);
    }
    const bool clash = tl_spans_clash(spans, n);
    if (spans != few) free(spans);
    if (clash) return tl_fail(TL_EINVAL, "evict: an output overlaps an input or another output");
    const hipStream_t st = (hipStream_t)stream;
    hipStreamCaptureStatus cap = hipStreamCaptureStatusNone;
    u32 n_long = 0, n_shared = 0;
    for (u32 i = 0; i < n_seq; i++) {
        n_long += seqs[i].len > EV_ONE * EV_THREADS;
        n_shared += seqs[i].len > EV_ONE * EV_THREADS && seqs[i].len <= EV_SEG * EV_MAX_SEG;
    }
    if (n_long) HIP_TRY(hipStreamIsCapturing(st, &cap));
    const bool shared = n_shared && cap == hipStreamCaptureStatusNone;
    /* short sessions join the long ones' launches where these have room for them
     * (8 of 1000 to 60000 positions, us: 28.4 with a launch of their own, 18.1 without) */
    const bool together = shared && (n_seq - n_long + n_shared + EV_MAX_SEQ - 1) / EV_MAX_SEQ ==
                                        (n_shared + EV_MAX_SEQ - 1) / EV_MAX_SEQ;
    /* three kinds of sessions: one workgroup's registers, several workgroups, neither */
    for (int kind = 0; kind < 3; kind++) {
        for (u32 i = 0; i < n_seq;) {
            EvParams p;
            memset(&p, 0, sizeof(p));
            u32 wgs = 0;
            for (; i < n_seq && p.n_seq < EV_MAX_SEQ; i++) {
                const tl_evict_seq &q = seqs[i];
                const int mine = q.len <= EV_ONE * EV_THREADS ? together : shared && q.len <= EV_SEG * EV_MAX_SEG ? 1 : 2;
                if (mine != kind) continue;
                EvSeq &s = p.seq[p.n_seq++];
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
                s.wg0 = wgs;
                wgs += kind == 1 ? (q.len + EV_SEG - 1) / EV_SEG : 1;
            }
            if (!p.n_seq) break;
            for (u32 j = 0; j < CK_MAX_SEQ; j++) p.wg0[j] = j < p.n_seq ? p.seq[j].wg0 : ~0u;
            if (kind == 0) {
                hipLaunchKernelGGL(evict_one_kernel, dim3(wgs), dim3(EV_THREADS), 0, st, p);
            } else if (kind == 2) {
                hipLaunchKernelGGL(evict_kernel, dim3(wgs), dim3(EV_THREADS), 0, st, p);
            } else {
                TlWorkspace *w;
                const int rc = tl_workspace_get(st, (size_t)wgs * EV_SEGW + p.n_seq * EV_AUX, 0, TL_MERGE_CNT_WORDS, &w);
                if (rc) return rc;
                for (u32 j = 0; j < p.n_seq; j++) {
                    p.seq[j].cnt = w->cnt + (size_t)j * EV_BINS;
                    p.seq[j].aux = (u32 *)w->acc + (size_t)wgs * EV_SEGW + j * EV_AUX;
                    p.seq[j].seg = (u32 *)w->acc + (size_t)p.seq[j].wg0 * EV_SEGW;
                }
                hipLaunchKernelGGL(evict_digit_kernel<0>, dim3(wgs), dim3(EV_THREADS), 0, st, p);
                hipLaunchKernelGGL(evict_digit_kernel<1>, dim3(wgs), dim3(EV_THREADS), 0, st, p);
                hipLaunchKernelGGL(evict_digit_kernel<2>, dim3(wgs), dim3(EV_THREADS), 0, st, p);
                hipLaunchKernelGGL(evict_write_kernel, dim3(wgs), dim3(EV_THREADS), 0, st, p);
            }
            HIP_TRY(hipGetLastError());
        }
    }
    return TL_OK;
}
