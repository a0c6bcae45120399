/*
 * tl_chunk.hip — batches of chunks over a paged cache: checks of arguments,
 * the norm + rotation + append of new rows, and the entry points and plans of
 * the attention (tl_chunk_attn_kernels.h) and of the attention weight
 * (tl_chunk_weight_kernels.h).
 */
#include "tl_chunk.h"
#include "tl_chunk_launch.h"

#include <math.h>
#include <stdlib.h>
#include <string.h>

/* ------------------------------------------------------------------------ */
/* checks                                                                    */
/* ------------------------------------------------------------------------ */

bool tl_ranges_overlap(const void *a, u64 a_bytes, const void *b, u64 b_bytes) {
    const uintptr_t x = (uintptr_t)a, y = (uintptr_t)b;
    return a && b && a_bytes && b_bytes && x < y + b_bytes && y < x + a_bytes;
}

static int by_start(const void *a, const void *b) {
    const u64 x = ((const TlSpan *)a)->at, y = ((const TlSpan *)b)->at;
    return x < y ? -1 : x > y;
}

bool tl_spans_clash(TlSpan *a, u32 n) {
    bool rising = true;
    for (u32 i = 1; i < n && rising; i++) rising = a[i - 1].at <= a[i].at;
    if (!rising) qsort(a, n, sizeof(*a), by_start);
    u64 end = 0, written = 0;      /* of the intervals so far */
    for (u32 i = 0; i < n; i++) {
        if (a[i].at == a[i].end) continue;
        if (a[i].at < (a[i].write ? end : written)) return true;
        if (a[i].end > end) end = a[i].end;
        if (a[i].write && a[i].end > written) written = a[i].end;
    }
    return false;
}

/* do the intervals [at(i), at(i) + len(i)) of chunks with len > 0 overlap? */
template <class At, class Len>
static bool any_overlap(u32 n, At at, Len len) {
    TlSpan a[CK_MAX_CHUNKS];
    u32 m = 0;
    for (u32 i = 0; i < n; i++)
        if (len(i)) a[m++] = {at(i), at(i) + len(i), true};
    return tl_spans_clash(a, m);
}

int tl_chunk_check(const LayerView &L, const tl_chunk *ch, u32 n_chunk, u32 rows, u32 page_size,
                   u32 *shift) {
    if (n_chunk > CK_MAX_CHUNKS || (n_chunk && !ch))
        return tl_fail(TL_EINVAL, "chunks: 0..%d chunks", CK_MAX_CHUNKS);
    if (!page_size || (page_size & (page_size - 1)) || page_size > TL_MAX_PAGE)
        return tl_fail(TL_EINVAL, "chunks: page size %u is no power of two up to %d", page_size, TL_MAX_PAGE);
    *shift = (u32)__builtin_ctz(page_size);
    if (L.ring) return tl_fail(TL_EINVAL, "chunks: ring layers have no pages");
    u32 live = 0, bare = 0;
    for (u32 i = 0; i < n_chunk; i++) {
        if (!ch[i].n) continue;
        live++;
        if ((u64)ch[i].row + ch[i].n > rows)
            return tl_fail(TL_ERANGE, "chunks: rows %u + %u of chunk %u exceed %u", ch[i].row, ch[i].n, i, rows);
        if ((u64)ch[i].pos + ch[i].n > 0x7fffffffull ||
            (u64)ch[i].pos + ch[i].n + ch[i].rope_skip > 0xffffffffull)
            return tl_fail(TL_ERANGE, "chunks: positions of chunk %u", i);
        if ((uintptr_t)ch[i].pages & 3) return tl_fail(TL_EINVAL, "chunks: page table of chunk %u not aligned", i);
        if (!ch[i].pages) {
            bare++;
            if ((u64)ch[i].pos + ch[i].n > L.cap)
                return tl_fail(TL_ERANGE, "chunks: pos %u + n %u exceeds cap %u", ch[i].pos, ch[i].n, L.cap);
        }
    }
    if (bare && live > 1) return tl_fail(TL_EINVAL, "chunks: more than one chunk needs page tables");
    if (any_overlap(n_chunk, [&](u32 i) { return (u64)ch[i].row; }, [&](u32 i) { return (u64)ch[i].n; }))
        return tl_fail(TL_EINVAL, "chunks: two chunks share batch rows");
    return TL_OK;
}

/* the starts of the launch's chunks side by side */
template <class P>
static void starts(P &p) {
    for (u32 i = 0; i < CK_MAX_SEQ; i++) p.wg0[i] = i < p.n_seq ? p.seq[i].wg0 : ~0u;
}

static CkCache cache_of(const LayerView &L, u32 shift) {
    CkCache c;
    c.k = (const u16 *)L.k;
    c.v = (const u16 *)L.v;
    c.ks = L.ks;
    c.vs = L.vs;
    c.cap = L.cap;
    c.n_kv = L.n_kv_head;
    c.shift = shift;
    return c;
}

static void seq_of(CkSeq &s, const tl_chunk &c) {
    memset(&s, 0, sizeof(s));
    s.pages = c.pages;
    s.weight = c.weight;
    s.pos = c.pos;
    s.n = c.n;
    s.row = c.row;
    s.prefix = c.prefix;
    s.rope_skip = c.rope_skip;
}

/* rows x stride floats starting at p, of which each row holds `width` */
static u64 span(u32 rows, u32 stride, u32 width) {
    return rows ? ((u64)(rows - 1) * stride + width) * sizeof(float) : 0;
}

/* Do the rows of two buffers share floats?  Buffers of one stride may lie side
 * by side in each row (q, k and v of one projection). */
static bool rows_overlap(u32 rows, const float *a, u32 a_stride, u32 a_width, const float *b, u32 b_stride,
                         u32 b_width) {
    if (!tl_ranges_overlap(a, span(rows, a_stride, a_width), b, span(rows, b_stride, b_width))) return false;
    if (a_stride != b_stride) return true;
    const long long d = b - a, s = a_stride;
    const u64 at = (u64)((d % s + s) % s);      /* column of b in a's rows */
    return at < a_width || at + b_width > a_stride;
}

static int check_rows(const char *what, const void *p, u32 stride, u64 width) {
    if (!p) return tl_fail(TL_EINVAL, "chunks: null %s", what);
    if (stride < width || (stride & 3) || ((uintptr_t)p & 15))
        return tl_fail(TL_EINVAL, "chunks: %s rows must be 16-byte aligned, of at least %llu floats", what,
                       (unsigned long long)width);
    return TL_OK;
}

/* ------------------------------------------------------------------------ */
/* norm + rotation + append                                                  */
/* ------------------------------------------------------------------------ */

struct CkAppendParams {
    u32 wg0[CK_MAX_SEQ];
    CkSeq seq[CK_MAX_SEQ];
    CkCache c;
    const float *q, *k, *v, *qw, *kw;
    float *q_out;
    float eps;
    u32 n_seq, n_head, q_stride, kv_stride, q_out_stride;
    u32 rdim;
    int neox;
    double step;             /* log2(theta) * 2 / rdim */
};

/* One workgroup per batch row and share of its heads (grid.y): the row's
 * rotation table goes to LDS once, then every group of D / 8 lanes takes head
 * rows of q, k and v in turn, eight elements to a lane: sum of squares over
 * the group by DPP, norm, rotation with the partner's elements (in the lane
 * for adjacent pairs, from memory again for half pairs), store.  Bound by the
 * traffic, f32 in and f32 q, f16 K and V out: 2100 rows at 32/8/128 23.3 us, 4.2
 * TB/s of 5.1 that a copy reaches; 16 rows at 8/4/256 5.2 us (a launch and one
 * round trip).  One row to a workgroup keeps the rotation table to one row and a
 * row's requests together; few rows share their heads out, up to 1024 workgroups. */
template <int D, bool Q8>
__global__ __launch_bounds__(256) void chunk_append_kernel(const CkAppendParams p) {
    constexpr u32 LPR = D / 8, GRP = 256 / LPR;
    __shared__ float2 s_cs[D / 2];
    const CkSeq &sq = p.seq[ck_find(p.wg0, p.n_seq, blockIdx.x)];
    const u32 r = blockIdx.x - sq.wg0;
    const u32 key = sq.pos + r;
    const u64 brow = (u64)sq.row + r;
    const u32 e0 = (threadIdx.x % LPR) * 8;
    const u32 units = p.n_head + 2 * p.c.n_kv;
    auto row_of = [&](u32 u) -> const float * {
        const u32 kv = p.n_head + p.c.n_kv;
        return u < p.n_head ? p.q + brow * p.q_stride + (u64)u * D
             : u < kv ? p.k + brow * p.kv_stride + (u64)(u - p.n_head) * D
                      : p.v + brow * p.kv_stride + (u64)(u - kv) * D;
    };
    const u32 u0 = blockIdx.y * GRP + threadIdx.x / LPR;
    /* the first head row is on its way while the table is made */
    const float *src = row_of(min(u0, units - 1));
    float4 a = *(const float4 *)(src + e0), b = *(const float4 *)(src + e0 + 4);
    const u32 prow = ck_row(p.c, sq.pages, key);
    if (threadIdx.x < p.rdim / 2) {
        /* turns in 64 bits: the fraction is good at any position */
        const double turns = (double)(key + sq.rope_skip) * (exp2(-p.step * (double)threadIdx.x) * 0.15915494309189535);
        float s, c;
        sincospif(2.f * (float)(turns - rint(turns)), &s, &c);
        s_cs[threadIdx.x] = make_float2(c, s);
    }
    __syncthreads();
    const u32 half = p.rdim >> 1;
    for (u32 u = u0; u < units; u += gridDim.y * GRP) {
        const bool is_q = u < p.n_head, is_v = u >= p.n_head + p.c.n_kv;
        const u32 h = is_q ? u : is_v ? u - p.n_head - p.c.n_kv : u - p.n_head;
        if (u != u0) {
            src = row_of(u);
            a = *(const float4 *)(src + e0);
            b = *(const float4 *)(src + e0 + 4);
        }
        float x[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
        float ss = 0.f;
#pragma unroll
        for (int j = 0; j < 8; j++) ss = fmaf(x[j], x[j], ss);
        ss = group_sum<LPR>(ss);
        if (!is_v) {
            const float inv = 1.f / sqrtf(ss * (1.f / D) + p.eps);
            const float *w = is_q ? p.qw : p.kw;
            float g[8] = {1.f, 1.f, 1.f, 1.f, 1.f, 1.f, 1.f, 1.f};
            if (w) {
                const float4 c = *(const float4 *)(w + e0), d = *(const float4 *)(w + e0 + 4);
                g[0] = c.x; g[1] = c.y; g[2] = c.z; g[3] = c.w;
                g[4] = d.x; g[5] = d.y; g[6] = d.z; g[7] = d.w;
            }
            float y[8];
#pragma unroll
            for (int j = 0; j < 8; j++) y[j] = x[j] * inv * g[j];
            if (p.rdim && !p.neox) {
#pragma unroll
                for (int j = 0; j < 8; j += 2)
                    if (e0 + j < p.rdim) {
                        const float2 cs = s_cs[(e0 + j) >> 1];
                        rope_rot(y[j], y[j + 1], cs.x, cs.y, x[j], x[j + 1]);
                    } else {
                        x[j] = y[j];
                        x[j + 1] = y[j + 1];
                    }
            } else if (p.rdim) {
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const u32 e = e0 + j;
                    if (e >= p.rdim) {
                        x[j] = y[j];
                        continue;
                    }
                    const bool low = e < half;
                    const u32 pe = low ? e + half : e - half;
                    const float o = src[pe] * inv * (w ? w[pe] : 1.f);
                    const float2 cs = s_cs[low ? e : pe];
                    float nx, ny;
                    rope_rot(low ? y[j] : o, low ? o : y[j], cs.x, cs.y, nx, ny);
                    x[j] = low ? nx : ny;
                }
            } else {
#pragma unroll
                for (int j = 0; j < 8; j++) x[j] = y[j];
            }
        }
        if (is_q) {
            float *d = p.q_out + brow * p.q_out_stride + (u64)h * D + e0;
            *(float4 *)d = make_float4(x[0], x[1], x[2], x[3]);
            *(float4 *)(d + 4) = make_float4(x[4], x[5], x[6], x[7]);
        } else if constexpr (Q8) {
            const float m = group_max<4>(amax8(x));
            const float d = m / 127.f, id = d > 0.f ? 1.f / d : 0.f;
            if (prow < p.c.cap) {
                const u64 at = (u64)h * p.c.cap + prow;
                char *dst = (char *)(is_v ? p.c.v : p.c.k) + at * D + e0;
                *(uint2 *)dst = q8_pack8(x, id);
                if ((e0 & 31) == 0)
                    ((u16 *)(is_v ? p.c.vs : p.c.ks))[at * (D / 32) + (e0 >> 5)] = (u16)f32_to_f16_bits(d);
            }
        } else if (prow < p.c.cap) {
            u16 *dst = (u16 *)(is_v ? p.c.v : p.c.k) + ((u64)h * p.c.cap + prow) * D + e0;
            *(uint4 *)dst = cvt8_f16_regs(make_float4(x[0], x[1], x[2], x[3]), make_float4(x[4], x[5], x[6], x[7]));
        }
    }
}

template <bool Q8>
static void launch_append(u32 head_dim, dim3 grid, hipStream_t st, const CkAppendParams &p) {
    if (head_dim == 64) hipLaunchKernelGGL((chunk_append_kernel<64, Q8>), grid, dim3(256), 0, st, p);
    else if (head_dim == 128) hipLaunchKernelGGL((chunk_append_kernel<128, Q8>), grid, dim3(256), 0, st, p);
    else hipLaunchKernelGGL((chunk_append_kernel<256, Q8>), grid, dim3(256), 0, st, p);
}

static int norm_append(const LayerView &L, const tl_qk_norm_args *a, const tl_chunk *ch, u32 n_chunk,
                       hipStream_t st) {
    if (!a) return tl_fail(TL_EINVAL, "qk_norm: null arguments");
    if (!a->n_head || a->n_head % L.n_kv_head)
        return tl_fail(TL_EINVAL, "qk_norm: n_head %u not a multiple of n_kv %u", a->n_head, L.n_kv_head);
    const u64 qw = (u64)a->n_head * L.head_dim, kw = (u64)L.n_kv_head * L.head_dim;
    u32 shift;
    int rc = tl_chunk_check(L, ch, n_chunk, a->rows, a->page_size, &shift);
    if (!rc) rc = check_rows("q", a->q, a->q_stride, qw);
    if (!rc) rc = check_rows("q_out", a->q_out, a->q_out_stride, qw);
    if (!rc) rc = check_rows("k", a->k, a->kv_stride, kw);
    if (!rc) rc = check_rows("v", a->v, a->kv_stride, kw);
    if (rc) return rc;
    if (((uintptr_t)a->q_weight | (uintptr_t)a->k_weight) & 15)
        return tl_fail(TL_EINVAL, "qk_norm: weights not 16-byte aligned");
    if (!(a->eps >= 0.f) || !isfinite(a->eps)) return tl_fail(TL_EINVAL, "qk_norm: eps %g", (double)a->eps);
    const bool place = a->q_out == a->q && a->q_out_stride == a->q_stride;
    if ((!place && rows_overlap(a->rows, a->q, a->q_stride, (u32)qw, a->q_out, a->q_out_stride, (u32)qw)) ||
        rows_overlap(a->rows, a->k, a->kv_stride, (u32)kw, a->q_out, a->q_out_stride, (u32)qw) ||
        rows_overlap(a->rows, a->v, a->kv_stride, (u32)kw, a->q_out, a->q_out_stride, (u32)qw))
        return tl_fail(TL_EINVAL, "qk_norm: q_out overlaps q, k or v");
    RopeCfg rope;
    rope.rdim = 0;
    if (a->rope.rope_dim) {
        rc = tl_rope_cfg(L.head_dim, &a->rope, rope);
        if (rc) return rc;
        if (!isfinite(a->rope.theta)) return tl_fail(TL_EINVAL, "rope: theta");
    }
    CkAppendParams p;
    memset(&p, 0, sizeof(p));
    p.c = cache_of(L, shift);
    p.q = a->q;
    p.k = a->k;
    p.v = a->v;
    p.qw = a->q_weight;
    p.kw = a->k_weight;
    p.q_out = a->q_out;
    p.eps = a->eps;
    p.n_head = a->n_head;
    p.q_stride = a->q_stride;
    p.kv_stride = a->kv_stride;
    p.q_out_stride = a->q_out_stride;
    p.rdim = rope.rdim;
    p.neox = rope.rdim ? rope.neox : 0;
    p.step = rope.rdim ? log2((double)rope.theta) * 2.0 / rope.rdim : 0.0;
    for (u32 i = 0; i < n_chunk;) {
        u32 m = 0;
        u64 wgs = 0;
        for (; i < n_chunk && m < CK_MAX_SEQ; i++) {
            if (!ch[i].n) continue;
            if (wgs + ch[i].n > 0x7fffffffull) break;
            seq_of(p.seq[m], ch[i]);
            p.seq[m++].wg0 = (u32)wgs;
            wgs += ch[i].n;
        }
        if (!m) break;
        p.n_seq = m;
        starts(p);
        /* few rows: their heads over several workgroups */
        const u32 units = a->n_head + 2 * L.n_kv_head, per = 256 / (L.head_dim / 8);
        u32 split = (units + per - 1) / per;
        while (split > 1 && wgs * split > 1024) split--;
        if (L.q8) launch_append<true>(L.head_dim, dim3((u32)wgs, split), st, p);
        else launch_append<false>(L.head_dim, dim3((u32)wgs, split), st, p);
        HIP_TRY(hipGetLastError());
    }
    return TL_OK;
}

extern "C" int tl_qk_norm_append(const tl_kv_layer *L, const tl_qk_norm_args *a, const tl_chunk *chunks,
                                 uint32_t n_chunk, void *stream) {
    const int rc = tl_check_layer(L);
    return rc ? rc : norm_append(tl_view(L), a, chunks, n_chunk, (hipStream_t)stream);
}

extern "C" int tl_qk_norm_append_q8(const tl_kv_layer_q8 *L, const tl_qk_norm_args *a,
                                    const tl_chunk *chunks, uint32_t n_chunk, void *stream) {
    const int rc = tl_check_layer_q8(L);
    return rc ? rc : norm_append(tl_view_q8(L), a, chunks, n_chunk, (hipStream_t)stream);
}

/* ------------------------------------------------------------------------ */
/* attention                                                                 */
/* ------------------------------------------------------------------------ */

/* keys that a launch may have to go through for rows [r0, r1) of a chunk (the
 * documents' starts are known on the device only) */
static u64 span_tiles(const tl_chunk &c, u32 window, u32 r0, u32 r1) {
    const u64 end = (u64)c.pos + c.n;
    const u64 pre = c.prefix < end ? c.prefix : end;
    const u64 hi = (u64)c.pos + r1;
    u64 lo = window && (u64)c.pos + r0 + 1 > window ? (u64)c.pos + r0 + 1 - window : 0;
    if (lo < pre) lo = pre;
    return (pre + CK_KEYS - 1) / CK_KEYS + (hi > lo ? (hi + CK_KEYS - 1) / CK_KEYS - lo / CK_KEYS : 0);
}

/* One launch of the narrow kernel and one of the wide, and their workspace. */
struct AttnPlan {
    CkSeq seq[2][CK_MAX_SEQ];   /* [0]: narrow, [1]: wide */
    u32 n[2], wgs[2];
    u64 parts;                  /* partial rows */
    u32 groups;                 /* their counters (narrow) */
};

/* Chunks of more columns than this take the wide kernel, unless the whole batch
 * is cheaper on the narrow one.  Its cost (us) is a round of up to 256 groups at a
 * time plus a time per 1000 tiles of 32 keys x 16 columns; the wide kernel's a
 * start (with the join of its splits) plus a time per 1000 tiles of 32 keys x 128
 * columns.  Fitted to both sides of 120 shapes; us narrow / wide at 32/8/128: 9
 * rows at 6000 keys 17 / 34, 60 rows 36 / 38, 200 rows 117 / 62; 128 rows at 500
 * keys 13 / 24; a first prompt of 300 rows 24 / 22; 8 sessions of 100 rows at 1000
 * keys 103 / 54; 6 of 1 to 200 rows at 64 to 6000 keys 35 / 25. */
#define CK_WIDE_MIN 32
struct AttnCost {
    float base, round, tile;     /* narrow */
    float start, wtile;          /* wide */
};
static const AttnCost g_attn_cost[3][2] = {
    /* f16, Q8_0 */
    {{2.f, 4.f, 0.78f, 17.f, 2.8f}, {2.f, 4.f, 0.87f, 19.f, 3.4f}},       /* head_dim 64 */
    {{3.f, 5.5f, 1.2f, 23.f, 3.6f}, {3.f, 5.5f, 1.5f, 24.f, 5.4f}},       /* 128 */
    {{10.f, 5.f, 3.2f, 22.f, 9.f}, {10.f, 5.f, 3.9f, 25.f, 11.f}},        /* 256 */
};

/* all of the batch on the narrow kernel? */
static bool all_narrow(const tl_chunk *const *ch, u32 n, u32 n_kv, u32 gqa, u32 head_dim, bool q8, u32 window) {
    const AttnCost &c = g_attn_cost[head_dim == 64 ? 0 : head_dim == 128 ? 1 : 2][q8];
    double groups = 0, small = 0, big = 0, wide = 0, most = 0;
    for (u32 i = 0; i < n; i++) {
        const u64 cols = (u64)ch[i]->n * gqa;
        const u32 step = (CK_COLS + gqa - 1) / gqa, rows = ch[i]->n;
        /* keys of the first and the last column block, on average */
        const double keys = 0.5e-3 * n_kv * (double)(span_tiles(*ch[i], window, 0, step < rows ? step : rows) +
                                                     span_tiles(*ch[i], window, rows > step ? rows - step : 0, rows));
        const double last = 1e-3 * (double)span_tiles(*ch[i], window, 0, rows);
        groups += (double)n_kv * ((cols + CK_COLS - 1) / CK_COLS);
        most = last > most ? last : most;
        (cols > CK_WIDE_MIN ? big : small) += keys * ((cols + CK_COLS - 1) / CK_COLS);
        if (cols > CK_WIDE_MIN) wide += keys * ((cols + CK_WCOLS - 1) / CK_WCOLS);
    }
    if (big == 0) return true;
    /* more than a round of groups of unequal lengths: the last one to start is late */
    const double late = groups > 256 ? 128 * most : 0;
    return c.base + c.round * ceil(groups / 256) + c.tile * (small + big + late) <=
           c.start + c.wtile * wide + 0.6 * c.tile * small;
}

/* As many splits as fill the chip (narrow: one workgroup to a CU, wide: two, at
 * head_dim 256 one), none of fewer tiles than a narrow workgroup has waves, or of
 * fewer keys than 128 (wide).  In one launch of both, up to head_dim 128, the
 * narrow ones are of half the size; a wide tile takes three times as long as one of
 * theirs, so the 512 places are shared out by that, and the wide ones have 192 keys
 * at least.  us, all places for the wide ones / shared: 24 sessions of 1 to 150
 * rows at up to 6000 keys, 32/8/128, 70.9 / 44.4; 12 of up to 30 at 8000 49.9 / 40.7;
 * 6 of up to 200 26.4 / 25.4; the worst of 30, 20 of up to 400 rows, 48.7 / 52.3. */
static bool plan_attn(AttnPlan &pl, const tl_chunk *const *ch, u32 n, u32 n_kv, u32 gqa, u32 head_dim, bool q8,
                      u32 window) {
    pl.n[0] = pl.n[1] = pl.wgs[0] = pl.wgs[1] = pl.groups = 0;
    pl.parts = 0;
    u64 tiles[2][CK_MAX_SEQ], total[2] = {0, 0};
    const u64 wide_min = all_narrow(ch, n, n_kv, gqa, head_dim, q8, window) ? ~0ull : CK_WIDE_MIN;
    u32 n_wide = 0;
    for (u32 i = 0; i < n; i++) n_wide += (u64)ch[i]->n * gqa > wide_min;
    for (u32 i = 0; i < n; i++) {
        const u64 cols = (u64)ch[i]->n * gqa;
        const int w = cols > wide_min;
        const u32 per = w ? CK_WCOLS : CK_COLS;
        const u32 ncb = (u32)((cols + per - 1) / per);
        /* bands of a wide chunk, each with splits by its own keys: its last rows see
         * more than its first */
        const u32 room = w ? 1 + (CK_MAX_SEQ - n) / n_wide : 1;
        const u32 bands = room < ncb ? (room < 8 ? room : 8) : (ncb < 8 ? ncb : 8);
        for (u32 b = 0; b < (w ? bands : 1); b++) {
            CkSeq &s = pl.seq[w][pl.n[w]];
            seq_of(s, *ch[i]);
            const u32 b0 = w ? (u32)((u64)ncb * b / bands) : 0, b1 = w ? (u32)((u64)ncb * (b + 1) / bands) : ncb;
            const u64 r1 = ((u64)b1 * per + gqa - 1) / gqa;
            s.cb0 = b0;
            s.ncb = b1 - b0;
            tiles[w][pl.n[w]] = span_tiles(*ch[i], window, (u32)((u64)b0 * per / gqa), r1 < ch[i]->n ? (u32)r1 : ch[i]->n);
            total[w] += tiles[w][pl.n[w]++] * s.ncb * n_kv;
        }
    }
    const bool both = pl.n[0] && pl.n[1] && head_dim != 256;
    for (int w = 1; w >= 0; w--) {
        u32 fill = w && head_dim != 256 ? 512 : 256;
        if (both && w) {
            fill = (u32)(512.0 * 3 * total[1] / (3.0 * total[1] + total[0]));
            if (fill < 64) fill = 64;
        }
        if (both && !w) fill = pl.wgs[1] < 384 ? 512 - pl.wgs[1] : 128;
        u64 per = (total[w] + fill - 1) / fill, wgs = 0;
        const u64 least = both ? (w ? 6 : 4) : !w && head_dim != 256 ? 8 : 4;
        if (per < least) per = least;
        /* the smallest share whose workgroups all run at once, if there is one */
        u64 all = 0, most = 0;
        for (u32 i = 0; i < pl.n[w]; i++) {
            all += (u64)pl.seq[w][i].ncb * n_kv;
            most = tiles[w][i] > most ? tiles[w][i] : most;
        }
        for (; all <= fill && per < most; per += 1 + per / 32) {
            u64 at_once = 0;
            for (u32 i = 0; i < pl.n[w]; i++)
                at_once += (u64)pl.seq[w][i].ncb * n_kv * ((tiles[w][i] + per - 1) / per);
            if (at_once <= fill) break;
        }
        for (u32 i = 0; i < pl.n[w]; i++) {
            CkSeq &s = pl.seq[w][i];
            u64 ns = (tiles[w][i] + per - 1) / per;
            /* two tiles to a wave cost less than a join at head_dim 64: 4 sessions of 5 rows at
             * 300 keys 7.8 us / 9.4; at 128 one of 500 keys 11.1 / 10.1 */
            if (!w && !both && head_dim == 64 && tiles[w][i] <= 2 * CK_WAVES(64)) ns = 1;
            const u64 groups = (u64)s.ncb * n_kv;
            const u64 cols = (u64)s.n * gqa;
            const u32 counters = ck_join_counters((u32)ns, cols < CK_COLS ? (u32)cols : CK_COLS, head_dim,
                                            both ? 4 : CK_WAVES(head_dim));
            if (ns < 1 || (!w && pl.groups + groups * counters > CK_MAX_GROUPS)) ns = 1;
            s.ns = (u32)ns;
            s.counters = counters;
            s.wg0 = (u32)wgs;
            s.part0 = (u32)pl.parts;
            s.grp0 = pl.groups;
            wgs += groups * ns;
            if (ns > 1) {
                pl.parts += groups * ns * (w ? CK_WCOLS : CK_COLS);
                if (!w) pl.groups += (u32)(groups * counters);
            }
        }
        if (wgs > 0x7fffffffull || pl.parts > 0xffffffffull) return false;
        pl.wgs[w] = (u32)wgs;
    }
    return true;
}

#define CK_WS_HEAD ((u64)CK_CNT_WORDS * sizeof(u32))
static u64 ws_need(u64 parts, u32 head_dim) {
    return CK_WS_HEAD + parts * (sizeof(float2) + (u64)head_dim * sizeof(float));
}

static int check_attn(const LayerView &L, const tl_chunk_attn_args *a, const tl_chunk *ch, u32 n_chunk,
                      bool weight, u32 *shift) {
    if (!a) return tl_fail(TL_EINVAL, "attn_chunks: null arguments");
    if (!a->n_head || a->n_head % L.n_kv_head)
        return tl_fail(TL_EINVAL, "attn_chunks: n_head %u not a multiple of n_kv %u", a->n_head, L.n_kv_head);
    const u64 width = (u64)a->n_head * L.head_dim;
    int rc = tl_chunk_check(L, ch, n_chunk, a->rows, a->page_size, shift);
    if (!rc) rc = check_rows("q", a->q, a->q_stride, width);
    if (!rc && !weight) rc = check_rows("dst", a->dst, a->q_stride, width);
    if (rc) return rc;
    if (((uintptr_t)a->lse | (uintptr_t)a->first | (uintptr_t)a->slopes) & 3)
        return tl_fail(TL_EINVAL, "attn_chunks: lse, first or slopes not aligned");
    if (!(a->scale > 0.f) || !isfinite(a->scale) || !(a->softcap == 0.f || a->softcap >= 1e-6f) ||
        !isfinite(a->softcap))
        return tl_fail(TL_EINVAL, "attn_chunks: scale %g softcap %g", (double)a->scale, (double)a->softcap);
    const u64 gqa = a->n_head / L.n_kv_head;
    for (u32 i = 0; i < n_chunk; i++)
        if (ch[i].n * gqa + CK_WCOLS > 0xffffffffull / gqa)
            return tl_fail(TL_ERANGE, "attn_chunks: %u rows of gqa %llu in a chunk", ch[i].n, (unsigned long long)gqa);
    if ((uintptr_t)a->ws & 15) return tl_fail(TL_EINVAL, "attn_chunks: workspace not 16-byte aligned");
    return TL_OK;
}

/* the call's chunks with rows, at most CK_MAX_SEQ of them from *at on */
static u32 next_chunks(const tl_chunk *ch, u32 n_chunk, u32 *at, const tl_chunk **of) {
    u32 m = 0;
    for (; *at < n_chunk && m < CK_MAX_SEQ; (*at)++)
        if (ch[*at].n) of[m++] = &ch[*at];
    return m;
}

/* most partial rows that the attention's launches of one group of chunks take */
static bool most_parts(u32 n_kv, u32 gqa, u32 head_dim, bool q8, u32 window, const tl_chunk *ch, u32 n_chunk,
                       u64 *parts) {
    AttnPlan pl;
    const tl_chunk *of[CK_MAX_SEQ];
    *parts = 0;
    for (u32 i = 0; i < n_chunk;) {
        const u32 m = next_chunks(ch, n_chunk, &i, of);
        if (!m) break;
        if (!plan_attn(pl, of, m, n_kv, gqa, head_dim, q8, window)) return false;
        *parts = pl.parts > *parts ? pl.parts : *parts;
    }
    return true;
}

/* The attention weight's launches of one group of chunks: [0] few columns, [1]
 * many, whose sums take `floats` of workspace. */
struct WeightPlan {
    CkSeq seq[2][CK_MAX_SEQ];
    u32 n[2], wgs[2], blocks;
    u64 floats;
};

/* More columns than this keep keys of one head to a workgroup; fewer go
 * through all heads of a run of keys, where reading K is the work. */
#define CK_WEIGHT_WIDE_MIN CK_COLS

static bool plan_weight(WeightPlan &pl, const tl_chunk *const *ch, u32 n, u32 n_kv, u32 gqa, u32 head_dim,
                        bool q8, u32 window) {
    pl.n[0] = pl.n[1] = pl.wgs[0] = pl.wgs[1] = pl.blocks = 0;
    pl.floats = 0;
    const u32 wkeys = (u32)ck_weight_keys((int)head_dim, q8);
    u64 wgs[2] = {0, 0}, blocks = 0, shares = 0, tiles = 0;
    for (u32 i = 0; i < n; i++) {
        const u64 cols = (u64)ch[i]->n * gqa, end = (u64)ch[i]->pos + ch[i]->n;
        const int w = cols > CK_WEIGHT_WIDE_MIN;
        CkSeq &s = pl.seq[w][pl.n[w]++];
        seq_of(s, *ch[i]);
        /* first key that a window leaves (documents' starts are known on the device only) */
        u64 lo = window && (u64)ch[i]->pos + 1 > window && !ch[i]->prefix ? (u64)ch[i]->pos + 1 - window : 0;
        if (!w) {
            s.part0 = (u32)(lo / CK_KEYS * CK_KEYS);
            tiles += (end - s.part0 + CK_KEYS - 1) / CK_KEYS;
        } else {
            s.part0 = (u32)(lo / wkeys * wkeys);
            s.ncb = (u32)((end - s.part0 + wkeys - 1) / wkeys);
            blocks += s.ncb;
            shares += (u64)s.ncb * ((cols + 127) / 128);
        }
    }
    /* few columns: the smallest run of tiles whose workgroups all run at once */
    u64 run = (tiles + 255) / 256;
    for (; pl.n[0]; run += 1 + run / 32) {
        u64 at_once = 0;
        for (u32 i = 0; i < pl.n[0]; i++) {
            const CkSeq &s = pl.seq[0][i];
            at_once += ((u64)s.pos + s.n - s.part0 + run * CK_KEYS - 1) / (run * CK_KEYS);
        }
        if (at_once <= 256 || run >= tiles) break;
    }
    for (u32 i = 0; i < pl.n[0]; i++) {
        CkSeq &s = pl.seq[0][i];
        s.ncb = (u32)run;
        s.wg0 = (u32)wgs[0];
        wgs[0] += ((u64)s.pos + s.n - s.part0 + run * CK_KEYS - 1) / (run * CK_KEYS);
    }
    /* Shares of the columns, in units of 128: those for which rounds of
     * workgroups x (the largest share + what a workgroup costs by itself) is least.
     * 512 rows over 4608 keys, 32/8/128 Q8_0, us: one share (144 workgroups) 102,
     * three (432, two rounds) 82; f16, three (216) 61, six (432, two rounds) 67. */
    const u32 fill = head_dim == 64 && !q8 ? 512 : 256;
    u64 per = 1;
    double least = 0;
    for (u64 x = 1 + shares * n_kv / (4 * fill); pl.n[1]; x += 1 + x / 32) {
        u64 at_once = 0;
        double most = 0;
        bool one = true;
        for (u32 i = 0; i < pl.n[1]; i++) {
            const u64 parts = ((u64)pl.seq[1][i].n * gqa + 127) / 128, k = (parts + x - 1) / x;
            at_once += (u64)pl.seq[1][i].ncb * n_kv * k;
            most = (double)parts / k > most ? (double)parts / k : most;
            one = one && k == 1;
        }
        const double cost = (double)((at_once + fill - 1) / fill) * (most + 0.55);
        if (!least || cost < least) {
            least = cost;
            per = x;
        }
        if (one) break;
    }
    for (u32 i = 0; i < pl.n[1]; i++) {
        CkSeq &s = pl.seq[1][i];
        const u64 parts = ((u64)s.n * gqa + 127) / 128;
        s.ns = (u32)((parts + per - 1) / per);
        s.wg0 = (u32)wgs[1];
        s.grp0 = (u32)(pl.floats / wkeys);
        wgs[1] += (u64)s.ncb * n_kv * s.ns;
        pl.floats += (u64)s.ncb * n_kv * s.ns * wkeys;
    }
    if (wgs[0] > 0x7fffffffull || wgs[1] > 0x7fffffffull) return false;
    pl.wgs[0] = (u32)wgs[0];
    pl.wgs[1] = (u32)wgs[1];
    pl.blocks = (u32)blocks;
    return true;
}

static bool most_sums(u32 n_kv, u32 gqa, u32 head_dim, bool q8, u32 window, const tl_chunk *ch, u32 n_chunk,
                      u64 *floats) {
    WeightPlan pl;
    const tl_chunk *of[CK_MAX_SEQ];
    *floats = 0;
    for (u32 i = 0; i < n_chunk;) {
        const u32 m = next_chunks(ch, n_chunk, &i, of);
        if (!m) break;
        if (!plan_weight(pl, of, m, n_kv, gqa, head_dim, q8, window)) return false;
        *floats = pl.floats > *floats ? pl.floats : *floats;
    }
    return true;
}

extern "C" int tl_attn_chunks_ws(uint32_t n_kv_head, uint32_t head_dim, const tl_chunk_attn_args *a,
                                 const tl_chunk *chunks, uint32_t n_chunk, uint64_t *bytes) {
    if (!a || !bytes || (n_chunk && !chunks) || n_chunk > CK_MAX_CHUNKS || !n_kv_head || !a->n_head ||
        a->n_head % n_kv_head || (head_dim != 64 && head_dim != 128 && head_dim != 256))
        return tl_fail(TL_EINVAL, "attn_chunks_ws: arguments");
    u64 parts[2], floats[2];
    if (!most_parts(n_kv_head, a->n_head / n_kv_head, head_dim, false, a->window, chunks, n_chunk, &parts[0]) ||
        !most_parts(n_kv_head, a->n_head / n_kv_head, head_dim, true, a->window, chunks, n_chunk, &parts[1]) ||
        !most_sums(n_kv_head, a->n_head / n_kv_head, head_dim, false, a->window, chunks, n_chunk, &floats[0]) ||
        !most_sums(n_kv_head, a->n_head / n_kv_head, head_dim, true, a->window, chunks, n_chunk, &floats[1]))
        return tl_fail(TL_ERANGE, "attn_chunks: too many workgroups");
    const u64 attn = ws_need(parts[0] > parts[1] ? parts[0] : parts[1], head_dim), weight = CK_WS_HEAD + (floats[0] > floats[1] ? floats[0] : floats[1]) * sizeof(float);
    *bytes = attn > weight ? attn : weight;
    return TL_OK;
}

/* where the call's counters, (max, sum) pairs and partial floats lie (its
 * launches take them one after another) */
static int take_ws(const tl_chunk_attn_args *a, u64 pairs, u64 floats, hipStream_t st, CkAttnParams &p) {
    if (!floats) return TL_OK;
    if (a->ws) {
        const u64 need = CK_WS_HEAD + pairs * sizeof(float2) + floats * sizeof(float);
        if (a->ws_bytes < need)
            return tl_fail(TL_ERANGE, "attn_chunks: workspace of %llu bytes, %llu needed",
                           (unsigned long long)a->ws_bytes, (unsigned long long)need);
        p.cnt = (u32 *)a->ws;
        p.ws_ml = (float2 *)((char *)a->ws + CK_WS_HEAD);
        p.ws_acc = (float *)(p.ws_ml + pairs);
        return TL_OK;
    }
    hipStreamCaptureStatus cs = hipStreamCaptureStatusNone;
    HIP_TRY(hipStreamIsCapturing(st, &cs));
    if (cs != hipStreamCaptureStatusNone)
        return tl_fail(TL_EINVAL, "attn_chunks: a captured call takes its own workspace (ws)");
    TlWorkspace *w;
    const int rc = tl_workspace_get(st, floats, pairs, TL_MERGE_CNT_WORDS, &w);
    if (rc) return rc;
    p.cnt = w->cnt;
    p.ws_ml = (float2 *)w->ml;
    p.ws_acc = w->acc;
    return TL_OK;
}

static void fill_attn(CkAttnParams &p, const LayerView &L, const tl_chunk_attn_args *a, u32 shift) {
    memset(&p, 0, sizeof(p));
    p.c = cache_of(L, shift);
    p.q = a->q;
    p.dst = a->dst;
    p.lse = a->lse;
    p.first = a->first;
    p.slopes = a->slopes;
    p.n_head = a->n_head;
    p.gqa = a->n_head / L.n_kv_head;
    p.q_stride = a->q_stride;
    p.window = a->window;
    p.scale = a->scale;
    p.softcap = a->softcap;
    p.inv_cap = a->softcap > 0.f ? 1.f / a->softcap : 0.f;
    p.gqa_mul = p.gqa > 1 ? (u32)((1ull << 32) / p.gqa) + 1 : 0;
}

static int attn_chunks(const LayerView &L, const tl_chunk_attn_args *a, const tl_chunk *ch, u32 n_chunk,
                       hipStream_t st) {
    u32 shift;
    int rc = check_attn(L, a, ch, n_chunk, false, &shift);
    if (rc) return rc;
    const u32 width = a->n_head * L.head_dim;
    if (rows_overlap(a->rows, a->q, a->q_stride, width, a->dst, a->q_stride, width))
        return tl_fail(TL_EINVAL, "attn_chunks: dst overlaps q");
    const u64 lse = (u64)a->rows * a->n_head * sizeof(float);
    if (tl_ranges_overlap(a->lse, lse, a->q, span(a->rows, a->q_stride, width)) ||
        tl_ranges_overlap(a->lse, lse, a->dst, span(a->rows, a->q_stride, width)))
        return tl_fail(TL_EINVAL, "attn_chunks: lse overlaps q or dst");
    CkAttnParams p;
    fill_attn(p, L, a, shift);
    u64 parts;
    if (!most_parts(L.n_kv_head, p.gqa, L.head_dim, L.q8, a->window, ch, n_chunk, &parts))
        return tl_fail(TL_ERANGE, "attn_chunks: too many workgroups");
    rc = take_ws(a, parts, parts * L.head_dim, st, p);
    if (rc) return rc;
    const tl_chunk *of[CK_MAX_SEQ];
    AttnPlan pl;
    for (u32 i = 0; i < n_chunk;) {
        const u32 m = next_chunks(ch, n_chunk, &i, of);
        if (!m) break;
        plan_attn(pl, of, m, L.n_kv_head, p.gqa, L.head_dim, L.q8, a->window);
        const bool both = pl.n[0] && pl.n[1] && L.head_dim != 256;
        for (int w = 1; w >= (both ? 1 : 0); w--) {
            if (!pl.wgs[w]) continue;
            p.n_seq = pl.n[w];
            memcpy(p.seq, pl.seq[w], pl.n[w] * sizeof(CkSeq));
            if (both) {
                /* the wide ones first: they take longer */
                for (u32 j = 0; j < pl.n[1]; j++) p.seq[j].wide = 1;
                for (u32 j = 0; j < pl.n[0]; j++) {
                    p.seq[p.n_seq] = pl.seq[0][j];
                    p.seq[p.n_seq++].wg0 += pl.wgs[1];
                }
            }
            starts(p);
            if (both) ck_launch_both(p, L.head_dim, L.q8, pl.wgs[0] + pl.wgs[1], st);
            else if (w) ck_launch_wide(p, L.head_dim, L.q8, pl.wgs[w], st);
            else ck_launch_attn(p, L.head_dim, L.q8, pl.wgs[w], st);
            HIP_TRY(hipGetLastError());
            if (!w) continue;
            /* the wide chunks with several splits are joined */
            u32 k = 0;
            u64 blocks = 0;
            const u32 per = 1024 / L.head_dim;      /* columns of a block */
            for (u32 j = 0; j < pl.n[1]; j++)
                if (pl.seq[1][j].ns > 1) {
                    p.seq[k] = pl.seq[1][j];
                    p.seq[k++].wg0 = (u32)blocks;
                    const u64 left = (u64)pl.seq[1][j].n * p.gqa - (u64)pl.seq[1][j].cb0 * CK_WCOLS;
                    const u64 cols = left < (u64)pl.seq[1][j].ncb * CK_WCOLS ? left : (u64)pl.seq[1][j].ncb * CK_WCOLS;
                    blocks += (cols * L.n_kv_head + per - 1) / per;
                }
            if (!k) continue;
            p.n_seq = k;
            starts(p);
            ck_launch_merge(p, L.head_dim, (u32)blocks, st);
            HIP_TRY(hipGetLastError());
        }
    }
    return TL_OK;
}

extern "C" int tl_attn_chunks(const tl_kv_layer *L, const tl_chunk_attn_args *a, const tl_chunk *chunks,
                              uint32_t n_chunk, void *stream) {
    const int rc = tl_check_layer(L);
    return rc ? rc : attn_chunks(tl_view(L), a, chunks, n_chunk, (hipStream_t)stream);
}

extern "C" int tl_attn_chunks_q8(const tl_kv_layer_q8 *L, const tl_chunk_attn_args *a, const tl_chunk *chunks,
                                 uint32_t n_chunk, void *stream) {
    const int rc = tl_check_layer_q8(L);
    return rc ? rc : attn_chunks(tl_view_q8(L), a, chunks, n_chunk, (hipStream_t)stream);
}

/* ------------------------------------------------------------------------ */
/* attention weight                                                          */
/* ------------------------------------------------------------------------ */

/* weight[key] += the sums of the kv heads and column shares, in order */
__global__ __launch_bounds__(256) void chunk_weight_sum_kernel(const CkAttnParams p, u32 wkeys) {
    const CkSeq &sq = p.seq[ck_find(p.wg0, p.n_seq, blockIdx.x)];
    /* the sums of a workgroup's keys lie side by side: sets of wkeys */
    const u32 key = (blockIdx.x - sq.wg0) * 256 + threadIdx.x;
    const u32 kblk = key / wkeys;
    if (sq.part0 + key >= sq.pos + sq.n) return;
    const float *in = p.ws_acc + ((u64)sq.grp0 + kblk) * wkeys + key % wkeys;
    const u32 n = sq.ns * p.c.n_kv;
    const float old = sq.weight[sq.part0 + key];
    float sum = 0.f;
    for (u32 x = 0; x < n; x += 8) {
        float v[8];
#pragma unroll
        for (u32 j = 0; j < 8; j++) v[j] = in[(u64)min(x + j, n - 1) * sq.ncb * wkeys];
#pragma unroll
        for (u32 j = 0; j < 8; j++) sum += x + j < n ? v[j] : 0.f;
    }
    sq.weight[sq.part0 + key] = old + sum;
}

static int attn_weight(const LayerView &L, const tl_chunk_attn_args *a, const tl_chunk *ch, u32 n_chunk,
                       hipStream_t st) {
    u32 shift;
    int rc = check_attn(L, a, ch, n_chunk, true, &shift);
    if (rc) return rc;
    if (!a->lse) return tl_fail(TL_EINVAL, "attn_weight: null lse");
    for (u32 i = 0; i < n_chunk; i++)
        if (ch[i].n && (!ch[i].weight || ((uintptr_t)ch[i].weight & 3)))
            return tl_fail(TL_EINVAL, "attn_weight: weight of chunk %u", i);
    if (any_overlap(n_chunk, [&](u32 i) { return (u64)(uintptr_t)ch[i].weight; },
                    [&](u32 i) { return ch[i].n ? ((u64)ch[i].pos + ch[i].n) * 4 : 0; }))
        return tl_fail(TL_EINVAL, "attn_weight: two chunks share weights");
    for (u32 i = 0; i < n_chunk; i++) {
        const u64 bytes = ch[i].n ? ((u64)ch[i].pos + ch[i].n) * sizeof(float) : 0;
        if (tl_ranges_overlap(ch[i].weight, bytes, a->lse, (u64)a->rows * a->n_head * sizeof(float)) ||
            tl_ranges_overlap(ch[i].weight, bytes, a->q, span(a->rows, a->q_stride, a->n_head * L.head_dim)))
            return tl_fail(TL_EINVAL, "attn_weight: weight of chunk %u overlaps q or lse", i);
    }
    CkAttnParams p;
    fill_attn(p, L, a, shift);
    u64 floats;
    if (!most_sums(L.n_kv_head, p.gqa, L.head_dim, L.q8, a->window, ch, n_chunk, &floats))
        return tl_fail(TL_ERANGE, "attn_weight: too many keys");
    rc = take_ws(a, 0, floats, st, p);
    if (rc) return rc;
    const tl_chunk *of[CK_MAX_SEQ];
    WeightPlan pl;
    for (u32 i = 0; i < n_chunk;) {
        const u32 m = next_chunks(ch, n_chunk, &i, of);
        if (!m) break;
        plan_weight(pl, of, m, L.n_kv_head, p.gqa, L.head_dim, L.q8, a->window);
        for (int w = 1; w >= 0; w--) {
            if (!pl.n[w]) continue;
            p.n_seq = pl.n[w];
            memcpy(p.seq, pl.seq[w], pl.n[w] * sizeof(CkSeq));
            starts(p);
            if (w) ck_launch_weight_wide(p, L.head_dim, L.q8, pl.wgs[w], st);
            else ck_launch_weight(p, L.head_dim, L.q8, pl.wgs[w], st);
            HIP_TRY(hipGetLastError());
            if (!w) continue;
            u32 at = 0;
            for (u32 j = 0; j < pl.n[1]; j++) {
                p.seq[j].wg0 = at;
                at += (p.seq[j].pos + p.seq[j].n - p.seq[j].part0 + 255) / 256;
            }
            starts(p);
            hipLaunchKernelGGL(chunk_weight_sum_kernel, dim3(at), dim3(256), 0, st, p, (u32)ck_weight_keys((int)L.head_dim, L.q8));
            HIP_TRY(hipGetLastError());
        }
    }
    return TL_OK;
}

extern "C" int tl_attn_weight(const tl_kv_layer *L, const tl_chunk_attn_args *a, const tl_chunk *chunks,
                              uint32_t n_chunk, void *stream) {
    const int rc = tl_check_layer(L);
    return rc ? rc : attn_weight(tl_view(L), a, chunks, n_chunk, (hipStream_t)stream);
}

extern "C" int tl_attn_weight_q8(const tl_kv_layer_q8 *L, const tl_chunk_attn_args *a, const tl_chunk *chunks,
                                 uint32_t n_chunk, void *stream) {
    const int rc = tl_check_layer_q8(L);
    return rc ? rc : attn_weight(tl_view_q8(L), a, chunks, n_chunk, (hipStream_t)stream);
}

/* ------------------------------------------------------------------------ */
/* instances                                                                 */
/* ------------------------------------------------------------------------ */

void ck_launch_attn(const CkAttnParams &p, u32 head_dim, bool q8, u32 wgs, hipStream_t st) {
    if (head_dim == 64) q8 ? ck_launch_attn_t<64, true>(p, wgs, st) : ck_launch_attn_t<64, false>(p, wgs, st);
    else if (head_dim == 128) q8 ? ck_launch_attn_t<128, true>(p, wgs, st) : ck_launch_attn_t<128, false>(p, wgs, st);
    else q8 ? ck_launch_attn_t<256, true>(p, wgs, st) : ck_launch_attn_t<256, false>(p, wgs, st);
}

void ck_launch_wide(const CkAttnParams &p, u32 head_dim, bool q8, u32 wgs, hipStream_t st) {
    if (head_dim == 64) q8 ? ck_launch_wide_t<64, true>(p, wgs, st) : ck_launch_wide_t<64, false>(p, wgs, st);
    else if (head_dim == 128) q8 ? ck_launch_wide_t<128, true>(p, wgs, st) : ck_launch_wide_t<128, false>(p, wgs, st);
    else q8 ? ck_launch_wide_t<256, true>(p, wgs, st) : ck_launch_wide_t<256, false>(p, wgs, st);
}

void ck_launch_both(const CkAttnParams &p, u32 head_dim, bool q8, u32 wgs, hipStream_t st) {
    if (head_dim == 64) q8 ? ck_launch_both_t<64, true>(p, wgs, st) : ck_launch_both_t<64, false>(p, wgs, st);
    else q8 ? ck_launch_both_t<128, true>(p, wgs, st) : ck_launch_both_t<128, false>(p, wgs, st);
}

void ck_launch_weight_wide(const CkAttnParams &p, u32 head_dim, bool q8, u32 wgs, hipStream_t st) {
    if (head_dim == 64) q8 ? ck_launch_weight_wide_t<64, true>(p, wgs, st) : ck_launch_weight_wide_t<64, false>(p, wgs, st);
    else if (head_dim == 128) q8 ? ck_launch_weight_wide_t<128, true>(p, wgs, st) : ck_launch_weight_wide_t<128, false>(p, wgs, st);
    else q8 ? ck_launch_weight_wide_t<256, true>(p, wgs, st) : ck_launch_weight_wide_t<256, false>(p, wgs, st);
}

void ck_launch_weight(const CkAttnParams &p, u32 head_dim, bool q8, u32 wgs, hipStream_t st) {
    if (head_dim == 64) q8 ? ck_launch_weight_t<64, true>(p, wgs, st) : ck_launch_weight_t<64, false>(p, wgs, st);
    else if (head_dim == 128) q8 ? ck_launch_weight_t<128, true>(p, wgs, st) : ck_launch_weight_t<128, false>(p, wgs, st);
    else q8 ? ck_launch_weight_t<256, true>(p, wgs, st) : ck_launch_weight_t<256, false>(p, wgs, st);
}
