"""The operators on batches of chunks over a paged KV cache, as cases that can be
timed and checked: norm + rotation + append of new rows (`append`), attention
with score caps, distance biases and masks (`attn`), the attention weight that
each cached position has received (`weight`), and the eviction of the positions
that received least (`evict`).

`run` computes them either from elementary torch operations in 32 bits
(own = False) or by the library's entry points (own = True); `exact` is the
definition in 64 bits, session by session.

A batch holds `n_seq` sessions.  Session i has `pos` positions in the cache and
brings `n` new rows; both are spread geometrically over the sessions, the
sessions with the longest contexts bringing the fewest rows.  The sessions'
pages are dealt out of one pool in random order.
"""
import ctypes
import math
import os
import sys

import torch

own = False
DEV = "cuda"

# (n_head, n_kv, head_dim, theta, neox): the shapes of the benchmark's configs
SHAPES = {
    "1b": (32, 8, 64, 5e5, 0),        # Llama-3.2-1B-shaped
    "8b": (32, 8, 128, 5e5, 0),       # Llama-3-8B-shaped
    "qwen": (28, 4, 128, 1e6, 1),     # Qwen2.5-7B-shaped (gqa 7)
    "gemma": (8, 4, 256, 1e4, 1),     # Gemma-3-4B-shaped
    "mha": (8, 8, 128, 5e5, 0),       # one query head per kv head
}
TAIL = 3          # batch rows behind the last session's: no call touches them
EPS = 1e-6


def _batch(op, shape, n_seq, pos, n, pos_min=0, n_min=0, page=16, q8=False, window=0, cap=0.0,
           alibi=False, prefix=0, doc=0, pad=0):
    return dict(op=op, shape=shape, n_seq=n_seq, pos=pos, pos_min=pos_min or pos, n=n,
                n_min=n_min or n, page=page, q8=q8, window=window, cap=cap, alibi=alibi,
                prefix=prefix, doc=doc, pad=pad)


def listed():
    return [
        # a server's decode step on a model that norms its heads: 16 sessions, one new token each
        dict(_batch("append", "gemma", 16, 8192, 1, pos_min=512), name="append-decode"),
        # a step that packs the prompts of three sessions (ragged, 2100 rows together)
        dict(_batch("append", "8b", 3, 4099, 1201, pos_min=17, n_min=333, pad=32),
             name="append-prompts"),
        # a server's decode step: 16 sessions of ragged lengths
        dict(_batch("attn", "qwen", 16, 8192, 1, pos_min=512), name="attn-decode"),
        # long-context decode of one session with capped scores, 64-row pages
        dict(_batch("attn", "8b", 1, 32781, 1, page=64, cap=30.0), name="attn-decode-cap"),
        # draft tokens of 4 small-model sessions with distance biases, slot table (pages of one row)
        dict(_batch("attn", "1b", 4, 1500, 5, pos_min=300, page=1, alibi=True),
             name="attn-draft-bias"),
        # a mixed step over the quantized cache: sessions that decode beside one that reads its prompt
        dict(_batch("attn", "8b", 6, 6000, 200, pos_min=64, n_min=1, q8=True),
             name="attn-mixed-q8"),
        # a prompt chunk of a deep context, packed documents of 9000 tokens
        dict(_batch("attn", "8b", 1, 16384, 512, doc=9000), name="attn-chunk-doc"),
        # first prompts behind an image-like prefix that sees itself both ways, windowed layer
        dict(_batch("attn", "gemma", 2, 0, 700, n_min=333, window=512, prefix=256, page=32),
             name="attn-prefix"),
        # the weight that a decode step of 8 sessions adds to every cached position
        dict(_batch("weight", "8b", 8, 12000, 1, pos_min=3000), name="weight-decode"),
        # the same for a prompt chunk, capped scores
        dict(_batch("weight", "1b", 1, 4096, 512, cap=50.0), name="weight-chunk"),
        # 8 sessions cut back to half of their positions
        dict(op="evict", n_seq=8, len=8192, len_min=3001, keep=0.5, sink=4, recent=256, page=16,
             name="evict-batch"),
        # one very long session cut back to a quarter
        dict(op="evict", n_seq=1, len=131072, len_min=131072, keep=0.25, sink=16, recent=1024,
             page=1, name="evict-long"),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(["append", "attn", "attn", "attn", "weight", "evict"])
    if op == "evict":
        n = _log_int(rng, 1, 16)
        top = _log_int(rng, 64, 131072 // n)
        return dict(op=op, n_seq=n, len=top, len_min=_log_int(rng, 33, top),
                    keep=round(rng.uniform(0.1, 0.9), 3), sink=rng.choice([0, 4, 16]),
                    recent=_log_int(rng, 1, max(2, top // 16)), page=rng.choice([1, 16, 64]))
    shape = rng.choice(list(SHAPES))
    H, KV, D, _, _ = SHAPES[shape]
    while True:
        n_seq = _log_int(rng, 1, 16)
        n = 1 if rng.random() < 0.4 else _log_int(rng, 2, 700)
        pos = _log_int(rng, 1, 32000)
        if op == "append":
            if n * n_seq <= 2100 and (pos + n) * n_seq <= 60000:
                break
        elif (n_seq * n * (pos + n) * H <= 1 << 28 and n_seq * n * (pos + n) * H * D * 4 <= 6 << 33
              and n_seq * (pos + n) * KV * D <= 1 << 27):
            break
    c = _batch(op, shape, n_seq, pos, n, pos_min=_log_int(rng, 1, pos), n_min=_log_int(rng, 1, n),
               page=rng.choice([1, 16, 32, 64]), q8=rng.random() < 0.3,
               pad=rng.choice([0, 0, 32]))
    if op != "append":
        if rng.random() < 0.3:
            c["window"] = _log_int(rng, 16, 4096)
        if rng.random() < 0.35:
            c["cap"] = rng.choice([15.0, 30.0, 50.0])
        if rng.random() < 0.3:
            c["alibi"] = True
        if rng.random() < 0.25:
            c["doc"] = _log_int(rng, 8, 8000)
        if rng.random() < 0.25:
            c["prefix"] = _log_int(rng, 1, max(2, pos // 2 + n // 2))
    return c


# ---- what a case holds -----------------------------------------------------------


def _spread(lo, hi, m):
    if m == 1:
        return [hi]
    return [int(round(lo * (hi / lo) ** (i / (m - 1)))) if lo else hi * i // (m - 1) for i in range(m)]


def _sizes(c):
    """(pos, n) of every session; long and short sessions side by side."""
    m = c["n_seq"]
    at = list(zip(_spread(c["pos_min"], c["pos"], m), _spread(c["n_min"], c["n"], m)[::-1]))
    return at[::2] + at[1::2]


def _lens(c):
    at = _spread(c["len_min"], c["len"], c["n_seq"])
    return at[::2] + at[1::2]


def _keeps(c):
    return [max(1, int(n * c["keep"])) for n in _lens(c)]


def _holds(c):
    """(first, last) positions of every session that stay whatever their weight."""
    return [(min(c["sink"], k), min(c["recent"], (k - min(c["sink"], k)) // 2)) for k in _keeps(c)]


def _visible(c, pos, n):
    """Scores that the masks leave, and keys that any row of the session sees."""
    pairs, low, base, first = 0, pos + n, pos + n, min(c["prefix"], pos + n)
    for p in range(pos, pos + n):
        start = p - p % c["doc"] if c["doc"] else 0
        a = max(start, p + 1 - c["window"] if c["window"] else 0)
        pairs += p + 1 - a + max(0, min(first, a) - start) + max(0, first - p - 1)
        low, base = min(low, a), min(base, start)
    return pairs, pos + n - low + max(0, min(first, low) - base)


def work(c):
    if c["op"] == "evict":
        # every weight and page entry is read, kept and freed rows and kept weights are written
        total, kept = sum(_lens(c)), sum(_keeps(c))
        return {"bytes": 4 * (total + total // c["page"] + 3 * kept + total - kept), "flops": 0}
    H, KV, D, _, _ = SHAPES[c["shape"]]
    rows = sum(n for _, n in _sizes(c))
    row = KV * (D + D // 16 if c["q8"] else 2 * D)        # bytes of one position's K (or V)
    if c["op"] == "append":
        return {"bytes": rows * (2 * H * D * 4 + 2 * KV * D * 4 + 2 * row), "flops": 0}
    pairs = keys = 0
    for pos, n in _sizes(c):
        p, k = _visible(c, pos, n)
        pairs, keys = pairs + p, keys + k
    if c["op"] == "weight":
        return {"bytes": keys * (row + 8) + rows * H * (D + 1) * 4, "flops": 2 * pairs * H * D}
    return {"bytes": keys * 2 * row + rows * H * (2 * D + 1) * 4, "flops": 4 * pairs * H * D}


# ---- inputs -----------------------------------------------------------------------


def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed))
    return g


def _quantize(x):
    """Q8_0 blocks of x[..., D]: int8 values and binary16 scales."""
    b = x.reshape(*x.shape[:-1], -1, 32)
    d = b.abs().amax(-1) / 127
    q = torch.round(b * torch.where(d > 0, 1 / d, torch.zeros_like(d))[..., None])
    return q.to(torch.int8).reshape(x.shape), d.to(torch.float16)


def _dequantize(v, s, t):
    return (v.to(t).reshape(*s.shape, 32) * s.to(t)[..., None]).reshape(v.shape)


def _pages(c, lens, g):
    """[n_seq][most pages] page tables out of one pool, and the pool's rows."""
    per = [-(-n // c["page"]) for n in lens]
    total = sum(per) + 1
    deal = torch.randperm(total, generator=g, device=DEV).to(torch.int32)
    table = torch.zeros((len(lens), max(per)), dtype=torch.int32, device=DEV)
    at = 0
    for i, k in enumerate(per):
        table[i, :k] = deal[at:at + k]
        at += k
    return table, total * c["page"]


def prepare(c, seed):
    g = _gen(seed)
    s = _prepare_evict(c, g) if c["op"] == "evict" else _prepare_batch(c, g)
    if own:
        # the argument blocks, which a program lays out once and then moves along with its sessions
        s["calls"] = (_calls_evict if c["op"] == "evict" else _calls_batch)(c, s)
    return s


def _prepare_evict(c, g):
    lens, keeps = _lens(c), _keeps(c)
    table, _ = _pages(c, lens, g)
    # a few positions hold most of the weight, many hold none
    w = torch.exp(2 * torch.randn((len(lens), max(lens)), generator=g, device=DEV))
    w = torch.round(w * 64) / 64
    free = max(a - b for a, b in zip(lens, keeps))
    out = {k: torch.zeros((len(lens), n), dtype=torch.int32, device=DEV)
           for k, n in (("kept", max(keeps)), ("rows", max(keeps)), ("freed", free))}
    out["weight"] = torch.zeros((len(lens), max(keeps)), device=DEV)
    at = torch.tensor(lens, device=DEV)[:, None]
    sink, recent = (torch.tensor(x, device=DEV)[:, None] for x in zip(*_holds(c)))
    return dict(c=c, table=table, w=w, out=out, lens=at, sink=sink, recent=recent,
                keeps=torch.tensor(keeps, device=DEV)[:, None])


def _prepare_batch(c, g):
    H, KV, D, theta, _ = SHAPES[c["shape"]]
    sizes = _sizes(c)
    lens = [p + n for p, n in sizes]
    table, cap = _pages(c, lens, g)
    rows = sum(n for _, n in sizes) + TAIL
    s = dict(c=c, table=table, cap=cap, rows=rows)

    def fresh(width):
        return torch.randn((rows, width + c["pad"]), generator=g, device=DEV)

    for x in "kv":
        if c["q8"]:
            s[x] = torch.empty((KV, cap, D), dtype=torch.int8, device=DEV)
            s[x + "s"] = torch.empty((KV, cap, D // 32), dtype=torch.float16, device=DEV)
            for h in range(KV):
                s[x][h], s[x + "s"][h] = _quantize(torch.randn((cap, D), generator=g, device=DEV))
        else:
            s[x] = torch.randn((KV, cap, D), generator=g, device=DEV, dtype=torch.float16)
    s["pos"] = torch.tensor([p for p, _ in sizes], device=DEV)
    s["n"] = torch.tensor([n for _, n in sizes], device=DEV)
    s["row"] = torch.cumsum(s["n"], 0) - s["n"]
    s["dst"] = torch.zeros((rows, H * D + c["pad"]), device=DEV)
    if c["op"] == "append":
        # activations of a projection; norm weights near one
        s.update(q=fresh(H * D), kin=fresh(KV * D), vin=fresh(KV * D))
        s["qw"] = 1 + 0.2 * torch.randn(D, generator=g, device=DEV)
        s["kw"] = 1 + 0.2 * torch.randn(D, generator=g, device=DEV)
        return s
    s["q"] = 2 * fresh(H * D)                      # sharper than noise: scores of spread 2
    s["lse"] = torch.zeros((rows, H), device=DEV)
    s["slopes"] = 2.0 ** (-8.0 * torch.arange(1, H + 1, device=DEV) / H) if c["alibi"] else None
    s["first"] = None
    if c["doc"]:
        s["first"] = torch.zeros(rows, dtype=torch.int32, device=DEV)
        for (p, n), r in zip(sizes, s["row"].tolist()):
            at = torch.arange(p, p + n, device=DEV)
            s["first"][r:r + n] = (at - at % c["doc"]).to(torch.int32)
    if c["op"] == "weight":
        s["weight"] = torch.rand((len(sizes), max(lens)), generator=g, device=DEV)
        _scores_lse(s)                             # the forward pass has run: its row sums are kept
    return s


# ---- the library's calls ------------------------------------------------------------


def _tlkv():
    at = os.path.join(os.getcwd(), "tinyllama.c_amd")
    if at not in sys.path:
        sys.path.insert(0, at)
    import tlkv
    if not getattr(_tlkv, "ready", False):
        tlkv.check(tlkv.lib().tl_init(0))
        _tlkv.ready = True
    return tlkv


def _calls_evict(c, s):
    t = _tlkv()
    o = s["out"]
    seqs = (t.EvictSeq * c["n_seq"])(*[
        t.EvictSeq(weight=s["w"][i].data_ptr(), pages=s["table"][i].data_ptr(), len=n, keep=k,
                   sink=a, recent=b, page_size=c["page"],
                   kept=o["kept"][i].data_ptr(), rows=o["rows"][i].data_ptr(),
                   freed=o["freed"][i].data_ptr(), weight_out=o["weight"][i].data_ptr())
        for i, (n, k, (a, b)) in enumerate(zip(_lens(c), _keeps(c), _holds(c)))])
    return [(t.lib().tl_kv_evict, [seqs, c["n_seq"], t.stream_handle()])]


def _calls_batch(c, s):
    t = _tlkv()
    L, (H, KV, D, theta, neox) = t.lib(), SHAPES[c["shape"]]
    if c["q8"]:
        layer = t.KvLayerQ8(s["k"].data_ptr(), s["v"].data_ptr(), s["ks"].data_ptr(),
                            s["vs"].data_ptr(), s["cap"], KV, D, 0)
    else:
        layer = t.KvLayer(s["k"].data_ptr(), s["v"].data_ptr(), s["cap"], KV, D, 0)
    chunks = (t.Chunk * c["n_seq"])(*[
        t.Chunk(pages=s["table"][i].data_ptr(), pos=p, n=n, row=r, prefix=c["prefix"],
                weight=s["weight"][i].data_ptr() if c["op"] == "weight" else None)
        for i, ((p, n), r) in enumerate(zip(_sizes(c), s["row"].tolist()))])
    if c["op"] == "append":
        a = t.QkNormArgs(q=s["q"].data_ptr(), k=s["kin"].data_ptr(), v=s["vin"].data_ptr(),
                         q_out=s["dst"].data_ptr(), q_weight=s["qw"].data_ptr(),
                         k_weight=s["kw"].data_ptr(), eps=EPS, rows=s["rows"], n_head=H,
                         q_stride=H * D + c["pad"], kv_stride=KV * D + c["pad"],
                         q_out_stride=H * D + c["pad"], page_size=c["page"],
                         rope=t.RopeParams(D, theta, neox))
        fn = L.tl_qk_norm_append_q8 if c["q8"] else L.tl_qk_norm_append
    else:
        a = t.ChunkAttnArgs(q=s["q"].data_ptr(), dst=s["dst"].data_ptr(), lse=s["lse"].data_ptr(),
                            first=None if s["first"] is None else s["first"].data_ptr(),
                            slopes=None if s["slopes"] is None else s["slopes"].data_ptr(),
                            rows=s["rows"], n_head=H, q_stride=H * D + c["pad"],
                            page_size=c["page"], window=c["window"], scale=1 / math.sqrt(D),
                            softcap=c["cap"])
        fn = {("attn", False): L.tl_attn_chunks, ("attn", True): L.tl_attn_chunks_q8,
              ("weight", False): L.tl_attn_weight, ("weight", True): L.tl_attn_weight_q8}[
                  c["op"], c["q8"]]
    return [(fn, [ctypes.byref(layer), ctypes.byref(a), chunks, c["n_seq"], t.stream_handle()])]


# ---- one pass ---------------------------------------------------------------------


def run(s):
    c = s["c"]
    if own:
        for fn, args in s["calls"]:
            rc = fn(*args)
            if rc:
                _tlkv().check(rc)
    elif c["op"] == "evict":
        _plain_evict(s)
    elif c["op"] == "append":
        _plain_append(s)
    elif c["op"] == "attn":
        _plain_attn(s)
    else:
        _plain_weight(s)
    if c["op"] == "evict":
        return s["out"]
    if c["op"] == "weight":
        return s["weight"]
    if c["op"] == "attn":
        return s["dst"], s["lse"]
    if c["q8"]:     # the quantized rows as the values that they stand for, in their scales' type
        return (s["dst"], _dequantize(s["k"], s["ks"], torch.float16),
                _dequantize(s["v"], s["vs"], torch.float16))
    return s["dst"], s["k"], s["v"]


def _plain_evict(s):
    c, w, o, lens = s["c"], s["w"], s["out"], s["lens"]
    S, N = w.shape
    at = torch.arange(N, device=DEV)[None, :]
    hold = (at < s["sink"]) | (at >= lens - s["recent"])
    rank_by = torch.where(hold, float("inf"), w).masked_fill(at >= lens, -1.0)
    order = torch.sort(rank_by, dim=1, descending=True, stable=True).indices
    rank = torch.empty_like(order).scatter_(1, order, at.expand(S, N))
    keep = rank < s["keeps"]
    rows = torch.gather(s["table"].long(), 1, (at // c["page"]).clamp(max=s["table"].shape[1] - 1).expand(S, N))
    rows = rows * c["page"] + at % c["page"]
    # the kept ones to the front, in the order of their positions, then the others
    front = torch.sort((~keep).to(torch.int8) + (at >= lens).to(torch.int8), dim=1, stable=True).indices
    K, F = o["kept"].shape[1], o["freed"].shape[1]
    slot = torch.arange(N, device=DEV)[None, :]
    here = (slot < s["keeps"])[:, :K]
    o["kept"].copy_(torch.where(here, front[:, :K], 0))
    o["rows"].copy_(torch.where(here, torch.gather(rows, 1, front[:, :K]), 0))
    o["weight"].copy_(torch.where(here, torch.gather(w, 1, front[:, :K]), 0.0))
    gone = (s["keeps"] + slot[:, :F]).clamp(max=N - 1)
    there = slot[:, :F] < lens - s["keeps"]
    o["freed"].copy_(torch.where(there, torch.gather(rows, 1, torch.gather(front, 1, gone)), 0))


def _grid(s):
    """[S, N] batch row and position of every session's new rows, and which of them exist."""
    n = torch.arange(s["c"]["n"], device=DEV)[None, :]
    real = n < s["n"][:, None]
    row = torch.where(real, s["row"][:, None] + n, s["rows"] - 1)
    return row, s["pos"][:, None] + n, real


def _rows_of(s, at):
    """Pool rows of positions at[S, K] (those behind a session's end: some row)."""
    page = (at // s["c"]["page"]).clamp(max=s["table"].shape[1] - 1)
    return torch.gather(s["table"].long(), 1, page.expand(s["table"].shape[0], -1)) * s["c"]["page"] + at % s["c"]["page"]


def _normed(x, w):
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w


def _rotated(x, pos, D, theta, neox):
    """x[rows, heads, D] rotated at pos[rows]; angles in 64 bits, the rotation in x's type."""
    i = torch.arange(D // 2, device=DEV, dtype=torch.float64)
    ang = pos.to(torch.float64)[:, None] * theta ** (-2 * i / D)
    co, si = torch.cos(ang).to(x.dtype)[:, None], torch.sin(ang).to(x.dtype)[:, None]
    a, b = (x[..., : D // 2], x[..., D // 2:]) if neox else (x[..., 0::2], x[..., 1::2])
    ra, rb = a * co - b * si, a * si + b * co
    return torch.cat([ra, rb], -1) if neox else torch.stack([ra, rb], -1).reshape(x.shape)


def _plain_append(s):
    c = s["c"]
    H, KV, D, theta, neox = SHAPES[c["shape"]]
    row, pos, real = _grid(s)
    at = _rows_of(s, pos)[real]
    row, pos = row[real], pos[real]
    q = _normed(s["q"][row, :H * D].reshape(-1, H, D), s["qw"])
    k = _normed(s["kin"][row, :KV * D].reshape(-1, KV, D), s["kw"])
    s["dst"][row, :H * D] = _rotated(q, pos, D, theta, neox).reshape(-1, H * D)
    k = _rotated(k, pos, D, theta, neox).transpose(0, 1)
    v = s["vin"][row, :KV * D].reshape(-1, KV, D).transpose(0, 1)
    if c["q8"]:
        s["k"][:, at], s["ks"][:, at] = _quantize(k)
        s["v"][:, at], s["vs"][:, at] = _quantize(v)
    else:
        s["k"][:, at] = k.to(torch.float16)
        s["v"][:, at] = v.to(torch.float16)


def _cached(s, x, at):
    """[S, KV, K, D] f32 of pool rows at[S, K]."""
    if s["c"]["q8"]:
        r = _dequantize(s[x][:, at], s[x + "s"][:, at], torch.float32)
    else:
        r = s[x][:, at].float()
    return r.transpose(0, 1).contiguous()


def _scores(s):
    """[S, KV, G, N, K] scores, -inf where the masks hide them, and the grids."""
    c = s["c"]
    H, KV, D, _, _ = SHAPES[c["shape"]]
    row, pos, real = _grid(s)
    S, N = row.shape
    ends = s["pos"] + s["n"]
    key = torch.arange(max(p + n for p, n in _sizes(c)), device=DEV)[None, :]
    at = _rows_of(s, key)
    q = s["q"][row, :H * D].reshape(S, N, KV, H // KV, D).permute(0, 2, 3, 1, 4)
    x = torch.matmul(q.reshape(S, KV, -1, D), _cached(s, "k", at).transpose(2, 3))
    x = x.reshape(S, KV, H // KV, N, -1) * (1 / math.sqrt(D))
    if c["cap"]:
        x = torch.tanh(x / c["cap"]) * c["cap"]
    p, k = pos[:, :, None], key[:, None, :]
    if s["slopes"] is not None:
        far = (p - k).abs().float()[:, None, None]
        x = x - s["slopes"].reshape(1, KV, -1, 1, 1) * far
    see = k <= p
    if c["window"]:
        see = see & (p - k < c["window"])
    if c["prefix"]:
        see = see | (k < c["prefix"])
    if s["first"] is not None:
        see = see & (k >= s["first"][row][:, :, None])
    see = see & (k < ends[:, None, None]) & real[:, :, None]
    return x.masked_fill(~see[:, None, None], float("-inf")), row, real, key, at


def _scores_lse(s):
    x, row, real, _, _ = _scores(s)
    s["lse"][row[real]] = torch.logsumexp(x, -1).permute(0, 3, 1, 2).flatten(2)[real]


def _plain_attn(s):
    c = s["c"]
    H, KV, D, _, _ = SHAPES[c["shape"]]
    x, row, real, _, at = _scores(s)
    S, _, _, N, K = x.shape
    top = x.amax(-1, keepdim=True)
    top = torch.where(top > float("-inf"), top, torch.zeros_like(top))
    p = torch.exp(x - top)
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p.reshape(S, KV, -1, K), _cached(s, "v", at)).reshape(S, KV, -1, N, D)
    out = out / torch.where(total > 0, total, torch.ones_like(total))
    lse = (top + torch.log(total))[..., 0]
    s["dst"][row[real], :H * D] = out.permute(0, 3, 1, 2, 4).flatten(2)[real]
    s["lse"][row[real]] = lse.permute(0, 3, 1, 2).flatten(2)[real]


def _plain_weight(s):
    c = s["c"]
    H, KV, _, _, _ = SHAPES[c["shape"]]
    x, row, _, key, _ = _scores(s)
    S, _, G, N, K = x.shape
    lse = s["lse"][row].reshape(S, N, KV, G).permute(0, 2, 3, 1)[..., None]
    p = torch.where(x > float("-inf"), torch.exp(x - lse), torch.zeros_like(x))
    s["weight"][:, :K] += p.sum((1, 2, 3))


# ---- 64 bits, session by session ---------------------------------------------------


def exact(c, seed):
    global own
    was, own = own, False
    try:
        s = prepare(c, seed)
    finally:
        own = was
    return {"evict": _exact_evict, "append": _exact_append, "attn": _exact_attn,
            "weight": _exact_weight}[c["op"]](c, s)


def _exact_evict(c, s):
    out = {k: torch.zeros(v.shape, dtype=torch.int64) for k, v in s["out"].items()}
    out["weight"] = torch.zeros(s["out"]["weight"].shape, dtype=torch.float64)
    w, table = s["w"].double().cpu(), s["table"].long().cpu()
    for i, (n, k, (a, b)) in enumerate(zip(_lens(c), _keeps(c), _holds(c))):
        v = w[i].tolist()
        best = sorted(range(n), key=lambda j: (a <= j < n - b, -v[j], j))
        kept = torch.tensor(sorted(best[:k]))
        gone = torch.tensor(sorted(best[k:]))
        out["kept"][i, :k] = kept
        out["weight"][i, :k] = w[i, kept]
        out["rows"][i, :k] = table[i, kept // c["page"]] * c["page"] + kept % c["page"]
        out["freed"][i, :n - k] = table[i, gone // c["page"]] * c["page"] + gone % c["page"]
    return {k: v.to(torch.int32) if k != "weight" else v for k, v in out.items()}


def _exact_append(c, s):
    H, KV, D, theta, neox = SHAPES[c["shape"]]
    dst = s["dst"].double()
    if c["q8"]:
        kc, vc = (_dequantize(s[x], s[x + "s"], torch.float64) for x in "kv")
    else:
        kc, vc = s["k"].double(), s["v"].double()
    for i, ((pos, n), r) in enumerate(zip(_sizes(c), s["row"].tolist())):
        p = torch.arange(pos, pos + n, device=DEV)
        at = s["table"][i].long()[p // c["page"]] * c["page"] + p % c["page"]
        for x, w, heads in (("q", "qw", H), ("kin", "kw", KV)):
            y = s[x][r:r + n, :heads * D].double().reshape(n, heads, D)
            y = y / torch.sqrt((y ** 2).sum(-1, keepdim=True) / D + EPS) * s[w].double()
            z = y.clone()
            for j in range(D // 2):
                a, b = (j, j + D // 2) if neox else (2 * j, 2 * j + 1)
                ang = p.double() * float(theta) ** (-2.0 * j / D)
                co, si = torch.cos(ang)[:, None], torch.sin(ang)[:, None]
                z[..., a] = y[..., a] * co - y[..., b] * si
                z[..., b] = y[..., a] * si + y[..., b] * co
            if x == "q":
                dst[r:r + n, :H * D] = z.reshape(n, H * D)
            else:
                kc[:, at] = z.transpose(0, 1)
        vc[:, at] = s["vin"][r:r + n, :KV * D].double().reshape(n, KV, D).transpose(0, 1)
    return dst, kc, vc


def _exact_sessions(c, s):
    """For every session and head: (session, rows, head, probabilities, log sums, values)."""
    H, KV, D, _, _ = SHAPES[c["shape"]]
    for i, ((pos, n), r) in enumerate(zip(_sizes(c), s["row"].tolist())):
        end = pos + n
        j = torch.arange(end, device=DEV)
        at = s["table"][i].long()[j // c["page"]] * c["page"] + j % c["page"]
        p = torch.arange(pos, end, device=DEV)[:, None]
        see = j[None, :] <= p
        if c["window"]:
            see &= j[None, :] > p - c["window"]
        see |= j[None, :] < c["prefix"]
        if c["doc"]:
            see &= j[None, :] >= s["first"][r:r + n, None]
        for h in range(H):
            kv = h // (H // KV)
            if c["q8"]:
                K, V = (_dequantize(s[x][kv, at], s[x + "s"][kv, at], torch.float64) for x in "kv")
            else:
                K, V = s["k"][kv, at].double(), s["v"][kv, at].double()
            x = s["q"][r:r + n, h * D:(h + 1) * D].double() @ K.T.contiguous() / math.sqrt(D)
            if c["cap"]:
                x = c["cap"] * torch.tanh(x / c["cap"])
            if c["alibi"]:
                x = x - s["slopes"][h].double() * (p - j[None, :]).abs().double()
            x = x.masked_fill(~see, -math.inf)
            lse = torch.logsumexp(x, -1)
            prob = torch.where(see, torch.exp(x - lse[:, None]), 0.0)
            yield i, slice(r, r + n), h, prob, lse, V


def _exact_attn(c, s):
    D = SHAPES[c["shape"]][2]
    dst, sums = s["dst"].double(), s["lse"].double()
    for _, rows, h, prob, lse, V in _exact_sessions(c, s):
        dst[rows, h * D:(h + 1) * D] = prob @ V
        sums[rows, h] = lse
    return dst, sums


def _exact_weight(c, s):
    w = s["weight"].double()
    for i, _, _, prob, _, _ in _exact_sessions(c, s):
        w[i, :prob.shape[1]] += prob.sum(0)
    return w
