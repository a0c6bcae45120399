"""Batches of chunks over a paged cache (include/tlkv.h, tl_chunk): norm +
rotation + append, attention, attention weight and eviction, each against its
definition in 64 bits (chunk_ref.py), and a run of them together."""
import ctypes
import math

import numpy as np
import pytest

import chunk_ref as R

pytestmark = pytest.mark.gpu

SHAPES = {"1b": (32, 8, 64), "8b": (32, 8, 128), "qwen": (28, 4, 128), "gemma": (8, 4, 256),
          "mha": (8, 8, 128), "mqa": (20, 1, 64), "kv12": (12, 12, 64), "kv3": (9, 3, 128),
          "mqa40": (40, 1, 128)}


@pytest.fixture(scope="module")
def T():
    import torch
    assert torch.cuda.is_available(), "GPU tests need a HIP device"
    import tlkv
    tlkv.check(tlkv.lib().tl_init(0))
    return torch


class Dev:
    """Device copies of a Batch and its argument blocks."""

    def __init__(self, T, B):
        import tlkv
        self.T, self.B, self.t = T, B, tlkv
        self.x = {}
        for f in ("q", "kin", "vin", "k", "v") + (("ks", "vs") if B.q8 else ()):
            self.put(f, getattr(B, f))
        self.tab = [None if t is None or not t.size else T.from_numpy(t.view(np.int32)).cuda()
                    for t in B.tables]
        k = self.x
        if B.q8:
            self.layer = tlkv.KvLayerQ8(*(k[f].data_ptr() for f in ("k", "v", "ks", "vs")), B.cap, B.KV, B.D, 0)
        else:
            self.layer = tlkv.KvLayer(k["k"].data_ptr(), k["v"].data_ptr(), B.cap, B.KV, B.D, 0)
        self.dst = T.full((B.rows, B.q_stride), 7.5, device="cuda")
        self.lse = T.full((B.rows, B.H), 7.5, device="cuda")

    def put(self, name, a):
        a = np.ascontiguousarray(a)
        self.x[name] = self.T.from_numpy(a.view(np.int32) if a.dtype == np.uint32 else a).cuda()
        return self.x[name]

    def chunks(self, prefix=None, weight=None, skip=None):
        B = self.B
        return (self.t.Chunk * max(1, len(B.sizes)))(*[
            self.t.Chunk(pages=None if self.tab[i] is None else self.tab[i].data_ptr(), pos=p, n=n,
                         row=B.row[i], prefix=prefix[i] if prefix else 0,
                         rope_skip=skip[i] if skip else 0,
                         weight=weight[i].data_ptr() if weight else None)
            for i, (p, n) in enumerate(B.sizes)])

    def attn_args(self, scale, window=0, first=None, softcap=0.0, slopes=None, ws=None, lse=True):
        B = self.B
        if first is not None:
            self.put("first", first)
        if slopes is not None:
            self.put("slopes", np.asarray(slopes, dtype=np.float32))
        return self.t.ChunkAttnArgs(
            q=self.x["q"].data_ptr(), dst=self.dst.data_ptr(), lse=self.lse.data_ptr() if lse else None,
            first=None if first is None else self.x["first"].data_ptr(),
            slopes=None if slopes is None else self.x["slopes"].data_ptr(), rows=B.rows, n_head=B.H,
            q_stride=B.q_stride, page_size=B.page, window=window, scale=scale, softcap=softcap,
            ws=None if ws is None else ws.data_ptr(),
            ws_bytes=0 if ws is None else ws.numel() * ws.element_size())

    def call(self, name, args, chunks, stream=None):
        fn = getattr(self.t.lib(), name + ("_q8" if self.B.q8 else ""))
        self.t.check(fn(self.layer, args, chunks, len(self.B.sizes), stream))

    def attn(self, scale, prefix=None, **kw):
        self.call("tl_attn_chunks", self.attn_args(scale, **kw), self.chunks(prefix))
        self.T.cuda.synchronize()
        return self.dst.cpu().numpy().astype(np.float64), self.lse.cpu().numpy().astype(np.float64)


def rel(a, b):
    return np.linalg.norm(a - b) / max(np.linalg.norm(b), 1e-300)


def real_rows(B):
    m = np.zeros(B.rows, dtype=bool)
    for i in B.live:
        m[B.row[i]:B.row[i] + B.sizes[i][1]] = True
    return m


def check_attn(B, got, ref):
    dst, lse = got
    want, sums, tol = ref
    m, W = real_rows(B), B.H * B.D
    assert np.all(dst[~m] == 7.5) and np.all(dst[:, W:] == 7.5) and np.all(lse[~m] == 7.5)
    assert np.isfinite(dst[m][:, :W]).all()
    assert rel(dst[m][:, :W], want[m]) <= tol
    # a wrong column or row shows here, however many others there are
    assert np.abs(dst[m][:, :W] - want[m]).max() <= 40 * tol * max(1.0, np.abs(want[m]).max())
    empty = np.isneginf(sums[m])
    assert np.array_equal(np.isneginf(lse[m]), empty)
    assert np.all(dst[m][:, :W].reshape(-1, B.H, B.D)[empty] == 0)
    # an absolute score error is an absolute error of the log sum
    assert np.abs(lse[m][~empty] - sums[m][~empty]).max(initial=0) <= tol + 4 * R.U24 * np.abs(sums[m][~empty]).max(initial=0)


ATTN = [
    # shape, sizes (pos, n), page, q8, options
    ("8b", [(0, 1)], 16, False, {}),
    ("8b", [(31, 1), (0, 1), (64, 1), (777, 1)], 16, False, {}),
    ("qwen", [(5, 3), (40, 0), (200, 1), (33, 9)], 1, False, dict(pad=32)),
    ("gemma", [(100, 5), (0, 7)], 32, False, dict(window=20)),
    ("1b", [(63, 2), (64, 33)], 64, False, dict(softcap=15.0)),
    ("mha", [(95, 1), (17, 20)], 16, False, dict(slopes=True)),
    ("mqa", [(50, 3), (0, 2)], 2, False, dict(softcap=8.0, slopes=True)),
    ("8b", [(0, 70), (90, 40)], 16, False, dict(first=True, gap=1)),
    ("gemma", [(0, 45), (30, 50)], 16, False, dict(prefix=[17, 64], window=9)),
    ("qwen", [(3000, 1), (17, 2)], 16, False, dict(softcap=30.0)),
    ("1b", [(5000, 4)], 16, False, dict(window=700, prefix=[40])),
    ("8b", [(31, 1), (130, 2), (0, 1)], 16, True, {}),
    ("gemma", [(100, 5), (0, 7)], 32, True, dict(window=20, softcap=20.0)),
    ("1b", [(63, 2), (64, 33)], 1, True, dict(slopes=True)),
    ("mha", [(10, 40)], 16, True, dict(first=True, prefix=[30])),
    ("qwen", [(2500, 2)], 16, True, {}),
    ("8b", [(40, 150), (300, 1), (0, 260)], 16, False, {}),
    ("1b", [(0, 300)], 16, False, dict(first=True, softcap=30.0, slopes=True)),
    ("gemma", [(77, 140)], 16, False, dict(window=64)),
    ("8b", [(513, 129)], 16, True, dict(window=300, prefix=[600])),
    ("mqa", [(11, 60)], 16, False, {}),
    ("kv12", [(100, 1), (3, 2), (70, 40)], 16, False, dict(window=33)),
    ("kv3", [(300, 1), (3, 2), (70, 4)], 16, True, dict(softcap=10.0)),
    ("mqa40", [(40, 1), (3, 2)], 16, False, dict(prefix=[9, 2])),
    ("8b", [(40, 60), (700, 1), (0, 3), (1300, 2)], 16, True, dict(slopes=True)),
    ("1b", [(0, 200), (2000, 1), (31, 16)], 16, False, dict(first=True, window=90)),
    ("gemma", [(0, 1), (600, 70), (1200, 1)], 16, True, dict(prefix=[0, 300, 7])),
    ("qwen", [(700, 300)], 64, False, dict(window=200, prefix=[100])),
    ("8b", [(0, 400)], 16, False, {}),
    ("mha", [(1000, 140), (20, 17)], 1, True, dict(softcap=20.0, first=True)),
]


def options(B, opt):
    kw = {k: v for k, v in opt.items() if k in ("window", "softcap")}
    if opt.get("slopes"):
        kw["slopes"] = (2.0 ** (-8.0 * np.arange(1, B.H + 1) / B.H)).astype(np.float32)
    if opt.get("first"):
        # documents of several lengths; a few rows whose document begins behind them see nothing
        f = np.zeros(B.rows, dtype=np.uint32)
        for i in B.live:
            pos, n = B.sizes[i]
            p = np.arange(pos, pos + n)
            f[B.row[i]:B.row[i] + n] = p - p % 23
            f[B.row[i] + n // 2] = pos + n // 2 + 1
            f[B.row[i] + n - 1] = 0xffffffff
        kw["first"] = f
    return kw


@pytest.mark.parametrize("shape,sizes,page,q8,opt", ATTN)
def test_attn_chunks(T, shape, sizes, page, q8, opt):
    B = R.Batch(len(sizes) * 7 + page, SHAPES[shape], sizes, page, q8, pad=opt.get("pad", 0), gap=opt.get("gap", 0))
    kw = options(B, opt)
    scale = 1 / math.sqrt(B.D)
    D = Dev(T, B)
    check_attn(B, D.attn(scale, prefix=opt.get("prefix"), **kw),
               R.attn(B, scale, prefix=opt.get("prefix"), **kw))


def test_attn_chunks_null_table_and_no_lse(T):
    B = R.Batch(3, SHAPES["8b"], [(70, 6)], 16)
    B.tables = [None]
    D = Dev(T, B)
    D.call("tl_attn_chunks", D.attn_args(0.1, lse=False), D.chunks())
    T.cuda.synchronize()
    want, _, tol = R.attn(B, 0.1)
    assert rel(D.dst.cpu().numpy()[:6], want[:6]) <= tol
    assert np.all(D.lse.cpu().numpy() == 7.5)


@pytest.mark.parametrize("n,pos", [(1, 40), (3, 90), (150, 90)])
@pytest.mark.parametrize("q8", [False, True])
def test_attn_chunks_unseen_rows_hold_anything(T, q8, n, pos):
    """Infinities and NaN in rows that a query does not see (later rows of the chunk, other
    documents, rows behind the window, rows behind the end of a page) leave no trace in it."""
    B = R.Batch(5, SHAPES["8b"], [(pos, n), (13, n)], 16, q8)
    first = np.zeros(B.rows, dtype=np.uint32)
    for i in (0, 1):
        p = np.arange(*np.cumsum(B.sizes[i]))
        first[B.row[i]:B.row[i] + n] = np.where(p % 3 == 0, p - np.minimum(p, 4), 3)
    scale = 1 / math.sqrt(B.D)
    want = R.attn(B, scale, first=first, window=30)
    # poison: for the chunk's rows but the last, K and V of the last position; all of rows 0..2;
    # everything that no position maps to
    B2 = R.Batch(5, SHAPES["8b"], [(pos, n), (13, n)], 16, q8)
    mapped = np.concatenate([B2.phys(i, np.arange(sum(B2.sizes[i]))) for i in (0, 1)])
    spoil = np.setdiff1d(np.arange(B2.cap), mapped)
    gone = [B2.phys(i, np.arange(3)) for i in (0, 1)]
    for x in ("k", "v"):
        a = getattr(B2, x + "s" if q8 else x)
        a[:, spoil] = np.nan
        a[:, spoil[::2]] = np.inf
        last = B2.phys(0, pos + n - 1)
        if n > 1:
            a[:, last, 0] = np.nan
            a[:, last, 1] = -np.inf
    p0 = np.arange(pos, pos + n)
    hidden = first[:n] == 3
    D = Dev(T, B2)
    dst, lse = D.attn(scale, first=first, window=30)
    ok = real_rows(B)
    if n > 1:
        ok[n - 1] = False      # sees the spoilt position
    assert np.isfinite(dst[ok]).all()
    if n > 1:
        assert not np.isfinite(dst[n - 1]).all()
    assert rel(dst[ok], want[0][ok]) <= want[2]
    assert np.abs(lse[ok] - want[1][ok]).max() <= want[2] + 4 * R.U24 * 10


@pytest.mark.parametrize("n", [2, 100])
def test_attn_chunks_bad_pages_are_not_seen(T, n):
    B = R.Batch(9, SHAPES["1b"], [(60, n), (20, 1)], 16)
    B.tables[0][1] = 0xffffffff
    B.tables[0][2] = B.cap // 16
    B.tables[1][:] = 1 << 28
    scale = 1 / math.sqrt(B.D)
    D = Dev(T, B)
    check_attn(B, D.attn(scale), R.attn(B, scale))


def test_attn_chunks_many_chunks(T):
    """More chunks than one launch takes, some without rows, their rows in another order."""
    rng = np.random.default_rng(1)
    sizes = [(int(rng.integers(0, 90)), int(rng.integers(0, 4))) for _ in range(75)]
    B = R.Batch(11, (8, 2, 64), sizes, 16)
    order = rng.permutation(75)
    at = 0
    for i in order:
        B.row[i] = at
        at += sizes[i][1]
    D = Dev(T, B)
    check_attn(B, D.attn(0.125), R.attn(B, 0.125))


@pytest.mark.parametrize("mag", [1e-30, 1e-3, 1.0, 3e4])
def test_attn_chunks_query_ranges(T, mag):
    """Queries of any size: the row's power of two keeps both halves of the pair in range."""
    B = R.Batch(13, SHAPES["8b"], [(200, 3)], 16)
    B.q *= np.float32(mag)
    scale = 1 / (mag * math.sqrt(B.D))
    D = Dev(T, B)
    check_attn(B, D.attn(scale), R.attn(B, scale))


def ws_of(T, D, args, chunks):
    need = ctypes.c_uint64()
    B = D.B
    D.t.check(D.t.lib().tl_attn_chunks_ws(B.KV, B.D, args, chunks, len(B.sizes), ctypes.byref(need)))
    return T.zeros(need.value, dtype=T.uint8, device="cuda")


@pytest.mark.parametrize("q8", [False, True])
def test_attn_chunks_repeats_and_graphs(T, q8):
    """Split launches give the same bits every time: eagerly, with a workspace of their own, and
    replayed from two graphs with eager work between; a captured call without one is refused."""
    B = R.Batch(17, SHAPES["qwen"], [(4000, 1), (900, 3), (20, 60)], 16, q8)
    D = Dev(T, B)
    scale = 1 / math.sqrt(B.D)
    base = D.attn(scale)
    check_attn(B, base, R.attn(B, scale))
    for _ in range(3):
        D.dst.fill_(7.5)
        again = D.attn(scale)
        assert all(np.array_equal(a, b) for a, b in zip(base, again))
    ch = D.chunks()
    wss = [ws_of(T, D, D.attn_args(scale), ch) for _ in range(2)]
    graphs = []
    s = T.cuda.Stream()
    for ws in wss:
        g = T.cuda.CUDAGraph()
        with T.cuda.graph(g, stream=s):
            h = D.t.stream_handle(s)
            D.call("tl_attn_chunks", D.attn_args(scale, ws=ws), ch, h)
        graphs.append(g)
    for _ in range(3):
        for g in graphs:
            D.dst.fill_(7.5)
            D.lse.fill_(7.5)
            g.replay()
            T.cuda.synchronize()
            assert np.array_equal(base[0], D.dst.cpu().numpy().astype(np.float64))
            assert np.array_equal(base[1], D.lse.cpu().numpy().astype(np.float64))
        assert all(np.array_equal(a, b) for a, b in zip(base, D.attn(scale)))
    g = T.cuda.CUDAGraph()
    with T.cuda.graph(g, stream=s):
        with pytest.raises(D.t.TlError, match="workspace"):
            D.call("tl_attn_chunks", D.attn_args(scale), ch, D.t.stream_handle(s))
        D.dst.fill_(1.0)


@pytest.mark.parametrize("shape,sizes,q8,opt", [
    ("gemma", [(5000, 8)], False, {}),
    ("gemma", [(9000, 1), (4000, 3)], True, dict(softcap=30.0)),
    ("qwen", [(6001, 2)], False, dict(slopes=True)),
    ("qwen", [(9000, 1)], True, dict(first=True)),
    ("1b", [(12000, 4)], False, dict(window=9000, prefix=[50])),
    ("mqa", [(2500, 2)], False, {}),
])
def test_attn_chunks_many_splits(T, shape, sizes, q8, opt):
    """One session whose keys are dealt out to many workgroups: joined in two steps, with the same
    bits every time, and every counter of the workspace back at zero."""
    B = R.Batch(23, SHAPES[shape], sizes, 16, q8)
    D = Dev(T, B)
    scale = 1 / math.sqrt(B.D)
    kw = options(B, opt)
    base = D.attn(scale, prefix=opt.get("prefix"), **kw)
    check_attn(B, base, R.attn(B, scale, prefix=opt.get("prefix"), **kw))
    ws = ws_of(T, D, D.attn_args(scale, **kw), D.chunks(opt.get("prefix")))
    for _ in range(3):
        D.dst.fill_(7.5)
        again = D.attn(scale, prefix=opt.get("prefix"), ws=ws, **kw)
        assert all(np.array_equal(a, b) for a, b in zip(base, again))
        assert not ws[:65536].any()


def test_attn_chunks_two_streams(T):
    """Calls on two streams at once do not share partials."""
    scale = 1 / math.sqrt(128)
    Bs = [R.Batch(19 + k, SHAPES["qwen"], [(3000 + 500 * k, 2)], 16) for k in range(2)]
    Ds = [Dev(T, B) for B in Bs]
    base = [D.attn(scale) for D in Ds]
    streams = [T.cuda.Stream(), T.cuda.Stream()]
    for D in Ds:
        D.dst.zero_()
    T.cuda.synchronize()
    args = [(D.attn_args(scale), D.chunks()) for D in Ds]
    for _ in range(20):
        for D, s, (a, c) in zip(Ds, streams, args):
            D.call("tl_attn_chunks", a, c, D.t.stream_handle(s))
    T.cuda.synchronize()
    for D, b in zip(Ds, base):
        assert np.array_equal(D.dst.cpu().numpy()[:2], b[0][:2].astype(np.float32))


# ---- weight ------------------------------------------------------------------------


@pytest.mark.parametrize("shape,sizes,page,q8,opt", ATTN)
def test_attn_weight(T, shape, sizes, page, q8, opt):
    B = R.Batch(len(sizes) * 7 + page, SHAPES[shape], sizes, page, q8, pad=opt.get("pad", 0), gap=opt.get("gap", 0))
    kw = options(B, opt)
    scale = 1 / math.sqrt(B.D)
    D = Dev(T, B)
    D.attn(scale, prefix=opt.get("prefix"), **kw)
    base = [B.rng.random(p + n + 5).astype(np.float32) for p, n in sizes]
    w = [T.from_numpy(b).cuda() for b in base]
    D.call("tl_attn_weight", D.attn_args(scale, **kw), D.chunks(opt.get("prefix"), w))
    T.cuda.synchronize()
    want, tol = R.weight(B, D.lse.cpu().numpy(), scale, prefix=opt.get("prefix"), **kw)
    for i, (p, n) in enumerate(sizes):
        got = w[i].cpu().numpy()
        assert np.array_equal(got[p + n:], base[i][p + n:])
        if not n:
            assert np.array_equal(got, base[i])
            continue
        # each addend within tol of itself; the sums of N of them and of the base to N roundings,
        # taken as 2 sqrt(N) units
        N = n * B.H
        bound = (tol + 2 * math.sqrt(N) * R.U24) * want[i] + 2 * R.U24 * (base[i][:p + n] + want[i])
        assert np.all(np.abs(got[:p + n] - base[i][:p + n] - want[i]) <= bound + 1e-30)
    # the same bits again
    w2 = [T.from_numpy(b).cuda() for b in base]
    D.call("tl_attn_weight", D.attn_args(scale, **kw), D.chunks(opt.get("prefix"), w2))
    T.cuda.synchronize()
    assert all(T.equal(a, b) for a, b in zip(w, w2))


def mixed_batch(seed):
    """A batch of any shapes, lengths and masks together."""
    r = np.random.default_rng(1000 + seed)
    shape = list(SHAPES)[r.integers(len(SHAPES))]
    top = int(r.choice([3, 40, 150]))
    sizes = [(int(r.choice([0, r.integers(1, 70), r.integers(70, 900), r.integers(900, 2500)])),
              int(r.choice([0, 1, 1, r.integers(1, 1 + top)]))) for _ in range(r.integers(1, 7))]
    if not any(n for _, n in sizes):
        sizes[0] = (sizes[0][0], 1)
    opt = {}
    if r.random() < 0.4:
        opt["window"] = int(r.integers(1, 600))
    if r.random() < 0.4:
        opt["prefix"] = [int(r.integers(0, p + n + 40)) for p, n in sizes]
    if r.random() < 0.3:
        opt["softcap"] = float(r.uniform(2, 40))
    if r.random() < 0.3:
        opt["slopes"] = True
    if r.random() < 0.4:
        opt["first"] = True
    return shape, sizes, int(r.choice([1, 2, 16, 64])), bool(r.random() < 0.4), opt


@pytest.mark.parametrize("seed", range(40))
def test_mixed_batches(T, seed):
    """Attention and weight of batches whose shapes, lengths and masks come together by chance."""
    shape, sizes, page, q8, opt = mixed_batch(seed)
    test_attn_chunks(T, shape, sizes, page, q8, opt)
    test_attn_weight(T, shape, sizes, page, q8, opt)


def test_attn_weight_unseen_rows_hold_anything(T):
    B = R.Batch(23, SHAPES["8b"], [(40, 3)], 16)
    last = B.phys(0, 42)
    mapped = B.phys(0, np.arange(43))
    D = Dev(T, B)
    D.attn(0.1, first=np.array([2, 2, 0xffffffff, 0, 0], dtype=np.uint32))
    lse = D.lse.cpu().numpy()
    B.k[:, np.setdiff1d(np.arange(B.cap), mapped)] = np.nan
    B.k[:, B.phys(0, np.array([0, 1, 42]))] = np.inf
    D.put("k", B.k)
    D.layer.k = D.x["k"].data_ptr()
    w = [T.zeros(43, device="cuda")]
    D.call("tl_attn_weight", D.attn_args(0.1, first=np.array([2, 2, 0xffffffff, 0, 0], dtype=np.uint32)),
           D.chunks(None, w))
    T.cuda.synchronize()
    got = w[0].cpu().numpy()
    assert np.isfinite(got).all() and np.all(got[[0, 1, 42]] == 0)
    assert abs(got.sum() - 2 * B.H) < 1e-3


@pytest.mark.parametrize("q8", [False, True])
def test_attn_and_weight_share_a_workspace_in_a_graph(T, q8):
    """One workspace for the attention and the weight of a step, captured together and replayed
    with eager calls between: every replay equals the eager step."""
    B = R.Batch(37, SHAPES["8b"], [(2500, 1), (300, 70), (40, 3)], 16, q8)
    D = Dev(T, B)
    scale = 1 / math.sqrt(B.D)
    w = [T.zeros(p + n, device="cuda") for p, n in B.sizes]
    ch = D.chunks(weight=w)
    ws = ws_of(T, D, D.attn_args(scale), ch)
    args = D.attn_args(scale, ws=ws)
    D.attn(scale)
    D.call("tl_attn_weight", D.attn_args(scale), ch)
    T.cuda.synchronize()
    base = [x.clone() for x in w]
    out = D.dst.clone()
    s = T.cuda.Stream()
    g = T.cuda.CUDAGraph()
    with T.cuda.graph(g, stream=s):
        h = D.t.stream_handle(s)
        D.call("tl_attn_chunks", args, ch, h)
        D.call("tl_attn_weight", args, ch, h)
    for _ in range(3):
        for x in w + [D.dst, D.lse]:
            x.zero_()
        g.replay()
        T.cuda.synchronize()
        m = real_rows(B)
        assert all(T.equal(a, b) for a, b in zip(w, base))
        assert np.array_equal(D.dst.cpu().numpy()[m], out.cpu().numpy()[m])
        D.attn(scale)
    with T.cuda.graph(T.cuda.CUDAGraph(), stream=s):
        with pytest.raises(D.t.TlError, match="workspace"):
            D.call("tl_attn_weight", D.attn_args(scale), ch, D.t.stream_handle(s))
        D.dst.fill_(1.0)


@pytest.mark.parametrize("n", [1, 60])
def test_pool_of_four_gib_per_head(T, n):
    """Rows at the end of the largest pool that a layer may have: offsets within a head pass 31
    bits, the heads' bases 32."""
    H, KV, Dm = 4, 2, 128
    cap = (1 << 32) // (Dm * 2) - 16
    sizes = [(90, n)]
    B = R.Batch(41, (H, KV, Dm), sizes, 16, spare=0)
    pages = -(-(90 + n) // 16)
    k = T.empty((KV, cap, Dm), dtype=T.float16, device="cuda")
    v = T.empty_like(k)
    D = Dev(T, B)
    small, B.cap = B.tables[0].copy(), cap
    B.tables[0] = (cap // 16 - 1 - np.arange(pages)).astype(np.uint32)
    far = T.from_numpy(B.phys(0, np.arange(90 + n))).cuda()
    near = T.from_numpy((small[np.arange(90 + n) // 16].astype(np.int64) * 16 + np.arange(90 + n) % 16)).cuda()
    k[:, far], v[:, far] = D.x["k"][:, near], D.x["v"][:, near]
    D.tab = [T.from_numpy(B.tables[0].view(np.int32)).cuda()]
    D.layer = D.t.KvLayer(k.data_ptr(), v.data_ptr(), cap, KV, Dm, 0)
    B.tables[0], B.cap = small, pages * 16
    want = R.attn(B, 0.1)
    got = D.attn(0.1)
    check_attn(B, got, want)
    w = [T.zeros(90 + n, device="cuda")]
    D.call("tl_attn_weight", D.attn_args(0.1), D.chunks(weight=w))
    a = D.t.QkNormArgs(q=D.x["q"].data_ptr(), k=D.x["kin"].data_ptr(), v=D.x["vin"].data_ptr(),
                       q_out=D.dst.data_ptr(), eps=1e-6, rows=B.rows, n_head=H, q_stride=B.q_stride,
                       kv_stride=B.kv_stride, q_out_stride=B.q_stride, page_size=16)
    D.call("tl_qk_norm_append", a, D.chunks())
    T.cuda.synchronize()
    assert abs(float(w[0].sum()) - n * H) <= 1e-3 * n * H
    assert T.equal(v[:, far[90:]].cpu(), T.from_numpy(B.vin[:n].reshape(n, KV, Dm).transpose(1, 0, 2).astype(np.float16)))


# ---- norm + rotation + append --------------------------------------------------------


@pytest.mark.parametrize("shape,sizes,page,q8,rdim,neox,opt", [
    ("8b", [(0, 1)], 16, False, 128, 0, {}),
    ("8b", [(31, 3), (5, 0), (100, 20)], 16, False, 128, 1, dict(pad=32)),
    ("gemma", [(8190, 1), (100000, 2)], 16, False, 256, 1, {}),
    ("1b", [(7, 40)], 1, False, 64, 0, dict(place=True)),
    ("qwen", [(3, 5), (64, 1)], 16, False, 36, 1, dict(place=True)),
    ("qwen", [(3, 5)], 16, False, 34, 0, dict(skip=[1000000])),
    ("mqa", [(3, 5)], 4, False, 0, 0, dict(noweight=True)),
    ("8b", [(31, 3), (100, 20)], 16, True, 128, 0, {}),
    ("gemma", [(9, 2)], 16, True, 64, 1, {}),
    ("1b", [(9, 700), (3, 2)], 16, True, 64, 1, {}),
    ("mha", [(9, 400), (30, 300)], 16, False, 128, 1, {}),
])
def test_qk_norm_append(T, shape, sizes, page, q8, rdim, neox, opt):
    B = R.Batch(sum(map(sum, sizes)) + page, SHAPES[shape], sizes, page, q8, pad=opt.get("pad", 0))
    B.q[0, :B.D] = 0                                     # a head of zeros
    qw = (1 + 0.3 * B.rng.standard_normal(B.D)).astype(np.float32)
    kw = (1 + 0.3 * B.rng.standard_normal(B.D)).astype(np.float32)
    theta, eps = 1e6, 1e-5
    D = Dev(T, B)
    skip = opt.get("skip") or [0] * len(sizes)
    out = D.x["q"] if opt.get("place") else D.dst
    a = D.t.QkNormArgs(q=D.x["q"].data_ptr(), k=D.x["kin"].data_ptr(), v=D.x["vin"].data_ptr(),
                       q_out=out.data_ptr(),
                       q_weight=None if opt.get("noweight") else D.put("qw", qw).data_ptr(),
                       k_weight=None if opt.get("noweight") else D.put("kw", kw).data_ptr(),
                       eps=eps, rows=B.rows, n_head=B.H, q_stride=B.q_stride, kv_stride=B.kv_stride,
                       q_out_stride=B.q_stride, page_size=page, rope=D.t.RopeParams(rdim, theta, neox))
    if opt.get("noweight"):
        qw = kw = None
    D.call("tl_qk_norm_append", a, D.chunks(skip=skip))
    T.cuda.synchronize()
    got, m = out.cpu().numpy(), real_rows(B)
    W = B.H * B.D
    before = B.q if opt.get("place") else np.full_like(B.q, 7.5)
    assert np.array_equal(got[~m], before[~m]) and np.array_equal(got[:, W:], before[:, W:])
    kc, vc = B.k.copy(), B.v.copy()
    cache = {f: D.x[f].cpu().numpy() for f in ("k", "v") + (("ks", "vs") if q8 else ())}
    touched = np.zeros(B.cap, dtype=bool)
    # an element's error: the norm's factor (sum of squares, root, two products: 8 units), the
    # rotation (angle to 2^-23 of a turn's 2 pi, sine and cosine and three roundings: 16 units),
    # relative to the pair's size
    for i in B.live:
        pos, n = sizes[i]
        r = slice(B.row[i], B.row[i] + n)
        p = np.arange(pos, pos + n) + skip[i]
        q = R.rotated(R.normed(B.q[r, :W].reshape(n, B.H, B.D), qw, eps), p, rdim, theta, neox)
        big = np.abs(q).max()
        assert np.abs(got[r, :W].reshape(n, B.H, B.D) - q).max() <= 24 * R.U24 * math.sqrt(2) * big
        k = R.rotated(R.normed(B.kin[r, :B.KV * B.D].reshape(n, B.KV, B.D), kw, eps), p, rdim, theta, neox)
        v = B.vin[r, :B.KV * B.D].reshape(n, B.KV, B.D).astype(np.float64)
        at = B.phys(i, np.arange(pos, pos + n))
        touched[at] = True
        for x, y in (("k", k), ("v", v)):
            c = cache[x][:, at].transpose(1, 0, 2).astype(np.float64)
            if q8:
                s = cache[x + "s"][:, at].transpose(1, 0, 2).astype(np.float64)
                c = (c.reshape(*s.shape, 32) * s[..., None]).reshape(c.shape)
                amax = np.abs(y.reshape(n, B.KV, -1, 32)).max(-1)
                # half a step of the quantizer, and the scale's rounding to f16 (2^-11, and half
                # of the smallest step of f16) on values of up to 127 steps
                step = np.repeat(amax / 127 * (0.5 + 127 * 2.0 ** -11) + 127 * 2.0 ** -25, 32, -1).reshape(y.shape)
                assert np.all(np.abs(c - y) <= step * (1 + 1e-3) + 64 * R.U24 * np.abs(y).max())
            else:
                assert np.all(np.abs(c - y) <= 2.0 ** -11 * np.abs(y) * (1 + 1e-3) + 2.0 ** -25 + 24 * R.U24 * math.sqrt(2) * np.abs(y).max() * (x == "k"))
    for x in cache:
        assert np.array_equal(cache[x][:, ~touched].view(np.uint8), getattr(B, x)[:, ~touched].view(np.uint8))


def test_qk_norm_append_bad_pages(T):
    B = R.Batch(29, SHAPES["1b"], [(14, 4)], 16)
    B.tables[0][1] = B.cap // 16
    D = Dev(T, B)
    a = D.t.QkNormArgs(q=D.x["q"].data_ptr(), k=D.x["kin"].data_ptr(), v=D.x["vin"].data_ptr(),
                       q_out=D.dst.data_ptr(), eps=1e-6, rows=B.rows, n_head=B.H, q_stride=B.q_stride,
                       kv_stride=B.kv_stride, q_out_stride=B.q_stride, page_size=16)
    D.call("tl_qk_norm_append", a, D.chunks())
    T.cuda.synchronize()
    k = D.x["k"].cpu().numpy()
    at = B.phys(0, np.array([14, 15]))
    rest = np.setdiff1d(np.arange(B.cap), at)
    assert np.array_equal(k[:, rest], B.k[:, rest]) and not np.array_equal(k[:, at], B.k[:, at])


# ---- eviction ----------------------------------------------------------------------


def run_evict(T, w, tables, page, lens, keeps, holds):
    import tlkv
    dev = lambda a: T.from_numpy(np.ascontiguousarray(a)).cuda()
    ws = [dev(x) for x in w]
    tabs = [None if t is None else dev(t.view(np.int32)) for t in tables]
    out = [[T.full((k + 1,), -7, dtype=T.int32, device="cuda"), T.full((k + 1,), -7, dtype=T.int32, device="cuda"),
            T.full((n - k + 1,), -7, dtype=T.int32, device="cuda"), T.full((k + 1,), -7.0, device="cuda")]
           for n, k in zip(lens, keeps)]
    seqs = (tlkv.EvictSeq * len(lens))(*[
        tlkv.EvictSeq(weight=ws[i].data_ptr(), pages=None if tabs[i] is None else tabs[i].data_ptr(),
                      len=lens[i], keep=keeps[i], sink=holds[i][0], recent=holds[i][1], page_size=page,
                      kept=out[i][0].data_ptr(), rows=out[i][1].data_ptr(), freed=out[i][2].data_ptr(),
                      weight_out=out[i][3].data_ptr()) for i in range(len(lens))])
    tlkv.check(tlkv.lib().tl_kv_evict(seqs, len(lens), None))
    T.cuda.synchronize()
    return [[x.cpu().numpy() for x in o] for o in out]


@pytest.mark.parametrize("page", [1, 16])
@pytest.mark.parametrize("lens,keeps,holds", [
    ([1], [1], [(0, 0)]),
    ([2, 65], [1, 64], [(0, 1), (0, 0)]),
    ([1000, 1023, 1024, 1025], [1, 1000, 512, 1025], [(1, 0), (4, 100), (0, 0), (25, 1000)]),
    ([5000], [700], [(4, 696)]),
    ([16384, 16385], [9000, 3], [(0, 0), (1, 1)]),
    ([100003], [40001], [(16, 500)]),
    ([40000] * 3 + [17] * 20, [13] * 3 + [5] * 20, [(2, 3)] * 23),
])
def test_kv_evict(T, lens, keeps, holds, page):
    rng = np.random.default_rng(sum(lens))
    w, tables = [], []
    for i, n in enumerate(lens):
        x = np.round(np.exp(2 * rng.standard_normal(n)) * 4).astype(np.float32) / 4      # many ties
        if i % 3 == 1:
            x = rng.standard_normal(n).astype(np.float32)
        sp = np.array([np.nan, np.inf, -np.inf, -0.0, 0.0, 1e-45, -1e-45, np.nan], dtype=np.float32)
        if n > 40:
            x[rng.permutation(n)[:24]] = np.tile(sp, 3)
        w.append(x)
        tables.append(rng.permutation(4 * n + 64)[:-(-n // page)].astype(np.uint32) if i % 4 != 3 else None)
    got = run_evict(T, w, tables, page, lens, keeps, holds)
    for i, n in enumerate(lens):
        kept, gone = R.evict(w[i], n, keeps[i], *holds[i])
        row = lambda j: j if tables[i] is None else tables[i][j // page].astype(np.int64) * page + j % page
        k, r, f, o = got[i]
        assert np.array_equal(k[:-1], kept) and np.array_equal(r[:-1], row(kept))
        assert np.array_equal(f[:-1], row(gone))
        assert np.array_equal(o[:-1].view(np.uint32), w[i][kept].view(np.uint32))
        assert k[-1] == r[-1] == f[-1] == -7 and o[-1] == -7.0


@pytest.mark.parametrize("lens", [[9000, 100, 1, 8192, 2049], [1, 8193], [30, 40] * 7 + [20000, 8200],
                                  [30, 40] * 8 + [20000], [5, 2048, 70000, 2047, 8191]])
def test_kv_evict_short_beside_long(T, lens):
    """Short sessions in the long ones' launches, where there is room, and beside them."""
    test_kv_evict(T, lens, [n // 3 + 1 for n in lens], [(min(n // 9, 4), min(n // 9, 100)) for n in lens], 16)


def test_kv_evict_between_split_attention(T):
    """Long sessions, more than one launch takes, beside short ones, and attention with many splits
    before and after on the same stream's workspace: each call gives what it gives alone."""
    rng = np.random.default_rng(4)
    lens = [8193 + 1111 * i if i % 5 else 200 + i for i in range(24)]
    keeps = [n // 3 + 1 for n in lens]
    w = [rng.standard_normal(n).astype(np.float32) for n in lens]
    B = R.Batch(5, SHAPES["gemma"], [(5000, 8)], 16, False)
    D = Dev(T, B)
    base = D.attn(1 / 16)
    for _ in range(2):
        got = run_evict(T, w, [None] * 24, 1, lens, keeps, [(2, 50)] * 24)
        for i, n in enumerate(lens):
            kept, gone = R.evict(w[i], n, keeps[i], 2, 50)
            assert np.array_equal(got[i][0][:-1], kept) and np.array_equal(got[i][2][:-1], gone)
        assert all(np.array_equal(a, b) for a, b in zip(base, D.attn(1 / 16)))


@pytest.mark.parametrize("value", [0.0, np.nan, np.inf, -np.inf])
def test_kv_evict_all_alike(T, value):
    """Equal weights: the lower positions stay."""
    n, keep = 3000, 1001
    got = run_evict(T, [np.full(n, value, dtype=np.float32)], [None], 1, [n], [keep], [(3, 10)])[0]
    assert np.array_equal(got[0][:-1], np.concatenate([np.arange(keep - 10), np.arange(n - 10, n)]))


# ---- together ------------------------------------------------------------------------


@pytest.mark.parametrize("q8", [False, True])
def test_prompt_evict_decode(T, q8):
    """Two sessions read a prompt in chunks, gather the weight of their positions, are cut back,
    and go on decoding over what is left: norm and append, attention, weight, eviction as a server
    runs them, against the same steps in 64 bits (over the cache rows that the device holds)."""
    import tlkv
    H, KV, D = 8, 2, 64
    B = R.Batch(31, (H, KV, D), [(0, 40), (0, 25)], page=1, q8=q8, spare=20)
    scale, theta, eps = 1 / 8, 1e4, 1e-6
    spare = np.setdiff1d(np.arange(B.cap), np.concatenate(B.tables)).astype(np.uint32)
    # tables long enough for the tokens to come
    B.tables = [np.concatenate([t, spare[8 * i:8 * i + 8]]) for i, t in enumerate(B.tables)]
    total = [np.zeros(48, dtype=np.float64), np.zeros(33, dtype=np.float64)]
    Dv = Dev(T, B)
    w = [T.zeros(48, device="cuda"), T.zeros(33, device="cuda")]
    qw = Dv.put("qw", (1 + 0.1 * B.rng.standard_normal(D)).astype(np.float32))
    skip = [0, 0]

    def step(sizes):
        rows = sum(n for _, n in sizes)
        B.sizes, B.row, B.rows = sizes, [0, sizes[0][1]], rows
        B.live = [i for i, (_, n) in enumerate(sizes) if n]
        B.q = raw = (2 * B.rng.standard_normal((rows, H * D))).astype(np.float32)
        kin = B.rng.standard_normal((rows, KV * D)).astype(np.float32)
        vin = B.rng.standard_normal((rows, KV * D)).astype(np.float32)
        for f, x in (("q", raw), ("kin", kin), ("vin", vin)):
            Dv.put(f, x)
        Dv.tab = [T.from_numpy(t.view(np.int32)).cuda() for t in B.tables]
        Dv.dst = T.zeros((rows, H * D), device="cuda")
        Dv.lse = T.zeros((rows, H), device="cuda")
        a = tlkv.QkNormArgs(q=Dv.x["q"].data_ptr(), k=Dv.x["kin"].data_ptr(), v=Dv.x["vin"].data_ptr(),
                            q_out=Dv.x["q"].data_ptr(), q_weight=qw.data_ptr(), eps=eps, rows=rows, n_head=H,
                            q_stride=H * D, kv_stride=KV * D, q_out_stride=H * D, page_size=1,
                            rope=tlkv.RopeParams(D, theta, 1))
        ch = Dv.chunks(weight=w, skip=skip)
        Dv.call("tl_qk_norm_append", a, ch)
        at = Dv.attn_args(scale, softcap=20.0)
        Dv.call("tl_attn_chunks", at, ch)
        Dv.call("tl_attn_weight", at, ch)
        T.cuda.synchronize()
        B.q = Dv.x["q"].cpu().numpy()
        for i in B.live:
            p, n = sizes[i]
            r = slice(B.row[i], B.row[i] + n)
            want = R.rotated(R.normed(raw[r].reshape(n, H, D), qw.cpu().numpy(), eps),
                             np.arange(p, p + n) + skip[i], D, theta, 1)
            assert rel(B.q[r].reshape(n, H, D), want) <= 16 * R.U24
        for f in ("k", "v") + (("ks", "vs") if q8 else ()):
            setattr(B, f, Dv.x[f].cpu().numpy())
        want, sums, tol = R.attn(B, scale, softcap=20.0)
        got = Dv.dst.cpu().numpy()
        assert rel(got, want) <= tol
        ww, wt = R.weight(B, Dv.lse.cpu().numpy(), scale, softcap=20.0)
        for i in B.live:
            total[i][:ww[i].size] += ww[i]
            assert np.abs(w[i].cpu().numpy()[:ww[i].size] - total[i][:ww[i].size]).max() <= 8 * (wt + 64 * R.U24) * total[i].max()

    step([(0, 20), (0, 25)])
    step([(20, 20), (25, 1)])
    lens, keeps, holds = [40, 26], [17, 26], [(2, 5), (0, 4)]
    host = [x.cpu().numpy() for x in w]
    got = run_evict(T, host, B.tables, 1, lens, keeps, holds)
    for i in (0, 1):
        kept, gone = R.evict(host[i], lens[i], keeps[i], *holds[i])
        assert np.array_equal(got[i][0][:-1], kept)
        # single-row pages: the kept rows are the new table, the freed ones go to its end
        free = np.concatenate([got[i][2][:-1], B.tables[i][lens[i]:].view(np.int32)])
        B.tables[i] = np.concatenate([got[i][1][:-1], free]).astype(np.uint32)
        new = np.zeros_like(host[i])
        new[:keeps[i]] = got[i][3][:-1]
        w[i] = T.from_numpy(new).cuda()
        total[i][:] = 0
        total[i][:keeps[i]] = new[:keeps[i]]
        skip[i] += lens[i] - keeps[i]
    for k in range(3):
        step([(17 + k, 1), (26 + k, 1)])


def test_kv_evict_captured(T):
    """A captured eviction (which takes no workspace) replays to the eager call's result, short
    and long, also with eager evictions on the same stream between."""
    import tlkv
    rng = np.random.default_rng(3)
    lens, keeps = [700, 30000], [300, 12000]
    w = [T.from_numpy(np.round(rng.standard_normal(n) * 8).astype(np.float32)).cuda() for n in lens]
    kept = [T.zeros(k, dtype=T.int32, device="cuda") for k in keeps]
    seqs = (tlkv.EvictSeq * 2)(*[
        tlkv.EvictSeq(weight=w[i].data_ptr(), len=lens[i], keep=keeps[i], sink=1, recent=9, page_size=1,
                      kept=kept[i].data_ptr()) for i in (0, 1)])
    s = T.cuda.Stream()
    h = tlkv.stream_handle(s)
    T.cuda.synchronize()
    g = T.cuda.CUDAGraph()
    with T.cuda.graph(g, stream=s):
        tlkv.check(tlkv.lib().tl_kv_evict(seqs, 2, h))
    want = [R.evict(x.cpu().numpy(), n, k, 1, 9)[0] for x, n, k in zip(w, lens, keeps)]
    for _ in range(3):
        for run in (g.replay, lambda: tlkv.check(tlkv.lib().tl_kv_evict(seqs, 2, h))):
            for x in kept:
                x.zero_()
            T.cuda.synchronize()
            run()
            T.cuda.synchronize()
            assert all(np.array_equal(x.cpu().numpy(), y) for x, y in zip(kept, want))
