"""Refusals of the calls on batches of chunks (include/tlkv.h): every rule that
the host can check is checked before anything reaches the device, so these run
without one.  Addresses are made up and never read."""
import ctypes

import pytest

import tlkv

P = 0x10000


def layer(**kw):
    a = dict(k=P, v=2 * P, cap=1024, n_kv_head=8, head_dim=128, ring=0)
    a.update(kw)
    return tlkv.KvLayer(**a)


def layer_q8(**kw):
    a = dict(k=P, v=2 * P, ks=3 * P, vs=4 * P, cap=1024, n_kv_head=8, head_dim=128, ring=0)
    a.update(kw)
    return tlkv.KvLayerQ8(**a)


def attn(**kw):
    a = dict(q=1 << 30, dst=1 << 31, lse=P, rows=64, n_head=32, q_stride=4096, page_size=16, scale=0.1)
    a.update(kw)
    return tlkv.ChunkAttnArgs(**a)


def norm(**kw):
    a = dict(q=1 << 30, k=5 * P, v=6 * P, q_out=1 << 31, eps=1e-6, rows=64, n_head=32, q_stride=4096,
             kv_stride=1024, q_out_stride=4096, page_size=16, rope=tlkv.RopeParams(128, 1e4, 0))
    a.update(kw)
    return tlkv.QkNormArgs(**a)


def chunks(*cs):
    full = [dict(dict(pages=P, pos=10, n=2, row=2 * i, weight=(64 + i) * P), **c) for i, c in enumerate(cs)]
    return (tlkv.Chunk * max(1, len(cs)))(*[tlkv.Chunk(**c) for c in full]), len(cs)


ONE = {}
CHUNKS = [
    ([dict(row=63)], -2), ([dict(row=0xffffffff)], -2), ([dict(pos=0x7fffffff)], -2),
    ([dict(pos=0xffffffff, n=1)], -2), ([dict(pos=0x7ffffff0, rope_skip=0x80000010)], -2),
    ([dict(pages=P + 2)], -1), ([dict(pages=None, pos=1023)], -2),
    ([dict(pages=None), dict()], -1), ([dict(), dict(row=1)], -1),
    ([dict(row=8), dict(row=0, n=9)], -1), ([dict(row=8), dict(row=4), dict(row=5)], -1),
]


@pytest.mark.parametrize("cs,code", CHUNKS)
@pytest.mark.parametrize("name", ["tl_qk_norm_append", "tl_attn_chunks", "tl_attn_weight"])
def test_chunks_refused(name, cs, code):
    L, (ch, n) = tlkv.lib(), chunks(*cs)
    a = norm() if name == "tl_qk_norm_append" else attn()
    assert getattr(L, name)(layer(), a, ch, n, None) == code
    assert getattr(L, name + "_q8")(layer_q8(), a, ch, n, None) == code
    assert L.tl_last_error()


@pytest.mark.parametrize("bad", [
    dict(q=None), dict(dst=None), dict(q=P + 4), dict(dst=P + 8), dict(lse=P + 2), dict(first=P + 1),
    dict(slopes=P + 3), dict(n_head=0), dict(n_head=12), dict(q_stride=4092), dict(q_stride=4098),
    dict(page_size=0), dict(page_size=24), dict(page_size=8192), dict(scale=0.0), dict(scale=-1.0),
    dict(scale=float("nan")), dict(scale=float("inf")), dict(softcap=-1.0), dict(softcap=float("nan")),
    dict(softcap=float("inf")), dict(softcap=1e-7), dict(ws=P + 8), dict(dst=1 << 30), dict(dst=(1 << 30) + 4096 * 16)])
def test_attn_args_refused(bad):
    L, (ch, n) = tlkv.lib(), chunks(ONE)
    assert L.tl_attn_chunks(layer(), attn(**bad), ch, n, None) == -1
    assert L.tl_attn_chunks_q8(layer_q8(), attn(**bad), ch, n, None) == -1


def test_lse_and_weight_apart():
    """Outputs that lie over another buffer of the call."""
    L, (ch, n) = tlkv.lib(), chunks(ONE)
    q, rows = 1 << 30, 64 * 4096 * 4
    for lse in (q, q + rows - 4, q - 64 * 32 * 4 + 4, 1 << 31, (1 << 31) + rows - 4):
        assert L.tl_attn_chunks(layer(), attn(lse=lse), ch, n, None) == -1
        assert L.tl_attn_chunks_q8(layer_q8(), attn(lse=lse), ch, n, None) == -1
    for w in (q, q + rows - 4, q - 44, P, P + 64 * 32 * 4 - 4):
        ch, n = chunks(dict(), dict(weight=w))
        assert L.tl_attn_weight(layer(), attn(), ch, n, None) == -1
        assert L.tl_attn_weight_q8(layer_q8(), attn(), ch, n, None) == -1


def test_many_heads_refused():
    """More q heads to a kv head than 32 bits hold columns of."""
    one = layer(n_kv_head=1, head_dim=64)
    L, (ch, n) = tlkv.lib(), chunks(dict(n=1, row=0))
    for name in ("tl_attn_chunks", "tl_attn_weight"):
        for heads in (1 << 16, (1 << 26) - 1):
            a = attn(rows=1, n_head=heads, q_stride=heads * 64, q=1 << 40, dst=1 << 45)
            assert getattr(L, name)(one, a, ch, n, None) == -2


def test_many_chunks_out_of_order():
    L = tlkv.lib()
    cs = [dict(row=3 * (i * 1237 % 4096), n=3, weight=P * (64 + i)) for i in range(4096)]
    for at, bad in ((17, dict(row=cs[4000]["row"] + 2)), (4095, dict(row=cs[9]["row"], n=1))):
        ch, n = chunks(*(cs[:at] + [dict(cs[at], **bad)] + cs[at + 1:]))
        assert L.tl_attn_chunks(layer(), attn(rows=3 * 4096 + 8, dst=1 << 45), ch, n, None) == -1


def test_attn_workspace_refused():
    L, (ch, n) = tlkv.lib(), chunks(dict(pos=5000, n=1))
    need = ctypes.c_uint64()
    assert L.tl_attn_chunks_ws(8, 128, attn(), ch, n, ctypes.byref(need)) == 0
    assert need.value > 64 << 10
    assert L.tl_attn_chunks(layer(), attn(ws=1 << 33, ws_bytes=need.value - 1), ch, n, None) == -2
    for args in ((0, 128), (8, 96), (5, 128)):
        assert L.tl_attn_chunks_ws(*args, attn(), ch, n, ctypes.byref(need)) == -1
    assert L.tl_attn_chunks_ws(8, 128, attn(), ch, n, None) == -1


@pytest.mark.parametrize("bad", [
    dict(q=None), dict(k=None), dict(v=None), dict(q_out=None), dict(k=P + 4), dict(q_weight=P + 4),
    dict(k_weight=P + 8), dict(n_head=0), dict(n_head=12), dict(q_stride=4092), dict(kv_stride=1020),
    dict(kv_stride=1026), dict(q_out_stride=4000), dict(page_size=3), dict(eps=-1.0), dict(eps=float("nan")),
    dict(eps=float("inf")), dict(rope=tlkv.RopeParams(130, 1e4, 0)), dict(rope=tlkv.RopeParams(63, 1e4, 0)),
    dict(rope=tlkv.RopeParams(64, 0.0, 0)), dict(rope=tlkv.RopeParams(64, float("inf"), 0)),
    dict(q_out=(1 << 30) + 16), dict(q_out=1 << 30, q_out_stride=4100), dict(q_out=5 * P, k=5 * P + 4096 * 8),
    dict(q_out=6 * P + 16), dict(q=1 << 30, q_stride=6144, q_out_stride=6144, q_out=(1 << 30) + 2064 * 4)])
def test_norm_args_refused(bad):
    L, (ch, n) = tlkv.lib(), chunks(ONE)
    assert L.tl_qk_norm_append(layer(), norm(**bad), ch, n, None) == -1
    assert L.tl_qk_norm_append_q8(layer_q8(), norm(**bad), ch, n, None) == -1


@pytest.mark.parametrize("bad", [dict(k=None), dict(head_dim=96), dict(cap=0), dict(ring=64), dict(v=P + 8)])
def test_layers_refused(bad):
    L, (ch, n) = tlkv.lib(), chunks(ONE)
    for name, a in (("tl_qk_norm_append", norm()), ("tl_attn_chunks", attn()), ("tl_attn_weight", attn())):
        assert getattr(L, name)(layer(**bad), a, ch, n, None) == -1
        assert getattr(L, name + "_q8")(layer_q8(**bad), a, ch, n, None) == -1
        assert getattr(L, name)(None, a, ch, n, None) == -1
        assert getattr(L, name)(layer(), None, ch, n, None) == -1
        assert getattr(L, name)(layer(), a, None, 1, None) == -1
        assert getattr(L, name)(layer(), a, ch, 5000, None) == -1


def test_weight_refused():
    L = tlkv.lib()
    for cs, a in (([dict(weight=None)], attn()), ([dict(weight=P + 2)], attn()), ([ONE], attn(lse=None)),
                  ([dict(), dict(weight=64 * P)], attn()), ([dict(), dict(weight=64 * P + 40)], attn()),
                  ([dict(), dict(weight=64 * P - 4)], attn())):
        ch, n = chunks(*cs)
        assert L.tl_attn_weight(layer(), a, ch, n, None) == -1
        assert L.tl_attn_weight_q8(layer_q8(), a, ch, n, None) == -1


def test_too_many_columns_refused():
    """Rows x gqa^2 past 32 bits: the kernels divide by multiplication."""
    L, (ch, n) = tlkv.lib(), chunks(dict(n=1 << 20, row=0))
    for name in ("tl_attn_chunks", "tl_attn_weight"):
        a = attn(rows=1 << 20, n_head=512, q_stride=65536, dst=1 << 45)
        assert getattr(L, name)(layer(), a, ch, n, None) == -2


def test_nothing_to_do():
    L, (ch, n) = tlkv.lib(), chunks(dict(n=0, row=99, weight=None))
    for name, a in (("tl_qk_norm_append", norm()), ("tl_attn_chunks", attn()), ("tl_attn_weight", attn())):
        for c, k in ((ch, n), (None, 0)):
            assert getattr(L, name)(layer(), a, c, k, None) == 0
            assert getattr(L, name + "_q8")(layer_q8(), a, c, k, None) == 0
    assert L.tl_kv_evict(None, 0, None) == 0


@pytest.mark.parametrize("bad", [
    dict(weight=None), dict(len=0), dict(keep=0), dict(keep=101), dict(sink=30, recent=21),
    dict(sink=0xffffffff, recent=2), dict(page_size=0), dict(page_size=12), dict(len=0x80000000),
    dict(kept=P + 2), dict(weight=P + 1), dict(weight_out=P), dict(kept=P + 396), dict(rows=2 * P + 20),
    dict(rows=4 * P + 100), dict(freed=4 * P), dict(weight_out=5 * P + 196)])
def test_evict_refused(bad):
    a = dict(weight=P, pages=2 * P, len=100, keep=50, sink=4, recent=10, page_size=16, kept=4 * P,
             rows=5 * P, freed=6 * P, weight_out=7 * P)
    a.update(bad)
    assert tlkv.lib().tl_kv_evict((tlkv.EvictSeq * 1)(tlkv.EvictSeq(**a)), 1, None) == -1
    two = (tlkv.EvictSeq * 2)(tlkv.EvictSeq(**dict(a, **dict(weight=P, len=100, keep=50, sink=0, recent=0, page_size=1,
                                                              kept=None, rows=None, freed=None, weight_out=None))),
                              tlkv.EvictSeq(**a))
    assert tlkv.lib().tl_kv_evict(two, 2, None) == -1
    assert tlkv.lib().tl_kv_evict(None, 1, None) == -1


def test_evict_sessions_apart():
    """An output of one session over an input or an output of another."""
    L = tlkv.lib()
    a = dict(weight=P, pages=2 * P, len=100, keep=50, sink=4, recent=10, page_size=16, kept=4 * P,
             rows=5 * P, freed=6 * P, weight_out=7 * P)
    b = {k: v + 16 * P if v >= P else v for k, v in a.items()}
    for bad in (dict(kept=P), dict(rows=2 * P), dict(freed=4 * P), dict(weight_out=6 * P + 196),
                dict(weight=5 * P), dict(pages=6 * P + 196)):
        assert L.tl_kv_evict((tlkv.EvictSeq * 2)(tlkv.EvictSeq(**a), tlkv.EvictSeq(**dict(b, **bad))), 2, None) == -1
        many = [dict(b, **{k: v + 16 * P * i for k, v in b.items() if v >= P}) for i in range(1, 40)]
        assert L.tl_kv_evict((tlkv.EvictSeq * 41)(*[tlkv.EvictSeq(**x) for x in many + [a, dict(b, **bad)]]), 41, None) == -1
    assert L.tl_kv_evict((tlkv.EvictSeq * 1)(tlkv.EvictSeq(**a)), 4097, None) == -1
