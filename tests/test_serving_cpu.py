"""The serving operators on a machine without a GPU: plans, sizes and everything that is refused before a launch."""
import ctypes

import numpy as np
import pytest

from m3_avm_b200 import _lib
from m3_avm_b200._lib import M3GError
from tests.conftest import HAS_CUDA

EINVAL = _lib.M3G_EINVAL


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def layout(**kw):
    d = dict(dtype=8, n_layers=2, n_kv_heads=4, head_dim=128, page_size=16, n_pages=10)
    d.update(kw)
    return _lib.KvLayout(*[d[f] for f, _ in _lib.KvLayout._fields_])


def test_structures_match_the_header_sizes():
    # 8-byte alignment of the C structures: the sizes a C compiler gives them
    assert ctypes.sizeof(_lib.RopeConfig) == 80
    assert ctypes.sizeof(_lib.RopeRows) == 56
    assert ctypes.sizeof(_lib.KvLayout) == 32
    assert ctypes.sizeof(_lib.KvBatchArgs) == 48
    assert ctypes.sizeof(_lib.Rows) == 24


@pytest.mark.parametrize("bad", [
    dict(head_dim=0), dict(head_dim=65), dict(head_dim=514), dict(rot_dim=0), dict(rot_dim=3), dict(rot_dim=66),
    dict(head_dim=512, rot_dim=258), dict(theta=1.0), dict(theta=float("nan")), dict(theta=float("inf")),
    dict(factor=2.0), dict(scaling="linear", factor=0.5), dict(scaling="yarn", factor=2.0),
    dict(scaling="llama3", factor=2.0, orig_ctx=8192, low_freq=4.0, high_freq=4.0),
    dict(scaling="yarn", factor=2.0, orig_ctx=8192, beta_fast=1.0, beta_slow=32.0), dict(magnitude=-1.0),
    dict(scaling="ntk", factor=2.0, rot_dim=2), dict(scaling="spiral"),
])
def test_rope_plan_refusals(bad):
    from m3_avm_b200.attention import Rope

    kw = dict(head_dim=64)
    kw.update(bad)
    with pytest.raises(M3GError) as e:
        Rope(**kw)
    assert e.value.code == EINVAL


def test_rope_call_refusals(lib):
    h = ctypes.c_void_p()
    cfg = _lib.RopeConfig(64, 64, 0, 0, 10000.0, 1.0, 0, 1.0, 4.0, 32.0, 1.0, 0.0)
    assert lib.m3g_rope_create(ctypes.byref(cfg), ctypes.byref(h)) == 0
    buf = np.zeros(4096, np.float32)
    p = buf.ctypes.data

    def call(dtype=0, pos=p, n=4, q=(p, p, 2, 128, 64, 128, 64), k=None, plan=h):
        rq = _lib.RopeRows(*q) if q else None
        rk = _lib.RopeRows(*k) if k else None
        return lib.m3g_rope_dev(plan, dtype, pos, n, ctypes.byref(rq) if rq else None,
                                ctypes.byref(rk) if rk else None, 0, None)

    assert call(plan=None) == EINVAL
    assert call(q=None) == EINVAL
    assert call(dtype=8) == EINVAL
    assert call(n=2 ** 31) == EINVAL
    assert call(pos=None) == EINVAL
    assert call(q=(None, p, 2, 128, 64, 128, 64)) == EINVAL
    assert call(q=(p, p, 2, 128, 64, 256, 64)) == EINVAL       # in place with other strides
    assert call(q=(p, p, 2, -128, 64, -128, 64)) == EINVAL
    assert call(q=(p, p + 4096, 2, 128, 64, 128, 32)) == EINVAL  # result heads overlap
    assert call(q=(p, p + 4096, 2, 0, 64, 0, 64)) == EINVAL      # result tokens overlap
    assert call(k=(p, None, 2, 128, 64, 128, 64)) == EINVAL
    assert call(n=0, pos=None) == 0                              # nothing to do
    assert call(q=(None, None, 0, 0, 0, 0, 0), pos=None) == 0
    if not HAS_CUDA:
        assert call() == _lib.M3G_ECUDA
    lib.m3g_rope_destroy(h)
    lib.m3g_rope_destroy(None)


@pytest.mark.parametrize("q8", [True, False])
def test_cache_bytes(lib, q8):
    out = ctypes.c_uint64()
    for hd in (64, 128):
        assert lib.m3g_kv_bytes(ctypes.byref(layout(dtype=8 if q8 else 2, head_dim=hd)), ctypes.byref(out)) == 0
        assert out.value == 2 * 10 * 4 * 16 * 2 * ((hd if q8 else hd // 2) + hd // 16)


BAD_LAYOUTS = [dict(dtype=0), dict(dtype=12), dict(head_dim=96), dict(head_dim=256), dict(n_layers=0),
               dict(n_kv_heads=0), dict(n_kv_heads=2000), dict(page_size=8), dict(page_size=48), dict(page_size=2048),
               dict(n_pages=0), dict(n_pages=2 ** 31)]


@pytest.mark.parametrize("bad", BAD_LAYOUTS)
def test_cache_layout_refusals(lib, bad):
    out = ctypes.c_uint64(7)
    assert lib.m3g_kv_bytes(ctypes.byref(layout(**bad)), ctypes.byref(out)) == EINVAL
    assert out.value == 0
    ws = ctypes.c_uint64(7)
    assert lib.m3g_tree_attn_workspace(ctypes.byref(layout(**bad)), 0, 8, 1, ctypes.byref(ws)) == EINVAL


def test_cache_too_large(lib):
    out = ctypes.c_uint64()
    assert lib.m3g_kv_bytes(ctypes.byref(layout(n_layers=4096, n_kv_heads=1024, page_size=1024, n_pages=2 ** 31 - 1)),
                            ctypes.byref(out)) == EINVAL


def _calls(lib):
    """The cache's and attention's calls with one argument changed at a time."""
    buf = np.zeros(1 << 16, np.uint8)
    p = (buf.ctypes.data + 63) // 64 * 64
    ints = np.zeros(64, np.int32)
    ip = ints.ctypes.data

    def args(lay=None, pool=p, layer=0, batch=None, dtype=0, a=None, b=None):
        lay = lay or layout(n_pages=1, n_layers=1)
        bt = dict(q_start=ip, ctx_len=ip, page_table=ip, n_seqs=1, max_pages=1, n_tokens=1, max_tokens=1, max_len=16)
        bt.update(batch or {})
        bat = _lib.KvBatchArgs(*[bt[f] for f, _ in _lib.KvBatchArgs._fields_])
        return lay, pool, layer, bat, dtype, a or (p, 512, 128), b or (p + 8192, 512, 128)

    def write(read=False, **kw):
        lay, pool, layer, bat, dtype, a, b = args(**kw)
        fn = lib.m3g_kv_read_dev if read else lib.m3g_kv_write_dev
        ra, rb = _lib.Rows(*a), _lib.Rows(*b)
        return fn(ctypes.byref(lay), pool, layer, ctypes.byref(bat), dtype, ctypes.byref(ra), ctypes.byref(rb), None)

    def attn(heads=4, mask=None, words=0, scale=0.0, ws=p + 16384, ws_bytes=1 << 40, **kw):
        lay, pool, layer, bat, dtype, a, b = args(**kw)
        ra, rb = _lib.Rows(*a), _lib.Rows(*b)
        return lib.m3g_tree_attn_dev(ctypes.byref(lay), pool, layer, ctypes.byref(bat), dtype, ctypes.byref(ra),
                                     heads, mask, words, scale, ctypes.byref(rb), ws, ws_bytes, None)

    return write, attn, p, buf


@pytest.mark.skipif(HAS_CUDA, reason="host pointers: only where nothing can be launched")
def test_cache_and_attention_refusals(lib):
    write, attn, p, _keep = _calls(lib)
    for f in (write, lambda **kw: write(read=True, **kw), attn):
        assert f() == _lib.M3G_ECUDA  # passes every check of arguments, and there is no device
        assert f(pool=None) == EINVAL
        assert f(pool=p + 8) == EINVAL
        assert f(layer=1) == EINVAL
        assert f(dtype=8) == EINVAL
        assert f(a=(None, 512, 128)) == EINVAL
        assert f(b=(None, 512, 128)) == EINVAL
        assert f(a=(p, -512, 128)) == EINVAL
        for name in ("q_start", "ctx_len", "page_table"):
            assert f(batch={name: None}) == EINVAL
        assert f(batch=dict(max_pages=0)) == EINVAL
        assert f(batch=dict(n_seqs=2 ** 21)) == EINVAL
        assert f(batch=dict(max_len=2 ** 31 - 1)) == EINVAL
        for bad in BAD_LAYOUTS:
            assert f(lay=layout(**dict(dict(n_pages=1, n_layers=1), **bad))) == EINVAL
    assert write(read=True, a=(p, 512, 64)) == EINVAL  # result rows overlap
    assert write(a=(p, 512, 0)) == _lib.M3G_ECUDA      # a broadcast input is fine
    assert attn(heads=0) == EINVAL
    assert attn(heads=6) == EINVAL
    assert attn(scale=-1.0) == EINVAL
    assert attn(scale=float("nan")) == EINVAL
    assert attn(mask=p, words=0) == EINVAL
    assert attn(mask=p, words=1, batch=dict(max_tokens=33)) == EINVAL
    assert attn(ws=None) == EINVAL
    assert attn(ws=p + 8) == EINVAL
    assert attn(ws_bytes=8) == EINVAL
    assert attn(b=(p + 8192, 512, 64)) == EINVAL
    assert attn(a=(p, 512, 128), b=(p, 512, 256)) == EINVAL  # in place with other strides
    assert attn(batch=dict(n_tokens=0), ws=None) == 0


def test_logprobs_refusals(lib):
    buf = np.zeros(4096, np.float32)
    p = buf.ctypes.data

    def call(dtype=0, x=p, rows=1, vocab=100, stride=100, tok=p, n=1, lp=p, ent=None, k=0, ids=None, tops=None):
        return lib.m3g_token_logprobs_dev(dtype, x, rows, vocab, stride, tok, n, lp, ent, k, ids, tops, None)

    assert call(dtype=8) == EINVAL
    assert call(vocab=0) == EINVAL
    assert call(vocab=2 ** 30 + 1) == EINVAL
    assert call(rows=2 ** 28) == EINVAL
    assert call(stride=-1) == EINVAL
    assert call(n=513) == EINVAL
    assert call(k=33, ids=p, tops=p) == EINVAL
    assert call(k=11, vocab=10, ids=p, tops=p) == EINVAL
    assert call(x=None) == EINVAL
    assert call(tok=None) == EINVAL
    assert call(lp=None) == EINVAL
    assert call(k=1, ids=None, tops=p) == EINVAL
    assert call(rows=0, x=None, tok=None) == 0
    if not HAS_CUDA:
        assert call() == _lib.M3G_ECUDA


def test_python_checks_without_a_device():
    import torch

    from m3_avm_b200.attention import KvBatch, KvCache, Rope
    from m3_avm_b200.logprobs import token_logprobs

    i32 = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
    r = Rope(64)
    q = torch.zeros(3, 2, 64)
    for pos, x in ((i32(2), q), (torch.zeros(3, dtype=torch.int64), q), (i32(3), q[..., :32]),
                   (i32(3), torch.zeros(3, 64, 2).transpose(1, 2)), (i32(3), q.double()), (i32(3), q)):
        with pytest.raises(M3GError):
            r.apply(pos, x)
    with pytest.raises(M3GError):
        KvBatch(i32(3), i32(3), i32(3, 2), 4, 4, 32)
    with pytest.raises(M3GError):
        KvBatch(i32(4), i32(3), i32(3, 4)[:, ::2], 4, 4, 32)
    with pytest.raises(M3GError):
        KvBatch(i32(4), i32(3), i32(3, 4), -1, 4, 32)
    with pytest.raises(M3GError):
        KvCache(8, 1, 2, 64, 16, 4, pool=torch.zeros(16, dtype=torch.uint8))
    cache = KvCache(8, 1, 2, 64, 16, 4, pool=torch.zeros(4 * 2 * 16 * 2 * 68, dtype=torch.uint8))
    batch = KvBatch(i32(2), i32(1), i32(1, 4), 3, 3, 64)
    with pytest.raises(M3GError):
        cache.write(0, q[:2], q[:2], batch)
    with pytest.raises(M3GError):
        cache.write(0, q, q.half(), batch)
    with pytest.raises(M3GError):
        cache.write(0, q, q, batch)  # not on a GPU
    x = torch.zeros(2, 100)
    for bad in (dict(logits=x.t()), dict(logits=x[0]), dict(logits=x, n_top=-1), dict(logits=x, tokens=i32(3, 1)),
                dict(logits=x, tokens=i32(2)), dict(logits=x.double(), n_top=1), dict(logits=x, n_top=1)):
        with pytest.raises(M3GError):
            token_logprobs(**bad)


def test_decoder_score_without_a_decoder(lib):
    assert lib.m3g_decoder_score(None, None, 0, None, None, 0, None, None) == EINVAL


def test_sizes_past_32_bits_are_refused():
    from m3_avm_b200.attention import KvBatch, KvCache, Rope
    from m3_avm_b200.logprobs import token_logprobs
    import torch

    i32 = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
    for args in ((1, 1, 2 ** 32 + 16), (1, 2 ** 32 + 1, 16), (2 ** 32 + 1, 1, 16)):
        with pytest.raises(M3GError):
            KvBatch(i32(2), i32(1), i32(1, 4), *args)
    for args in ((8, 2 ** 32 + 1, 2, 64, 16, 4), (8, 1, 2, 64, 2 ** 32 + 16, 4), (8, 1, 2, 2 ** 32 + 64, 16, 4)):
        with pytest.raises(M3GError):
            KvCache(*args, pool=torch.zeros(1 << 16, dtype=torch.uint8))
    with pytest.raises(M3GError):
        Rope(2 ** 32 + 64)
    with pytest.raises(M3GError):
        token_logprobs(torch.zeros(1, 4), n_top=2 ** 32 + 1)


def test_pointers_off_their_types_alignment_are_refused(lib):
    write, attn, p, _keep = _calls(lib)
    for f in (write, lambda **kw: write(read=True, **kw), attn):
        assert f(a=(p + 2, 512, 128)) == EINVAL
        assert f(b=(p + 8193, 512, 128), dtype=30) == EINVAL
        for name in ("q_start", "ctx_len", "page_table"):
            assert f(batch={name: p + 2}) == EINVAL
    assert attn(mask=p + 2, words=1) == EINVAL
    h = ctypes.c_void_p()
    cfg = _lib.RopeConfig(64, 64, 0, 0, 10000.0, 1.0, 0, 1.0, 4.0, 32.0, 1.0, 0.0)
    assert lib.m3g_rope_create(ctypes.byref(cfg), ctypes.byref(h)) == 0
    for x, y, pos, dtype in ((p + 2, p + 4096, p, 0), (p, p + 4097, p, 1), (p, p + 4096, p + 1, 30)):
        rows = _lib.RopeRows(x, y, 2, 128, 64, 128, 64)
        assert lib.m3g_rope_dev(h, dtype, pos, 4, ctypes.byref(rows), None, 0, None) == EINVAL
    lib.m3g_rope_destroy(h)


def test_logits_off_their_types_alignment_are_refused(lib):
    buf = (ctypes.c_uint8 * 64)()
    at = ctypes.addressof(buf) // 16 * 16 + 16
    for dtype, off in ((0, 2), (1, 1), (30, 1)):
        assert lib.m3g_token_logprobs_dev(dtype, at + off, 1, 4, 4, None, 0, None, at, 0, None, None, None) == EINVAL
