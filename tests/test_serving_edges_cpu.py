"""Edges of the serving operators that need no GPU: whose memory results are, and what is refused."""
import contextlib

import pytest
import torch

from m3_avm_b200 import attention as A
from m3_avm_b200 import logprobs as L
from m3_avm_b200._lib import M3GError


def i32(*s):
    return torch.zeros(s, dtype=torch.int32)


# ---------------------------------------------------------------- results of a call on another stream
class Streams:
    """Stands in for the device: the current stream is 0, launches do nothing, allocations say where they were made."""

    def __init__(self, monkeypatch):
        self.current, self.made, self.kept, self.launched = 0, [], [], []
        for name in ("empty", "empty_like"):
            monkeypatch.setattr(torch, name, self._noted(getattr(torch, name)))
        new_empty = torch.Tensor.new_empty
        monkeypatch.setattr(torch.Tensor, "new_empty", self._noted(new_empty))
        monkeypatch.setattr(torch.cuda, "ExternalStream", lambda stream, device=None: stream)
        monkeypatch.setattr(torch.cuda, "default_stream", lambda device=None: 0)
        monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: self.current)
        monkeypatch.setattr(torch.cuda, "stream", self._on)
        monkeypatch.setattr(torch.Tensor, "record_stream", lambda t, s: self.kept.append((t.data_ptr(), s)))
        A._need_torch()
        monkeypatch.setattr(A, "_need_torch", lambda: None)
        monkeypatch.setattr(A, "_current_stream", lambda device: 0)
        for module in (A, L):
            monkeypatch.setattr(module, "_device", lambda t: -1)
            monkeypatch.setattr(module, "_call", lambda fn, device, stream, *args: self.launched.append(stream))

    def _noted(self, make):
        def run(*args, **kw):
            t = make(*args, **kw)
            self.made.append((t.data_ptr(), self.current))
            return t
        return run

    @contextlib.contextmanager
    def _on(self, stream):
        before, self.current = self.current, stream
        yield
        self.current = before


def calls():
    q, k = torch.randn(3, 4, 64), torch.randn(3, 2, 64)
    cache = A.KvCache(8, 1, 2, 64, 16, 4, pool=torch.zeros(4 * 2 * 16 * 2 * 68, dtype=torch.uint8))
    batch = A.KvBatch(i32(2), i32(1), i32(1, 4), 3, 3, 64)
    x = torch.randn(3, 40)
    rope = A.Rope(64)
    return {
        "rope": lambda s: rope.apply(i32(3), q, k, stream=s),
        "rope of strided rows": lambda s: rope.apply(i32(3), q[:, ::2], stream=s)[:1],
        "read": lambda s: cache.read(0, batch, stream=s),
        "attention": lambda s: (A.tree_attention(q, cache, 0, batch, stream=s),),
        "logprobs": lambda s: L.token_logprobs(x, i32(3, 2), n_top=4, entropy=True, stream=s),
    }


@pytest.mark.parametrize("stream", [None, 0, 7])
@pytest.mark.parametrize("name", list(calls()))
def test_results_are_memory_of_the_calls_stream(monkeypatch, name, stream):
    """The allocator gives a block to the work of one stream: results have to come from the stream that writes them, and
    stay until the current stream is done with them."""
    call = calls()[name]
    dev = Streams(monkeypatch)
    results = call(stream)
    assert dev.launched == [stream]
    where = dict(dev.made)
    assert dev.made and all(s == (stream or 0) for s in where.values())
    assert all(t.data_ptr() in where for t in results)
    for t in results:
        assert ((t.data_ptr(), 0) in dev.kept) == (stream == 7)


# ---------------------------------------------------------------- refusals
@pytest.mark.parametrize("scale", [0.0, -1.0, float("nan"), 1e-50])
def test_scales_that_are_not_positive_in_32_bits(scale):
    """1e-50 is 0 in 32 bits, which the library takes for 1 / sqrt(head_dim)."""
    cache = A.KvCache(8, 1, 2, 64, 16, 4, pool=torch.zeros(4 * 2 * 16 * 2 * 68, dtype=torch.uint8))
    batch = A.KvBatch(i32(2), i32(1), i32(1, 4), 3, 3, 64)
    with pytest.raises(M3GError, match="scale must be positive"):
        A.tree_attention(torch.zeros(3, 4, 64), cache, 0, batch, scale=scale)


def test_attention_bounds_that_are_and_are_not_too_large():
    """Bounds count as what the batch's tokens could come to, not as if every sequence had the most of all."""
    import ctypes

    from m3_avm_b200 import _lib
    from tests.conftest import HAS_CUDA

    if HAS_CUDA:
        pytest.skip("host pointers: only where nothing can be launched")
    buf = (ctypes.c_uint8 * (1 << 16))()
    p = ctypes.addressof(buf) // 64 * 64 + 64

    def call(n_seqs, n_tokens, max_tokens, max_len, dtype):
        lay = _lib.KvLayout(8, 1, 8, 128, 64, 1000)
        bat = _lib.KvBatchArgs(p, p, p, n_seqs, 1 << 14, n_tokens, max_tokens, max_len)
        a, b = _lib.Rows(p, 4096, 128), _lib.Rows(p + 8192, 4096, 128)
        return _lib.load().m3g_tree_attn_dev(ctypes.byref(lay), p, 0, ctypes.byref(bat), dtype, ctypes.byref(a), 32,
                                             None, 0, 0.0, ctypes.byref(b), p, 1 << 40, None)

    for dtype in (0, 1, 30):
        # one prompt chunk beside single tokens
        assert call(256, 2303, 2048, 131072, dtype) == _lib.M3G_ECUDA
        assert call(1000, 1999, 1000, 1 << 20, dtype) == _lib.M3G_ECUDA
        # 2^31 chunks and more
        assert call(1 << 20, 1 << 20, 1, 1 << 20, dtype) == _lib.M3G_EINVAL
        assert call(4096, 1 << 24, 1 << 12, 1 << 20, dtype) == _lib.M3G_EINVAL
        assert call(1, 1 << 30, 1 << 30, 64, dtype) == _lib.M3G_EINVAL


def test_tensors_that_require_a_gradient_are_refused(monkeypatch):
    """Autograd sees none of the calls: the gradient would be lost (in place, a leaf changed behind its back)."""
    dev = Streams(monkeypatch)
    cache = A.KvCache(8, 1, 2, 64, 16, 4, pool=torch.zeros(4 * 2 * 16 * 2 * 68, dtype=torch.uint8))
    batch, rope = A.KvBatch(i32(2), i32(1), i32(1, 4), 3, 3, 64), A.Rope(64)
    leaf = lambda *s: torch.randn(*s, requires_grad=True)  # noqa: E731
    q, k, x = leaf(3, 4, 64), leaf(3, 2, 64), leaf(3, 40)
    calls_of = [
        lambda q, k, x: rope.apply(i32(3), q, k.detach()),
        lambda q, k, x: rope.apply(i32(3), q.detach(), k),
        lambda q, k, x: rope.apply(i32(3), q.detach(), q_out=q),
        lambda q, k, x: cache.write(0, k, k.detach(), batch),
        lambda q, k, x: cache.write(0, k.detach(), k, batch),
        lambda q, k, x: A.tree_attention(q, cache, 0, batch),
        lambda q, k, x: L.token_logprobs(x, n_top=2),
    ]
    for call in calls_of:
        with pytest.raises(M3GError, match="gradient"):
            call(q, k, x)
    assert not dev.launched
    with torch.no_grad():
        for call in calls_of:
            call(q, k, x)
    for call in calls_of:
        call(q.detach(), k.detach(), x.detach())
    assert len(dev.launched) == 2 * len(calls_of)


def test_numbers_past_32_bits_are_refused_not_cut(monkeypatch):
    from m3_avm_b200.decoder import GpuDecoder

    dev = Streams(monkeypatch)
    cache = A.KvCache(8, 2, 2, 64, 16, 4, pool=torch.zeros(2 * 4 * 2 * 16 * 2 * 68, dtype=torch.uint8))
    batch, q, k = A.KvBatch(i32(2), i32(1), i32(1, 4), 3, 3, 64), torch.zeros(3, 4, 64), torch.zeros(3, 2, 64)
    for layer in (2, -1, 2 ** 32, 2 ** 32 + 1, -2 ** 32):
        for call in (lambda: cache.write(layer, k, k, batch), lambda: cache.read(layer, batch),
                     lambda: A.tree_attention(q, cache, layer, batch)):
            with pytest.raises(M3GError, match="layer"):
                call()
    assert not dev.launched
    for args in ((2 ** 32 + 4, None, 1), (4, None, 2 ** 32 + 1), (4, None, -1), (4, torch.float64, 1)):
        with pytest.raises(M3GError):
            cache.attention_workspace(*args)
    for n_top in (-1, 33, 2 ** 32 + 1):
        with pytest.raises(M3GError, match="alternatives"):
            GpuDecoder.score(GpuDecoder.__new__(GpuDecoder), [], n_top=n_top)


def test_what_the_library_was_told_cannot_be_changed_behind_its_back():
    cache = A.KvCache(8, 1, 2, 64, 16, 4, pool=torch.zeros(4 * 2 * 16 * 2 * 68, dtype=torch.uint8))
    batch, rope = A.KvBatch(i32(2), i32(1), i32(1, 4), 3, 3, 64), A.Rope(64)
    for obj, name, value in ((batch, "n_tokens", 5), (batch, "ctx_len", i32(1)), (batch, "max_len", 128),
                             (cache, "pool", torch.zeros(16, dtype=torch.uint8)), (cache, "n_layers", 9),
                             (rope, "head_dim", 128)):
        before = getattr(obj, name)
        with pytest.raises(M3GError, match="cannot be changed"):
            setattr(obj, name, value)
        assert getattr(obj, name) is before
    batch.ctx_len[0] = 7  # the contents are the caller's

    class Mine(A.KvCache):  # and so are attributes of their own
        def __init__(self, *args, **kw):
            super().__init__(*args, **kw)
            self.free = [1]

    mine = Mine(8, 1, 2, 64, 16, 4, pool=cache.pool)
    mine.free = []
    with pytest.raises(M3GError, match="cannot be changed"):
        mine.head_dim = 128
    rope.close()
