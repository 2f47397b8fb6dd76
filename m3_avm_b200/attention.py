"""Rotary positions, the paged quantised KV cache and attention of drafted
tokens over it, on CUDA tensors (the serving operators of include/m3gemv.h).

A step of a batch: ``Rope.apply`` turns q and k, ``KvCache.write`` puts the new
tokens' K and V into the cache, ``tree_attention`` attends over it; ``KvBatch``
says which tokens belong to which sequence.  Tensors are f32, f16 or bf16 of
shape (tokens, heads, head_dim), any strides with a contiguous last dimension.
Everything runs on `stream` (the current one of the tensors' device by
default), enqueued without waiting, and raises M3GError for what the library
refuses.
"""
from __future__ import annotations

import ctypes

from . import _lib

SCALINGS = {"none": 0, "linear": 1, "ntk": 2, "yarn": 3, "llama3": 4}
Q4_0, Q8_0 = 2, 8
_dtypes: dict = {}


def act_dtype(t) -> int:
    """ggml number of an activation tensor's type."""
    if not _dtypes:
        import torch

        _dtypes.update({torch.float32: 0, torch.float16: 1, torch.bfloat16: 30})
    try:
        return _dtypes[t.dtype]
    except KeyError:
        raise _lib.M3GError(_lib.M3G_EINVAL, f"activations of type {t.dtype} (f32, f16 and bf16 are supported)") from None


class _OnDevice:
    """Makes the tensors' device current for a call, where it is not."""

    def __init__(self, t):
        import torch

        if not t.is_cuda:
            raise _lib.M3GError(_lib.M3G_EINVAL, "the operators need CUDA tensors")
        cur = torch.cuda.current_device()
        self._guard = torch.cuda.device(t.device) if t.device.index != cur else None

    def __enter__(self):
        if self._guard:
            self._guard.__enter__()

    def __exit__(self, *exc):
        if self._guard:
            self._guard.__exit__(*exc)


def _stream(t, stream):
    import torch

    return stream if stream is not None else torch.cuda.current_stream(t.device).cuda_stream


def _fail(msg):
    raise _lib.M3GError(_lib.M3G_EINVAL, msg)


def _check_rows(name, t, like, heads=None, head_dim=None, tokens=None):
    """t is (tokens, heads, head_dim) with a contiguous last dimension, on like's device."""
    if t.dim() != 3 or (t.shape[2] > 1 and t.stride(2) != 1):
        _fail(f"{name}: (tokens, heads, head_dim) with a contiguous last dimension is wanted, got {tuple(t.shape)}")
    if t.device != like.device:
        _fail(f"{name} is on {t.device}, not on {like.device}")
    for what, got, want in (("tokens", t.shape[0], tokens), ("heads", t.shape[1], heads),
                            ("head_dim", t.shape[2], head_dim)):
        if want is not None and got != want:
            _fail(f"{name} has {got} {what}, not {want}")


def _check_ints(name, t, like, shape):
    import torch

    if t.dtype != torch.int32 or not t.is_contiguous() or tuple(t.shape) != shape or t.device != like.device:
        _fail(f"{name}: a contiguous int32 tensor of shape {shape} on {like.device} is wanted")


def _rows(t):
    return _lib.Rows(t.data_ptr(), t.stride(0), t.stride(1))


class Rope:
    """A plan of rotary positions (m3g_rope_config); host arithmetic, usable on every device."""

    def __init__(self, head_dim: int, rot_dim: int | None = None, theta: float = 10000.0, interleaved: bool = False,
                 scaling: str = "none", factor: float = 1.0, orig_ctx: int = 0, low_freq: float = 1.0,
                 high_freq: float = 4.0, beta_fast: float = 32.0, beta_slow: float = 1.0, magnitude: float = 0.0):
        if scaling not in SCALINGS:
            _fail(f"scaling {scaling!r}: one of {', '.join(SCALINGS)} is wanted")
        self.head_dim = head_dim
        cfg = _lib.RopeConfig(head_dim, rot_dim if rot_dim is not None else head_dim, 1 if interleaved else 0,
                              SCALINGS[scaling], theta, factor, orig_ctx, low_freq, high_freq, beta_fast, beta_slow,
                              magnitude)
        h = ctypes.c_void_p()
        _lib.check(_lib.load().m3g_rope_create(ctypes.byref(cfg), ctypes.byref(h)))
        self._h = h

    def apply(self, positions, q, k=None, q_out=None, k_out=None, inverse: bool = False, stream=None):
        """Turns q and k (k may be None) at int32 `positions` (tokens,); q_out, k_out may be q and k themselves.
        inverse: by the opposite angles, the gradient of the forward call."""
        import torch

        n = positions.numel()
        _check_ints("positions", positions, q, (n,))
        _check_rows("q", q, q, head_dim=self.head_dim, tokens=n)
        if q_out is None:
            q_out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        pairs = [(q, q_out)]
        if k is not None:
            _check_rows("k", k, q, head_dim=self.head_dim, tokens=n)
            if k_out is None:
                k_out = torch.empty(k.shape, dtype=k.dtype, device=k.device)
            pairs.append((k, k_out))
        args = []
        for x, y in pairs:
            if x.dtype != q.dtype or y.dtype != q.dtype:
                _fail("q, k and their results have one type")
            _check_rows("result", y, q, heads=x.shape[1], head_dim=self.head_dim, tokens=n)
            args.append(_lib.RopeRows(x.data_ptr(), y.data_ptr(), x.shape[1], x.stride(0), x.stride(1), y.stride(0),
                                      y.stride(1)))
        with _OnDevice(q):
            _lib.check(_lib.load().m3g_rope_dev(self._h, act_dtype(q), positions.data_ptr(), n, ctypes.byref(args[0]),
                                                ctypes.byref(args[1]) if k is not None else None,
                                                1 if inverse else 0, _stream(q, stream)))
        return q_out, k_out

    def close(self) -> None:
        if getattr(self, "_h", None) and self._h.value:
            _lib.load().m3g_rope_destroy(self._h)
            self._h = ctypes.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


class KvBatch:
    """The new tokens of a batch of sequences (m3g_kv_batch).  `q_start` (n + 1,), `ctx_len` (n,) and `page_table`
    (n, max_pages) are int32 tensors of the GPU, read when an operator runs (a captured step replays with what they
    hold then); max_tokens and max_len bound what they may say."""

    def __init__(self, q_start, ctx_len, page_table, n_tokens: int, max_tokens: int, max_len: int):
        n = ctx_len.numel()
        _check_ints("q_start", q_start, q_start, (n + 1,))
        _check_ints("ctx_len", ctx_len, q_start, (n,))
        _check_ints("page_table", page_table, q_start, (n, page_table.shape[-1]))
        if min(n_tokens, max_tokens, max_len) < 0:
            _fail("negative size of the batch")
        self.q_start, self.ctx_len, self.page_table = q_start, ctx_len, page_table
        self.n_tokens, self.max_tokens, self.max_len = n_tokens, max_tokens, max_len
        self.args = _lib.KvBatchArgs(q_start.data_ptr(), ctx_len.data_ptr(), page_table.data_ptr(), n,
                                     page_table.shape[1], n_tokens, max_tokens, max_len)


class KvCache:
    """A paged cache of K and V rows in Q8_0 or Q4_0 blocks (m3g_kv_layout).  Its memory is one uint8 tensor, `pool`,
    allocated here (zeros) or the caller's own."""

    def __init__(self, dtype: int, n_layers: int, n_kv_heads: int, head_dim: int, page_size: int, n_pages: int,
                 device: int = 0, pool=None):
        import torch

        if min(n_layers, n_kv_heads, head_dim, page_size, n_pages) < 0:
            _fail("negative size of the cache")
        self.dtype, self.n_layers, self.n_kv_heads, self.head_dim = dtype, n_layers, n_kv_heads, head_dim
        self.page_size, self.n_pages = page_size, n_pages
        self.layout = _lib.KvLayout(dtype, n_layers, n_kv_heads, head_dim, page_size, n_pages)
        need = ctypes.c_uint64()
        _lib.check(_lib.load().m3g_kv_bytes(ctypes.byref(self.layout), ctypes.byref(need)))
        if pool is None:
            pool = torch.zeros(need.value, dtype=torch.uint8, device=f"cuda:{device}")
        elif pool.dtype != torch.uint8 or not pool.is_contiguous() or pool.numel() < need.value:
            _fail(f"the pool: a contiguous uint8 tensor of {need.value} bytes is wanted")
        self.pool = pool
        self._workspace_bytes: dict[int, int] = {}

    def _io(self, fn, layer, k, v, batch, stream):
        for name, t in (("k", k), ("v", v)):
            _check_rows(name, t, self.pool, self.n_kv_heads, self.head_dim, batch.n_tokens)
        if k.dtype != v.dtype:
            _fail("k and v have one type")
        if batch.q_start.device != self.pool.device:
            _fail("the batch is on another device than the cache")
        rk, rv = _rows(k), _rows(v)
        with _OnDevice(self.pool):
            _lib.check(fn(ctypes.byref(self.layout), self.pool.data_ptr(), layer, ctypes.byref(batch.args),
                          act_dtype(k), ctypes.byref(rk), ctypes.byref(rv), _stream(self.pool, stream)))

    def write(self, layer: int, k, v, batch: KvBatch, stream=None) -> None:
        """Quantises the new tokens' rows into their places."""
        self._io(_lib.load().m3g_kv_write_dev, layer, k, v, batch, stream)

    def read(self, layer: int, batch: KvBatch, dtype=None, k_out=None, v_out=None, stream=None):
        """The values held at the new tokens' places, as (k, v) of `dtype` (f32 by default)."""
        import torch

        shape = (batch.n_tokens, self.n_kv_heads, self.head_dim)
        if k_out is None:
            k_out = torch.empty(shape, dtype=dtype or torch.float32, device=self.pool.device)
        if v_out is None:
            v_out = torch.empty(shape, dtype=k_out.dtype, device=self.pool.device)
        self._io(_lib.load().m3g_kv_read_dev, layer, k_out, v_out, batch, stream)
        return k_out, v_out

    def attention_workspace(self, n_heads: int) -> int:
        """Bytes of workspace that attention of n_heads query heads needs."""
        got = self._workspace_bytes.get(n_heads)
        if got is None:
            need = ctypes.c_uint64()
            _lib.check(_lib.load().m3g_tree_attn_workspace(ctypes.byref(self.layout), n_heads, ctypes.byref(need)))
            got = self._workspace_bytes[n_heads] = need.value
        return got


def tree_attention(q, cache: KvCache, layer: int, batch: KvBatch, mask=None, scale: float | None = None, out=None,
                   workspace=None, stream=None):
    """Attention of the batch's new tokens (already written) over the cache.  `mask`: int32 (tokens, words), bit i % 32
    of word i / 32 says whether the token sees new token i of its sequence; None: all up to and including itself.
    `workspace`: a uint8 tensor of cache.attention_workspace(heads) bytes, used by one call at a time (allocated here
    when None)."""
    import torch

    _check_rows("q", q, cache.pool, head_dim=cache.head_dim, tokens=batch.n_tokens)
    heads = q.shape[1]
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    else:
        _check_rows("out", out, q, heads, cache.head_dim, batch.n_tokens)
        if out.dtype != q.dtype:
            _fail("q and out have one type")
    if batch.q_start.device != q.device:
        _fail("the batch is on another device than q")
    words = 0
    if mask is not None:
        words = mask.shape[-1] if mask.dim() == 2 else 0
        _check_ints("mask", mask, q, (batch.n_tokens, words))
    if scale is not None and not scale > 0:
        _fail("scale must be positive")
    if stream is not None and workspace is None:
        _fail("a call on a stream of its own needs its own workspace")
    with _OnDevice(q):
        if workspace is None:
            workspace = torch.empty(cache.attention_workspace(heads), dtype=torch.uint8, device=q.device)
        elif workspace.dtype != torch.uint8 or workspace.device != q.device or not workspace.is_contiguous():
            _fail("workspace: a contiguous uint8 tensor on q's device is wanted")
        rq, ro = _rows(q), _rows(out)
        _lib.check(_lib.load().m3g_tree_attn_dev(
            ctypes.byref(cache.layout), cache.pool.data_ptr(), layer, ctypes.byref(batch.args), act_dtype(q),
            ctypes.byref(rq), heads, mask.data_ptr() if mask is not None else None, words, scale or 0.0,
            ctypes.byref(ro), workspace.data_ptr(), workspace.numel(), _stream(q, stream)))
    return out
