"""Rotary positions, the paged quantised KV cache and attention of drafted
tokens over it, on CUDA tensors (the serving operators of include/m3gemv.h).

A step of a batch: ``Rope.apply`` turns q and k, ``KvCache.write`` puts the new
tokens' K and V into the cache, ``tree_attention`` attends over it; ``KvBatch``
says which tokens belong to which sequence.  Tensors are f32, f16 or bf16 of
shape (tokens, heads, head_dim), any strides with a contiguous last dimension.
Everything runs on `stream` (a raw handle; the current one of the tensors'
device by default), enqueued without waiting, and raises M3GError for what the
library refuses.  Given another stream than the current one, a call expects
its inputs to be ready there; results and workspaces that it allocates are
that stream's memory, kept until the current stream's work on them is done
too, and whoever reads them elsewhere waits for the stream first.  What the
kernels skip on the device (a sequence past the batch's limits, a page outside
the pool, a wait that ran out) raises nothing: matvec_quant.device_status says
so, and the rows stay as they were, which in a result allocated by the call,
as in its rows of no sequence, is whatever its memory held.  Autograd
does not see the calls: a tensor that requires a gradient is refused while
gradients are recorded, since the gradient would be lost without a word.
"""
from __future__ import annotations

import ctypes

from . import _lib

SCALINGS = {"none": 0, "linear": 1, "ntk": 2, "yarn": 3, "llama3": 4}
Q4_0, Q8_0 = 2, 8

# torch is imported at the first use: the host-side rules work without it.
torch = None
_dtypes: dict = {}


def _need_torch():
    """Binds torch and what each call needs of it (the raw getters cost a tenth of the checked ones)."""
    global torch, _int32, _current_device, _current_stream
    import torch as t

    torch, _int32 = t, t.int32
    _dtypes.update({t.float32: 0, t.float16: 1, t.bfloat16: 30})
    _current_device = getattr(t._C, "_cuda_getDevice", t.cuda.current_device)
    _current_stream = getattr(t._C, "_cuda_getCurrentRawStream", lambda i: t.cuda.current_stream(i).cuda_stream)


def act_dtype(t) -> int:
    """ggml number of an activation tensor's type."""
    if torch is None:
        _need_torch()
    number = _dtypes.get(t.dtype)
    if number is None:
        _fail(f"activations of type {t.dtype} (f32, f16 and bf16 are supported)")
    return number


def _device(t) -> int:
    if torch is None:
        _need_torch()
    i = t.get_device()
    if i < 0:
        _fail("the operators need CUDA tensors")
    return i


def _call(fn, device: int, stream, *args) -> None:
    """fn(*args, stream) with `device` current; stream None: the current one."""
    if stream is None:
        stream = _current_stream(device)
    if device == _current_device():
        rc = fn(*args, stream)
    else:
        with torch.cuda.device(device):
            rc = fn(*args, stream)
    if rc:
        _lib.check(rc)


def _fail(msg):
    raise _lib.M3GError(_lib.M3G_EINVAL, msg)


def _check_no_grad(name, t):
    if t.requires_grad and torch.is_grad_enabled():
        _fail(f"{name} requires a gradient, which this call does not record: torch.no_grad() or detach()")


def _check_rows(name, t, device=None, heads=None, head_dim=None, tokens=None):
    """t is (tokens, heads, head_dim) with a contiguous last dimension on `device`; returns its shape and strides."""
    shape = t.shape
    if len(shape) != 3:
        _fail(f"{name}: (tokens, heads, head_dim) is wanted, got {tuple(shape)}")
    _check_no_grad(name, t)
    strides = t.stride()
    if strides[2] != 1 and shape[2] > 1:
        _fail(f"{name}: the last dimension has to be contiguous")
    if device is not None and t.get_device() != device:
        _fail(f"{name} is on {t.device}, not on cuda:{device}")
    if (tokens is not None and shape[0] != tokens or heads is not None and shape[1] != heads
            or head_dim is not None and shape[2] != head_dim):
        _fail(f"{name} is {tuple(shape)}, not ({tokens}, {heads or 'heads'}, {head_dim})")
    return shape, strides


def _new_like(t):
    """An uninitialised contiguous tensor of t's shape and type (empty_like takes two thirds of new_empty's time)."""
    return torch.empty_like(t) if t.is_contiguous() else t.new_empty(t.shape)


def _on(device, stream, make, /, *args, **kw):
    """make(*args, **kw), a new tensor, for a call on `stream`.  The allocator takes it that a block is used on the stream
    that was current when it was handed out: a result made under another one could share its memory with that stream's
    pending work, or be handed out again before the call has written it."""
    if stream is None or stream == _current_stream(device):
        return make(*args, **kw)
    own = torch.cuda.ExternalStream(stream, device=device) if stream else torch.cuda.default_stream(device)
    with torch.cuda.stream(own):
        t = make(*args, **kw)
    t.record_stream(torch.cuda.current_stream(device))
    return t


def _check_sizes(what, *sizes):
    """Sizes that the library takes as 32 bits (ctypes would cut them)."""
    if min(sizes) < 0 or max(sizes) >= 2 ** 31:
        _fail(f"size of the {what} out of range")


def _check_ints(name, t, device, shape):
    if torch is None:
        _need_torch()
    if t.dtype is not _int32 or tuple(t.shape) != shape or not t.is_contiguous() or t.get_device() != device:
        _fail(f"{name}: a contiguous int32 tensor of shape {shape} on the device of the other tensors is wanted")


class _Told:
    """What the library was told once, by value and by address: the attributes made here stay.  (A changed n_tokens
    would pass the checks of the tensors, and the kernels would still go by the old one.)"""

    _told = frozenset()

    def _seal(self):
        self._told = frozenset(name for name in self.__dict__ if not name.startswith("_"))

    def __setattr__(self, name, value):
        if name in self._told:
            _fail(f"{type(self).__name__}.{name} cannot be changed: make a new {type(self).__name__}")
        object.__setattr__(self, name, value)


class Rope(_Told):
    """A plan of rotary positions (m3g_rope_config); host arithmetic, usable on every device.  The gradient of
    apply(...) is apply(..., inverse=True) of the results' gradients."""

    def __init__(self, head_dim: int, rot_dim: int | None = None, theta: float = 10000.0, interleaved: bool = False,
                 scaling: str = "none", factor: float = 1.0, orig_ctx: int = 0, low_freq: float = 1.0,
                 high_freq: float = 4.0, beta_fast: float = 32.0, beta_slow: float = 1.0, magnitude: float = 0.0):
        if scaling not in SCALINGS:
            _fail(f"scaling {scaling!r}: one of {', '.join(SCALINGS)} is wanted")
        rot_dim = head_dim if rot_dim is None else rot_dim
        _check_sizes("head", head_dim, rot_dim)
        self.head_dim = head_dim
        cfg = _lib.RopeConfig(head_dim, rot_dim, 1 if interleaved else 0,
                              SCALINGS[scaling], theta, factor, orig_ctx, low_freq, high_freq, beta_fast, beta_slow,
                              magnitude)
        h = ctypes.c_void_p()
        _lib.check(_lib.load().m3g_rope_create(ctypes.byref(cfg), ctypes.byref(h)))
        self._h = h
        self._seal()

    def apply(self, positions, q, k=None, q_out=None, k_out=None, inverse: bool = False, stream=None):
        """Turns q and k (k may be None) at int32 `positions` (tokens,); q_out, k_out may be q and k themselves.
        inverse: by the opposite angles, the gradient of the forward call."""
        dtype, n = act_dtype(q), positions.numel()
        device = _device(q)
        _check_ints("positions", positions, device, (n,))
        args, results = [], []
        for name, x, y in (("q", q, q_out), ("k", k, k_out)):
            if x is None:
                args.append(None)
                results.append(None)
                continue
            shape, sx = _check_rows(name, x, device, None, self.head_dim, n)
            heads = shape[1]
            if y is None:
                y, sy = _on(device, stream, _new_like, x), (heads * self.head_dim, self.head_dim)
            else:
                _, sy = _check_rows(name + "_out", y, device, heads, self.head_dim, n)
            if x.dtype is not q.dtype or y.dtype is not q.dtype:
                _fail("q, k and their results have one type")
            args.append(_lib.RopeRows(x.data_ptr(), y.data_ptr(), heads, sx[0], sx[1], sy[0], sy[1]))
            results.append(y)
        _call(_lib.load().m3g_rope_dev, device, stream, self._h, dtype, positions.data_ptr(), n, ctypes.byref(args[0]),
              ctypes.byref(args[1]) if args[1] is not None else None, 1 if inverse else 0)
        return results[0], results[1]

    def close(self) -> None:
        if getattr(self, "_h", None) and self._h.value:
            _lib.load().m3g_rope_destroy(self._h)
            self._h = ctypes.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


class KvBatch(_Told):
    """The new tokens of a batch of sequences (m3g_kv_batch).  `q_start` (n + 1,), `ctx_len` (n,) and `page_table`
    (n, max_pages) are int32 tensors of the GPU, read when an operator runs (a captured step replays with what they
    hold then); max_tokens and max_len bound what they may say."""

    def __init__(self, q_start, ctx_len, page_table, n_tokens: int, max_tokens: int, max_len: int):
        n = ctx_len.numel()
        self.device = q_start.get_device()
        _check_ints("q_start", q_start, self.device, (n + 1,))
        _check_ints("ctx_len", ctx_len, self.device, (n,))
        if page_table.dim() != 2:
            _fail("page_table: (sequences, pages) is wanted")
        _check_ints("page_table", page_table, self.device, (n, page_table.shape[1]))
        _check_sizes("batch", n_tokens, max_tokens, max_len)
        self.q_start, self.ctx_len, self.page_table = q_start, ctx_len, page_table
        self.n_tokens, self.max_tokens, self.max_len = n_tokens, max_tokens, max_len
        self.args = _lib.KvBatchArgs(q_start.data_ptr(), ctx_len.data_ptr(), page_table.data_ptr(), n,
                                     page_table.shape[1], n_tokens, max_tokens, max_len)
        self._seal()


class KvCache(_Told):
    """A paged cache of K and V rows in Q8_0 or Q4_0 blocks (m3g_kv_layout).  Its memory is one uint8 tensor, `pool`,
    allocated here (zeros) or the caller's own."""

    def __init__(self, dtype: int, n_layers: int, n_kv_heads: int, head_dim: int, page_size: int, n_pages: int,
                 device: int = 0, pool=None):
        if torch is None:
            _need_torch()
        _check_sizes("cache", n_layers, n_kv_heads, head_dim, page_size, n_pages)
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
        self.device = pool.get_device()
        self._workspace_bytes: dict[tuple, int] = {}
        self._seal()

    def _check_layer(self, layer):
        if not 0 <= layer < self.n_layers:  # here: the library would get its low 32 bits
            _fail(f"layer {layer} of {self.n_layers}")

    def _io(self, fn, layer, k, v, batch, stream):
        self._check_layer(layer)
        device, dtype = _device(self.pool), act_dtype(k)
        if k.dtype is not v.dtype:
            _fail("k and v have one type")
        if batch.device != device:
            _fail("the batch is on another device than the cache")
        rows = []
        for name, t in (("k", k), ("v", v)):
            _, strides = _check_rows(name, t, device, self.n_kv_heads, self.head_dim, batch.n_tokens)
            rows.append(_lib.Rows(t.data_ptr(), strides[0], strides[1]))
        _call(fn, device, stream, ctypes.byref(self.layout), self.pool.data_ptr(), layer, ctypes.byref(batch.args),
              dtype, ctypes.byref(rows[0]), ctypes.byref(rows[1]))

    def write(self, layer: int, k, v, batch: KvBatch, stream=None) -> None:
        """Quantises the new tokens' rows into their places."""
        self._io(_lib.load().m3g_kv_write_dev, layer, k, v, batch, stream)

    def read(self, layer: int, batch: KvBatch, dtype=None, k_out=None, v_out=None, stream=None):
        """The values held at the new tokens' places, as (k, v) of `dtype` (f32 by default)."""
        device, shape = _device(self.pool), (batch.n_tokens, self.n_kv_heads, self.head_dim)
        if k_out is None:
            k_out = _on(device, stream, torch.empty, shape, dtype=dtype or torch.float32, device=self.pool.device)
        if v_out is None:
            v_out = _on(device, stream, _new_like, k_out)
        self._io(_lib.load().m3g_kv_read_dev, layer, k_out, v_out, batch, stream)
        return k_out, v_out

    def attention_workspace(self, n_heads: int, dtype=None, max_tokens: int = 1) -> int:
        """Bytes of workspace that attention of n_heads query heads of `dtype` (f32 by default) over at most max_tokens
        new tokens of a sequence needs."""
        number = 0 if dtype is None else _dtypes.get(dtype)
        key = (n_heads, number, max_tokens)
        got = self._workspace_bytes.get(key)
        if got is None:
            if number is None:
                _fail(f"attention of type {dtype} (f32, f16 and bf16 are supported)")
            _check_sizes("attention", n_heads, max_tokens)
            need = ctypes.c_uint64()
            _lib.check(_lib.load().m3g_tree_attn_workspace(ctypes.byref(self.layout), key[1], n_heads, max_tokens,
                                                           ctypes.byref(need)))
            got = self._workspace_bytes[key] = need.value
        return got


def tree_attention(q, cache: KvCache, layer: int, batch: KvBatch, mask=None, scale: float | None = None, out=None,
                   workspace=None, stream=None):
    """Attention of the batch's new tokens (already written) over the cache.  `mask`: int32 (tokens, words), bit i % 32
    of word i / 32 says whether the token sees new token i of its sequence; None: all up to and including itself.
    `workspace`: a uint8 tensor of cache.attention_workspace(heads, q.dtype, batch.max_tokens) bytes, used by one call
    at a time (allocated here when None)."""
    if scale is not None and not ctypes.c_float(scale).value > 0:  # in 32 bits, where 0 stands for the default
        _fail("scale must be positive")
    cache._check_layer(layer)
    device, dtype = _device(q), act_dtype(q)
    shape, sq = _check_rows("q", q, cache.device, None, cache.head_dim, batch.n_tokens)
    heads = shape[1]
    if out is None:
        out, so = _on(device, stream, _new_like, q), (heads * cache.head_dim, cache.head_dim)
    else:
        if out.dtype is not q.dtype:
            _fail("q and out have one type")
        _, so = _check_rows("out", out, device, heads, cache.head_dim, batch.n_tokens)
    if batch.device != device:
        _fail("the batch is on another device than q")
    words, bits = 0, None
    if mask is not None:
        words = mask.shape[-1] if mask.dim() == 2 else 0
        _check_ints("mask", mask, device, (batch.n_tokens, words))
        bits = mask.data_ptr()
    if workspace is None:
        workspace = _on(device, stream, cache.pool.new_empty,
                        cache.attention_workspace(heads, q.dtype, batch.max_tokens))
    elif workspace.dtype is not torch.uint8 or workspace.get_device() != device or not workspace.is_contiguous():
        _fail("workspace: a contiguous uint8 tensor on q's device is wanted")
    rq, ro = _lib.Rows(q.data_ptr(), sq[0], sq[1]), _lib.Rows(out.data_ptr(), so[0], so[1])
    _call(_lib.load().m3g_tree_attn_dev, device, stream, ctypes.byref(cache.layout), cache.pool.data_ptr(), layer,
          ctypes.byref(batch.args), dtype, ctypes.byref(rq), heads, bits, words, scale or 0.0, ctypes.byref(ro),
          workspace.data_ptr(), workspace.numel())
    return out
