"""Log probabilities of given tokens, entropy and the most probable
alternatives of rows of logits, on CUDA tensors (m3g_token_logprobs_dev)."""
from __future__ import annotations

from typing import NamedTuple

from . import _lib
from .attention import _call, _check_ints, _check_no_grad, _device, _fail, _on, act_dtype


class TokenLogprobs(NamedTuple):
    logprob: object       # (rows, tokens) f32, None without tokens
    entropy: object       # (rows,) f32, None unless asked for
    top_ids: object       # (rows, n_top) int32, None with n_top 0
    top_logprobs: object  # (rows, n_top) f32, None with n_top 0


def token_logprobs(logits, tokens=None, n_top: int = 0, entropy: bool = False, stream=None) -> TokenLogprobs:
    """logits (rows, vocab) f32, f16 or bf16 with a contiguous last dimension; tokens int32 (rows, n) ids whose log
    probabilities are wanted (-inf for an id outside the vocabulary), at most 512 a row; n_top <= 32 most probable ids
    of each row.  `stream` as in m3_avm_b200.attention."""
    import torch

    if logits.dim() != 2 or (logits.shape[1] > 1 and logits.stride(1) != 1):
        _fail("logits: (rows, vocab) with a contiguous last dimension is wanted")
    if not 0 <= n_top <= 32:
        _fail(f"{n_top} alternatives (at most 32)")
    rows, vocab = logits.shape
    device, dtype = _device(logits), act_dtype(logits)
    _check_no_grad("logits", logits)
    n = 0
    lp = ent = ids = tops = None
    if tokens is not None:
        n = tokens.shape[-1] if tokens.dim() == 2 else -1
        _check_ints("tokens", tokens, device, (rows, n))
        lp = _on(device, stream, torch.empty_like, tokens, dtype=torch.float32)
    if entropy:
        ent = _on(device, stream, logits.new_empty, (rows,), dtype=torch.float32)
    if n_top:
        ids = _on(device, stream, logits.new_empty, (rows, n_top), dtype=torch.int32)
        tops = _on(device, stream, torch.empty_like, ids, dtype=torch.float32)
    ptr = lambda t: t.data_ptr() if t is not None else None  # noqa: E731
    _call(_lib.load().m3g_token_logprobs_dev, device, stream, dtype, logits.data_ptr(), rows, vocab, logits.stride(0),
          ptr(tokens), n, ptr(lp), ptr(ent), n_top, ptr(ids), ptr(tops))
    return TokenLogprobs(lp, ent, ids, tops)
