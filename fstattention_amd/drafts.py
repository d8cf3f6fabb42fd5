"""Which drafted tokens stand: trees or chains of drafts against the model's logits, from given random numbers.

The reference stops at the attention of a tree's nodes (``fstattention.py:153-181``); what a program of speculative decoding does
with the logits behind it is here.  The compute is ``libfsta.so``'s (``include/fsta.h``), on torch's current stream; there is no
CPU fallback."""
from __future__ import annotations

from typing import NamedTuple, Optional, Union

import torch

from . import _lib
from . import attention as _attention
from .attention import _on_device, _stream_ptr

_FLOATS = {torch.float32: _lib.F32, torch.float16: _lib.F16, torch.bfloat16: _lib.BF16}


class Verified(NamedTuple):
    """``path`` int32 ``[B, max_path]``: the accepted nodes' numbers within their tree from the root, -1 behind them; ``counts`` int32
    ``[B]``: how many; ``next_tokens`` int64 ``[B]``: the token behind each path."""
    path: torch.Tensor
    counts: torch.Tensor
    next_tokens: torch.Tensor


def _calls():
    return _attention._CALLS or _attention._calls()


def _check_rows(t: torch.Tensor, name: str, like: torch.Tensor):
    if t.dim() != 2 or t.dtype not in _FLOATS:
        raise ValueError(f"{name} must be [nodes, vocabulary] of float32, float16 or bfloat16")
    if t.device != like.device:
        raise ValueError("all tensors must live on the same device")
    if t.numel() and t.shape[1] > 1 and t.stride(1) != 1:
        raise ValueError(f"{name}'s rows must be contiguous")
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _check_array(t: torch.Tensor, name: str, dtype: torch.dtype, size: int, like: torch.Tensor):
    if t.dtype != dtype or tuple(t.shape) != (size,) or not t.is_contiguous() or t.device != like.device:
        raise ValueError(f"{name} must be a contiguous {str(dtype).split('.')[1]} tensor [{size}] on the logits' device")
    return t.data_ptr()


def verify_drafts(logits: torch.Tensor, tokens: torch.Tensor, parent: torch.Tensor, q_starts: torch.Tensor, u_accept: torch.Tensor,
                  u_next: torch.Tensor, max_path: int, *, temperature: Union[float, torch.Tensor] = 1.0,
                  draft_probs: Optional[torch.Tensor] = None) -> Verified:
    """The accepted path of every draft tree of a batch, and the token behind it.

    ``logits [T, V]`` (float32, float16 or bfloat16; rows may be slices of longer ones): row ``t`` is what the model says behind node
    ``t``.  ``tokens, parent`` int64 ``[T]`` and ``q_starts`` int32 ``[B + 1]``: the trees, packed as :func:`tree_mask_bits` takes them
    (a chain of drafts is a tree whose parents are 0, 1, 2, ..).  Node 0 of a tree stands: it is the newest token of its conversation;
    other roots are never reached.  ``u_accept [T], u_next [B]`` float32: random numbers in [0, 1), one for each node's acceptance, one
    for each next token.  ``temperature``: a number, or float32 ``[B]`` on the GPU; 0 (or less, or NaN, in a tensor) takes the largest
    logit, the first of equals.  Tokens that may not be chosen (top-k, top-p, a grammar) have logits of -inf.

    ``draft_probs [T, V]``: row ``t`` holds the probabilities from which node ``t``'s children were drawn, one after the other in the
    order of their numbers, no token twice (rows of leaves are not read).  Without it the children are taken for a given list, such as a
    draft head's best guesses.  In both cases the token behind what was committed so far is distributed as the model's own: a drafted one
    where a child stands, ``next_tokens`` otherwise.  Answers are those of sums and comparisons in 64 bits: equal inputs give equal answers,
    whatever the batch.

    A path ends at ``max_path`` nodes (the depth of the trees plus 1 loses nothing, and more costs launches); of a node's children the first
    2048 are asked.  A row of nothing but -inf (or NaN, which counts as that) leaves no token: ``next_tokens`` is -1; logits of +inf share all
    mass.  Sequences without nodes have no path and no token (0 and -1).  ``path`` and ``counts`` are what :func:`compact_paged_kv` takes."""
    out = _calls().verify_drafts(logits, tokens, parent, q_starts, u_accept, u_next, max_path, temperature, draft_probs)
    if out is not NotImplemented:
        return Verified(*out)
    if not logits.is_cuda:
        raise ValueError("verify_drafts runs on the GPU only (no CPU fallback)")
    stride = _check_rows(logits, "logits", logits)
    nodes, vocabulary = logits.shape
    if vocabulary < 1:
        raise ValueError("logits must have a vocabulary")
    draft_stride = 0
    if draft_probs is not None:
        draft_stride = _check_rows(draft_probs, "draft_probs", logits)
        if draft_probs.shape != logits.shape:
            raise ValueError(f"draft_probs must be [{nodes}, {vocabulary}] like logits, got {tuple(draft_probs.shape)}")
    if q_starts.dim() != 1 or q_starts.shape[0] < 1:
        raise ValueError("q_starts must be int32 [batch + 1]")
    batch = q_starts.shape[0] - 1
    if max_path < 1:
        raise ValueError(f"max_path={max_path} must be at least 1")
    pointers = [_check_array(tokens, "tokens", torch.int64, nodes, logits), _check_array(parent, "parent", torch.int64, nodes, logits),
                _check_array(q_starts, "q_starts", torch.int32, batch + 1, logits), _check_array(u_accept, "u_accept", torch.float32, nodes, logits),
                _check_array(u_next, "u_next", torch.float32, batch, logits)]
    if isinstance(temperature, torch.Tensor):
        temperatures, value = _check_array(temperature, "temperature", torch.float32, batch, logits), 0.0
    else:
        temperatures, value = None, float(temperature)
        if not 0 <= value < float("inf"):
            raise ValueError(f"temperature={temperature} must be 0 or more")
    lib = _lib.load()
    dev = logits.device
    path = torch.empty((batch, max_path), dtype=torch.int32, device=dev)
    counts = torch.empty((batch,), dtype=torch.int32, device=dev)
    next_tokens = torch.empty((batch,), dtype=torch.int64, device=dev)
    code = _FLOATS[logits.dtype]
    need = lib.fsta_verify_workspace_bytes(batch, nodes, vocabulary, max_path, draft_probs is not None)
    work = torch.empty((need,), dtype=torch.uint8, device=dev)
    with _on_device(dev):
        _lib.check(lib.fsta_verify_drafts(logits.data_ptr(), stride, code, None if draft_probs is None else draft_probs.data_ptr(), draft_stride,
                                          _lib.F32 if draft_probs is None else _FLOATS[draft_probs.dtype], *pointers, temperatures, value,
                                          path.data_ptr(), counts.data_ptr(), next_tokens.data_ptr(), batch, nodes, vocabulary, max_path,
                                          work.data_ptr() if need else None, need, _stream_ptr(dev)))
    return Verified(path, counts, next_tokens)
