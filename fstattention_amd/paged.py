"""A KV cache in pages: writing new tokens to it, attending to it, reading it back.

The reference's K and V are dense ``[prefix | tree]`` tensors (``fstattention.py:188-196``); a program that serves
several sequences keeps theirs in pages.  Three arrays describe a batch, on the GPU and never read by the host:

* ``page_table`` int32 ``[B, W]``: position ``p`` of sequence ``b`` is row ``p % page_size`` of page
  ``page_table[b, p // page_size]``; entries outside ``[0, num_pages)`` name no page.
* ``kv_lens`` int32 ``[B]``: positions of every sequence, its new tokens included.
* ``q_starts`` int32 ``[B + 1]``, ascending: tokens ``q_starts[b]`` to ``q_starts[b + 1] - 1`` of the packed tensors
  (``q [T, H, D]``, ``k, v [T, Hkv, D]``) are sequence ``b``'s new ones, at its last positions.

The compute is ``libfsta.so``'s (``include/fsta.h``), on torch's current stream; there is no CPU fallback.  No operator has a
derivative: rows or caches that require a gradient, or carry a tangent, are refused.
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch
from torch.autograd import forward_ad
from torch.autograd.graph import increment_version

from . import _lib
from . import attention as _attention
from .attention import _on_device, _stream_ptr

_HALF = {torch.float16: _lib.F16, torch.bfloat16: _lib.BF16}
_CACHE = {**_HALF, torch.float8_e4m3fn: _lib.FP8}


class PagedKV(NamedTuple):
    """The cache of one layer: ``k, v [num_pages, Hkv, page_size, D]`` (float16, bfloat16, or float8_e4m3fn), and for 8-bit
    rows ``k_exponent, v_exponent`` uint8 ``[num_pages, Hkv, page_size]``: a row's value is ``k * 2.0 ** (k_exponent - 127)``."""
    k: torch.Tensor
    v: torch.Tensor
    k_exponent: Optional[torch.Tensor] = None
    v_exponent: Optional[torch.Tensor] = None


def _calls():
    """The module of plain C functions: what it takes of a call it has launched, for anything else it answers NotImplemented and
    the checks below say why (or launch what it did not want to judge)."""
    return _attention._CALLS or _attention._calls()


def paged_kv_cache(num_pages: int, kv_heads: int, page_size: int, head_dim: int, dtype: torch.dtype = torch.bfloat16,
                   device="cuda") -> PagedKV:
    """An empty cache.  ``page_size``: a power of two from 16 to 4096; ``head_dim``: 64 or 128; ``dtype``: float16, bfloat16, or
    float8_e4m3fn (half the memory and traffic; rows are kept as e4m3 bytes times a power of two each)."""
    if dtype not in _CACHE:
        raise ValueError("a paged cache is float16, bfloat16 or float8_e4m3fn")
    shape = (num_pages, kv_heads, page_size, head_dim)
    k, v = torch.zeros(shape, dtype=dtype, device=device), torch.zeros(shape, dtype=dtype, device=device)
    if dtype != torch.float8_e4m3fn:
        return PagedKV(k, v)
    return PagedKV(k, v, *(torch.full(shape[:3], 127, dtype=torch.uint8, device=device) for _ in range(2)))


def _refuse_derivatives(name: str, t: torch.Tensor):
    if t.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{name} requires a gradient: the paged cache's operators have no backward pass")
    if forward_ad.unpack_dual(t).tangent is not None:
        raise ValueError(f"{name} carries a tangent: the paged cache's operators have no forward-mode derivative")


def _check_cache(cache: PagedKV):
    """(num_pages, kv_heads, page_size, head_dim, dtype code, exponent pointers)"""
    k, v = cache.k, cache.v
    if k.dim() != 4 or v.shape != k.shape or v.dtype != k.dtype:
        raise ValueError("the cache's k and v must be [num_pages, kv_heads, page_size, head_dim] of one shape and dtype")
    if k.dtype not in _CACHE:
        raise ValueError("a paged cache is float16, bfloat16 or float8_e4m3fn")
    if not k.is_cuda or v.device != k.device:
        raise ValueError("a paged cache lives on the GPU (no CPU fallback)")
    if not (k.is_contiguous() and v.is_contiguous()):
        raise ValueError("the cache's k and v must be contiguous")
    _refuse_derivatives("the cache's k", k)
    _refuse_derivatives("the cache's v", v)
    exponents = (cache.k_exponent, cache.v_exponent)
    if k.dtype == torch.float8_e4m3fn:
        for e in exponents:
            if e is None or e.dtype != torch.uint8 or e.shape != k.shape[:3] or not e.is_contiguous() or e.device != k.device:
                raise ValueError("an 8-bit cache needs contiguous uint8 k_exponent and v_exponent [num_pages, kv_heads, page_size]")
    elif any(e is not None for e in exponents):
        raise ValueError("k_exponent / v_exponent belong to an 8-bit cache (float8_e4m3fn)")
    return (*k.shape, _CACHE[k.dtype], *(None if e is None else e.data_ptr() for e in exponents))


def _check_arrays(cache: PagedKV, page_table, kv_lens, q_starts=None):
    """(batch, width)"""
    if page_table.dim() != 2 or kv_lens.shape != page_table.shape[:1]:
        raise ValueError("page_table must be [batch, width] and kv_lens [batch]")
    if q_starts is not None and tuple(q_starts.shape) != (page_table.shape[0] + 1,):
        raise ValueError("q_starts must be [batch + 1]")
    for t in (page_table, kv_lens) + (() if q_starts is None else (q_starts,)):
        if t.dtype != torch.int32 or not t.is_contiguous() or t.device != cache.k.device:
            raise ValueError("page_table, kv_lens and q_starts must be contiguous int32 tensors on the cache's device")
    return page_table.shape


def _check_rows(t: torch.Tensor, name: str, cache: PagedKV):
    """(token stride, head stride) of packed rows [tokens, heads, head_dim]"""
    if t.dim() != 3 or t.shape[2] != cache.k.shape[3]:
        raise ValueError(f"{name} must be [tokens, heads, head_dim={cache.k.shape[3]}], got {tuple(t.shape)}")
    if t.dtype not in _HALF or (cache.k.dtype != torch.float8_e4m3fn and t.dtype != cache.k.dtype):
        raise ValueError(f"{name} must be float16 or bfloat16, and of the cache's dtype unless that is 8 bits")
    if t.device != cache.k.device:
        raise ValueError("all tensors must live on the same device")
    _refuse_derivatives(name, t)
    strides = [t.stride(d) if t.shape[d] > 1 else 0 for d in (0, 1)]
    if t.numel() and (t.stride(2) != 1 or any(s % 8 for s in strides) or t.data_ptr() % 16):
        raise ValueError(f"{name}'s rows must be contiguous and 16-byte aligned (strides that are multiples of 8)")
    return strides


def write_paged_kv(cache: PagedKV, k: torch.Tensor, v: torch.Tensor, page_table: torch.Tensor, kv_lens: torch.Tensor,
                   q_starts: torch.Tensor) -> None:
    """Rows ``k, v [T, Hkv, D]`` of the new tokens (views with strides that are multiples of 8 elements are fine: slices of a
    fused projection) to their places in the pages; tokens without a place are left out.

    An 8-bit cache gets, per row, the smallest exponent ``e`` with ``max |x| <= 448 * 2**e`` over the row's finite values
    (kept within [-110, 120]; 0 for a row of zeros) and bytes rounded to nearest even; infinities and NaNs become NaN.  The version
    counters of the tensors written to move, as by an operation in place of torch's own."""
    if _calls().paged_write(cache, k, v, page_table, kv_lens, q_starts) is None:
        return
    pages, heads, page_size, d, code, k_exp, v_exp = _check_cache(cache)
    batch, width = _check_arrays(cache, page_table, kv_lens, q_starts)
    k_strides, v_strides = _check_rows(k, "k", cache), _check_rows(v, "v", cache)
    if k.shape != v.shape or k.shape[1] != heads or k.dtype != v.dtype:
        raise ValueError(f"k and v must both be [tokens, {heads}, {d}] of one dtype")
    lib = _lib.load()
    with _on_device(cache.k.device):
        _lib.check(lib.fsta_paged_write(k.data_ptr(), v.data_ptr(), *k_strides, *v_strides, cache.k.data_ptr(), cache.v.data_ptr(),
                                        k_exp, v_exp, page_table.data_ptr(), kv_lens.data_ptr(), q_starts.data_ptr(), batch, width,
                                        k.shape[0], pages, page_size, heads, d, _HALF[k.dtype], code, _stream_ptr(cache.k.device)))
    # autograd is told, as by torch's own operations in place (inference tensors have no version counter)
    increment_version([t for t in cache if t is not None and not t.is_inference()])


def read_paged_kv(cache: PagedKV, page_table: torch.Tensor, kv_lens: torch.Tensor, max_len: int,
                  dtype: Optional[torch.dtype] = None):
    """The pages of a batch as dense ``k, v [B, Hkv, max_len, D]`` (the layout ``fst_attention`` takes), zeros where a sequence
    has no position.  ``dtype``: the cache's, or float16 / bfloat16 for an 8-bit one (bfloat16 if not given, which holds its values
    exactly; float16 rounds them, beyond 65504 to infinities)."""
    out = _calls().paged_read(cache, page_table, kv_lens, max_len, dtype)
    if out is not NotImplemented:
        return out
    pages, heads, page_size, d, code, k_exp, v_exp = _check_cache(cache)
    batch, width = _check_arrays(cache, page_table, kv_lens)
    fp8 = cache.k.dtype == torch.float8_e4m3fn
    dtype = dtype or (torch.bfloat16 if fp8 else cache.k.dtype)
    if dtype not in _HALF or (not fp8 and dtype != cache.k.dtype):
        raise ValueError("dtype must be float16 or bfloat16, and the cache's own unless that is 8 bits")
    if max_len < 0:
        raise ValueError(f"max_len={max_len}")
    lib = _lib.load()
    k = torch.empty((batch, heads, max_len, d), dtype=dtype, device=cache.k.device)
    v = torch.empty_like(k)
    with _on_device(cache.k.device):
        _lib.check(lib.fsta_paged_read(cache.k.data_ptr(), cache.v.data_ptr(), k_exp, v_exp, page_table.data_ptr(), kv_lens.data_ptr(),
                                       k.data_ptr(), v.data_ptr(), batch, width, max_len, pages, page_size, heads, d, _HALF[dtype],
                                       code, _stream_ptr(cache.k.device)))
    return k, v


def paged_attention(q: torch.Tensor, cache: PagedKV, page_table: torch.Tensor, kv_lens: torch.Tensor, q_starts: torch.Tensor,
                    sm_scale: float, *, causal: bool = True, tree_bits: Optional[torch.Tensor] = None,
                    max_q_len: Optional[int] = None, return_lse: bool = False):
    """Attention of a batch's new tokens ``q [T, H, D]`` over each sequence's pages -> ``o [T, H, D]``, typed like ``q``.

    The new tokens' own keys and values are in the cache already (:func:`write_paged_kv`); ``H`` is a multiple of the cache's
    ``Hkv``, query head ``h`` sees K/V head ``h // (H // Hkv)``.  A sequence may bring one token, a chunk of a prompt or a draft
    tree.  With ``causal`` a token sees the positions up to its own; with ``tree_bits`` (:func:`tree_mask_bits`: int32
    ``[T, words]``) all positions in front of the new tokens and, among those, the ones of its row of bits; with neither, every
    position of its sequence.  ``return_lse``: also the base-2 log-sum-exp ``[T, H]`` float32, e.g. to join the result with
    another part's by :func:`merge_attention_states`.  ``max_q_len``: the most new tokens a sequence has, if the caller knows.  It
    steers the choice of kernel, and by that the rounding of the weights (below), nothing else; without it every sequence is taken
    to bring a token, unless there are fewer tokens than sequences: a batch of mostly empty slots is faster with it (256 slots,
    260 tokens of one behind 8000 keys: 73 us instead of 111).

    Tokens that see nothing get zeros (and ``-inf``); rows of tokens that ``q_starts`` gives to no sequence are not written.
    Sums and softmax statistics are float32 (finite values of up to 1e24 in magnitude do not leave it).  The weights' rounding: where
    a workgroup takes up to 64 rows (tokens times query heads per K/V head: short chunks, and small calls; the longest chunk of a
    batch decides for all), bfloat16 weights go to the matrix cores as pairs (2^-16 relative at most), elsewhere rounded once (2^-8
    at most, as the output itself).  float16 weights over a 16-bit cache are rounded once everywhere (2^-11, those below 2^-14 of the
    running maximum's to 2^-25 of it), over an 8-bit cache they are pairs of bfloat16."""
    out = _calls().paged_attention(q, cache, page_table, kv_lens, q_starts, sm_scale, causal, tree_bits, max_q_len, return_lse)
    if out is not NotImplemented:
        return out
    pages, heads_kv, page_size, d, code, k_exp, v_exp = _check_cache(cache)
    batch, width = _check_arrays(cache, page_table, kv_lens, q_starts)
    q_strides = _check_rows(q, "q", cache)
    tokens, heads = q.shape[0], q.shape[1]
    if heads == 0 or heads_kv == 0 or heads % heads_kv:
        raise ValueError(f"{heads} query heads do not share {heads_kv} K/V heads evenly")
    if not sm_scale > 0 or sm_scale == float("inf"):
        raise ValueError(f"sm_scale={sm_scale} must be positive")
    if max_q_len is not None and max_q_len < 0:
        raise ValueError(f"max_q_len={max_q_len}")
    words, bits, mask = 0, None, _lib.PAGED_CAUSAL if causal else _lib.PAGED_ALL
    if tree_bits is not None:
        if tree_bits.dtype != torch.int32 or tree_bits.dim() != 2 or tree_bits.shape[0] != tokens or not tree_bits.is_contiguous() or \
                tree_bits.device != q.device:
            raise ValueError("tree_bits must be a contiguous int32 tensor [tokens, words] on q's device")
        words, bits, mask = tree_bits.shape[1], tree_bits.data_ptr(), _lib.PAGED_TREE
    if tokens and (batch == 0 or width == 0 or pages == 0):
        raise ValueError(f"{tokens} tokens need sequences and a cache with pages")
    lib = _lib.load()
    max_q_len = max_q_len or 0
    o = torch.empty((tokens, heads, d), dtype=q.dtype, device=q.device)
    lse = torch.empty((tokens, heads), dtype=torch.float32, device=q.device) if return_lse else None
    need = lib.fsta_paged_attention_workspace_bytes(batch, tokens, max_q_len, heads, heads_kv, d, code)
    work = torch.empty((need,), dtype=torch.uint8, device=q.device)
    with _on_device(q.device):
        _lib.check(lib.fsta_paged_attention(q.data_ptr(), *q_strides, cache.k.data_ptr(), cache.v.data_ptr(), k_exp, v_exp,
                                            page_table.data_ptr(), kv_lens.data_ptr(), q_starts.data_ptr(), bits, words, o.data_ptr(),
                                            None if lse is None else lse.data_ptr(), batch, width, tokens, max_q_len, pages, page_size,
                                            heads, heads_kv, d, _HALF[q.dtype], code, mask, sm_scale, work.data_ptr(), need,
                                            _stream_ptr(q.device)))
    return (o, lse) if return_lse else o


def tree_mask_bits(parent: torch.Tensor, q_starts: Optional[torch.Tensor] = None, max_nodes: Optional[int] = None) -> torch.Tensor:
    """Masks of a batch of draft trees for :func:`paged_attention`: int32 ``[T, ceil(max_nodes / 32)]``, bit ``j % 32`` of word
    ``j // 32`` of a node's row set where ``j`` is the node or one of its ancestors.

    ``parent`` int64 ``[T]``: every node's parent by its number within its tree, smaller than its own, -1 for a root (as in
    ``lineage_from_parents``; anything else counts as a root).  ``q_starts`` int32 ``[B + 1]``: tree ``b``'s nodes (one tree if
    not given).  ``max_nodes``: the most nodes a tree has (``T`` if not given; below 2^31); bits beyond it are dropped."""
    bits = _calls().tree_bits(parent, q_starts, max_nodes)
    if bits is not NotImplemented:
        return bits
    if parent.dim() != 1 or parent.dtype != torch.int64:
        raise ValueError("parent must be int64 [tokens]")
    if not parent.is_cuda:
        raise ValueError("tree_mask_bits runs on the GPU only (no CPU fallback)")
    tokens = parent.shape[0]
    if q_starts is None:
        q_starts = torch.arange(2, dtype=torch.int32, device=parent.device) * tokens      # (made there: a copy cannot be captured)
    if q_starts.dim() != 1 or q_starts.dtype != torch.int32 or q_starts.shape[0] < 2 or q_starts.device != parent.device:
        raise ValueError("q_starts must be int32 [batch + 1] on parent's device, of at least one sequence")
    max_nodes = tokens if max_nodes is None else max_nodes
    if not 0 <= max_nodes < 2 ** 31:
        raise ValueError(f"max_nodes={max_nodes}")
    lib = _lib.load()
    parent, q_starts = parent.contiguous(), q_starts.contiguous()
    bits = torch.empty((tokens, (max_nodes + 31) // 32), dtype=torch.int32, device=parent.device)
    with _on_device(parent.device):
        _lib.check(lib.fsta_tree_bits(parent.data_ptr(), q_starts.data_ptr(), q_starts.shape[0] - 1, tokens, bits.shape[1],
                                      bits.data_ptr(), _stream_ptr(parent.device)))
    return bits
