"""The pages of a paged KV cache between two passes of a model: rows of accepted drafts moved together, pages given to sequences,
shared among them, copied, taken back.

The arrays are those of :mod:`fstattention_amd.paged`, and like there the host reads none of them: nothing here waits for the GPU.
Beside them a program keeps ``refs`` int32 ``[num_pages]``: by how many entries of the page table a page is held.  A page with 0 is free,
so ``torch.zeros`` (and a page table of -1) is where a server starts; from then on only the calls here change both.  ``caches`` is a
:class:`PagedKV` or a list or tuple of them, one per layer (a plain tuple of its four tensors will do); they share ``num_pages`` and
``page_size``, so that one page table serves all, and may differ in heads, head_dim and dtype.  All layers go in one launch (32 at a time).

The compute is ``libfsta.so``'s (``include/fsta.h``), on torch's current stream; there is no CPU fallback.  Tensors are changed in place,
and their version counters move, as by an operation in place of torch's own; caches that require a gradient, or carry a tangent, are refused.
"""
from __future__ import annotations

from typing import List, Optional, Sequence, Union

import torch
from torch.autograd.graph import increment_version

from . import _lib
from .attention import _on_device, _stream_ptr
from .paged import PagedKV, _calls, _check_cache

Caches = Union[PagedKV, Sequence[PagedKV]]


def _check_caches(caches: Caches, name: str = "caches"):
    """(layers, num_pages, page_size, the host array of fsta_paged_pool)"""
    layers: List[PagedKV] = [caches] if isinstance(caches, PagedKV) else [PagedKV(*c) for c in caches]
    if not layers:
        raise ValueError(f"{name} must hold at least one layer's cache")
    pools = (_lib.PagedPool * len(layers))()
    for c, pool in zip(layers, pools):
        pages, heads, page_size, d, code, k_exp, v_exp = _check_cache(c)
        if (pages, page_size) != (layers[0].k.shape[0], layers[0].k.shape[2]):
            raise ValueError(f"{name} must share num_pages and page_size")
        if c.k.device != layers[0].k.device:
            raise ValueError("all tensors must live on the same device")
        pool.k, pool.v, pool.k_exponent, pool.v_exponent = c.k.data_ptr(), c.v.data_ptr(), k_exp, v_exp
        pool.kv_heads, pool.head_dim, pool.cache_dtype = heads, d, code
    return layers, layers[0].k.shape[0], layers[0].k.shape[2], pools


def _check_int32(t: torch.Tensor, name: str, shape, like: torch.Tensor) -> int:
    if t.dtype != torch.int32 or tuple(t.shape) != tuple(shape) or not t.is_contiguous() or t.device != like.device:
        raise ValueError(f"{name} must be a contiguous int32 tensor {list(shape)} on the caches' device")
    return t.data_ptr()


def _written(layers, *arrays):
    increment_version([t for c in layers for t in c if t is not None and not t.is_inference()] + [t for t in arrays if not t.is_inference()])


def compact_paged_kv(caches: Caches, path: torch.Tensor, counts: torch.Tensor, page_table: torch.Tensor, kv_lens: torch.Tensor,
                     q_starts: torch.Tensor) -> torch.Tensor:
    """The rows of each sequence's accepted nodes move to the places directly behind what it had before the tree, in all layers;
    returns the lengths ``[B]`` that this leaves.

    ``kv_lens`` and ``q_starts`` are those of the pass that wrote the tree (new tokens included); ``path`` int32 ``[B, P]`` and ``counts`` int32
    ``[B]`` are :func:`verify_drafts`' (node numbers within each tree, ascending): row ``base + path[b, i]`` goes to ``base + i`` for the first
    ``counts[b]``, ``base = kv_lens[b]`` minus its new tokens.  Entries outside the new tokens, and rows without a page, move nothing.
    Rows move in place: no layer may be there twice."""
    out = _calls().compact_paged_kv(caches, path, counts, page_table, kv_lens, q_starts)
    if out is not NotImplemented:
        return out
    layers, pages, page_size, pools = _check_caches(caches)
    k = layers[0].k
    if page_table.dim() != 2 or path.dim() != 2:
        raise ValueError("page_table must be [batch, width] and path [batch, most nodes]")
    batch, width = page_table.shape
    pointers = [_check_int32(path, "path", (batch, path.shape[1]), k), _check_int32(counts, "counts", (batch,), k),
                _check_int32(page_table, "page_table", (batch, width), k), _check_int32(kv_lens, "kv_lens", (batch,), k),
                _check_int32(q_starts, "q_starts", (batch + 1,), k)]
    lens = torch.empty((batch,), dtype=torch.int32, device=k.device)
    with _on_device(k.device):
        _lib.check(_lib.load().fsta_compact_paged_kv(pools, len(layers), pages, page_size, pointers[0], path.shape[1], *pointers[1:], batch, width,
                                                     lens.data_ptr(), _stream_ptr(k.device)))
    _written(layers)
    return lens


def copy_pages(caches: Caches, sources: torch.Tensor, targets: torch.Tensor, into: Optional[Caches] = None) -> None:
    """Page ``sources[i]`` goes to page ``targets[i]`` (int32 ``[N]``), in all layers: within ``caches``, or to the same layers of other caches
    ``into`` (a larger pool, say).  Pairs with a number that names no page are left out.  No page may be the target of two pairs, or of one
    and the source of another: what it holds then is not defined."""
    if _calls().copy_pages(caches, sources, targets, into) is None:
        return
    layers, pages, page_size, pools = _check_caches(caches)
    others, into_pages, into_size, into_pools = (layers, pages, page_size, pools) if into is None else _check_caches(into, "into")
    k = layers[0].k
    if len(others) != len(layers) or into_size != page_size or any(
            a.k.shape[1] != b.k.shape[1] or a.k.shape[3] != b.k.shape[3] or a.k.dtype != b.k.dtype or a.k.device != b.k.device for a, b in zip(layers, others)):
        raise ValueError("into must have the layers of caches: heads, page_size, head_dim, dtype and device")
    if sources.dim() != 1:
        raise ValueError("sources and targets must be [pairs]")
    pointers = [_check_int32(sources, "sources", sources.shape, k), _check_int32(targets, "targets", sources.shape, k)]
    with _on_device(k.device):
        _lib.check(_lib.load().fsta_copy_pages(pools, into_pools, len(layers), pages, into_pages, page_size, *pointers, sources.shape[0],
                                               _stream_ptr(k.device)))
    _written(others)


def fit_pages(caches: Caches, refs: torch.Tensor, page_table: torch.Tensor, lens: torch.Tensor) -> torch.Tensor:
    """Makes ``page_table`` int32 ``[B, W]`` hold the pages that lengths ``lens`` int32 ``[B]`` need, and no others: before a pass with the
    lengths that it will write, after one with what is kept; a length of 0 frees a sequence's pages.

    Entries up to a sequence's last page that name none get a free one (the lowest-numbered, in order of sequence and position); entries
    behind it become -1, and their pages are held once less.  Where a sequence ends inside a page that others hold too
    (:func:`fork_pages`, then shortened), it gets its own copy of the rows it has there; so a sequence that shares pages and is cut short
    is fitted to the shorter length before it grows again.  Pages given back by a call are free for the next one.  Lengths are cut to
    what ``W`` entries hold.

    Returns int32 ``[B]``: how many pages each sequence wanted and did not get.  One with any must not be written to: nothing is
    given to it in another's place, and it may still end in a page of others."""
    out = _calls().fit_pages(caches, refs, page_table, lens)
    if out is not NotImplemented:
        return out
    layers, pages, page_size, pools = _check_caches(caches)
    k = layers[0].k
    if page_table.dim() != 2:
        raise ValueError("page_table must be [batch, width]")
    batch, width = page_table.shape
    pointers = [_check_int32(refs, "refs", (pages,), k), _check_int32(page_table, "page_table", (batch, width), k),
                _check_int32(lens, "lens", (batch,), k)]
    lib = _lib.load()
    missing = torch.empty((batch,), dtype=torch.int32, device=k.device)
    need = lib.fsta_fit_pages_workspace_bytes(batch, pages)
    work = torch.empty((need,), dtype=torch.uint8, device=k.device)
    with _on_device(k.device):
        _lib.check(lib.fsta_fit_pages(pools, len(layers), pages, page_size, *pointers, batch, width, missing.data_ptr(), work.data_ptr(), need,
                                      _stream_ptr(k.device)))
    _written(layers, refs, page_table)
    return missing


def fork_pages(caches: Caches, refs: torch.Tensor, page_table: torch.Tensor, lens: torch.Tensor, sources: torch.Tensor,
               targets: torch.Tensor) -> torch.Tensor:
    """Slot ``targets[i]`` of the batch gives up its pages and becomes a copy of slot ``sources[i]`` as it was before the call (int32
    ``[N]`` both): further answers to a prompt, the beams that a search goes on with.

    Full pages are shared (held once more); the rows of the last page, if it is not full, are copied to a free page, in all layers.
    ``page_table``, ``refs`` and ``lens`` int32 ``[B]`` are changed in place.  Where several pairs have one target the first counts; a pair of one
    slot twice, or with a number outside the batch, does nothing.

    Returns int32 ``[N]``: 1 where there was no free page for the last rows; that target is then empty (length 0, no pages)."""
    out = _calls().fork_pages(caches, refs, page_table, lens, sources, targets)
    if out is not NotImplemented:
        return out
    layers, pages, page_size, pools = _check_caches(caches)
    k = layers[0].k
    if page_table.dim() != 2 or sources.dim() != 1:
        raise ValueError("page_table must be [batch, width], sources and targets [pairs]")
    (batch, width), pairs = page_table.shape, sources.shape[0]
    pointers = [_check_int32(refs, "refs", (pages,), k), _check_int32(page_table, "page_table", (batch, width), k),
                _check_int32(lens, "lens", (batch,), k)]
    named = [_check_int32(sources, "sources", (pairs,), k), _check_int32(targets, "targets", (pairs,), k)]
    lib = _lib.load()
    missing = torch.empty((pairs,), dtype=torch.int32, device=k.device)
    need = lib.fsta_fork_pages_workspace_bytes(pairs, width, pages)
    work = torch.empty((need,), dtype=torch.uint8, device=k.device)
    with _on_device(k.device):
        _lib.check(lib.fsta_fork_pages(pools, len(layers), pages, page_size, *pointers, batch, width, *named, pairs, missing.data_ptr(),
                                       work.data_ptr(), need, _stream_ptr(k.device)))
    _written(layers, refs, page_table, lens)
    return missing
